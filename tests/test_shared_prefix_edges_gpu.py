"""Shared-prefix decode where its inputs are at the edge of what they may be.

Bounds as in ``test_shared_prefix_gpu`` (one softmax per sequence and head in 64 bits).
"""

from __future__ import annotations

import pytest
import torch

from tests.test_shared_prefix_gpu import DEV, check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import flashattntile_b200  # noqa: F401


def _edges(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("kind", ["f16", "int8"])
@pytest.mark.parametrize("most", [0, 1, 15, 16, 39])
def test_a_group_larger_than_announced(kind, most):
    """It is decoded without sharing, and named; the groups beside it share."""
    from flashattntile_b200 import SharedPrefix, device_error, shared_prefix_decode_attention, value_checks

    q, cache, scales = make(kind, [40, 2], [320, 96], [1 + i % 7 for i in range(42)], 32, 4, 128, 16, seed=most)
    shared = SharedPrefix(_edges(0, 40, 42), _edges(320, 96), most)
    with value_checks(False):
        out = shared_prefix_decode_attention(q, cache, shared, scales=scales)
        assert device_error() == 32
        check(out, q, cache, scales)


def test_edges_that_do_not_start_at_the_first_sequence():
    """Sequences before the first edge are in no group."""
    from flashattntile_b200 import SharedPrefix, shared_prefix_decode_attention, value_checks

    q, cache, _ = make("f16", [40], [320], [1 + i % 7 for i in range(40)], 32, 4, 128, 16, seed=1)
    for first in (1, 39):
        with value_checks(False):
            out = shared_prefix_decode_attention(q, cache, SharedPrefix(_edges(first, 40), _edges(320), 40))
        check(out, q, cache, None)


def test_edges_that_fall_or_leave_the_batch_are_named():
    from flashattntile_b200 import SharedPrefix, device_error, shared_prefix_decode_attention, value_checks

    q, cache, _ = make("f16", [6], [64], [1, 2, 3, 4, 5, 6], 8, 2, 64, 16, seed=1)
    want = shared_prefix_decode_attention(q, cache, SharedPrefix(_edges(0, 6), _edges(64), 6))
    for edges in ((0, 4, 2), (0, 4, 9), (-3, 3, 6), (5, 0, 6), (7, 7, 7)):
        with value_checks(False):
            out = shared_prefix_decode_attention(q, cache, SharedPrefix(_edges(*edges), _edges(64, 64), 6))
            assert device_error() == 32
            assert out.shape == want.shape and out.isfinite().all()
    # A call after them is right.
    assert torch.equal(shared_prefix_decode_attention(q, cache, SharedPrefix(_edges(0, 6), _edges(64), 6)), want)


@pytest.mark.parametrize("kind", ["f16", "bf16", "int8", "e4m3"])
@pytest.mark.parametrize("rows,dim", [(3, 128), (40, 64), (3, 256), (5, 32)])  # one row tile, two, one stream
def test_any_scale_on_a_prefix_that_ends_inside_a_tile(kind, rows, dim):
    """Masked scores stay masked, also by a scale of 0 (then every token weighs the same)."""
    from flashattntile_b200 import find_shared_prefix, shared_prefix_decode_attention

    for tokens in (16, 80, 128, 656):
        q, cache, scales = make(kind, [rows], [tokens], [1 + i % 3 for i in range(rows)], 16, 4, dim, 16, seed=tokens)
        shared = find_shared_prefix(cache, [rows])
        for scale in (0.0, -0.0, 0.02, -0.3, 1e-38):
            check(shared_prefix_decode_attention(q, cache, shared, softmax_scale=scale, scales=scales), q, cache,
                  scales, scale)


@pytest.mark.parametrize("kind", ["f16", "bf16", "int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 256])
def test_sequences_that_ended_leave_the_others_right(kind, dim):
    """Any of a group's sequences may be released, the first ones too: their tables are not
    read, their outputs are zeros whatever their queries hold, and nothing is reported."""
    from flashattntile_b200 import find_shared_prefix, shared_prefix_decode_attention, value_checks

    n = 70
    q, cache, scales = make(kind, [n, 3], [656, 96], [1 + i % 9 for i in range(n + 3)], 8, 4, dim, 16, seed=dim)
    shared = find_shared_prefix(cache, [n, 3])
    # Page 0 is what a released row's table holds; here it would do harm.
    bad = int((set(range(cache.num_pages)) - set(cache.page_table.unique().tolist())).pop())
    if scales is None:
        cache.k_cache[bad], cache.v_cache[bad] = float("nan"), float("nan")
    for ended in ([0], [0, 1, 2, 33], list(range(64)), list(range(1, n)), [n], [n, n + 1], [0, n, n + 2]):
        lens, table = cache.seq_lens.clone(), cache.page_table.clone()
        lens[ended], table[ended] = 0, bad
        now = type(cache)(cache.k_cache, cache.v_cache, table, lens, 16)
        qs = q.clone()
        qs[ended] = float("nan")
        with value_checks(False):
            out = shared_prefix_decode_attention(qs, now, shared, scales=scales)
        assert not out[ended].any()
        check(out, q, now, scales)


def test_a_short_sequence_harms_no_other():
    from flashattntile_b200 import device_error, find_shared_prefix, shared_prefix_decode_attention, value_checks

    q, cache, _ = make("f16", [5], [320], [1, 2, 3, 4, 5], 8, 2, 64, 16, seed=1)
    shared = find_shared_prefix(cache, [5])
    want = shared_prefix_decode_attention(q, cache, shared)
    for short in (0, 2):
        lens, table = cache.seq_lens.clone(), cache.page_table.clone()
        lens[short], table[short, 7:] = 100, 0
        now = type(cache)(cache.k_cache, cache.v_cache, table, lens, 16)
        with value_checks(False):
            out = shared_prefix_decode_attention(q, now, shared)
            assert device_error() == 4
        rest = [i for i in range(5) if i != short]
        assert torch.equal(out[rest], want[rest])
