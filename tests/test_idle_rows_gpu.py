"""Rows that were released stay idle in a captured loop, until they are taken up again."""

from __future__ import annotations

import pytest
import torch

from tests.test_shared_loop_gpu import _BOUND, _dense, _exact

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import flashattntile_b200  # noqa: F401


def _rows(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _prompt(pool, row, tokens, gen):
    pool.reserve(tokens, rows=_rows(row))
    pages = pool.cache.page_table[row, : -(-tokens // pool.cache.page_size)].long()
    for x in (pool.cache.k_cache, pool.cache.v_cache):
        y = torch.randn((len(pages), *x.shape[1:]), generator=gen, device=DEV)
        x[pages] = (y if pool.scales is None else (y * 30).clamp(-120, 120)).to(x.dtype)
    if pool.scales is not None:
        for s in pool.scales.values():
            s[pages] = 0.03
    pool.cache.seq_lens[row] = tokens


@pytest.mark.parametrize("kind", ["f16", "int8"])
@pytest.mark.parametrize("sharing", [True, False])
def test_a_loop_goes_on_beside_released_rows(kind, sharing):
    import flashattntile_b200 as fat
    from flashattntile_b200.decode_loop import DecodeLoop

    gen = torch.Generator(device=DEV).manual_seed(3)
    rows, heads, kvh, dim, ps = 6, 8, 2, 64, 16
    pool = fat.PagePool.allocate(26, rows, 400, kvh, dim, ps, device=DEV,
                                 dtype=torch.float16 if kind == "f16" else torch.int8)
    _prompt(pool, 0, 150, gen)
    pool.fork(_rows(0, 0, 0, 0, 0), _rows(1, 2, 3, 4, 5))
    shared = fat.find_shared_prefix(pool.cache, [rows]) if sharing else None
    loop = DecodeLoop(pool.cache, heads, q_dtype=torch.float16, pool=pool, shared=shared)
    lens = [150] * rows

    def steps(n):
        for _ in range(n):
            q = torch.randn((rows, heads, dim), generator=gen, device=DEV).half()
            nk, nv = (torch.randn((rows, kvh, dim), generator=gen, device=DEV).half() for _ in range(2))
            idle = [b for b in range(rows) if not lens[b]]
            q[idle] = float("nan")
            got = loop.step(q, nk, nv)
            for b in range(rows):
                lens[b] += b not in idle
            assert pool.cache.seq_lens.tolist() == lens
            assert not got[idle].any()
            want = _exact(q, pool.cache, pool.scales, lens)
            live = [b for b in range(rows) if lens[b]]
            top = max(float(_dense(pool.cache, pool.scales, b, lens[b])[1].abs().max()) for b in live)
            assert float((got[live].double() - want[live]).abs().max()) <= _BOUND[torch.float16] * top

    steps(2)  # 9 shared pages, and one of each row's own
    assert pool.free_pages() == 26 - 9 - 6
    # The first row, whose prompt it was, and another end; their own pages are free again,
    # and stay so while the others cross a page's end.
    pool.release(_rows(0, 3))
    lens[0] = lens[3] = 0
    assert pool.released.tolist() == [1, 0, 0, 1, 0, 0]
    steps(20)
    assert pool.free_pages() == 26 - 9 - 2 * 4 and pool.owned.tolist()[0] == 0
    # One is forked to, the other starts a prompt of its own, after which nothing is shared.
    pool.fork(_rows(4), _rows(3))
    lens[3] = lens[4]
    steps(3)
    if sharing:
        shared.prefix_lens.zero_()
    _prompt(pool, 0, 21, gen)
    lens[0] = 21
    assert not pool.released.any()
    steps(3)
    assert loop.device_error() == 0 and fat.device_error() == 0


def test_marks():
    """Release sets them, forks copy them, a reserve by name clears them; eager calls go by them when asked to."""
    from flashattntile_b200 import PagePool, device_error

    pool = PagePool.allocate(16, 4, 32, 1, 8, 4, device=DEV)
    new = torch.ones(4, 1, 8, dtype=torch.float16, device=DEV)
    pool.reserve(1)
    pool.append(new, new)
    pool.release(_rows(1, 2))
    assert pool.released.tolist() == [0, 1, 1, 0]
    pool.fork(_rows(1, 0), _rows(3, 2))
    assert pool.released.tolist() == [0, 1, 0, 1]
    pool.reserve(5, skip_released=True)
    pool.append(new, new, skip_released=True)
    assert pool.cache.seq_lens.tolist() == [2, 0, 2, 0] and pool.owned.tolist() == [2, 0, 2, 0]
    pool.reserve(1, rows=_rows(3))
    assert pool.released.tolist() == [0, 1, 0, 0]
    pool.append(new, new, skip_released=True)
    assert pool.cache.seq_lens.tolist() == [3, 0, 3, 1]
    pool.reserve(1)  # all rows, released ones too; they stay marked
    pool.append(new, new)
    assert pool.cache.seq_lens.tolist() == [4, 1, 4, 2] and pool.released.tolist() == [0, 1, 0, 0]
    other = pool.compact(in_place=False)
    other.release(_rows(0))
    assert pool.released.tolist() == [1, 1, 0, 0] and device_error() == 0


def test_many_rows_with_some_released():
    """More rows than one round of a reserve takes."""
    from flashattntile_b200 import PagePool, device_error

    n = 2500
    pool = PagePool.allocate(n + 9, n, 8, 1, 8, 4, device=DEV)
    gone = torch.randperm(n, generator=torch.Generator().manual_seed(1))[:1100].sort().values.to(DEV, torch.int32)
    pool.release(gone)
    pool.reserve(3, skip_released=True)
    keep = torch.ones(n, dtype=torch.bool, device=DEV)
    keep[gone.long()] = False
    assert torch.equal(pool.owned, keep.to(torch.int32))
    assert pool.cache.page_table[keep, 0].tolist() == list(range(n - 1100))
    assert not pool.cache.page_table[~keep].any() and pool.free_pages() == 9 + 1100
    assert device_error() == 0
