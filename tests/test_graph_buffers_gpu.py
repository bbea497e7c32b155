"""What a CUDA graph was captured with stays its own, whatever is called afterwards."""

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


def _plain(q, cache, shared, out):
    from flashattntile_b200.kernels.decode import launch_decode

    launch_decode(q, cache.k_cache, cache.v_cache, cache.page_table, cache.seq_lens, cache.page_size,
                  q.shape[2] ** -0.5, out=out)


def _shared(q, cache, shared, out):
    from flashattntile_b200 import shared_prefix_decode_attention

    shared_prefix_decode_attention(q, cache, shared, out=out)


def _problem(n, heads=32, seed=0):
    from flashattntile_b200 import find_shared_prefix

    q, cache, _ = make("f16", [n], [512], [1 + i % 40 for i in range(n)], heads, heads // 4, 128, 16, seed=seed)
    return q, cache, find_shared_prefix(cache, [n]), torch.empty_like(q)


@pytest.mark.parametrize("call", [_plain, _shared])
@pytest.mark.parametrize("warm", [True, False])
def test_a_larger_call_leaves_an_earlier_graph_its_buffers(call, warm):
    """Captured after a call on the stream (whose buffers the graph goes on using), or as the
    stream's first (its buffers belong to the graph).  What the larger calls and others
    allocate afterwards stays as it is when the graph is replayed."""
    from flashattntile_b200 import value_checks

    small, big, bigger = _problem(2), _problem(90, seed=1), _problem(200, 64, seed=2)
    stream = torch.cuda.Stream()
    with value_checks(False):
        if warm:
            with torch.cuda.stream(stream):
                call(*small)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(*small)
            call(*small)
        for other in (big, bigger):
            with torch.cuda.stream(stream):
                call(*other)
            torch.cuda.synchronize()
            torch.cuda.empty_cache()
            fence = [torch.full((1 << 20,), 7, dtype=torch.uint8, device=DEV) for _ in range(64)]
            check(other[3], *other[:2], None)
            for _ in range(3):
                small[3].zero_()
                graph.replay()
                torch.cuda.synchronize()
                check(small[3], *small[:2], None)
            assert all(bool((x == 7).all()) for x in fence)
            with torch.cuda.stream(stream):
                call(*other)
            torch.cuda.synchronize()
            check(other[3], *other[:2], None)


@pytest.mark.parametrize("call", [_plain, _shared])
def test_a_graph_captured_first_and_not_replayed(call):
    """Its zeros are a node of the graph: nothing else may rely on them."""
    from flashattntile_b200 import value_checks

    one, two = _problem(3), _problem(40, seed=1)
    for _ in range(8):
        stream = torch.cuda.Stream()
        with value_checks(False):
            graphs = []
            for p in (one, two):
                graphs.append(torch.cuda.CUDAGraph())
                with torch.cuda.graph(graphs[-1], stream=stream):
                    call(*p)
            with torch.cuda.stream(stream):
                call(*two)
            torch.cuda.synchronize()
            check(two[3], *two[:2], None)
            for p, g in zip((two, one), graphs[::-1]):
                p[3].zero_()
                g.replay()
                torch.cuda.synchronize()
                check(p[3], *p[:2], None)


def test_loops_on_one_stream_replay_beside_each_other():
    """Streams come from a pool of 32; two loops may hold the same one."""
    from flashattntile_b200 import PagedKVCache, device_error
    from flashattntile_b200.decode_loop import DecodeLoop

    def loop(seed):
        q, cache, shared, _ = _problem(60, seed=seed)
        q2 = torch.randn_like(q)
        room = torch.cat([cache.page_table, cache.page_table[:, :2]], dim=1)
        cache = PagedKVCache(cache.k_cache, cache.v_cache, room, cache.seq_lens, cache.page_size)
        made = DecodeLoop(cache, q.shape[1], shared=shared)
        made.q.copy_(q2)
        return made

    first = loop(0)
    second = loop(1)
    for _ in range(64):
        if second.stream.cuda_stream == first.stream.cuda_stream:
            break
        second = loop(1)  # each takes the next stream of the pool
    assert second.stream.cuda_stream == first.stream.cuda_stream
    assert not set(t.data_ptr() for t in first._buffers.scratch.values()) \
        & set(t.data_ptr() for t in second._buffers.scratch.values())
    # The decode alone, over and over, both loops at once.
    from flashattntile_b200 import _lib, value_checks

    want = []
    for x in (first, second):
        with value_checks(False):
            x._decode()
        want.append(x.out.clone())
    graphs = []
    for x in (first, second):
        g = torch.cuda.CUDAGraph()
        with value_checks(False), _lib.own_buffers(x._buffers), torch.cuda.graph(g, stream=x.stream):
            for _ in range(10):
                x._decode()
        graphs.append(g)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(b):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(first.out, want[0]) and torch.equal(second.out, want[1])
    assert device_error() == 0 and first.device_error() == 0
