"""Shared-prefix decode over 8-bit caches whose scales are zero, of either sign, or far apart.

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


# sizes, prefixes, own tokens, heads, kv heads, dim, page: one row tile, two, one stream
SHAPES = [([3], [640], [0, 1, 40], 8, 2, 128, 16), ([40], [1040], [1 + i % 9 for i in range(40)], 16, 2, 64, 8),
          ([3, 2], [768, 512], [10, 30, 0, 1, 57], 4, 2, 256, 32)]


def _case(kind, shape, **kw):
    sizes, *rest = SHAPES[shape]
    return sizes, *make(kind, sizes, *rest, **kw)


def _prefix_pages(cache, shape):
    at, pages, (sizes, prefixes, *_) = 0, [], SHAPES[shape]
    for size, tokens in zip(sizes, prefixes):
        pages.append(cache.page_table[at, :tokens // cache.page_size])
        at += size
    return torch.cat(pages).long()


def _decode(q, cache, scales, sizes):
    from flashattntile_b200 import find_shared_prefix, shared_prefix_decode_attention

    out = torch.empty(q.shape, dtype=torch.float32, device=DEV)
    return shared_prefix_decode_attention(q, cache, find_shared_prefix(cache, sizes), scales=scales, out=out)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("size", [-12.0, 0.0, 8.0])  # log2 of the other scales' factor
def test_pages_whose_v_scale_is_zero(kind, shape, size):
    """Their codes count as zeros, whatever they hold; their weights count.  (By page and
    KV head, by whole pages from the start, and everywhere.)"""
    for seed, where in enumerate(("some", "first", "all")):
        sizes, q, cache, scales = _case(kind, shape, seed=seed, spread=2.0)
        scales["v"][_prefix_pages(cache, shape)] *= 2.0 ** size
        if where == "some":
            gen = torch.Generator(device=DEV).manual_seed(seed)
            scales["v"][torch.rand(scales["v"].shape, generator=gen, device=DEV) < 0.5] = 0.0
        elif where == "first":
            scales["v"][cache.page_table[0, :9].long()] = 0.0
        else:
            scales["v"].zero_()
        out = _decode(q, cache, scales, sizes)
        check(out, q, cache, scales)
        if where == "all":
            assert not out.any()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_scales_of_either_sign_and_k_scales_of_zero(kind, shape):
    sizes, q, cache, scales = _case(kind, shape, seed=3)
    gen = torch.Generator(device=DEV).manual_seed(9)
    scales["k"][torch.rand(scales["k"].shape, generator=gen, device=DEV) < 0.2] = 0.0
    sign = {n: torch.randint(0, 2, s.shape, generator=gen, device=DEV) * 2.0 - 1.0 for n, s in scales.items()}
    out = _decode(q, cache, {n: s * sign[n] for n, s in scales.items()}, sizes)
    # The same values with the signs in the codes.
    for n, x in (("k", cache.k_cache), ("v", cache.v_cache)):
        y = x.float().clamp(-127 if kind == "int8" else -448, 448) * sign[n][:, None, :, None]
        x.copy_(y.to(x.dtype))
    check(out, q, cache, scales)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("small,codes", [(1e-8, False), (1e-8, True), (2.0 ** -18, True), (2.0 ** -120, True)])
def test_v_scales_far_apart(kind, shape, small, codes):
    """Half of the pages hold values that are zero (``codes`` false) or next to nothing; 1e-8
    is the least scale that quantisation gives.  Their weights stay in the sum."""
    for seed in range(3):
        sizes, q, cache, scales = _case(kind, shape, seed=seed, spread=2.0)
        gen = torch.Generator(device=DEV).manual_seed(seed + 50)
        pages = torch.rand(cache.num_pages, generator=gen, device=DEV) < 0.5
        scales["v"][pages] = small
        if not codes:
            cache.v_cache.view(torch.uint8)[pages] = 0
        check(_decode(q, cache, scales, sizes), q, cache, scales)
