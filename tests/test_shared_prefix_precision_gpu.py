"""Shared-prefix decode keeps its weights to 32 bits, nearly: fp32 outputs against 64 bits.

With w the softmax weights and l = sum 2^(s - max), an output may differ by

* P in two parts: sum_t w_t |v_t| times 2^-16 (bf16) or 2^-20 (fp16), and where a part is
  subnormal in fp16 2^-24 of a unit that is at most 2^-7 of the heaviest: 2^-31 |v_t| / l each
  (8-bit caches: |code| times twice the largest V scale for |v_t|);
* scores: fp32 sums of dim products in steps of 16, of which each may lose 2^-23 of
  sum |q k| scale, and four more roundings; 2^x to 2^-21 with x up to 2^6 in fp32: a relative
  error of every weight, twice (numerator, sum);
* sums over n tokens, 16 at a time in two parts, each adding 2^-23 of sum w |v| at most, and
  32 more for rescaling and joining.
"""

from __future__ import annotations

import pytest
import torch

from tests.test_shared_prefix_gpu import DEV, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import flashattntile_b200  # noqa: F401


def _exact(q, cache, scales):
    """(out, bound) in 64 bits."""
    b, heads, dim = q.shape
    kvh, ps = cache.num_kv_heads, cache.page_size
    group, scale = heads // kvh, dim ** -0.5
    out = torch.zeros(b, heads, dim, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    parts = 2.0 ** -16 if cache.k_cache.dtype == torch.bfloat16 else 2.0 ** -20
    for i, n in enumerate(cache.seq_lens.tolist()):
        ids = cache.page_table[i, :-(-n // ps)].long()
        k, v = cache.k_cache[ids].double(), cache.v_cache[ids].double()
        codes, unit = v, torch.ones(kvh, dtype=torch.float64, device=DEV)
        if scales is not None:
            k = k * scales["k"][ids].double()[:, None, :, None]
            v = v * scales["v"][ids].double()[:, None, :, None]
            unit = 2 * scales["v"][ids].double().abs().amax(0)
        k, v, codes = (x.reshape(-1, kvh, dim)[:n] for x in (k, v, codes))
        for h in range(kvh):
            rows = slice(h * group, (h + 1) * group)
            qh = q[i, rows].double()
            s = qh @ k[:, h].T * scale
            most = (qh.abs() @ k[:, h].abs().T * scale).amax(-1, keepdim=True)
            e = torch.exp(s - s.amax(-1, keepdim=True))
            l = e.sum(-1, keepdim=True)
            w = e / l
            out[i, rows] = w @ v[:, h]
            score = 2.0 ** -23 * (dim / 16 + 4) * most + 2.0 ** -21 + 2.0 ** -18
            rel = parts + 2 * score + 2.0 ** -23 * (n / 8 + 32)
            tiny = 2.0 ** -31 * unit[h] * codes[:, h].abs().sum(0)[None] / l
            bound[i, rows] = rel * (w @ v[:, h].abs()) + tiny
    return out, bound


SHAPES = [  # sizes, prefixes, own tokens, heads, kv heads, dim, page
    ([3], [640], [0, 1, 40], 8, 2, 128, 16),                         # one row tile
    ([40], [1040], [1 + i % 9 for i in range(40)], 16, 2, 64, 8),    # two row tiles
    ([3, 2], [768, 512], [10, 30, 0, 1, 57], 4, 2, 256, 32),         # one stream
    ([6], [640], [1, 2, 3, 4, 5, 6], 8, 4, 32, 16),
    ([4, 2], [400, 96], [3, 40, 17, 90, 2, 70], 24, 2, 128, 8),      # 12 heads per KV head: two head groups
    ([2], [256], [100, 30], 64, 1, 64, 16),                          # 64: eight
    ([2, 1], [96, 0], [9, 300, 80], 128, 1, 64, 32),                 # 128: one sequence per row tile
    ([5], [336], [1, 20, 3, 40, 5], 27, 3, 64, 16),                  # 9: a head group of one
]


@pytest.mark.parametrize("kind", ["f16", "bf16", "int8", "e4m3"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_weights_are_kept(kind, shape):
    from flashattntile_b200 import device_error, find_shared_prefix, shared_prefix_decode_attention

    sizes, prefixes, owns, heads, kvh, dim, ps = SHAPES[shape]
    for seed, spread in enumerate((1.0, 3.0)):
        q_dtype = torch.bfloat16 if kind in ("int8", "e4m3") and seed else None
        q, cache, scales = make(kind, sizes, prefixes, owns, heads, kvh, dim, ps, seed=seed, q_dtype=q_dtype,
                                spread=spread)
        out = torch.empty(q.shape, dtype=torch.float32, device=DEV)
        shared_prefix_decode_attention(q, cache, find_shared_prefix(cache, sizes), scales=scales, out=out)
        want, bound = _exact(q, cache, scales)
        over = (out.double() - want).abs() / (bound + 2.0 ** -40)
        assert float(over.max()) <= 1.0, f"{float(over.max()):.2f} of its bound"
        assert device_error() == 0


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
@pytest.mark.parametrize("size", [-110, -30, -12, 12, 30])
def test_values_of_any_size(kind, dim, size):
    """V scales of 2^-125 to 2^30, in the prefix and in own tokens, rising and falling along them."""
    from flashattntile_b200 import device_error, find_shared_prefix, shared_prefix_decode_attention

    q, cache, scales = make(kind, [3], [320], [0, 40, 300], 8, 2, dim, 16, seed=dim, spread=2.0)
    scales["v"] *= 2.0 ** size
    for own in (1, 2):  # larger page by page, then smaller
        n = -(-int(cache.seq_lens[own]) // 16)
        steps = torch.arange(n, device=DEV, dtype=torch.float32)
        scales["v"][cache.page_table[own, :n].long()] *= torch.exp2(steps % 11 - 5 if own == 1 else 5 - steps % 11)[:, None]
    out = torch.empty(q.shape, dtype=torch.float32, device=DEV)
    shared_prefix_decode_attention(q, cache, find_shared_prefix(cache, [3]), scales=scales, out=out)
    want, bound = _exact(q, cache, scales)
    assert out.isfinite().all()
    assert float(((out.double() - want).abs() / (bound + 2.0 ** (size - 40))).max()) <= 1.0
    assert device_error() == 0
