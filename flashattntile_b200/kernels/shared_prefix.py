"""Decode attention for a batch whose sequences share long prefixes (``fat_shared_prefix_decode``).

Samples of one prompt, beams, conversations behind one system prompt: the page
tables of such sequences begin with the same pages (``page_pool.PagePool.fork``
makes them so).  ``paged_decode_attention`` reads those pages once per
sequence; here they are read once per group, and the queries of the whole group
are multiplied with them on the tensor cores:

    shared = find_shared_prefix(pool.cache, group_sizes=[32, 16])   # after a fork; kept between steps
    out = shared_prefix_decode_attention(q, pool.cache, shared)     # = paged_decode_attention(q, pool.cache)

The shared prefix does not change while its sequences only grow, so
``SharedPrefix`` is made when groups are formed and used for every step.  No
counterpart in FlashAttnTile (``kernels/decode.py:533-704`` reads every
sequence's pages on their own).
"""

from __future__ import annotations

import ctypes
import threading
from dataclasses import dataclass, field

import torch

from .. import _config, _lib
from ..paging import PagedKVCache, validate_cache_values, validate_metadata
from .decode import _QUANT_DTYPES, _aligned_q, _q_error, _require_cuda
from .pages import scales_of


@dataclass
class SharedPrefix:
    """Groups of consecutive sequences and the tokens that each group shares.

    ``cu_groups`` int32 ``[G + 1]``: group ``g`` is sequences ``cu_groups[g]`` to
    ``cu_groups[g + 1] - 1`` (from 0; sequences past the last group share nothing).
    ``prefix_lens`` int32 ``[G]``: shared tokens; a prefix that ends inside a page is
    used up to the page's start.  ``max_group``: no group has more sequences.
    """

    cu_groups: torch.Tensor
    prefix_lens: torch.Tensor
    max_group: int
    # The layout that the last call checked, and its argument struct (see _Packed).
    _packed: "_Packed | None" = field(default=None, init=False, repr=False, compare=False)

    @property
    def num_groups(self) -> int:
        return int(self.prefix_lens.shape[0])


class _Packed:
    """The argument struct of a layout -- shapes, strides, types, devices, page size and
    stream -- that passed every structural check, kept in the ``SharedPrefix`` that a
    decode loop holds.  A call with the same layout skips those checks; its pointers
    are taken from its own tensors, and nothing else of an earlier call is kept.  It is
    the thread's that made it: pointers are written into it before the library reads them."""

    __slots__ = ("layout", "call", "addr", "buffers", "index", "stream", "thread")

    @staticmethod
    def layout_of(q, cache, shared, k_scale, v_scale):
        k, v, table, lens, cu, pre = (cache.k_cache, cache.v_cache, cache.page_table, cache.seq_lens,
                                      shared.cu_groups, shared.prefix_lens)
        out = (q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(),
               v.dtype, v.device, table.shape, table.stride(), table.dtype, table.device, lens.shape, lens.stride(),
               lens.dtype, lens.device, cu.shape, cu.stride(), cu.dtype, cu.device, pre.shape, pre.stride(), pre.dtype,
               pre.device, cache.page_size, shared.max_group)
        if k_scale is None or v_scale is None:
            return out, k_scale is None, v_scale is None
        return out, (k_scale.shape, k_scale.stride(), k_scale.dtype, k_scale.device, v_scale.shape, v_scale.stride(),
                     v_scale.dtype, v_scale.device)


def _table_and_lens(cache: PagedKVCache):
    table = cache.page_table if cache.page_table.stride(1) == 1 else cache.page_table.contiguous()
    lens = cache.seq_lens if cache.seq_lens.is_contiguous() else cache.seq_lens.contiguous()
    return table, lens


def _find(cache: PagedKVCache, cu_groups: torch.Tensor, num_groups: int, min_sequences: int) -> torch.Tensor:
    table, lens = _table_and_lens(cache)
    out = torch.empty(num_groups, dtype=torch.int32, device=table.device)
    with torch.cuda.device(table.device):
        status = _lib.load().fat_find_shared_prefix(
            table.data_ptr(), table.stride(0), table.shape[1], lens.data_ptr(), lens.shape[0], cache.page_size,
            cu_groups.data_ptr(), num_groups, min_sequences, out.data_ptr(), _lib.stream_handle(table.device))
    _lib.check(status, "find_shared_prefix")
    return out


def find_shared_prefix(cache: PagedKVCache, group_sizes) -> SharedPrefix:
    """The prefix that each group of ``cache``'s sequences shares, read off the page
    tables on the device: whole pages in which all tables of the group agree.

    ``group_sizes``: sequences per group, in batch order (a list of ints).  A group of
    one shares nothing (its tokens are read once anyway)."""
    validate_metadata(cache)
    sizes = [int(n) for n in group_sizes]
    if any(n < 0 for n in sizes):
        raise ValueError("group_sizes must be non-negative")
    if sum(sizes) > cache.batch_size:
        raise ValueError(f"group_sizes add up to {sum(sizes)} sequences, the cache has {cache.batch_size}")
    _require_cuda(cache.page_table, cache.seq_lens)
    edges = [0]
    for n in sizes:
        edges.append(edges[-1] + n)
    cu_groups = torch.tensor(edges, dtype=torch.int32, device=cache.page_table.device)
    return SharedPrefix(cu_groups, _find(cache, cu_groups, len(sizes), 2), max(sizes, default=0))


def _check_shared(shared: SharedPrefix, device: torch.device) -> None:
    if not isinstance(shared, SharedPrefix):
        raise TypeError("shared must be a SharedPrefix")
    cu, lens = shared.cu_groups, shared.prefix_lens
    for name, t in (("cu_groups", cu), ("prefix_lens", lens)):
        if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous 1-D int32 tensor")
        if t.device != device:
            raise ValueError(f"{name} must be on the cache's device")
    if cu.shape[0] != lens.shape[0] + 1:
        raise ValueError(f"cu_groups must have {lens.shape[0] + 1} entries, got {cu.shape[0]}")
    if int(shared.max_group) < 0:
        raise ValueError("max_group must be non-negative")


def _check_values(cache: PagedKVCache, shared: SharedPrefix) -> None:
    """The value checks of a decode, and those of the groups (read back)."""
    stats = validate_cache_values(cache)
    if stats is not None and stats[0] <= 0:
        raise ValueError("decode requires every sequence to hold at least one cached token")
    if shared.num_groups == 0:
        return
    cu = shared.cu_groups.tolist()
    sizes = [b - a for a, b in zip(cu, cu[1:])]
    if cu[0] != 0 or min(sizes) < 0 or cu[-1] > cache.batch_size:
        raise ValueError(f"cu_groups must rise from 0 to at most {cache.batch_size}")
    if max(sizes) > shared.max_group:
        raise ValueError(f"a group has {max(sizes)} sequences, max_group is {shared.max_group}")
    agreed = _find(cache, shared.cu_groups, shared.num_groups, 1).tolist()
    for g, (want, have) in enumerate(zip(shared.prefix_lens.tolist(), agreed)):
        if want < 0:
            raise ValueError("prefix_lens must be non-negative")
        if sizes[g] and want // cache.page_size * cache.page_size > have:
            raise ValueError(f"group {g} shares {have} tokens, not {want}")


def shared_prefix_decode_attention(q: torch.Tensor, cache: PagedKVCache, shared: SharedPrefix,
                                   softmax_scale: float | None = None, scales=None,
                                   out: torch.Tensor | None = None) -> torch.Tensor:
    """One query per sequence against a paged cache whose groups of sequences share
    prefixes -> ``[B, H, D]`` in q's dtype (or in ``out``'s, q's or fp32).

    The result is that of ``paged_decode_attention`` (``paged_decode_attention_fp8``
    with ``scales`` for an INT8 / e4m3 cache) on the same cache."""
    packed = shared._packed if type(shared) is SharedPrefix else None
    if packed is not None and out is None and type(cache) is PagedKVCache and isinstance(q, torch.Tensor) \
            and not _config.validate_values():
        k_scale, v_scale = scales_of(scales)
        index = torch._C._cuda_getDevice()
        stream = torch._C._cuda_getCurrentRawStream(index)
        key = (index, stream)
        if packed.thread == threading.get_ident() and index == packed.index and stream == packed.stream and q.data_ptr() % 16 == 0 \
                and packed.layout == _Packed.layout_of(q, cache, shared, k_scale, v_scale) \
                and _lib._WS.get(key) is packed.buffers[0] and _lib._SCRATCH.get(key) is packed.buffers[1] \
                and _lib._ERR.get(key) is packed.buffers[2]:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            call = packed.call
            call.cu_groups, call.prefix_lens = shared.cu_groups.data_ptr(), shared.prefix_lens.data_ptr()
            call = call.decode
            call.q, call.out = q.data_ptr(), out.data_ptr()
            call.k_cache, call.v_cache = cache.k_cache.data_ptr(), cache.v_cache.data_ptr()
            call.page_table, call.seq_lens = cache.page_table.data_ptr(), cache.seq_lens.data_ptr()
            if k_scale is not None:
                call.k_scale, call.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
            call.softmax_scale = float(softmax_scale) if softmax_scale is not None else q.shape[2] ** -0.5
            _lib.check(_lib.load().fat_shared_prefix_decode(packed.addr), "shared_prefix_decode")
            return out
    if not isinstance(cache, PagedKVCache):
        raise TypeError("cache must be a PagedKVCache")
    validate_metadata(cache)
    err = _q_error(q, cache)
    if err is not None:
        raise err
    k, v = cache.k_cache, cache.v_cache
    k_scale, v_scale = scales_of(scales)
    given = (k, v, cache.page_table, cache.seq_lens, None, None, k_scale, v_scale)
    q_given, own_out = q, out is None
    _require_cuda(q, k, v, cache.page_table, cache.seq_lens)
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise NotImplementedError(f"paged decode has fp16/bf16 kernels only, got {q.dtype}")
    if k.dtype in _QUANT_DTYPES:
        expected = (cache.num_pages, cache.num_kv_heads)
        if k_scale is None or v_scale is None:
            raise ValueError("an int8/fp8 cache needs its scales")
        if tuple(k_scale.shape) != expected or tuple(v_scale.shape) != expected:
            raise ValueError(f"scales must have shape {expected}, got {tuple(k_scale.shape)}")
        _require_cuda(k_scale, v_scale)
        k_scale, v_scale = k_scale.float(), v_scale.float()
        if k_scale.stride(1) != 1 or v_scale.stride() != k_scale.stride():
            k_scale, v_scale = k_scale.contiguous(), v_scale.contiguous()
    elif k.dtype != q.dtype:
        raise ValueError(f"q dtype {q.dtype} must match cache dtype {k.dtype}")
    elif k_scale is not None:
        raise ValueError(f"scales belong to an int8/fp8 cache, got {k.dtype}")
    if k.stride() != v.stride():
        raise ValueError("k_cache and v_cache must have identical strides")
    if k.stride(3) != 1:
        raise ValueError("k_cache/v_cache must be contiguous along head_dim")
    _check_shared(shared, k.device)
    if _config.validate_values():
        _check_values(cache, shared)
    q = _aligned_q(q)
    table, lens = _table_and_lens(cache)
    batch, heads, dim = q.shape
    if out is None:
        out = torch.empty((batch, heads, dim), dtype=q.dtype, device=q.device)
    elif tuple(out.shape) != (batch, heads, dim) or out.device != q.device or out.dtype not in (q.dtype, torch.float32) \
            or out.stride(2) != 1:
        raise ValueError(f"out must be a {q.dtype} or float32 tensor of shape {(batch, heads, dim)} on q's device")
    lib = _lib.load()
    dev = q.device
    idx, stream = _lib._key(dev)
    kvh = cache.num_kv_heads
    ws = _lib.workspace_for(idx, stream, dev, lib.fat_paged_decode_workspace_size(idx, batch, heads, kvh, dim))
    scratch = _lib.scratch_for(idx, stream, dev, lib.fat_shared_prefix_scratch_size(idx, batch, heads, kvh, dim,
                                                                                   int(shared.max_group)))
    call = _lib.SharedPrefixCall(
        decode=_lib.DecodeCall(
            q=q.data_ptr(), q_stride_b=q.stride(0), q_stride_h=q.stride(1), k_cache=k.data_ptr(),
            v_cache=v.data_ptr(), kv_stride_page=k.stride(0), kv_stride_slot=k.stride(1), kv_stride_head=k.stride(2),
            num_pages=k.shape[0], page_table=table.data_ptr(), page_table_stride=table.stride(0),
            max_pages=table.shape[1], seq_lens=lens.data_ptr(), k_scale=_lib.ptr(k_scale), v_scale=_lib.ptr(v_scale),
            scale_stride_page=0 if k_scale is None else k_scale.stride(0), out=out.data_ptr(),
            out_stride_b=out.stride(0), out_stride_h=out.stride(1), batch=batch, num_heads=heads, num_kv_heads=kvh,
            head_dim=dim, page_size=cache.page_size, q_dtype=_lib.DTYPE_CODE[q.dtype],
            kv_dtype=_lib.DTYPE_CODE[k.dtype], out_dtype=_lib.DTYPE_CODE[out.dtype],
            softmax_scale=float(softmax_scale) if softmax_scale is not None else dim ** -0.5, split_k_hint=1,
            workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
            error_word=_lib.error_word_for(idx, stream, dev).data_ptr(), stream=stream),
        cu_groups=shared.cu_groups.data_ptr(), prefix_lens=shared.prefix_lens.data_ptr(),
        num_groups=shared.num_groups, max_group=int(shared.max_group), scratch=scratch.data_ptr(),
        scratch_bytes=scratch.numel())
    if idx == torch.cuda.current_device():
        status = lib.fat_shared_prefix_decode(ctypes.addressof(call))
    else:
        with torch.cuda.device(idx):
            status = lib.fat_shared_prefix_decode(ctypes.addressof(call))
    _lib.check(status, "shared_prefix_decode")
    if own_out and q is q_given and table is given[2] and lens is given[3] and k_scale is given[6] \
            and v_scale is given[7]:
        packed = _Packed()
        packed.layout = _Packed.layout_of(q, cache, shared, k_scale, v_scale)
        packed.call, packed.addr = call, ctypes.addressof(call)
        packed.index, packed.stream, packed.thread = idx, stream, threading.get_ident()
        packed.buffers = (ws, scratch, _lib._ERR[(idx, stream)])
        shared._packed = packed
    return out


__all__ = ["SharedPrefix", "find_shared_prefix", "shared_prefix_decode_attention"]
