"""Launchers of the page operations (``fat_copy_pages``, ``fat_fork_sequences``, ``fat_reserve_tokens``,
``fat_release_sequences``, ``fat_compact_pages``).

Arguments are packed once into a ``fat_page_pool`` struct (:func:`pool_call`);
a call sets the stream and its error word and launches on the stream current
now.  Nothing here synchronises; device-side problems are recorded in the
stream's error word (``flashattntile_b200.device_error``).
"""

from __future__ import annotations

import ctypes
import threading

import torch

from .. import _lib
from .append import _QUANT


def scales_of(scales):
    """``(k, v)`` of a ``QuantScales``, a dict with ``k``/``v``, or None."""
    if scales is None:
        return None, None
    return (scales["k"], scales["v"]) if isinstance(scales, dict) else (scales.k, scales.v)


def check_storage(what: str, k_cache, v_cache, k_scale, v_scale) -> None:
    for t in (k_cache, v_cache):
        if not t.is_cuda:
            raise RuntimeError(f"{what}: flashattntile_b200 runs on CUDA tensors only (no CPU path)")
    if k_cache.stride() != v_cache.stride() or k_cache.stride(3) != 1:
        raise ValueError(f"{what}: k_cache and v_cache need equal strides and a contiguous last dim")
    if k_cache.dtype in _QUANT:
        if k_scale is None or v_scale is None:
            raise ValueError(f"{what}: an int8/fp8 cache needs its scales (they move with the pages)")
    elif k_scale is not None or v_scale is not None:
        raise ValueError(f"{what}: scales belong to an int8/fp8 cache, got {k_cache.dtype}")
    if k_scale is not None:
        expected = (k_cache.shape[0], k_cache.shape[2])
        for s in (k_scale, v_scale):
            if tuple(s.shape) != expected or s.dtype != torch.float32 or s.stride(1) != 1 \
                    or s.stride() != k_scale.stride() or s.device != k_cache.device:
                raise ValueError(f"{what}: scales must be float32 {expected} on the cache's device with equal strides")


def check_rows(what: str, rows, device, name: str) -> torch.Tensor:
    if not isinstance(rows, torch.Tensor) or rows.dtype != torch.int32 or rows.dim() != 1:
        raise ValueError(f"{what}: {name} must be a 1-D int32 tensor")
    if rows.device != device:
        raise ValueError(f"{what}: {name} must be on the pool's device")
    return rows if rows.is_contiguous() else rows.contiguous()


def pool_call(k_cache, v_cache, page_size, k_scale=None, v_scale=None) -> _lib.PagePoolCall:
    """The struct with its storage fields filled."""
    eb = k_cache.element_size()
    return _lib.PagePoolCall(
        k_cache=k_cache.data_ptr(), v_cache=v_cache.data_ptr(), stride_page_bytes=k_cache.stride(0) * eb,
        stride_slot_bytes=k_cache.stride(1) * eb, stride_head_bytes=k_cache.stride(2) * eb,
        num_pages=k_cache.shape[0], row_bytes=k_cache.shape[3] * eb, k_scale=_lib.ptr(k_scale),
        v_scale=_lib.ptr(v_scale), scale_stride_page=0 if k_scale is None else k_scale.stride(0),
        num_kv_heads=k_cache.shape[2], page_size=int(page_size))


_LOCK = threading.Lock()


def launch(name: str, call: _lib.PagePoolCall, device: torch.device, *args, skip_released: bool = False) -> None:
    """Call library function ``name`` with the struct, on the stream current now."""
    fn = getattr(_lib.load(), name)
    index = device.index if device.index is not None else torch.cuda.current_device()
    stream = torch._C._cuda_getCurrentRawStream(index)
    err = _lib._ERR.get((index, stream))
    if err is None:
        err = _lib.error_word_for(index, stream, device)
    with _LOCK:  # the struct is its pool's: from its words to the library's reading of them
        call.stream = stream
        call.error_word = err.data_ptr()
        call.skip_released = skip_released
        if index == torch._C._cuda_getDevice():
            status = fn(ctypes.addressof(call), *args)
        else:
            with torch.cuda.device(index):
                status = fn(ctypes.addressof(call), *args)
    if status:
        _lib.check(status, name)


__all__ = ["check_rows", "check_storage", "launch", "pool_call", "scales_of"]
