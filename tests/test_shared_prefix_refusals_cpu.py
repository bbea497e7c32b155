"""Shared-prefix decode: what is refused before anything is launched."""

from __future__ import annotations

import ctypes

import pytest

from tests.test_shared_pages_cpu import _shared_call


@pytest.mark.parametrize("heads", [65536, 65537 * 2])
def test_more_kv_heads_than_the_join_has_blocks_for(heads):
    from flashattntile_b200 import _lib

    lib = _lib.load()
    call = _shared_call(_lib, {"num_heads": heads, "num_kv_heads": heads, "q_stride_b": heads * 128,
                               "out_stride_b": heads * 128})
    assert lib.fat_shared_prefix_decode(ctypes.addressof(call)) == _lib.FAT_ERR_UNSUPPORTED
    assert b"KV heads" in lib.fat_last_error()
