"""Sizes whose tiles 32 bits do not count are refused on the host."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lite_llama_b200 import _lib


@pytest.mark.skipif(torch.cuda.is_available(), reason="sizes that fit go on to a launch, over addresses that are no tensors")
@pytest.mark.parametrize("tiles,refused", [(65533, False), (65534, False), (65535, True), (65536, True), (100000, True)])
def test_tiles_of_a_decode_step(tiles, refused):
    """4096 rows of 8 kv heads, a tile of 16 tokens each: with the one that a row's start and end count for, 2^15 (tiles + 1) in all."""
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    stride = lib.b2l_kv_int4_row_bytes(8, 128, 32)
    lib.b2l_flash_decoding_int4(p, p, p, stride, 1 << 21, p, 1 << 21, 1, 1, 1 << 21, p, 4, p, 4, 4096, 512, 8, 128, 32, 16 * tiles,
                                ctypes.c_float(0.1), 65536, 128, 65536, 128, p, 1 << 50, 0, None)
    assert (b"too many tokens" in lib.b2l_last_error()) == refused
