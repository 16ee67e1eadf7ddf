"""The 4-bit cache's layout and refusals, as far as they need no GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import kv_int4_oracle as O
from lite_llama_b200 import _lib
from lite_llama_b200 import kernels as K


@pytest.mark.parametrize("heads,d,group", [(8, 128, 64), (4, 128, 128), (2, 64, 32), (1, 64, 64), (3, 32, 32), (5, 128, 32)])
def test_row_bytes(heads, d, group):
    assert K.kv_int4_row_bytes(heads, d, group) == O.row_bytes(heads, d, group)
    assert K.kv_int4_row_bytes(heads, d, group) % 16 == 0


@pytest.mark.parametrize("heads,d,group", [(8, 96, 32), (8, 256, 64), (8, 64, 128), (8, 128, 16), (0, 128, 64), (8, 128, 0)])
def test_rows_that_there_are_not(heads, d, group):
    with pytest.raises(ValueError, match="head_dim 32, 64 or 128"):
        K.kv_int4_row_bytes(heads, d, group)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_value_comes_back_within_half_a_step(dtype):
    x = torch.randn(40, 3, 128, dtype=torch.float64).to(dtype)
    y = torch.randn(40, 3, 128, dtype=torch.float64).to(dtype)
    k, v, _, _ = O.values(O.rows_of(x, y, 64), 3, 128, 64, dtype)
    for got, want in ((k, x), (v, y)):
        g = want.double().unflatten(-1, (-1, 64))
        step = (g.amax(-1) - g.amin(-1)) / 15
        # half a step, and 15 steps whose size was rounded
        bound = step * (0.5 + 15 * torch.finfo(dtype).eps / 2)
        assert ((got.unflatten(-1, (-1, 64)) - g).abs() <= bound[..., None] * (1 + 1e-9)).all()


def _tensors(n=3, hq=4, hkv=2, d=64, dtype=torch.float16):
    q, k, v = torch.zeros(n, hq, d, dtype=dtype), torch.zeros(n, hkv, d, dtype=dtype), torch.zeros(n, hkv, d, dtype=dtype)
    return q, k, v, torch.zeros(n, dtype=torch.int32), torch.zeros(9, O.row_bytes(hkv, d, 64), dtype=torch.uint8)


def test_shims_refuse_cpu_tensors():
    q, k, v, idx, cache = _tensors()
    table = torch.zeros(3, 8, dtype=torch.int32)
    cos = torch.zeros(1, 3, 64, dtype=torch.float16)
    for call in (lambda: K.update_kv_buffer_int4(k, v, idx, cache), lambda: K.rope_kv_write_int4(q, k, v, cos, cos, idx, cache, 1, 3),
                 lambda: K.read_kv_buffer_int4(cache, idx, 2, 64, torch.float16),
                 lambda: K.flash_decoding_int4(q, cache, 0.1, table, idx, idx, 8, 2),
                 lambda: K.flash_attention_int4(q, cache, 0.1, idx, idx, table, idx, idx, 2, 8, 2),
                 lambda: K.build_slot_maps(idx, idx, idx, table, 5)):
        with pytest.raises(ValueError, match="no CPU fallback"):
            call()


def test_writer_refuses_what_does_not_fit():
    q, k, v, idx, cache = _tensors()
    cos = torch.zeros(1, 3, 64, dtype=torch.float16)
    bad = [
        (lambda: K.update_kv_buffer_int4(k, v[:, :1], idx, cache), "one shape"),
        (lambda: K.update_kv_buffer_int4(k, v.bfloat16(), idx, cache), "one shape"),
        (lambda: K.update_kv_buffer_int4(k.float(), v.float(), idx, cache), "float16 or bfloat16"),
        (lambda: K.update_kv_buffer_int4(k, v, idx[:2], cache), "one entry per token"),
        (lambda: K.update_kv_buffer_int4(k, v, torch.zeros(6, dtype=torch.int32)[::2], cache), "contiguous vector"),
        (lambda: K.update_kv_buffer_int4(k, v, idx, cache.view(torch.int8)), "uint8 matrix"),
        (lambda: K.update_kv_buffer_int4(k, v, idx, cache[:, :-16]), "takes 144 bytes"),
        (lambda: K.update_kv_buffer_int4(k, v, idx, cache, 32), "takes 160 bytes"),
        (lambda: K.update_kv_buffer_int4(k, v, idx, cache.t()), "contiguous rows"),
        (lambda: K.update_kv_buffer_int4(k.transpose(1, 2), v, idx, cache), "contiguous head_dim"),
        (lambda: K.update_kv_buffer_int4(k, v, idx, cache, 48), "groups of 48"),
        (lambda: K.rope_kv_write_int4(q, k, v, cos, cos, idx, cache, 1, 2), "batch_size"),
        (lambda: K.rope_kv_write_int4(q, k, v, cos, cos.float(), idx, cache, 1, 3), "activation dtype"),
        (lambda: K.rope_kv_write_int4(q, k, v, cos[:, :2], cos[:, :2], idx, cache, 1, 3), "cos and sin"),
        (lambda: K.rope_kv_write_int4(q, k, v, cos[..., :16], cos[..., :16], idx, cache, 1, 3), "cos and sin"),
        (lambda: K.rope_kv_write_int4(q, k, v, cos, cos, idx, cache, 1, 3, out_k=q), "shapes of q and k"),
        (lambda: K.read_kv_buffer_int4(cache, idx.view(1, 3), 2, 64, torch.float16), "contiguous vector"),
    ]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()


def test_attention_and_maps_refuse_what_does_not_fit():
    q, k, v, idx, cache = _tensors()
    table = torch.zeros(3, 8, dtype=torch.int32)
    bad = [
        (lambda: K.flash_decoding_int4(q, cache, 0.1, table, idx, idx, 8, 3), "no multiple"),
        (lambda: K.flash_decoding_int4(q, cache, 0.1, table, idx, idx, 8, 0), "no multiple"),
        (lambda: K.flash_decoding_int4(q.float(), cache, 0.1, table, idx, idx, 8, 2), "float16 or bfloat16"),
        (lambda: K.flash_decoding_int4(q, cache, 0.1, table.long(), idx, idx, 8, 2), "int32 matrix"),
        (lambda: K.flash_decoding_int4(q, cache, 0.1, table, idx[:2], idx, 8, 2), "one entry per sequence"),
        (lambda: K.flash_decoding_int4(q, cache, 0.1, table, idx, idx, 8, 4), "takes 288 bytes"),
        (lambda: K.flash_decoding_int4(q, cache, 0.1, table, idx, idx, 8, 2, out=q[:2]), "shape and type of q"),
        (lambda: K.flash_decoding_int4(q, cache, 0.1, table, idx, idx, 8, 2, out=q.bfloat16()), "shape and type of q"),
        (lambda: K.flash_attention_int4(q, cache, 0.1, idx, idx, table, idx, idx, 2, 8, 3), "no multiple"),
        (lambda: K.flash_attention_int4(q, cache, 0.1, idx[:2], idx, table, idx, idx, 2, 8, 2), "one entry per sequence"),
        (lambda: K.flash_attention_int4(q, cache, 0.1, idx, idx, table, idx, idx, 2, 8, 2, out=q[:2]), "shape and type of q"),
        (lambda: K.flash_attention_int4(q, cache, 0.1, idx, idx, table, idx, idx, 2, 8, 2, 128), "groups of 128"),
        (lambda: K.flash_attention_int4(q, cache.view(-1), 0.1, idx, idx, table, idx, idx, 2, 8, 2), "uint8 matrix"),
        (lambda: K.build_slot_maps(idx, idx[:2], idx, table, 5), "one entry per sequence"),
        (lambda: K.build_slot_maps(idx, idx, idx, table.long(), 5), "int32 matrix"),
        (lambda: K.build_slot_maps(idx, idx, idx, table, -1), "total_tokens"),
        (lambda: K.build_slot_maps(idx, idx, idx, table, 5, idx), "at least total_tokens"),
    ]
    for call, match in bad:
        with pytest.raises(ValueError, match=match):
            call()


def test_c_entries_refuse_on_the_host():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    f = ctypes.c_float(0.1)

    def decode(cache=p, stride=144, tokens=9, hq=4, hkv=2, d=64, group=64, ws=p, nbytes=1 << 30, dtype=0, w=4):
        return lib.b2l_flash_decoding_int4(p, p, cache, stride, tokens, p, 8, 1, 3, 8, p, w, p, 4, 3, hq, hkv, d, group, 8, f, 256, 64, 256, 64,
                                           ws, nbytes, dtype, None)

    for kwargs, why in [({"hq": 5}, b"multiple of num_kv_heads"), ({"hq": 130}, b"more than 64 query heads"), ({"d": 48}, b"head_dim 48"),
                        ({"stride": 128}, b"hold 144 bytes"), ({"stride": 152}, b"16-byte aligned"), ({"cache": p + 8}, b"16-byte aligned"),
                        ({"ws": None}, b"workspace"), ({"nbytes": 64}, b"workspace"), ({"dtype": 2}, b"dtype 2"), ({"w": 2}, b"index widths"),
                        ({"cache": None}, b"null pointer"), ({"tokens": 0}, b"bad shape")]:
        assert decode(**kwargs) == -1 and why in lib.b2l_last_error(), (kwargs, lib.b2l_last_error())

    def write(k=p, cos=p, hq=4, d=64, group=64, stride=144, w=4, dtype=0):
        return lib.b2l_kv_int4_write(p, p, p, k, p, cos, p, p, w, p, stride, 9, 3, 3, hq, 2, d, group, 256, 64, 128, 64, 128, 64, 192, 64, 256, 64,
                                     128, 64, dtype, None)

    for kwargs, why in [({"k": None}, b"null pointer"), ({"cos": None}, b"without positions"), ({"d": 80}, b"head_dim 80"), ({"group": 128}, b"groups of 128"),
                        ({"stride": 136}, b"hold 144 bytes"), ({"w": 1}, b"index width"), ({"dtype": 2}, b"dtype 2")]:
        assert write(**kwargs) == -1 and why in lib.b2l_last_error(), (kwargs, lib.b2l_last_error())
    assert lib.b2l_kv_int4_read(p, p, 144, 9, p, 4, 3, 2, 64, 48, 0, None) == -1 and b"groups of 48" in lib.b2l_last_error()
    assert lib.b2l_slot_maps(p, p, p, p, p, 3, p, 4, p, 4, None, 0, p, 8, 1, 3, 8, 3, 5, None) == -1 and b"widths" in lib.b2l_last_error()
    assert lib.b2l_slot_maps(None, p, p, p, p, 4, p, 4, p, 4, None, 0, p, 8, 1, 3, 8, 3, 5, None) == -1


def test_workspace_is_a_function_of_sizes():
    lib = _lib.load()
    assert lib.b2l_flash_decoding_int4_workspace_bytes(0, 32, 8, 128, 64, 256) == 0
    assert lib.b2l_flash_decoding_int4_workspace_bytes(4, 32, 8, 128, 48, 256) == 0
    a = lib.b2l_flash_decoding_int4_workspace_bytes(1, 32, 8, 128, 64, 64)
    assert 0 < a <= lib.b2l_flash_decoding_int4_workspace_bytes(32, 32, 8, 128, 64, 4096)


def test_slot_maps_oracle():
    table = [[10, 11, 12, 13], [20, 21, 22, 23]]
    assert O.slot_maps([1, 0], [2, 0], [2, 1], table, 4) == ([22, 23, 10, -1], [2, 3, 0, 0], [0, 2], [4, 1])
    O.slot_maps([1], [1], [2], table, 2, [7, 8])
    assert table[1] == [20, 7, 8, 23]
