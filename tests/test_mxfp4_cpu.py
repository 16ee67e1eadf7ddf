"""Microscaled 4-bit floating point without a GPU: the oracle against the format's own rules, the layout, and refusals."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mxfp4_oracle as O
from lite_llama_b200 import _lib
from lite_llama_b200 import kernels as K
from lite_llama_b200.quantization import LINEAR_METHODS, make_linear_weights


# ------------------------------------------------------------------------------------------------- the oracle
def test_the_oracle_rounds_to_the_nearest_with_ties_to_the_even_code():
    t = torch.tensor([0.0, 0.25, 0.26, 0.5, 0.75, 1.0, 1.25, 1.26, 1.5, 1.75, 2.0, 2.5, 2.51, 3.0, 3.5, 4.0, 5.0, 5.01, 6.0, 7.9])
    want = torch.tensor([0, 0, 1, 1, 2, 2, 2, 3, 3, 4, 4, 4, 5, 5, 6, 6, 6, 7, 7, 7])
    x = torch.zeros(2, 32)
    x[0, :20], x[1, :20] = t, -t
    code, byte = O.quantise(x)
    assert torch.equal(byte, torch.full((2, 1), 127, dtype=torch.uint8))
    assert torch.equal(code[0, :20].long(), want) and torch.equal(code[1, :20].long() & 7, want)
    assert (O.values(code, byte)[0, :20] - t.double()).abs()[t <= 6].max() <= 1


def test_the_oracles_scale_is_the_power_of_two_below_the_largest_over_four():
    top = torch.tensor([1.0, 1.99, 2.0, 2.0 ** -126, 2.0 ** -130, 0.0, float("inf"), float("nan"), 3e38])
    x = torch.zeros(9, 32)
    x[:, 7] = top
    code, byte = O.quantise(x)
    assert byte[:, 0].tolist() == [125, 125, 126, 0, 0, 0, 255, 255, 252]
    assert not code[6:8].any()
    assert O.values(code, byte)[6:8].isnan().all()


def test_scale_tiles_hold_every_row_and_block_once():
    rows, k = 300, 32 * 11
    byte = torch.randint(0, 256, (2, rows, 11), dtype=torch.uint8)
    codes = torch.randint(0, 256, (2, rows, k // 2), dtype=torch.uint8)
    q = K.mxfp4_pack(codes, byte)
    assert q.scales.shape == (2, 3, 3, 32, 4, 4) and q.rows == rows and q.k == k and q.ready
    assert torch.equal(O.scale_rows(q.scales, rows, k), byte)
    assert q.scales.long().sum() == byte.long().sum()                    # and zeros elsewhere
    assert _lib.load().b2l_mxfp4_scale_bytes(rows, k) == q.scales[0].numel()
    assert q.nbytes() == codes.numel() + q.scales.numel()


def test_gate_and_up_rows_alternate_in_runs():
    gate, up = torch.arange(192.0)[:, None].repeat(1, 32), -torch.arange(192.0)[:, None].repeat(1, 32) - 1
    w = K.mxfp4_gate_up(gate, up)
    assert w.shape == (384, 32)
    assert torch.equal(w[64:128], up[:64]) and torch.equal(w[128:192], gate[64:128]) and torch.equal(w[320:], up[128:])
    stack = K.mxfp4_gate_up(gate.expand(3, 192, 32), up.expand(3, 192, 32))
    assert torch.equal(stack[2], w)


# ------------------------------------------------------------------------------------------------- refusals
def test_the_method_is_offered():
    assert "mxfp4" in LINEAR_METHODS
    with pytest.raises(ValueError, match="CUDA tensors only"):
        make_linear_weights(torch.zeros(64, 64), "mxfp4")


def packed(n=8, k=64):
    return K.mxfp4_pack(torch.zeros(n, k // 2, dtype=torch.uint8), torch.zeros(n, k // 32, dtype=torch.uint8))


def test_python_refusals():
    x = torch.zeros(2, 64, dtype=torch.float16)
    for call in (lambda: K.mxfp4_quantize(x), lambda: K.mxfp4_dequantize(packed()), lambda: K.mxfp4_matmul(x, packed()),
                 lambda: K.skip_rmsnorm_mxfp4(x, None, x[0]), lambda: K.fused_moe_mxfp4(x, packed(), packed(), x, x)):
        with pytest.raises(ValueError):
            call()
    for call, what in ((lambda: K.mxfp4_pack(torch.zeros(2, 16), torch.zeros(2, 1, dtype=torch.uint8)), "uint8"),
                       (lambda: K.mxfp4_pack(torch.zeros(2, 24, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8)), "belong"),
                       (lambda: K.mxfp4_pack(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)), "belong"),
                       (lambda: K.mxfp4_gate_up(torch.zeros(32, 64), torch.zeros(32, 64)), "multiple of 64"),
                       (lambda: K.mxfp4_gate_up(torch.zeros(64, 64), torch.zeros(64, 32)), "alike"),
                       (lambda: K.mxfp4_matmul(x, x), "must be MXFP4"), (lambda: K.mxfp4_dequantize(x), "must be MXFP4"),
                       (lambda: K.fused_moe_mxfp4(x, x, x, x, x), "must be MXFP4")):
        with pytest.raises(ValueError, match=what):
            call()


def test_host_entries_refuse_before_any_launch():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 127) // 128 * 128
    f = ctypes.c_float(1e-5)
    refused = [
        ("multiple of 32", lib.b2l_mxfp4_quantize, (p, p, p, 1, 1, 33, 40, 0, None)),
        ("null", lib.b2l_mxfp4_quantize, (None, p, p, 1, 1, 32, 32, 0, None)),
        ("16 bytes", lib.b2l_mxfp4_quantize, (p, p, p + 2, 1, 1, 32, 32, 0, None)),
        ("16 bytes", lib.b2l_mxfp4_quantize, (p, p, p, 1, 2, 32, 33, 0, None)),
        ("dtype", lib.b2l_mxfp4_quantize, (p, p, p, 1, 1, 32, 32, 7, None)),
        ("multiple of 32", lib.b2l_mxfp4_dequantize, (p, p, p, 1, 1, 16, 8, 0, None)),
        ("16384", lib.b2l_skip_rmsnorm_mxfp4, (p, p, p, p, p, p, 1, 16416, 16416, 16416, 16416, f, 0, None)),
        ("null", lib.b2l_skip_rmsnorm_mxfp4, (p, p, None, p, p, p, 1, 32, 32, 32, 32, f, 0, None)),
        ("dtype", lib.b2l_skip_rmsnorm_mxfp4, (p, p, p, p, p, p, 1, 32, 32, 32, 32, f, 2, None)),
        ("multiple of 32", lib.b2l_mxfp4_matmul, (p, None, p, p, p, p, None, 1, 8, 48, 32, 32, 8, 0, 0, 0, None)),
        ("runs of 64", lib.b2l_mxfp4_matmul, (p, p, p, p, p, p, None, 1, 64, 64, 32, 32, 16, 1, 0, 0, None)),
        ("null", lib.b2l_mxfp4_matmul, (p, None, p, p, p, p, None, 1, 128, 64, 32, 32, 32, 1, 0, 0, None)),
        ("16 bytes", lib.b2l_mxfp4_matmul, (p, None, p, p, p, p, None, 2, 8, 64, 24, 32, 8, 0, 0, 0, None)),
        ("quantiser first", lib.b2l_mxfp4_matmul, (p, None, p, None, p, p, None, 9, 8, 64, 64, 32, 8, 0, 0, 0, None)),
        ("dtype", lib.b2l_mxfp4_matmul, (p, None, p, p, p, p, None, 1, 8, 64, 32, 32, 8, 0, 0, 2, None)),
        ("tiles of", lib.b2l_mxfp4_grouped_matmul, (p, p, p, p, p, p, p, 1, 16, 1, 32, 64, 0, None)),
        ("units of 32", lib.b2l_mxfp4_grouped_matmul, (p, p, p, p, p, p, p, 1, 128, 1, 40, 64, 0, None)),
        ("null", lib.b2l_mxfp4_grouped_matmul, (p, None, p, p, p, p, p, 1, 128, 1, 32, 64, 0, None)),
        ("over 5000 experts", lib.b2l_mxfp4_moe_scatter, (p, p, p, p, p, p, 8, 1, 1, 64, 5000, 64, 64, 0, None)),
        ("int32 or int64", lib.b2l_mxfp4_moe_scatter, (p, p, p, p, p, p, 2, 1, 1, 64, 8, 64, 64, 0, None)),
        ("16777216 tokens", lib.b2l_mxfp4_moe_scatter, (p, p, p, p, p, p, 8, 1 << 24, 1, 64, 8, 64, 64, 0, None)),
        ("tiles of 48", lib.b2l_mxfp4_moe_scatter, (p, p, p, p, p, p, 8, 1, 1, 48, 8, 64, 64, 0, None)),
        ("null", lib.b2l_mxfp4_moe_scatter, (p, p, p, p, p, None, 8, 1, 1, 64, 8, 64, 64, 0, None)),
        ("multiple of 8", lib.b2l_mxfp4_moe_combine, (p, p, p, p, p, 0, 1, 1, 12, 0, None)),
    ]
    for what, entry, args in refused:
        rc = entry(*args)
        assert rc < 0 and what in lib.b2l_last_error().decode(), (what, rc, lib.b2l_last_error())
    # nothing to do is no error
    assert lib.b2l_mxfp4_quantize(None, None, None, 1, 0, 32, 32, 0, None) == 0
    assert lib.b2l_mxfp4_matmul(None, None, None, None, None, None, None, 0, 8, 64, 32, 32, 8, 0, 0, 0, None) == 0


def test_tiles_of_experts_hold_every_split_of_the_slots():
    lib = _lib.load()
    gen = torch.Generator().manual_seed(0)
    for slots, experts, rows in ((1, 1, 64), (5, 128, 64), (256, 128, 64), (6000, 150, 64), (1000, 7, 128), (16000, 128, 128), (33, 32, 64), (50000, 128, 256)):
        tile = lib.b2l_mxfp4_moe_tile_rows(slots, experts, 1536)
        assert tile == rows
        most = lib.b2l_mxfp4_moe_max_tiles(slots, tile, experts)
        for _ in range(20):
            skew = torch.rand(experts, generator=gen) ** 4 + 1e-9
            counts = torch.bincount(torch.multinomial(skew, slots, True, generator=gen), minlength=experts)
            assert int(((counts + tile - 1) // tile).sum()) <= most


def test_products_that_quantise_their_rows_have_room_for_them():
    """A CTA's part is at most 24 rows of 256 elements, by the same division as the launch."""
    lib = _lib.load()
    assert lib.b2l_mxfp4_matmul_takes_16bit(1, 6144, 4096) and lib.b2l_mxfp4_matmul_takes_16bit(3, 4096, 14336)
    assert not lib.b2l_mxfp4_matmul_takes_16bit(4, 4096, 14336) and lib.b2l_mxfp4_matmul_takes_16bit(8, 9728, 896)
    assert not lib.b2l_mxfp4_matmul_takes_16bit(9, 6144, 4096) and not lib.b2l_mxfp4_matmul_takes_16bit(0, 6144, 4096)
    assert lib.b2l_mxfp4_matmul_takes_16bit(1, 40000, 24 * 256) and not lib.b2l_mxfp4_matmul_takes_16bit(1, 40000, 24 * 256 + 32)
