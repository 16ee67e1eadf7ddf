"""Routed experts in every form (tiles of 64, 128 and 256 rows): a slot's outputs are 32-bit sums, whatever lies beside them and however many tokens
there are."""

from __future__ import annotations

import math

import pytest
import torch

import mxfp4_oracle as O
from lite_llama_b200 import kernels as K
from lite_llama_b200.kernels._common import lib

pytestmark = pytest.mark.gpu
EXPERTS, INNER = 4, 576
FORMS = ((3, 64), (200, 64), (550, 128), (900, 256))      # tokens with two slots each, rows of a tile


def gate_up(experts, inner, hidden):
    gate, up = (torch.randn(experts, inner, hidden, device="cuda") * 0.05 for _ in range(2))
    return K.mxfp4_quantize_weight(K.mxfp4_gate_up(gate, up))


def down_values(w2):
    return O.values(O.unpack_codes(w2.codes), O.scale_rows(w2.scales, w2.rows, w2.k))


def slots(x, w1, w2, weights, ids, dtype):
    """(result in 64 bits, how far off it may be) from the framework's own quantised activations: each slot is a sum of exact products in 32 bits
    (at most one unit of the last place of the magnitudes' sum for each addition), the slots are multiplied and added up in 32 bits, and the
    result is rounded once."""
    down = down_values(w2)
    out, off = (torch.zeros(x.shape[0], w2.rows, dtype=torch.float64, device="cuda") for _ in range(2))
    for e in range(w1.codes.shape[0]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if not t.numel():
            continue
        q = K.mxfp4_matmul(x[t], K.MXFP4(w1.codes[e], w1.scales[e]), swiglu=True)
        act = O.values(O.unpack_codes(q.codes), O.scale_rows(q.scales, q.rows, q.k))
        w = weights[t, j].double()[:, None]
        y, size = act @ down[e].t(), act.abs() @ down[e].abs().t()
        out.index_add_(0, t, w * y)
        off.index_add_(0, t, w.abs() * (INNER * 2.0 ** -23 * size + 4 * 2.0 ** -24 * y.abs()))
    info = torch.finfo(dtype)
    return out, off + out.abs() * info.eps / 2 + info.smallest_normal * info.eps


def inputs(tokens, hidden, dtype, tile, experts=EXPERTS):
    x = torch.randn(tokens, hidden, device="cuda").to(dtype)
    top = torch.softmax(torch.randn(tokens, experts, device="cuda"), -1).topk(2, -1)
    assert lib().b2l_mxfp4_moe_tile_rows(2 * tokens, experts, 2 * INNER) == tile
    return x, top.values, top.indices


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("tokens,tile", FORMS)
@pytest.mark.parametrize("strong", (1.0, 30.0, 300.0, 1000.0))
def test_a_strong_output_costs_its_neighbours_nothing(dtype, tokens, tile, strong):
    """One output of 64 is up to a thousand times the others: those are as exact as ever."""
    hidden = 256
    x, weights, ids = inputs(tokens, hidden, dtype, tile)
    down = torch.randn(EXPERTS, hidden, INNER, device="cuda") * 0.01
    down[:, 13::64] *= strong
    w1, w2 = gate_up(EXPERTS, INNER, hidden), K.mxfp4_quantize_weight(down)
    want, off = slots(x, w1, w2, weights, ids, dtype)
    assert ((K.fused_moe_mxfp4(x, w1, w2, weights, ids).double() - want).abs() <= off).all()


@pytest.mark.parametrize("tokens,tile", FORMS)
@pytest.mark.parametrize("hidden", (32, 96, 160, 256, 2048))
def test_any_number_of_outputs(tokens, tile, hidden):
    x, weights, ids = inputs(tokens, hidden, torch.bfloat16, tile)
    w1, w2 = gate_up(EXPERTS, INNER, hidden), K.mxfp4_quantize_weight(torch.randn(EXPERTS, hidden, INNER, device="cuda") * 0.05)
    want, off = slots(x, w1, w2, weights, ids, torch.bfloat16)
    assert ((K.fused_moe_mxfp4(x, w1, w2, weights, ids).double() - want).abs() <= off).all()


@pytest.mark.parametrize("tokens,tile", FORMS)
def test_outputs_at_both_ends_of_32_bits(tokens, tile):
    """bf16 outputs up to 2^127 and down to 2^-121, in blocks of their own."""
    hidden = 256
    x, weights, ids = inputs(tokens, hidden, torch.bfloat16, tile)
    weights = torch.ones_like(weights) / 2
    w1 = gate_up(EXPERTS, INNER, hidden)
    down = torch.randn(EXPERTS, hidden, INNER, device="cuda") * 0.01
    pair = K.mxfp4_quantize_weight(down)
    values, peak = down_values(pair), 0.0
    for e in range(EXPERTS):                                             # the largest slot
        q = K.mxfp4_matmul(x[(ids == e).any(1)], K.MXFP4(w1.codes[e], w1.scales[e]), swiglu=True)
        act = O.values(O.unpack_codes(q.codes), O.scale_rows(q.scales, q.rows, q.k))
        peak = max(peak, (act @ values[e, :64].t()).abs().max().item() if q.rows else 0.0)
    byte = O.scale_rows(pair.scales, hidden, INNER).int()
    up = math.floor(127.9 - math.log2(peak))
    byte[:, :64] += up
    byte[:, 64:128] += up - 3
    byte[:, 128:192] -= 112
    assert byte.min() >= 1 and byte.max() <= 254
    w2 = K.mxfp4_pack(pair.codes, byte.to(torch.uint8))
    want, off = slots(x, w1, w2, weights, ids, torch.bfloat16)
    assert 2.0 ** 125 < want.abs().max() < 2.0 ** 127.9 and want[:, 128:192].abs().amax() < 2.0 ** -105
    got = K.fused_moe_mxfp4(x, w1, w2, weights, ids)
    assert ((got.double() - want).abs() <= off).all()
    assert (got[:, 128:192] != 0).float().mean() > 0.99


@pytest.mark.parametrize("tokens,tile", FORMS)
def test_sums_beyond_32_bits_are_infinite(tokens, tile):
    hidden = 256
    x, weights, ids = inputs(tokens, hidden, torch.float16, tile)
    x = x.abs() + 1
    gate = torch.full((EXPERTS, INNER, hidden), 0.25, device="cuda")
    w1 = K.mxfp4_quantize_weight(K.mxfp4_gate_up(gate, gate))             # activations far above 1
    code = torch.zeros(EXPERTS, hidden, INNER, dtype=torch.uint8, device="cuda")
    byte = torch.full((EXPERTS, hidden, INNER // 32), 127, dtype=torch.uint8, device="cuda")
    code[:, :, 5] = 2
    code[:, 70, 5], code[:, 201, 5] = 7, 15
    byte[:, 70], byte[:, 201] = 253, 253
    w2 = K.mxfp4_pack(O.pack_codes(code), byte)
    got = K.fused_moe_mxfp4(x, w1, w2, weights, ids)
    plain = torch.ones(hidden, dtype=torch.bool, device="cuda")
    plain[70] = plain[201] = False
    assert (got[:, 70] == float("inf")).all() and (got[:, 201] == -float("inf")).all()
    code[:, 70], code[:, 201] = 0, 0
    byte[:, 70], byte[:, 201] = 127, 127
    other = K.fused_moe_mxfp4(x, w1, K.mxfp4_pack(O.pack_codes(code), byte), weights, ids)
    assert torch.equal(got[:, plain], other[:, plain]) and other.isfinite().all()
