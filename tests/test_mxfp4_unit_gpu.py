"""The gated unit next to the borders of the 4-bit format: its codes are those of 64-bit arithmetic on the product's sums."""

from __future__ import annotations

import pytest
import torch

import mxfp4_borders as B
import mxfp4_oracle as O
from lite_llama_b200 import kernels as K
from lite_llama_b200.kernels._common import lib

pytestmark = pytest.mark.gpu
HALVES = (torch.float16, torch.bfloat16)


def weights(numbers, k):
    code, byte = B.rows(numbers, k)
    return O.pack_codes(code), byte


def gate_up(g, u, k):
    (gc, gb), (uc, ub) = weights(g, k), weights(u, k)
    return K.mxfp4_gate_up(gc, uc), K.mxfp4_gate_up(gb, ub)


def packed(codes, byte):
    return K.mxfp4_pack(codes.cuda(), byte.cuda())


# few tokens quantised inside, one part of k to eight, tiles of 32, 64 and 128 tokens; pairs, narrow and wide
@pytest.mark.parametrize("t,inner,k", ((1, 1024, 384), (7, 1024, 2048), (20, 1024, 384), (32, 512, 4096), (5, 256, 8192), (33, 1024, 1024), (64, 512, 4096), (65, 1024, 384),
                                       (128, 256, 8192), (300, 1024, 384), (1000, 4096, 384), (700, 4160, 416)))
@pytest.mark.parametrize("biased", (False, True))
def test_values_next_to_borders(t, inner, k, biased):
    numbers = B.sums(inner, t, biased)
    g, u, bg, bu = numbers
    w = packed(*gate_up(g, u, k))
    bias = K.mxfp4_gate_up(bg[:, None], bu[:, None]).flatten().half().cuda() if biased else None
    q = K.mxfp4_matmul(B.ones(t, k).half().cuda(), w, bias, swiglu=True)
    code, byte = (v.cuda() for v in B.wanted(*numbers))
    assert torch.equal(O.scale_rows(q.scales, t, inner), byte.expand(t, -1))
    assert torch.equal(O.unpack_codes(q.codes), code.expand(t, -1))


@pytest.mark.parametrize("t", (1, 9, 40, 100, 300))
@pytest.mark.parametrize("biased", (False, True))
def test_gates_whose_exponential_32_bits_have_not(t, biased):
    """Blocks of gates around -106, times millions: 1e-38, where 32 bits give zero.  Beside them blocks of zeros."""
    inner, k = 1024, 384
    gen = torch.Generator().manual_seed(t)
    g = B.kept(-104 - 4 * torch.rand(inner, generator=gen, dtype=torch.float64))
    u = B.kept(1e6 * (1 + torch.rand(inner, generator=gen, dtype=torch.float64)))
    bg, bu = torch.full_like(g, -0.5 if biased else 0.0), torch.zeros_like(g)
    empty = torch.arange(inner) // 32 % 4 == 1
    g, bg = torch.where(empty, 0.0, g), torch.where(empty, 0.0, bg)
    w = packed(*gate_up(g, u, k))
    bias = K.mxfp4_gate_up(bg[:, None], bu[:, None]).flatten().half().cuda() if biased else None
    q = K.mxfp4_matmul(B.ones(t, k).half().cuda(), w, bias, swiglu=True)
    code, byte = (v.cuda() for v in B.wanted(g, u, bg, bu))
    assert (code[:, ~empty] & 7).any() and not (code[:, empty] & 7).any()
    assert torch.equal(O.scale_rows(q.scales, t, inner), byte.expand(t, -1))
    assert torch.equal(O.unpack_codes(q.codes), code.expand(t, -1))


@pytest.mark.parametrize("tokens,tile", ((3, 64), (700, 64), (2000, 128), (3000, 256)))
@pytest.mark.parametrize("dtype", HALVES)
def test_experts_next_to_borders(tokens, tile, dtype):
    """The down projection is the identity, so that an expert's output is its quantised activations, exact in 16 bits."""
    experts, k = 8, 384
    assert lib().b2l_mxfp4_moe_tile_rows(tokens, experts, 2 * k) == tile
    numbers = [B.sums(k, 50 + e) for e in range(experts)]
    for n in numbers:                                                    # no blocks far below: fp16 does not reach there
        low = torch.arange(k) // 32 % 3 == 2
        n[0][low] = B.kept(n[0][low] / 10)
    both = [gate_up(g, u, k) for g, u, _, _ in numbers]
    w1 = packed(torch.stack([c for c, _ in both]), torch.stack([b for _, b in both]))
    one = torch.zeros(k, k, dtype=torch.uint8)
    one[range(k), range(k)] = 2
    w2 = packed(O.pack_codes(one).expand(experts, -1, -1).contiguous(), torch.full((experts, k, k // 32), 127, dtype=torch.uint8))
    want = torch.stack([O.values(*B.wanted(*n))[0] for n in numbers]).cuda()
    ids = torch.randint(0, experts, (tokens, 1), device="cuda")
    out = K.fused_moe_mxfp4(B.ones(tokens, k).to(dtype).cuda(), w1, w2, torch.ones(tokens, 1, device="cuda"), ids)
    expected = want[ids[:, 0]].to(dtype)
    assert torch.equal(out, expected)
