"""Gated units whose activations lie next to the borders of the 4-bit format.

``silu(gate) * up`` is quantised from the product's sums.  Here every sum is a number of the test's choice: a row of weights has one element
in each of twelve blocks, digit j of a number of 24 bits to the base 4 with the scale 4^j, and every token has ones in those places.  All
partial sums are whole multiples of the last digit below 2^24 of it, so they are exact in 32 bits in any order."""

from __future__ import annotations

import torch

import mxfp4_oracle as O

BITS, DIGITS = 22, 12
TARGETS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
CODE = torch.tensor([0, 2, 4, 5], dtype=torch.uint8)      # 0, 1, 2, 3


def kept(v: torch.Tensor) -> torch.Tensor:
    """64-bit numbers rounded to 22 bits."""
    m, e = torch.frexp(v)
    return torch.ldexp(torch.round(torch.ldexp(m, torch.tensor(BITS))), e - BITS)


def rows(v: torch.Tensor, k: int):
    """Numbers of 22 bits -> (codes one per byte ``[n, k]``, scale bytes ``[n, k / 32]``) of rows that add up to them."""
    m, e = torch.frexp(v.double())
    whole, e = torch.ldexp(m, torch.tensor(BITS)).abs().long(), e.long() - BITS
    odd = e % 2 != 0
    whole, e = torch.where(odd, 2 * whole, whole), torch.where(odd, e - 1, e)
    code = torch.zeros(len(v), k, dtype=torch.uint8)
    byte = torch.full((len(v), k // 32), 127, dtype=torch.uint8)
    for j in range(DIGITS):
        digit = CODE[(whole >> (2 * j)) & 3]
        code[:, 32 * j] = torch.where(digit > 0, digit + 8 * (v < 0), 0).to(torch.uint8)
        place = e + 2 * j + 127
        used = digit > 0
        assert ((place >= 1) & (place <= 250))[used].all()
        byte[:, j] = place.clamp(1, 250).to(torch.uint8)
    return code, byte


def ones(t: int, k: int) -> torch.Tensor:
    x = torch.zeros(t, k)
    x[:, :32 * DIGITS:32] = 1
    return x


def silu(g: torch.Tensor) -> torch.Tensor:
    return g / (1 + torch.exp(-g))


def sums(inner: int, seed: int, biased: bool = False):
    """(gate sums, up sums, gate biases, up biases), 64-bit ``[inner]``: in turn blocks whose largest magnitude is 64 and whose other values lie within some
    2^-22 of a border, blocks whose largest lies that near to a power of two, and blocks far below."""
    gen = torch.Generator().manual_seed(seed)
    uniform = lambda lo, hi: lo + (hi - lo) * torch.rand(inner, generator=gen, dtype=torch.float64)  # noqa: E731
    number = torch.arange(inner)
    kind, first = number // 32 % 3, number % 32 == 0
    sign = torch.where(torch.rand(inner, generator=gen) < 0.5, -1.0, 1.0).double()
    g = kept(torch.where(torch.rand(inner, generator=gen) < 0.5, uniform(0.5, 12.0), uniform(-18.0, -0.5)))
    g = torch.where(kind == 2, kept(uniform(-100.0, -60.0)), g)
    bg = bu = torch.zeros(inner, dtype=torch.float64)
    if biased:
        bg, bu = uniform(-1, 1).half().double(), uniform(-1, 1).half().double()
    border = torch.tensor(TARGETS, dtype=torch.float64)[torch.randint(0, 7, (inner,), generator=gen)] * 16
    border = torch.where(kind == 1, torch.where(first, 64.0, border / 8), border)
    nudge = torch.ldexp(torch.randint(-1, 2, (inner,), generator=gen).double(), torch.tensor(-BITS))
    u = kept((sign * border / silu(g + bg)) * (1 + nudge) - bu)
    u = torch.where(kind == 2, kept(uniform(1, 1e4)) * sign, u)
    anchor = (kind == 0) & first
    g, u = torch.where(anchor, 64.0 - bg, g), torch.where(anchor, 1.0 - bu, u)      # silu(64) is 64 in 64 bits
    if biased:                                                                      # sums of 22 bits there, too
        bg, bu = torch.where(anchor, 0.0, bg), torch.where(anchor, 0.0, bu)
        g, u = torch.where(anchor, 64.0, g), torch.where(anchor, 1.0, u)
    return g, u, bg, bu


def wanted(g, u, bg, bu):
    """(codes, scale bytes) of the row of activations."""
    return O.quantise((silu(g + bg) * (u + bu))[None])
