"""Microscaled 4-bit floating point in 64 bits: what the operators' results are held against."""

from __future__ import annotations

import torch

MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantise(x: torch.Tensor):
    """``x [..., k]`` -> (codes one per byte ``[..., k]``, scale bytes ``[..., k / 32]``), by search among the eight magnitudes."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    bad = ~b.isfinite().all(-1)
    top = torch.where(bad, torch.ones_like(top), top)
    exponent = torch.frexp(top)[1] - 1                                   # of the power of two not above it
    byte = torch.where(top > 0, (exponent - 2 + 127).clamp(0, 254), torch.zeros_like(exponent))
    t = torch.where(bad[..., None], torch.zeros_like(b), b) * torch.exp2(127.0 - byte.double())[..., None]
    m = t.abs().clamp(max=6.0)
    grid = MAGNITUDES.to(x.device)
    far = (m[..., None] - grid).abs()                                    # exact: t has few bits more than the grid
    best = far.argmin(-1)                                                # a tie: the first is the lower code
    upper = (best + 1).clamp(max=7)
    tie = far.gather(-1, upper[..., None])[..., 0] == far.gather(-1, best[..., None])[..., 0]
    code = torch.where(tie & (upper > best) & (best % 2 == 1), upper, best)
    code = code + 8 * (torch.signbit(t)).long()
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    return code.flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def values(code: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    grid = MAGNITUDES.to(code.device)
    v = grid[(code & 7).long()] * torch.where(code >= 8, -1.0, 1.0)
    scale = torch.exp2(byte.double() - 127)
    scale = torch.where(byte == 255, torch.full_like(scale, float("nan")), scale)
    return (v.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def rounded(x: torch.Tensor) -> torch.Tensor:
    return values(*quantise(x))


def pack_codes(code: torch.Tensor) -> torch.Tensor:
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous()


def unpack_codes(codes: torch.Tensor) -> torch.Tensor:
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


def scale_rows(tiles: torch.Tensor, rows: int, k: int) -> torch.Tensor:
    """Scale bytes ``[..., rows, k / 32]`` of tiles, one index at a time."""
    r, b = torch.arange(rows, device=tiles.device)[:, None], torch.arange(k // 32, device=tiles.device)
    return tiles[..., r // 128, b // 4, r % 32, r % 128 // 32, b % 4]


def norm(x, residual, weight, eps):
    total = x.double() if residual is None else x.double() + residual.double()
    return total / torch.sqrt(total.square().mean(-1, keepdim=True) + eps) * weight.double(), total


def product_bound(x: torch.Tensor, w: torch.Tensor, y: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """How far a product of exact operands may be off: each of k additions in 32 bits loses at most one unit of the last place (the
    tensor cores may cut instead of round) of a partial sum, which no partial sum of magnitudes exceeds; then the rounding of the result
    (or half of the smallest step below the normal numbers)."""
    sums = x.double().abs() @ w.double().abs().transpose(-1, -2)
    info = torch.finfo(dtype)
    return x.shape[-1] * 2.0 ** -23 * sums + y.abs() * info.eps / 2 + info.smallest_normal * info.eps / 2


def slot_bound(x: torch.Tensor, w: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """The same for an expert's output that is held as a whole number of up to 32767 with a scale for 64: the sums' error; half a step of
    the block's largest / 32767, which may itself be off by its sum's error; and five roundings in 32 bits on the way there and back (the
    factor by a division of two units, the scale, its product with a weight)."""
    sums = x.shape[-1] * 2.0 ** -23 * (x.double().abs() @ w.double().abs().transpose(-1, -2))
    n = y.shape[-1]
    high = torch.nn.functional.pad(y.abs() + sums, (0, -n % 64)).unflatten(-1, (-1, 64)).amax(-1).repeat_interleave(64, -1)[..., :n]
    return sums + high / 65534 + (y.abs() + high / 65534) * 2.0 ** -20 + 2.0 ** -110
