"""The 4-bit cache in plain torch, in 64 bits: rows from values, values from rows, attention over rows, slot maps."""

from __future__ import annotations

import math

import torch


def row_bytes(kv_heads: int, d: int, group: int) -> int:
    return (kv_heads * (d + 8 * (d // group)) + 15) // 16 * 16


def quantise(x: torch.Tensor, group: int):
    """``x [..., D]`` -> codes ``[..., D/group, group]`` uint8, (scale, minimum) in ``x``'s type."""
    g = x.double().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = (((hi - lo) / 16).float() / 0.9375).to(x.dtype)   # the 32-bit quotient by 15, rounded (a range of bf16 may pass 32 bits)
    s = scale.double()[..., None]
    code = torch.where(s > 0, (g - lo[..., None]) / torch.where(s > 0, s, 1.0), 0.0).round().clamp(0, 15)
    bad = ~torch.isfinite(g).all(-1)
    scale, lo = scale.masked_fill(bad, math.nan), lo.to(x.dtype).masked_fill(bad, math.nan)
    return code.masked_fill(bad[..., None], 0).to(torch.uint8), scale, lo


def rows_of(k: torch.Tensor, v: torch.Tensor, group: int) -> torch.Tensor:
    """Cache rows of ``k, v [tokens, heads, D]``, byte by byte as documented."""
    n, heads, d = k.shape
    out = torch.zeros(n, row_bytes(heads, d, group), dtype=torch.uint8, device=k.device)
    per_head, groups = d + 8 * (d // group), d // group
    for h in range(heads):
        at = h * per_head
        for side, x in enumerate((k[:, h], v[:, h])):
            code, scale, lo = quantise(x, group)
            code = code.reshape(n, d)
            out[:, at + side * d // 2:at + (side + 1) * d // 2] = code[:, 0::2] | (code[:, 1::2] << 4)
            params = torch.stack((scale, lo), -1).reshape(n, 2 * groups).contiguous().view(torch.uint8)
            out[:, at + d + side * 4 * groups:at + d + (side + 1) * 4 * groups] = params
    return out


def values(rows: torch.Tensor, heads: int, d: int, group: int, dtype: torch.dtype):
    """``(k, v, reach)`` of rows ``[n, bytes]`` in 64 bits, ``[n, heads, D]``; reach = 15 scale + |minimum|, what an element's parts sum up to."""
    n, per_head, groups = rows.shape[0], d + 8 * (d // group), d // group
    r = rows[:, :heads * per_head].reshape(n, heads, per_head)
    out, reach = [], []
    for side in (0, 1):
        byte = r[..., side * d // 2:(side + 1) * d // 2].long()
        code = torch.stack((byte % 16, byte // 16), -1).reshape(n, heads, groups, group).double()
        params = r[..., d + side * 4 * groups:d + (side + 1) * 4 * groups].contiguous().view(dtype).view(n, heads, groups, 2).double()
        out.append((code * params[..., :1] + params[..., 1:]).reshape(n, heads, d))
        reach.append((15 * params[..., :1].abs() + params[..., 1:].abs()).expand(-1, -1, -1, group).reshape(n, heads, d))
    return out[0], out[1], reach[0], reach[1]


def attention(q, rows, heads: int, group: int, scale: float):
    """``q [m, Hq, D]``, the last ``m`` tokens of the sequence ``rows``; causal.  ``(out, error)``: error bounds what 32-bit sums and exponentials
    may be off, before the result's rounding: a score's products add up to at most A (its parts in absolute value) in fewer than
    32 sums that each lose 2^-23 of that, in base 2; the weights are off by as much and by 2^-21 for exponentials, for what is left of
    their rounding and for the sums, and so is each value's part."""
    m, hq, d = q.shape
    n, dtype = rows.shape[0], q.dtype
    if n == 0:
        return torch.zeros(m, hq, d, dtype=torch.float64, device=q.device), torch.zeros(m, hq, d, dtype=torch.float64, device=q.device)
    k, v, k_reach, v_reach = (t.repeat_interleave(hq // heads, 1) for t in values(rows, heads, d, group, dtype))
    x = q.double()
    s = torch.einsum("mhd,nhd->hmn", x, k) * scale
    seen = torch.arange(n, device=q.device) <= torch.arange(n - m, n, device=q.device)[:, None]
    s = s.masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    p = torch.where(seen.any(-1)[None, :, None], p, torch.zeros_like(p))      # a query that sees nothing
    big = (torch.einsum("mhd,nhd->hmn", x.abs(), k_reach) * scale * math.log2(math.e)).masked_fill(~seen, 0).amax(-1)   # [h, m]
    out = torch.einsum("hmn,nhd->mhd", p, v)
    weight = torch.einsum("hmn,nhd->mhd", p, v_reach)
    return out, weight * ((64 * 2.0**-23 * big + 2.0**-20).T[..., None])


def prompt_attention(q, rows, heads: int, group: int, scale: float):
    """``(out, error)`` as ``attention``, for operands and weights of 16 bits: keys, values, weights (and bf16 queries not at all) are rounded to
    halves, off by 2^-11 of themselves, so a score is off by 2^-11 of A' (its products in absolute value, base 2) and every weight by
    2 ln 2 times that and 2^-11, each value by 2^-11; what lies below the halves' range is off by 2^-25 a weight and a value, where weights
    are scaled up to 2^8."""
    out, error = attention(q, rows, heads, group, scale)
    m, hq, d = q.shape
    n = rows.shape[0]
    if n == 0:
        return out, error
    k, v, _, _ = (t.repeat_interleave(hq // heads, 1) for t in values(rows, heads, d, group, q.dtype))
    x = q.double()
    seen = torch.arange(n, device=q.device) <= torch.arange(n - m, n, device=q.device)[:, None]
    p = torch.nan_to_num(torch.softmax((torch.einsum("mhd,nhd->hmn", x, k) * scale).masked_fill(~seen, -math.inf), -1))
    big = (torch.einsum("mhd,nhd->hmn", x.abs(), k.abs()) * scale * math.log2(math.e)).masked_fill(~seen, 0).amax(-1).T[..., None]
    weight = torch.einsum("hmn,nhd->mhd", p, v.abs())
    tiny = n * 2.0**-25 * (v.abs().amax(0) + 1)
    return out, error + weight * 2.0**-11 * (2 + 2 * math.log(2) * big) * 1.01 + tiny


def within(got: torch.Tensor, want: torch.Tensor, error: torch.Tensor) -> torch.Tensor:
    """Where ``got`` is a rounding of something within ``error`` of ``want`` (64 bits)."""
    fi = torch.finfo(got.dtype)
    half_step = (want.abs() + error) * fi.eps / 2 + fi.smallest_normal * fi.eps / 2
    return (got.double() - want).abs() <= half_step + error


def slot_maps(req, ctx, new, table, total, pool=None):
    """Plain loops over Python ints; ``table`` is a list of lists and is changed."""
    rows, pos, start, length, at = [-1] * total, [0] * total, [], [], 0
    for r, c, n in zip(req, ctx, new):
        c, n = max(c, 0), max(n, 0)
        start.append(at)
        length.append(c + n)
        for j in range(n):
            t = at + j
            if t >= total:
                break
            pos[t] = c + j
            if 0 <= r < len(table) and c + j < len(table[r]):
                if pool is not None:
                    table[r][c + j] = pool[t]
                rows[t] = table[r][c + j]
        at += n
    return rows, pos, start, length
