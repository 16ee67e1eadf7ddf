"""flash_decoding_int4 over values whose scales lie far apart: by token, by group and by head, in any order (bounds: kv_int4_oracle.attention)."""

from __future__ import annotations

import pytest
import torch

import kv_int4_oracle as O
from lite_llama_b200 import kernels as K
from test_kv_int4_gpu import DTYPES, _normal

pytestmark = pytest.mark.gpu
SHAPES = [(8, 2, 128, 64), (16, 2, 128, 64), (4, 1, 128, 32), (8, 1, 64, 32), (9, 1, 64, 64), (4, 1, 128, 128), (8, 2, 32, 32)]


def _run(log2_weight, v, hq, heads, group, dtype, other=None):
    """A cache whose token t has the weight 2^log2_weight[t], up to a common factor; the heads of the upper half: other[t]."""
    n, d = v.shape[0], v.shape[2]
    k = torch.zeros(n, heads, d, device="cuda")
    k[:, :, 0] = log2_weight[:, None] / 8
    k[:, :, 1] = (log2_weight if other is None else other)[:, None] / 8
    q = torch.zeros(1, hq, d, device="cuda")
    q[0, :(hq + 1) // 2, 0] = q[0, (hq + 1) // 2:, 1] = 8.0
    q += _normal(1, hq, d) * 0.01
    rows = O.rows_of(k.to(dtype), v.to(dtype), group)
    table = torch.randperm(n, device="cuda", dtype=torch.int32)
    cache = torch.empty_like(rows)
    cache[table.long()] = rows
    one, q, scale = torch.ones(1, dtype=torch.int32, device="cuda"), q.to(dtype), 0.6931
    out = K.flash_decoding_int4(q, cache, scale, table[None], 0 * one, n * one, n, heads, group)
    want, error = O.attention(q, rows, heads, group, scale)
    assert torch.isfinite(want).all()
    ok = O.within(out, want, error)
    assert ok.all(), ((out.double() - want).abs().max().item(), (~ok).sum().item(), ok.numel())


@pytest.mark.parametrize("hq,heads,d,group", SHAPES)
@pytest.mark.parametrize("apart", [16, 20, 24, 28])
@pytest.mark.parametrize("where", ["first", "last", "middle"])
@pytest.mark.parametrize("n", [33, 700])
def test_a_wide_value_of_little_weight(n, where, apart, hq, heads, d, group):
    """Its products are no larger than the others': their digits stay."""
    at = {"first": 0, "last": n - 1, "middle": n // 2}[where]
    for dtype, wide in ((torch.float16, 4000.0), (torch.bfloat16, 1e6)):
        weight = torch.zeros(n, device="cuda")
        weight[at] = -float(apart)
        v = _normal(n, heads, d) * wide * 2.0**-apart
        v[at] *= 2.0**apart
        _run(weight, v, hq, heads, group, dtype)


@pytest.mark.parametrize("hq,heads,d,group", SHAPES)
@pytest.mark.parametrize("n", [40, 700])
def test_scales_that_fall_while_scores_rise(n, hq, heads, d, group):
    """Every token's products are level, each scale a little smaller than the one before; and the other way round."""
    for dtype, span in ((torch.float16, 26), (torch.bfloat16, 60)):
        fall = torch.linspace(0, span, n, device="cuda")
        for order in (fall, fall.flip(0), fall[torch.randperm(n, device="cuda")]):
            v = _normal(n, heads, d) * (torch.exp2(-order) * 2000)[:, None, None]
            _run(order - span, v, hq, heads, group, dtype)


@pytest.mark.parametrize("hq,heads,d,group", SHAPES)
def test_a_late_high_score_of_a_narrow_value(hq, heads, d, group):
    for n, at in ((20, 17), (300, 290)):
        weight = torch.full((n,), -30.0, device="cuda")
        weight[at] = 0
        for dtype in DTYPES:
            v = _normal(n, heads, d) * 1000
            v[at] *= 2.0**-27
            _run(weight, v, hq, heads, group, dtype)


@pytest.mark.parametrize("hq,heads,d,group", [s for s in SHAPES if s[2] > s[3]])
def test_one_wide_group_beside_narrow_ones(hq, heads, d, group):
    for n in (17, 400):
        for wide in range(d // group):
            v = _normal(n, heads, d)
            v[..., :wide * group] *= 2.0**-20
            v[..., (wide + 1) * group:] *= 2.0**-20
            for dtype in DTYPES:
                _run(torch.zeros(n, device="cuda"), v * 1000, hq, heads, group, dtype)


@pytest.mark.parametrize("hq,heads,d,group", SHAPES)
def test_heads_that_weigh_the_wide_value_differently(hq, heads, d, group):
    """It is everything to one half of the heads and nothing to the other."""
    for n, at in ((33, 5), (500, 499)):
        mine, other = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        mine[at], other[at] = 4.0, -26.0
        for dtype in DTYPES:
            v = _normal(n, heads, d) * 2000 * 2.0**-26
            v[at] *= 2.0**26
            _run(mine, v, hq, heads, group, dtype, other)


@pytest.mark.parametrize("magnitude", [1e-37, 1e-30, 1e30, 1e34])
def test_values_at_the_ends_of_bf16(magnitude):
    for hq, heads, d, group in SHAPES:
        for n in (5, 130):
            _run(torch.zeros(n, device="cuda"), _normal(n, heads, d) * magnitude, hq, heads, group, torch.bfloat16)
