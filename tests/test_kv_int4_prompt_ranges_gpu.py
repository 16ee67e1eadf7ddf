"""flash_attention_int4 over elements below the normal halves: each is off by 2^-25 at most, as documented."""

from __future__ import annotations

import math

import pytest
import torch

import kv_int4_oracle as O
from test_kv_int4_gpu import DTYPES, _normal
from test_kv_int4_prompt_gpu import LOOSE, _call, _run

pytestmark = pytest.mark.gpu


def _bound(q, rows, heads, group, scale):
    """``O.prompt_attention``, but for what lies below the halves' range: a value is off by 2^-25, and so is their mean under the weights;
    a weight by 2^-25; a key's element by 2^-25, so a score by that of the query's elements in absolute value, and the weights by 2 ln 2 of
    it (base 2)."""
    want, error = O.attention(q, rows, heads, group, scale)
    m, hq, d = q.shape
    n = rows.shape[0]
    k, v, _, _ = (t.repeat_interleave(hq // heads, 1) for t in O.values(rows, heads, d, group, q.dtype))
    x = q.double()
    seen = torch.arange(n, device=q.device) <= torch.arange(n - m, n, device=q.device)[:, None]
    p = torch.softmax((torch.einsum("mhd,nhd->hmn", x, k) * scale).masked_fill(~seen, -math.inf), -1)
    base2 = scale * math.log2(math.e)
    big = (torch.einsum("mhd,nhd->hmn", x.abs(), k.abs()) * base2).masked_fill(~seen, 0).amax(-1).T[..., None]
    small = (x.abs().sum(-1) * base2 * 2.0**-25)[..., None]
    weight = torch.einsum("hmn,nhd->mhd", p, v.abs())
    error = error + weight * (2.0**-11 * (2 + 2 * math.log(2) * big) + 2 * math.log(2) * small) * 1.01
    return want, error + 2.0**-25 * (1 + n * v.abs().amax(0))


def _check(step, heads, group, scale, max_len):
    q, rows, start, new, table, req, n = step
    out = _call(step, heads, group, scale, max_len=max_len)
    for s, m, r, c in zip(start.tolist(), new.tolist(), req.tolist(), n.tolist()):
        want, error = _bound(q[s:s + m], rows[table[r, :c].long()], heads, group, scale)
        ok = O.within(out[s:s + m], want, error)
        assert ok.all(), ((out[s:s + m].double() - want).abs().max().item(), want.abs().max().item(), (~ok).sum().item())


@pytest.mark.parametrize("new,lens,max_len", [([70, 3], [300, 9], 300), ([1400], [1500], LOOSE)], ids=["beside", "ready"])
@pytest.mark.parametrize("hq,heads,d,group", [(8, 2, 128, 64), (8, 2, 64, 32), (8, 2, 32, 32), (8, 2, 128, 128)])
@pytest.mark.parametrize("scale_v", [1e-4, 1e-5, 1e-6, 1e-7])
@pytest.mark.parametrize("dtype", DTYPES)
def test_small_values(dtype, scale_v, hq, heads, d, group, new, lens, max_len):
    _check(_run(new, lens, hq, heads, d, group, dtype, scale_v=scale_v), heads, group, d**-0.5, max_len)


@pytest.mark.parametrize("new,lens,max_len", [([70, 3], [300, 9], 300), ([1400], [1500], LOOSE)], ids=["beside", "ready"])
@pytest.mark.parametrize("scale_k", [1e-4, 1e-5, 1e-6])
def test_small_keys_under_large_queries(scale_k, new, lens, max_len):
    step = _run(new, lens, 8, 2, 128, 64, torch.bfloat16, scale_k=scale_k, q=(_normal(sum(new), 8, 128) / scale_k).bfloat16())
    _check(step, 2, 64, 0.088, max_len)


@pytest.mark.parametrize("new,lens,max_len", [([70, 3], [300, 9], 300), ([1400], [1500], LOOSE)], ids=["beside", "ready"])
def test_small_groups_beside_others(new, lens, max_len):
    """Groups of every size in one head, and constant ones, whose scale is zero."""
    q, rows, start, fresh, table, req, n = _run(new, lens, 8, 2, 128, 32, torch.bfloat16)
    k, v, _, _ = O.values(rows, 2, 128, 32, torch.bfloat16)
    size = torch.exp2(-torch.arange(0, 32, 8, device="cuda", dtype=torch.float64)).repeat_interleave(32)
    v = v * size
    v[::3, :, 96:] = 1e-6
    v[1::3, :, 64:96] = 0
    _check((q, O.rows_of(k.bfloat16(), v.bfloat16(), 32), start, fresh, table, req, n), 2, 32, 0.088, max_len)
