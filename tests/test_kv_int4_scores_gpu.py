"""flash_decoding_int4 where one element of a query or one channel of the keys is far larger than the others (bounds: kv_int4_oracle.attention)."""

from __future__ import annotations

import pytest
import torch

import kv_int4_oracle as O
from lite_llama_b200 import kernels as K
from test_kv_int4_gpu import DTYPES, _normal

pytestmark = pytest.mark.gpu
SHAPES = [(8, 2, 128, 64), (16, 2, 128, 64), (4, 1, 128, 32), (8, 1, 64, 32), (9, 1, 64, 64), (4, 1, 128, 128), (8, 2, 32, 32)]


def _check(q, k, v, heads, group, scale):
    n, dtype = k.shape[0], q.dtype
    rows = O.rows_of(k.to(dtype), v.to(dtype), group)
    table = torch.randperm(n, device="cuda", dtype=torch.int32)
    cache = torch.empty_like(rows)
    cache[table.long()] = rows
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    out = K.flash_decoding_int4(q, cache, scale, table[None], 0 * one, n * one, n, heads, group)
    want, error = O.attention(q, rows, heads, group, scale)
    ok = O.within(out, want, error)
    assert ok.all(), ((out.double() - want).abs().max().item(), (~ok).sum().item(), ok.numel())


@pytest.mark.parametrize("hq,heads,d,group", SHAPES)
@pytest.mark.parametrize("noise", [1e-3, 1e-2, 0.1])
@pytest.mark.parametrize("dtype", DTYPES)
def test_one_large_element_of_the_query(dtype, noise, hq, heads, d, group):
    """Beside it the others' products are small, and cancel; the value is the weight of one token."""
    for n, at in ((33, 5), (500, 499)):
        for seed in range(4):
            torch.manual_seed(seed)
            k = torch.zeros(n, heads, d, device="cuda")
            k[at, :, 0], k[at, :, 1] = 0.5, -25.0
            q = _normal(1, hq, d) * noise
            q[..., 1] = 0
            q[..., 0] += 8.0
            v = torch.zeros(n, heads, d, device="cuda")
            v[at] = 1.0
            _check(q.to(dtype), k, v, heads, group, 0.7)


@pytest.mark.parametrize("hq,heads,d,group", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_one_large_channel_of_the_keys(dtype, hq, heads, d, group):
    for n in (33, 500):
        k = _normal(n, heads, d)
        k[..., 3] += 60.0
        q = _normal(1, hq, d)
        q[..., 3] *= 20.0
        _check(q.to(dtype), k, _normal(n, heads, d), heads, group, d**-0.5)
