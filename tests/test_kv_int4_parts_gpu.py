"""What is not finite in a part of a row that several blocks share: it reaches the row whatever its weight, as in a row of one part."""

from __future__ import annotations

import math

import pytest
import torch

import kv_int4_oracle as O
from lite_llama_b200 import kernels as K
from test_kv_int4_gpu import DTYPES, _normal

pytestmark = pytest.mark.gpu


def _step(n, heads, hq, d, dtype, tokens, low):
    """Keys whose scores rise by 200 (base e) half way, so that what lies before has a weight of zero; queries with one element."""
    k = torch.zeros(n, heads, d, device="cuda")
    k[n // 2:, :, 0] = low
    q = torch.zeros(tokens, hq, d, device="cuda")
    q[..., 0] = 200.0 / low / 0.125
    return q.to(dtype), k.to(dtype), _normal(n, heads, d, dtype=dtype)


def _call(q, k, v, heads, group, bound):
    n, tokens = k.shape[0], q.shape[0]
    cache = O.rows_of(k, v, group)
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    table = torch.arange(n, dtype=torch.int32, device="cuda")[None]
    if tokens == 1:
        return K.flash_decoding_int4(q, cache, 0.125, table, 0 * one, n * one, bound, heads, group)
    return K.flash_attention_int4(q, cache, 0.125, 0 * one, tokens * one, table, 0 * one, n * one, tokens, bound, heads, group)


@pytest.mark.parametrize("tokens,n,bound", [(1, 900, 900), (1, 5000, 5000), (40, 200, 200), (40, 5000, 5000), (1000, 6000, 1 << 13)],
                         ids=["decode in a cluster", "decode in shares", "a portion", "a portion in parts", "ready operands"])
@pytest.mark.parametrize("side", ["key", "value"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_nan_of_no_weight(dtype, side, tokens, n, bound):
    heads, hq, d, group = 2, 8, 64, 32
    q, k, v = _step(n, heads, hq, d, dtype, tokens, 4.0)
    clean = _call(q, k, v, heads, group, bound)
    assert torch.isfinite(clean).all()
    for at in (0, n // 4):
        bad_k, bad_v = k.clone(), v.clone()
        (bad_k if side == "key" else bad_v)[at, 1, 40] = math.nan
        out = _call(q, bad_k, bad_v, heads, group, bound)
        nan = torch.zeros_like(out, dtype=torch.bool)
        nan[:, hq // 2:, 0 if side == "key" else 32:] = True
        assert torch.equal(out.isnan(), nan) and torch.equal(out[~nan], clean[~nan])


@pytest.mark.parametrize("tokens,n,bound", [(1, 900, 900), (1, 5000, 5000), (40, 5000, 5000), (1000, 6000, 1 << 13)])
def test_keys_of_a_whole_part_that_are_nan(tokens, n, bound):
    heads, hq, d, group = 2, 8, 64, 32
    q, k, v = _step(n, heads, hq, d, torch.float16, tokens, 4.0)
    clean = _call(q, k, v, heads, group, bound)
    k[:n // 2, 0, 3] = math.inf
    out = _call(q, k, v, heads, group, bound)
    nan = torch.zeros_like(out, dtype=torch.bool)
    nan[:, :hq // 2] = True
    assert torch.equal(out.isnan(), nan) and torch.equal(out[~nan], clean[~nan])
