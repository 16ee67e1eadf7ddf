"""Attention over the 4-bit cache with weights on one key: a key that is left out, or seen too early, changes the result by all of it.

A query is a multiple of one key, its target, whose weight is close to 1; where the first key that a query must not see is added to it,
that key would take half."""

from __future__ import annotations

import pytest
import torch

import kv_int4_oracle as O
from lite_llama_b200 import kernels as K
from test_kv_int4_gpu import _normal

pytestmark = pytest.mark.gpu


def _cached(lens, heads, d, group, dtype):
    """Rows in shuffled order, a table, and the keys as they are read."""
    total = sum(lens)
    rows = O.rows_of(_normal(total, heads, d, dtype=dtype), _normal(total, heads, d, dtype=dtype), group)
    table = torch.zeros(len(lens), max(lens), dtype=torch.int32, device="cuda")
    order, at = torch.randperm(total, device="cuda", dtype=torch.int32), 0
    for b, n in enumerate(lens):
        table[b, :n] = order[at:at + n]
        at += n
    return rows, table, O.values(rows, heads, d, group, dtype)[0]


def _toward(keys, target, hq, weight):
    """Queries ``[m, hq, D]`` along the keys ``target [m, hq]`` of their kv heads, with the score ``weight`` (base e, scale 1 / sqrt(D))."""
    n, heads, d = keys.shape
    head = torch.arange(hq, device="cuda") // (hq // heads)
    k = keys[target, head]
    return k * (weight * d**0.5 / (k * k).sum(-1, keepdim=True))


def _portions(new, lens, hq, heads, d, group, dtype, max_len, own):
    rows, table, keys = _cached(lens, heads, d, group, dtype)
    parts = []
    for b, (m, n) in enumerate(zip(new, lens)):
        mine = keys[table[b, :n].long()]
        pos = torch.arange(n - m, n, device="cuda")[:, None].expand(-1, hq)
        if own:
            x = _toward(mine, pos, hq, 20.0)
            unseen = (pos + 1).clamp(max=n - 1)
            parts.append(x + torch.where((pos + 1 < n)[..., None], _toward(mine, unseen, hq, 20.0), 0.0))
        else:
            parts.append(_toward(mine, (torch.rand(m, hq, device="cuda") * (pos + 1)).long().minimum(pos), hq, 20.0))
    q = torch.cat(parts).to(dtype)
    i32 = dict(dtype=torch.int32, device="cuda")
    starts = [sum(new[:b]) for b in range(len(new))]
    out = K.flash_attention_int4(q, rows, d**-0.5, torch.tensor(starts, **i32), torch.tensor(new, **i32), table, torch.arange(len(new), **i32),
                                 torch.tensor(lens, **i32), max(new), max_len, heads, group)
    for b, (s, m, n) in enumerate(zip(starts, new, lens)):
        for lo in range(0, m, 64):                       # a block of queries at a time: the last ones of the keys that they end with
            hi, end = min(lo + 64, m), n - m + min(lo + 64, m)
            want, error = O.prompt_attention(q[s + lo:s + hi], rows[table[b, :end].long()], heads, group, d**-0.5)
            assert error.mean() < 0.1                    # against values of 1
            ok = O.within(out[s + lo:s + hi], want, error)
            assert ok.all(), (b, lo, (out[s + lo:s + hi].double() - want).abs().max().item(), (~ok).sum().item())


STEPS = [([256], [6000], 6000), ([17], [3001], 3001), ([64, 5, 130], [1000, 2111, 130], 2111), ([5] * 7, [300 + 61 * i for i in range(7)], 900),
         ([1000], [4000], 1 << 14), ([512, 700], [640, 3700], 1 << 14)]


@pytest.mark.parametrize("own", [True, False], ids=["own key", "any key"])
@pytest.mark.parametrize("hq,heads,d,group", [(8, 2, 128, 64), (14, 2, 128, 32), (8, 2, 64, 32)])
@pytest.mark.parametrize("new,lens,max_len", STEPS, ids=str)
def test_portions(new, lens, max_len, hq, heads, d, group, own):
    _portions(new, lens, hq, heads, d, group, torch.float16, max_len, own)


@pytest.mark.parametrize("new,lens,max_len", STEPS[::2], ids=str)
def test_portions_of_bf16(new, lens, max_len):
    _portions(new, lens, 8, 2, 128, 64, torch.bfloat16, max_len, True)


@pytest.mark.parametrize("lens,max_len", [([201, 37, 128], 201), ([1000] * 4, 1000), ([1500, 3000, 1, 640], 4096), ([9000] * 3, 16384),
                                          ([i * 13 % 700 + 1 for i in range(200)], 700)], ids=["cluster", "cluster of 1000", "shares", "long", "many"])
@pytest.mark.parametrize("hq,heads,d,group", [(32, 8, 128, 64), (28, 4, 128, 128), (14, 2, 64, 32), (20, 1, 64, 64)])
def test_decode(lens, max_len, hq, heads, d, group):
    """Targets over all of a row, its first, its last; and a large key behind its end."""
    rows, table, keys = _cached([n + 1 for n in lens], heads, d, group, torch.float16)
    i32 = dict(dtype=torch.int32, device="cuda")
    n = torch.tensor(lens, **i32)
    for turn in range(4):
        q = []
        for b, c in enumerate(lens):
            mine = keys[table[b, :c + 1].long()]
            at = torch.randint(0, c, (1, hq), device="cuda") if turn < 2 else torch.full((1, hq), (0, c - 1)[turn - 2], device="cuda")
            q.append(_toward(mine, at, hq, 20.0) + _toward(mine, torch.full((1, hq), c, device="cuda"), hq, 20.0))
        q = torch.cat(q).half()
        out = K.flash_decoding_int4(q, rows, d**-0.5, table, torch.arange(len(lens), **i32), n, max_len, heads, group)
        for b, c in enumerate(lens):
            want, error = O.attention(q[b:b + 1], rows[table[b, :c].long()], heads, group, d**-0.5)
            ok = O.within(out[b:b + 1], want, error)
            assert ok.all(), (turn, b, (out[b].double() - want[0]).abs().max().item(), (~ok).sum().item())
