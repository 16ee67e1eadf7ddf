"""Prompt portions over a 4-bit cache (flash_attention_int4) against 64-bit attention; tolerances: kv_int4_oracle.prompt_attention."""

from __future__ import annotations

import math

import pytest
import torch

import kv_int4_oracle as O
from lite_llama_b200 import kernels as K
from lite_llama_b200.kernels import kv_int4 as KV
from lite_llama_b200.kernels import slot_maps as SM
from test_kv_int4_gpu import DTYPES, SHAPES, _normal, _step

pytestmark = pytest.mark.gpu


def _run(new, lens, hq, heads, d, group, dtype, q=None, gap=0, **kw):
    """A step whose sequence b ends with new[b] new tokens; gap rows of q between the sequences belong to none."""
    rows, table, req, n = _step(lens, heads, d, group, dtype, **kw)
    starts, at = [], gap
    for m in new:
        starts.append(at)
        at += m + gap
    if q is None:
        q = _normal(at, (hq + 2 * heads) * d, dtype=dtype)[:, :hq * d].view(at, hq, d)
    i32 = dict(dtype=torch.int32, device="cuda")
    return q, rows, torch.tensor(starts, **i32), torch.tensor(new, **i32), table, req, n


def _check(out, step, heads, group, scale, keep=None):
    q, rows, start, new, table, req, n = step
    mine = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    for b, (s, m, r, c) in enumerate(zip(start.tolist(), new.tolist(), req.tolist(), n.tolist())):
        want, error = O.prompt_attention(q[s:s + m], rows[table[r, :c].long()], heads, group, scale)
        ok = O.within(out[s:s + m], want, error)
        assert ok.all(), (b, m, c, (out[s:s + m].double() - want).abs().max().item(), (~ok).sum().item())
        mine[s:s + m] = True
    if keep is not None:
        assert torch.equal(out[~mine], keep[~mine])


def _call(step, heads, group, scale, **kw):
    q, rows, start, new, table, req, n = step
    max_new = kw.pop("max_new") if "max_new" in kw else int(new.max())
    max_len = kw.pop("max_len") if "max_len" in kw else int(n.max())
    return K.flash_attention_int4(q, rows, scale, start, new, table, req, n, max_new, max_len, heads, group, **kw)


# a bound on the lengths that makes many steps of a CTA: with it, portions of more than four row blocks on average have operands made ready
LOOSE = 1 << 13

STEPS = [([1], [1]), ([3], [3]), ([1], [130]), ([128], [128]), ([129, 2], [300, 2]), ([5, 0, 33, 1], [127, 40, 161, 129]), ([64, 200], [64, 1000])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,heads,d,group", SHAPES)
@pytest.mark.parametrize("new,lens", STEPS, ids=str)
def test_portions(hq, heads, d, group, dtype, new, lens):
    step = _run(new, lens, hq, heads, d, group, dtype)
    out = _call(step, heads, group, d**-0.5)
    _check(out, step, heads, group, d**-0.5)
    assert torch.equal(out, _call(step, heads, group, d**-0.5))


@pytest.mark.parametrize("hq,heads", [(1, 1), (7, 1), (64, 1), (100, 1), (32, 32), (30, 6)])
def test_head_layouts(hq, heads):
    step = _run([40, 3], [170, 90], hq, heads, 64, 32, torch.float16)
    _check(_call(step, heads, 32, 0.125), step, heads, 32, 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_ragged_portions_with_rows_of_none_between(dtype):
    new = [(i * 29) % 71 for i in range(40)]
    lens = [m + (i * 53) % 400 for i, m in enumerate(new)]
    step = _run(new, lens, 28, 4, 128, 64, dtype, gap=2)
    keep = _normal(*step[0].shape, dtype=dtype)
    out = keep.clone()
    got = _call(step, 4, 64, 0.09, out=out, max_new=100, max_len=2048)
    assert got is out
    _check(out, step, 4, 64, 0.09, keep)


def test_a_long_context_in_shares():
    step = _run([256, 17], [6000, 3001], 32, 8, 128, 64, torch.float16)
    _check(_call(step, 8, 64, 0.088), step, 8, 64, 0.088)


def test_a_whole_prompt():
    step = _run([1500], [1500], 8, 2, 128, 128, torch.bfloat16)
    _check(_call(step, 2, 128, 0.088), step, 2, 128, 0.088)


def test_more_sequences_than_one_launch_takes():
    new = [1 + i % 2 for i in range(1100)]
    lens = [m + i % 7 for i, m in enumerate(new)]
    step = _run(new, lens, 2, 1, 32, 32, torch.float16)
    out = _call(step, 1, 32, 0.2)
    q, rows, start, new_t, table, req, n = step
    pick = [0, 1, 1023, 1024, 1025, 1099]
    part = (q, rows, start[pick], new_t[pick], table, req[pick], n[pick])
    _check(out, part, 1, 32, 0.2)


@pytest.mark.parametrize("scale_q,scale_k,scale_v", [(30, 1, 1), (1e-3, 1, 1), (1, 30, 1), (1, 1, 1e-3), (1, 1, 1e3)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_and_small_values(dtype, scale_q, scale_k, scale_v):
    step = _run([70], [300], 8, 2, 128, 64, dtype, q=(_normal(70, 8, 128) * scale_q).to(dtype), scale_k=scale_k, scale_v=scale_v)
    _check(_call(step, 2, 64, 0.088), step, 2, 64, 0.088)


@pytest.mark.parametrize("wide", [0, 600, 1100])
def test_elements_past_the_range_of_halves(wide):
    """Of a bf16 cache: as 65504.  wide: beside a long portion, at 1100 tokens with ready operands."""
    step = _run([4, wide] if wide else [4], [40, wide + 100] if wide else [40], 2, 1, 64, 64, torch.bfloat16)
    q, rows, start, new, table, req, n = step
    k, v, _, _ = O.values(rows, 1, 64, 64, torch.bfloat16)
    v = v.bfloat16()
    at = int(table[int(req[0]), 3])
    v[at, 0] = torch.where(torch.arange(64, device="cuda") % 2 == 0, 1e6, -1e6)
    step = (q, O.rows_of(k.bfloat16(), v, 64), start, new, table, req, n)
    out = _call(step, 1, 64, 0.1, max_len=1 << 15 if wide == 1100 else int(n.max()))
    assert torch.isfinite(out).all()
    q, out = q[:4], out[:4]
    v[at, 0] = v[at, 0].clamp(-65504, 65504)
    w = torch.softmax(torch.einsum("mhd,nd->hmn", q.double(), O.values(step[1], 1, 64, 64, torch.bfloat16)[0][table[int(req[0]), :40].long(), 0]) * 0.1 +
                      torch.full((4, 40), -math.inf, device="cuda", dtype=torch.float64).triu(37), -1)
    assert ((out.double().abs().amax(-1) - w[:, :, 3].T * 65504).abs() <= 0.02 * w[:, :, 3].T * 65504 + 5).all()


@pytest.mark.parametrize("count", [48, 200, 600])        # a row block, several, and more than four on average: ready operands
def test_a_value_that_is_nan_reaches_only_the_rows_that_see_it(count):
    for where in (3, 60, count + 49):               # before the new tokens, among them, the last one
        q, rows, start, new, table, req, n = _run([count, 5], [count + 50, 20], 8, 2, 128, 64, torch.float16)
        k, v, _, _ = O.values(rows, 2, 128, 64, torch.float16)
        k, v = k.half(), v.half()
        bound = LOOSE if count == 600 else count + 50
        fine = _call((q, O.rows_of(k, v, 64), start, new, table, req, n), 2, 64, 0.1, max_len=bound)
        v[int(table[int(req[0]), where]), 1, 100] = math.nan
        out = _call((q, O.rows_of(k, v, 64), start, new, table, req, n), 2, 64, 0.1, max_len=bound)
        nan = torch.zeros_like(out, dtype=torch.bool)
        first = max(0, where - 50)
        nan[first:count, 4:, 64:] = True
        assert torch.equal(out.isnan(), nan), where
        # the NaN's group of the others is as before
        assert torch.equal(out[~nan], fine[~nan])


@pytest.mark.parametrize("count", [48, 200, 300])
def test_a_key_that_is_nan_reaches_only_the_rows_that_see_it(count):
    q, rows, start, new, table, req, n = _run([count], [count + 50], 8, 2, 128, 64, torch.bfloat16)
    k, v, _, _ = O.values(rows, 2, 128, 64, torch.bfloat16)
    k, v = k.bfloat16(), v.bfloat16()
    bound = 1 << 14 if count == 300 else count + 50                # ready operands
    fine = _call((q, O.rows_of(k, v, 64), start, new, table, req, n), 2, 64, 0.1, max_len=bound)
    k[int(table[int(req[0]), 70]), 0, 9] = math.inf
    out = _call((q, O.rows_of(k, v, 64), start, new, table, req, n), 2, 64, 0.1, max_len=bound)
    nan = torch.zeros_like(out, dtype=torch.bool)
    nan[20:, :4] = True
    assert torch.equal(out.isnan(), nan) and torch.equal(out[~nan], fine[~nan])


def test_what_lies_behind_the_length_does_not_count():
    q, rows, start, new, table, req, n = _run([9], [77], 4, 1, 64, 64, torch.float16, width=256)
    want = _call((q, rows, start, new, table, req, n), 1, 64, 0.1)
    used = torch.zeros(rows.shape[0], dtype=torch.bool, device="cuda")
    used[table[int(req[0]), :77].long()] = True
    spoiled = rows.clone()
    spoiled[~used] = 0xFF
    table[int(req[0]), 77:] = int((~used).nonzero()[0])
    assert torch.equal(_call((q, spoiled, start, new, table, req, n), 1, 64, 0.1, max_len=256), want)


def test_requests_pages_and_rows_that_are_not_there():
    q, rows, start, new, table, req, n = _run([4, 5, 6, 3], [40, 30, 20, 10], 4, 2, 64, 64, torch.float16, width=40)
    req[0], req[1] = -1, table.shape[0]
    table[int(req[2]), 3], table[int(req[2]), 8] = -1, rows.shape[0]
    keep = _normal(*q.shape, dtype=torch.float16)
    out = _call((q, rows, start, new, table, req, n), 2, 64, 0.1, out=keep.clone())
    assert not out[:9].any()
    table[int(req[2]), 3] = table[int(req[2]), 8] = 0
    _check(out, (q, rows, start[2:], new[2:], table, req[2:], n[2:]), 2, 64, 0.1)
    # a sequence that would end past q, one that begins past it, one that brings more than its length
    start[3], start[2], new[3], n[3] = 16, 18, 12, 10
    out = _call((q, rows, start, new, table, req, n), 2, 64, 0.1, out=keep.clone())
    table_row = table[int(req[3]), :10].long()
    assert not out[16:].any()                        # positions -2 and -1: nothing to see
    assert torch.equal(out[9:16], keep[9:16])
    start[3] = 0
    out = _call((q, rows, start[3:], new[3:], table, req[3:], n[3:]), 2, 64, 0.1, out=keep.clone())
    want, error = O.prompt_attention(q[:12], rows[table_row], 2, 64, 0.1)
    assert O.within(out[:12], want, error).all() and not out[:2].any()


def test_strides():
    q, rows, start, new, table, req, n = _run([5, 12], [30, 140], 4, 2, 64, 32, torch.bfloat16)
    wide = torch.zeros(rows.shape[0], rows.shape[1] + 32, dtype=torch.uint8, device="cuda")
    wide[:, 16:16 + rows.shape[1]] = rows
    odd = _normal(17, 4, 67, dtype=torch.bfloat16)[..., 3:]
    back = torch.empty(4, 17, 66, dtype=torch.bfloat16, device="cuda").transpose(0, 1)[..., 1:65]
    for q in (odd, _normal(4, 17, 64, dtype=torch.bfloat16).transpose(0, 1), _normal(17, 64, 4, dtype=torch.bfloat16).transpose(1, 2)):
        step = (q, wide[:, 16:16 + rows.shape[1]], start.long(), new, table.t().contiguous().t(), req.long(), n)
        _check(_call(step, 2, 32, 0.1, out=back), (q, rows, start, new, table, req, n), 2, 32, 0.1)


def test_captured_and_replayed_with_other_lengths():
    q, rows, start, new, table, req, n = _run([40, 8], [500, 1200], 28, 4, 128, 64, torch.float16)
    step = (q, rows, start, new, table, req, n)
    kw = dict(max_new=40, max_len=2048)
    _call(step, 4, 64, 0.1, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _call(step, 4, 64, 0.1, **kw)
    for cut in (0, 31):
        n.sub_(cut)
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        _check(out, step, 4, 64, 0.1)


def test_a_single_token_meets_decode_attention():
    """The two forms on one step, each within its bound."""
    rows, table, req, n = _step([333, 20, 1], 4, 128, 64, torch.float16)
    q = _normal(3, 28, 128, dtype=torch.float16)
    one = torch.ones(3, dtype=torch.int32, device="cuda")
    start = torch.arange(3, dtype=torch.int32, device="cuda")
    a = K.flash_decoding_int4(q, rows, 0.088, table, req, n, 333, 4)
    b = K.flash_attention_int4(q, rows, 0.088, start, one, table, req, n, 1, 333, 4)
    for i, (r, c) in enumerate(zip(req.tolist(), n.tolist())):
        _, error = O.prompt_attention(q[i:i + 1], rows[table[r, :c].long()], 4, 64, 0.088)
        assert O.within(b[i:i + 1], a[i:i + 1].double(), error + a[i:i + 1].double().abs() * 2.0**-11).all()


def test_scales_that_are_not_positive_are_refused():
    step = _run([2], [9], 2, 1, 64, 64, torch.float16)
    for scale in (0.0, -0.1, math.inf, math.nan):
        with pytest.raises(ValueError, match="qk_scale must be positive"):
            _call(step, 1, 64, scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,heads,d,group", SHAPES)
def test_long_portions_of_every_shape(hq, heads, d, group, dtype):
    """Several row blocks to a sequence beside short ones."""
    new, lens = [300, 3, 0, 520], [301, 400, 9, 1111]
    step = _run(new, lens, hq, heads, d, group, dtype, gap=1)
    keep = _normal(*step[0].shape, dtype=dtype)
    _check(_call(step, heads, group, d**-0.5, out=keep.clone(), max_len=1200), step, heads, group, d**-0.5, keep)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,heads,d,group", SHAPES)
def test_ready_operands_of_every_shape(hq, heads, d, group, dtype):
    """More than four row blocks to a sequence on average, of which one has none and sees nothing."""
    new, lens = [2000, 0, 1301], [2001, 40, 1500]
    step = _run(new, lens, hq, heads, d, group, dtype, gap=1)
    keep = _normal(*step[0].shape, dtype=dtype)
    _check(_call(step, heads, group, d**-0.5, out=keep.clone(), max_len=LOOSE), step, heads, group, d**-0.5, keep)


def test_ready_operands_of_a_sequence_that_sees_nothing():
    q, rows, start, new, table, req, n = _run([600, 600], [700, 600], 8, 2, 64, 32, torch.float16)
    n = n * torch.tensor([1, 0], device="cuda", dtype=n.dtype)
    out = _call((q, rows, start, new, table, req, n), 2, 32, 0.1, max_len=LOOSE)
    assert not out[600:].any()
    _check(out[:600], (q[:600], rows, start[:1], new[:1], table, req[:1], n[:1]), 2, 32, 0.1)


def test_ready_operands_do_not_outgrow_their_limit():
    """The same step under bounds that leave room for ready operands, and under bounds that do not."""
    step = _run([300, 250], [1300, 600], 8, 2, 128, 64, torch.float16)
    a = _call(step, 2, 64, 0.1, max_len=1 << 14)
    b = _call(step, 2, 64, 0.1, max_len=1 << 20)
    _check(a, step, 2, 64, 0.1)
    _check(b, step, 2, 64, 0.1)


def test_two_streams_and_a_graph_at_once():
    """Two long portions on streams of their own beside a replayed one: each has its own workspace."""
    steps = [_run([1400], [2000 + 100 * i], 8, 2, 128, 64, torch.float16) for i in range(3)]
    want = [_call(s, 2, 64, 0.1, max_len=LOOSE) for s in steps]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = _call(steps[2], 2, 64, 0.1, max_new=1400, max_len=LOOSE)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(_call(steps[i], 2, 64, 0.1, max_new=1400, max_len=LOOSE))
        with torch.cuda.stream(streams[2]):
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i]) and torch.equal(replayed, want[2])


@pytest.mark.parametrize("new,lens", [([5, 1, 40], [90, 300, 40]), ([2000], [2500])], ids=str)
def test_native_and_python_forms(new, lens):
    """Both make the same call."""
    step = _run(new, lens, 8, 2, 128, 64, torch.bfloat16, gap=1)
    q, rows, start, fresh, table, req, n = step
    keep = _normal(*q.shape, dtype=torch.bfloat16)
    args = (q, rows, 0.1, start, fresh, table, req, n, max(new), LOOSE, 2, 64)
    assert torch.equal(KV._flash_attention_int4(*args, keep.clone()), K.flash_attention_int4(*args, out=keep.clone()))
    args = (q[:len(new)], rows, 0.1, table, req, n, max(lens), 2, 64)
    assert torch.equal(KV._flash_decoding_int4(*args), K.flash_decoding_int4(*args))
    index = table[req[0].long(), :lens[0]].contiguous()
    assert torch.equal(KV._read_kv_buffer_int4(rows, index, 2, 128, torch.bfloat16, 64), K.read_kv_buffer_int4(rows, index, 2, 128, torch.bfloat16, 64))
    caches = [torch.zeros_like(rows) for _ in range(2)]
    for write, cache in zip((KV._rope_kv_write_int4, K.rope_kv_write_int4), caches):
        g = torch.Generator(device="cuda").manual_seed(1)
        a, b, c, cos = (torch.randn(m, x, 128, device="cuda", generator=g).bfloat16() for m, x in ((lens[0], 8), (lens[0], 2), (lens[0], 2), (1, lens[0])))
        write(a, b, c, cos.view(1, lens[0], 128), cos.view(1, lens[0], 128), index, cache, 1, lens[0], 64)
    assert torch.equal(*caches) and caches[0].any()
    total = sum(new)
    maps = [f(req, n - fresh, fresh, t, total, None) for f, t in ((SM._build_slot_maps, table.clone()), (K.build_slot_maps, table.clone()))]
    assert all(torch.equal(x, y) for x, y in zip(*maps))


def test_many_row_blocks_of_one_tile_to_a_cta():
    """More short sequences and heads than CTAs, by a factor: a CTA's second row tile has nothing to do in any of them."""
    new = [1 + i % 7 for i in range(128)]
    lens = [m + i % 50 for i, m in enumerate(new)]
    for d, group in ((64, 32), (128, 64)):
        step = _run(new, lens, 32, 16, d, group, torch.float16)
        _check(_call(step, 16, group, 0.1), step, 16, group, 0.1)


def test_a_short_sequence_of_many_heads_behind_long_portions():
    """The last CTA has the short one's eight heads, a row block of one tile each; operands are made ready."""
    new, lens = [512, 388, 512, 118, 512, 3], [1024, 900, 1024, 512, 512, 3]
    step = _run(new, lens, 32, 8, 128, 64, torch.float16)
    _check(_call(step, 8, 64, 0.088, max_len=LOOSE), step, 8, 64, 0.088)
    _check(_call(step, 8, 64, 0.088), step, 8, 64, 0.088)
