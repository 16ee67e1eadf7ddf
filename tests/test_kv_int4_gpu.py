"""The 4-bit cache on the GPU: writer, reader, decode attention and slot maps against 64-bit forms (kv_int4_oracle.py).

Tolerances: a stored row is met byte by byte; a value that was computed is a rounding (half a step of its type) of something within a
bound that the oracle derives from the operands (kv_int4_oracle.attention)."""

from __future__ import annotations

import math

import pytest
import torch

import kv_int4_oracle as O
from lite_llama_b200 import kernels as K

pytestmark = pytest.mark.gpu
SHAPES = [(32, 8, 128, 64), (28, 4, 128, 128), (14, 2, 64, 32), (8, 2, 32, 32), (8, 8, 64, 64), (15, 3, 128, 32), (6, 1, 64, 64)]
DTYPES = [torch.float16, torch.bfloat16]


def _normal(*shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda").to(dtype)


def _cache(tokens, heads, d, group):
    return torch.full((tokens, O.row_bytes(heads, d, group)), 0xA5, dtype=torch.uint8, device="cuda")


def _used(heads, d, group):
    return heads * (d + 8 * (d // group))


def _same_rows(got, want, used):
    """Bytes of rows; a NaN may be any."""
    assert torch.equal(got[:, :used], want[:, :used])


# ------------------------------------------------------------------------------------------------------------------ writer
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,heads,d,group", SHAPES)
def test_rows_are_stored_as_documented(hq, heads, d, group, dtype):
    n = 37
    kv = _normal(n, 2 * heads, d + 8, dtype=dtype)[..., :d]                      # rows of a wider tensor
    k, v = kv[:, :heads], kv[:, heads:]
    cache = _cache(50, heads, d, group)
    before = cache.clone()
    index = torch.randperm(50, device="cuda")[:n]
    K.update_kv_buffer_int4(k, v, index, cache, group)
    _same_rows(cache[index], O.rows_of(k, v, group), _used(heads, d, group))
    rest = torch.ones(50, dtype=torch.bool, device="cuda")
    rest[index] = False
    assert torch.equal(cache[rest], before[rest])


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_with_every_scale_and_ties(dtype):
    """Groups of whole numbers on the grid and between two of its points (ties go to the even code), constant, tiny, huge groups."""
    d, n = 128, 12
    k = _normal(n, 2, d, dtype=dtype)
    grid = torch.arange(d, device="cuda") % 31
    k[0, 0] = (grid * 0.5).to(dtype)                     # scale 1, every second element half way between two codes
    k[1, 0] = 3.25
    k[2, 0] = 0
    k[3, 0] = (k[3, 0].float() * 1e-6).to(dtype)
    k[4, 0] = (k[4, 0].float() * 1e4).to(dtype)
    k[5, 0, ::2], k[5, 0, 1::2] = torch.finfo(dtype).max, -torch.finfo(dtype).max
    k[6, 0] = 1e-7 if dtype == torch.float16 else 1e-38
    k[6, 0, 5] = 0
    cache = _cache(n, 2, d, 64)
    K.update_kv_buffer_int4(k, k, torch.arange(n, device="cuda"), cache)
    want = O.rows_of(k, k, 64)
    _same_rows(cache, want, _used(2, d, 64))
    back = K.read_kv_buffer_int4(cache, torch.arange(n, device="cuda"), 2, d, dtype)
    exact = torch.cat(O.values(want, 2, d, 64, dtype)[:2], 1).clamp(max=torch.finfo(dtype).max)   # nothing finite reads as infinite
    assert O.within(back, exact, exact.abs() * 2.0**-23).all()
    assert torch.equal(back[0, 0, :62], torch.round(k[0, 0, :62].float()).to(dtype))
    assert torch.equal(back[1, 0], k[1, 0]) and torch.equal(back[2, 0], k[2, 0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_half_steps_that_a_tiny_element_leaves(dtype):
    """Elements of +-2^-24 .. 2^-8 in groups whose minimum lies exactly k + 1/2 steps below zero: their sign decides the code."""
    groups = []
    for k in range(15):
        for base in (1.0, 3.0, 1024.0):                      # scale 2 base; the range is 15 of it, so that it is stored exactly (fp16: 29 * 1024 is finite)
            lo = -(2 * k + 1) * base
            tiny = [s * 2.0**-e for e in (8, 12, 14, 18, 24) for s in (1, -1)]
            groups.append([lo, lo + 30 * base] + tiny + [0.0] * 20)
    k = torch.tensor(groups, device="cuda", dtype=torch.float64).to(dtype).view(-1, 1, 32)
    cache = _cache(k.shape[0], 1, 32, 32)
    K.update_kv_buffer_int4(k, k.flip(0).contiguous(), torch.arange(k.shape[0], device="cuda"), cache, 32)
    _same_rows(cache, O.rows_of(k, k.flip(0), 32), _used(1, 32, 32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_group_that_is_not_finite_reads_as_nan(dtype, bad):
    k, v = _normal(5, 2, 128, dtype=dtype), _normal(5, 2, 128, dtype=dtype)
    k[1, 0, 3] = bad
    v[2, 1, 100] = bad
    cache = _cache(5, 2, 128, 64)
    index = torch.arange(5, device="cuda")
    K.update_kv_buffer_int4(k, v, index, cache)
    back = K.read_kv_buffer_int4(cache, index, 2, 128, dtype)
    nan = torch.zeros_like(back, dtype=torch.bool)
    nan[1, 0, :64] = nan[2, 3, 64:] = True
    assert torch.equal(back.isnan(), nan)


@pytest.mark.parametrize("width", [torch.int32, torch.int64])
def test_tokens_without_a_row_are_skipped(width):
    k = _normal(6, 2, 64, dtype=torch.float16)
    cache = _cache(10, 2, 64, 64)
    before = cache.clone()
    index = torch.tensor([3, -1, 10, 7, -5, 2**31 - 1], device="cuda").to(width)
    K.update_kv_buffer_int4(k, k, index, cache)
    want = before.clone()
    want[[3, 7], :144] = O.rows_of(k, k, 64)[[0, 3]]
    assert torch.equal(cache, want)
    back = K.read_kv_buffer_int4(cache, index, 2, 64, torch.float16)
    assert not back[[1, 2, 4, 5]].any() and back[[0, 3]].any()


def _rotation(batch, seq, d, dtype):
    angle = torch.rand(batch, seq, d // 2, device="cuda") * 6
    return torch.cat((angle.cos(), angle.cos()), -1).to(dtype), torch.cat((angle.sin(), angle.sin()), -1).to(dtype)


def _rotated(x, cos, sin):
    d = x.shape[-1]
    c, s = (t.reshape(-1, 1, t.shape[-1])[..., :d // 2].double() for t in (cos, sin))
    a, b = x[..., :d // 2].double(), x[..., d // 2:].double()
    want = torch.cat((a * c - b * s, b * c + a * s), -1)
    parts = torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()), -1)
    return want, parts * 2.0**-23                            # two products and a sum in 32 bits


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,heads,d,group", SHAPES)
@pytest.mark.parametrize("batch,seq,pad", [(1, 1, 0), (3, 1, 0), (2, 19, 0), (1, 5, 3)])
def test_rotation_and_store(hq, heads, d, group, dtype, batch, seq, pad):
    """From the projection's columns, in place; pad: rows that no 16-byte access fits."""
    n, wide = batch * seq, (hq + 2 * heads) * d + pad
    qkv = _normal(n, wide, dtype=dtype)
    q, k, v = (qkv[:, lo * d:hi * d].view(n, -1, d) if pad == 0 else qkv[:, pad + lo * d:pad + hi * d].unflatten(1, (-1, d))
               for lo, hi in ((0, hq), (hq, hq + heads), (hq + heads, hq + 2 * heads)))
    cos, sin = _rotation(batch, seq, d, dtype)
    want_q, want_k = _rotated(q, cos, sin), _rotated(k, cos, sin)
    kept_v = v.clone()
    cache = _cache(n + 4, heads, d, group)
    index = torch.randperm(n + 4, device="cuda", dtype=torch.int32)[:n]
    out_q, out_k = K.rope_kv_write_int4(q, k, v, cos, sin, index, cache, batch, seq, group)
    assert out_q.data_ptr() == q.data_ptr() and out_k.data_ptr() == k.data_ptr() and torch.equal(v, kept_v)
    assert O.within(q, *want_q).all() and O.within(k, *want_k).all()
    _same_rows(cache[index.long()], O.rows_of(k, v, group), _used(heads, d, group))


def test_rotation_into_other_tensors():
    n, hq, heads, d = 7, 4, 2, 64
    q, k, v = _normal(n, hq, d, dtype=torch.float16), _normal(n, heads, d, dtype=torch.float16), _normal(n, heads, d, dtype=torch.float16)
    cos, sin = _rotation(1, n, d, torch.float16)
    kept = q.clone(), k.clone()
    new_q, new_k = torch.empty_like(q), torch.empty(n, heads + 1, d, dtype=torch.float16, device="cuda")[:, 1:]
    cache, other = _cache(n, heads, d, 64), _cache(n, heads, d, 64)
    index = torch.arange(n, device="cuda")
    a, b = K.rope_kv_write_int4(q, k, v, cos, sin, index, cache, 1, n, out_q=new_q, out_k=new_k)
    assert a is new_q and b is new_k and torch.equal(q, kept[0]) and torch.equal(k, kept[1])
    K.rope_kv_write_int4(q, k, v, cos, sin, index, other, 1, n)
    assert torch.equal(q, new_q) and torch.equal(k, new_k) and torch.equal(cache, other)


def test_nothing_to_write_or_read():
    e = torch.empty(0, 2, 64, dtype=torch.float16, device="cuda")
    cache, idx = _cache(3, 2, 64, 64), torch.empty(0, dtype=torch.int32, device="cuda")
    K.update_kv_buffer_int4(e, e, idx, cache)
    assert K.read_kv_buffer_int4(cache, idx, 2, 64, torch.float16).shape == (0, 4, 64)
    assert (cache == 0xA5).all()


# ------------------------------------------------------------------------------------------------------------------ decode
def _step(lens, heads, d, group, dtype, width=None, scale_v=1.0, scale_k=1.0, extra=7):
    """A filled cache in shuffled rows, a table and lengths for one step."""
    lens = list(lens)
    total = sum(lens) + extra
    rows = O.rows_of((_normal(total, heads, d) * scale_k).to(dtype), (_normal(total, heads, d) * scale_v + 0.3 * scale_v).to(dtype), group)
    width = max(1, max(lens)) if width is None else width
    table = torch.full((len(lens) + 2, width), -7, dtype=torch.int32, device="cuda")
    order, req = torch.randperm(total, device="cuda", dtype=torch.int32), torch.randperm(len(lens) + 2)[:len(lens)].tolist()
    at = 0
    for r, n in zip(req, lens):
        table[r, :n] = order[at:at + n]
        at += n
    return rows, table, torch.tensor(req, device="cuda", dtype=torch.int32), torch.tensor(lens, device="cuda", dtype=torch.int32)


def _check(out, q, rows, table, req, lens, heads, group, scale):
    for b, (r, n) in enumerate(zip(req.tolist(), lens.tolist())):
        want, error = O.attention(q[b:b + 1], rows[table[r, :n].long()], heads, group, scale)
        ok = O.within(out[b:b + 1], want, error)
        assert ok.all(), (b, n, (out[b].double() - want[0]).abs().max().item(), (~ok).sum().item())


LENGTHS = [[1], [0, 3, 0], [15, 16, 17], [63, 64, 65, 1, 128], [201], [1000, 77, 0, 513], [4097]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,heads,d,group", SHAPES)
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
def test_decode(hq, heads, d, group, dtype, lens):
    rows, table, req, n = _step(lens, heads, d, group, dtype)
    q = _normal(len(lens), hq * d + 2 * heads * d, dtype=dtype)[:, :hq * d].view(len(lens), hq, d)
    out = K.flash_decoding_int4(q, rows, d**-0.5, table, req, n, max(lens) + 5, heads, group)
    _check(out, q, rows, table, req, n, heads, group, d**-0.5)
    assert torch.equal(out, K.flash_decoding_int4(q, rows, d**-0.5, table, req, n, max(lens) + 5, heads, group))


@pytest.mark.parametrize("hq,heads", [(1, 1), (3, 1), (4, 1), (5, 1), (8, 1), (9, 1), (20, 1), (64, 1), (32, 32), (18, 9), (44, 11), (30, 6), (48, 24)])
def test_decode_head_layouts(hq, heads):
    lens = [130, 33]
    for d, group in ((64, 64), (128, 128)):
        rows, table, req, n = _step(lens, heads, d, group, torch.bfloat16)
        q = _normal(2, hq, d, dtype=torch.bfloat16)
        _check(K.flash_decoding_int4(q, rows, d**-0.5, table, req, n, 130, heads, group), q, rows, table, req, n, heads, group, d**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_of_a_large_uneven_batch(dtype):
    """More tiles than CTAs; rows that several CTAs share beside rows that share one."""
    lens = [(i * 37) % 211 for i in range(300)] + [9000, 0, 3000]
    rows, table, req, n = _step(lens, 8, 128, 64, dtype)
    q = _normal(len(lens), 32, 128, dtype=dtype)
    out = K.flash_decoding_int4(q, rows, 0.09, table, req.long(), n.long(), 16384, 8)
    _check(out, q, rows, table, req, n, 8, 64, 0.09)


def test_decode_of_more_rows_than_one_launch_takes():
    lens = [1 + i % 5 for i in range(4100)]
    rows, table, req, n = _step(lens, 1, 32, 32, torch.float16)
    q = _normal(len(lens), 2, 32, dtype=torch.float16)
    out = K.flash_decoding_int4(q, rows, 0.2, table, req, n, 5, 1, 32)
    pick = [0, 1, 4095, 4096, 4099]
    _check(out[pick], q[pick], rows, table, req[pick], n[pick], 1, 32, 0.2)


@pytest.mark.parametrize("scale_q,scale_k,scale_v", [(30, 1, 1), (1e-3, 1, 1), (1, 60, 1), (1, 1, 1e-4), (1, 1, 1e3), (300, 1e-2, 30)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_with_large_and_small_values(dtype, scale_q, scale_k, scale_v):
    """Scores far apart, where one token takes everything, and scales at both ends."""
    rows, table, req, n = _step([300, 41], 2, 128, 64, dtype, scale_k=scale_k, scale_v=scale_v)
    q = (_normal(2, 8, 128) * scale_q).to(dtype)
    _check(K.flash_decoding_int4(q, rows, 0.088, table, req, n, 300, 2), q, rows, table, req, n, 2, 64, 0.088)


def test_decode_with_value_scales_that_rise_along_the_row():
    rows, table, req, n = _step([400], 1, 64, 32, torch.bfloat16)
    k, v, _, _ = O.values(rows, 1, 64, 32, torch.bfloat16)
    order = torch.empty(407, device="cuda")
    order[table[int(req[0]), :400].long()] = torch.arange(400, device="cuda").float()
    rows = O.rows_of(k.bfloat16(), (v * torch.exp2((order - 200) / 12)[:, None, None]).bfloat16(), 32)
    for hq in (4, 8):
        q = _normal(1, hq, 64, dtype=torch.bfloat16)
        _check(K.flash_decoding_int4(q, rows, 0.125, table, req, n, 400, 1, 32), q, rows, table, req, n, 1, 32, 0.125)


def test_decode_reads_only_what_counts():
    """Behind a row's length, in rows of other requests and in tokens that no table names there may be NaN."""
    lens = [70, 0, 33]
    rows, table, req, n = _step(lens, 2, 64, 64, torch.float16, width=128)
    used = torch.zeros(rows.shape[0], dtype=torch.bool, device="cuda")
    for r, c in zip(req.tolist(), lens):
        used[table[r, :c].long()] = True
        table[r, c:] = int((~used).nonzero()[0]) if (~used).any() else 0
    spoiled = rows.clone()
    spoiled[~used] = 0xFF
    for r, c in zip(req.tolist(), lens):
        table[r, c:] = int((~used).nonzero()[0])
    q = _normal(3, 8, 64, dtype=torch.float16)
    out = K.flash_decoding_int4(q, spoiled, 0.1, table, req, n, 128, 2)
    _check(out, q, rows, table, req, n, 2, 64, 0.1)
    assert not out[1].any()


def test_decode_where_a_cached_group_is_nan():
    """As in plain attention: a key that is not finite spoils its kv head's outputs, a value's group its elements; nothing else."""
    rows, table, req, n = _step([50, 20], 2, 128, 64, torch.float16)
    k, v, _, _ = O.values(rows, 2, 128, 64, torch.float16)
    k, v = k.half(), v.half()
    clean = O.rows_of(k, v, 64)
    k[int(table[int(req[0]), 7]), 1, 5] = math.inf
    v[int(table[int(req[0]), 30]), 0, 70] = math.nan
    rows = O.rows_of(k, v, 64)
    for hq in (8, 16):
        q = _normal(2, hq, 128, dtype=torch.float16)
        out, fine = (K.flash_decoding_int4(q, c, 0.1, table, req, n, 50, 2) for c in (rows, clean))
        g = hq // 2
        nan = torch.zeros_like(out, dtype=torch.bool)
        nan[0, g:] = True
        nan[0, :g, 64:] = True
        assert torch.equal(out.isnan(), nan)
        assert torch.equal(out[1], fine[1]) and torch.equal(out[0, :g, :64], fine[0, :g, :64])


def test_decode_where_one_query_is_not_finite():
    rows, table, req, n = _step([50], 1, 64, 64, torch.float16)
    q = _normal(1, 4, 64, dtype=torch.float16)
    q[0, 2, 9] = math.nan
    out = K.flash_decoding_int4(q, rows, 0.1, table, req, n, 50, 1)
    assert torch.equal(out.isnan().any(-1), torch.tensor([[False, False, True, False]], device="cuda"))
    q[0, 2] = 0
    _check(torch.where(out.isnan(), K.flash_decoding_int4(q, rows, 0.1, table, req, n, 50, 1), out), q, rows, table, req, n, 1, 64, 0.1)


def test_decode_of_requests_and_pages_that_are_not_there():
    rows, table, req, n = _step([40, 30, 20], 2, 64, 64, torch.float16, width=40)
    q = _normal(3, 4, 64, dtype=torch.float16)
    req[0], req[1] = -1, table.shape[0]
    table[int(req[2]), 3], table[int(req[2]), 8] = -1, rows.shape[0]
    out = K.flash_decoding_int4(q, rows, 0.1, table, req, n, 40, 2)
    assert not out[:2].any()
    table[int(req[2]), 3] = table[int(req[2]), 8] = 0
    _check(out[2:], q[2:], rows, table, req[2:], n[2:], 2, 64, 0.1)
    n[2] = 1000                                       # past the table: its width counts
    out = K.flash_decoding_int4(q, rows, 0.1, table.clamp(min=0), req, n, 2000, 2)
    n[2] = 40
    _check(out[2:], q[2:], rows, table.clamp(min=0), req[2:], n[2:], 2, 64, 0.1)


def test_decode_with_strides():
    """A cache with rows of a wider tensor, a transposed table, queries with a foreign stride."""
    rows, table, req, n = _step([70, 20], 2, 128, 32, torch.bfloat16)
    wide = torch.zeros(rows.shape[0], rows.shape[1] + 48, dtype=torch.uint8, device="cuda")
    wide[:, 16:16 + rows.shape[1]] = rows
    turned = table.t().contiguous().t()
    for q in (_normal(2, 4, 130, dtype=torch.bfloat16)[..., 1:129], _normal(4, 2, 128, dtype=torch.bfloat16).transpose(0, 1),
              _normal(2, 128, 4, dtype=torch.bfloat16).transpose(1, 2)):
        out = K.flash_decoding_int4(q, wide[:, 16:16 + rows.shape[1]], 0.1, turned, req, n, 70, 2, 32)
        _check(out, q, rows, table, req, n, 2, 32, 0.1)


@pytest.mark.parametrize("batch,max_len", [(1, 0), (1, 5), (3, 1), (3, 2000), (200, 64), (70, 3000)])
def test_decode_of_rows_that_see_nothing(batch, max_len):
    rows, table, req, n = _step([1] * batch, 2, 64, 32, torch.float16, width=1)
    q = _normal(batch, 4, 64, dtype=torch.float16)
    assert not K.flash_decoding_int4(q, rows, 0.1, table, req, torch.zeros_like(n) if max_len else n, max_len, 2, 32).any()


@pytest.mark.parametrize("lens", [[201, 17], [1500, 3000]], ids=str)
def test_decode_into_a_tensor(lens):
    """A part of a larger tensor; the query itself."""
    rows, table, req, n = _step(lens, 4, 128, 64, torch.float16)
    q, keep = _normal(2, 8, 128, dtype=torch.float16), _normal(5, 10, 136, dtype=torch.float16)
    want = K.flash_decoding_int4(q, rows, 0.1, table, req, n, max(lens), 4, 64)
    to = keep.clone()
    view = to[1:3, 2:, 4:132]
    assert K.flash_decoding_int4(q, rows, 0.1, table, req, n, max(lens), 4, 64, view) is view and torch.equal(view, want)
    keep[1:3, 2:, 4:132] = want
    assert torch.equal(to, keep)
    assert K.flash_decoding_int4(q, rows, 0.1, table, req, n, max(lens), 4, 64, out=q) is q and torch.equal(q, want)


def test_decode_of_rows_past_32_bits():
    heads, d = 8, 128
    row = O.row_bytes(heads, d, 64)
    tokens = 2**31 // row + 4000                       # the last ones lie past 2^31 bytes
    if torch.cuda.mem_get_info()[0] < 2 * tokens * row:
        pytest.skip("not enough memory")
    small, table, req, n = _step([300, 100], heads, d, 64, torch.float16)
    cache = torch.zeros(tokens, row, dtype=torch.uint8, device="cuda")
    cache[-small.shape[0]:] = small
    q = _normal(2, 32, d, dtype=torch.float16)
    want = K.flash_decoding_int4(q, small, 0.1, table, req, n, 300, heads)
    far = torch.where(table >= 0, table + (tokens - small.shape[0]), table)
    assert torch.equal(K.flash_decoding_int4(q, cache, 0.1, far, req, n, 300, heads), want)
    k = _normal(3, heads, d, dtype=torch.float16)
    index = torch.tensor([tokens - 1, tokens - 2, 0], device="cuda")
    K.update_kv_buffer_int4(k, k, index, cache)
    assert torch.equal(cache[index], O.rows_of(k, k, 64))


def test_decode_captured_and_replayed_beside_another():
    """Two graphs with workspaces of their own, replayed in turn and on two streams with new lengths."""
    steps = []
    for lens in ([900, 50, 333], [64, 2000]):
        rows, table, req, n = _step(lens, 4, 128, 64, torch.float16)
        q = _normal(len(lens), 28, 128, dtype=torch.float16)
        K.flash_decoding_int4(q, rows, 0.1, table, req, n, 4096, 4)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = K.flash_decoding_int4(q, rows, 0.1, table, req, n, 4096, 4)
        steps.append((graph, out, q, rows, table, req, n))
    for cut in (0, 13):
        for s in steps:
            s[6].sub_(cut)
            s[2].normal_()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        for _ in range(5):
            steps[0][0].replay()
            with torch.cuda.stream(side):
                steps[1][0].replay()
        torch.cuda.synchronize()
        for _, out, q, rows, table, req, n in steps:
            _check(out, q, rows, table, req, n, 4, 64, 0.1)


def test_an_operand_on_no_or_another_device_is_refused():
    rows, table, req, n = _step([5], 1, 64, 64, torch.float16)
    q = _normal(1, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="no CPU fallback"):
        K.flash_decoding_int4(q, rows, 0.1, table.cpu(), req, n, 5, 1)


# ------------------------------------------------------------------------------------------------------------------ slot maps
def _maps(req, ctx, new, width, total, requests, pool=False, types=(torch.int32, torch.int32, torch.int32)):
    table = torch.randperm(requests * width, device="cuda", dtype=torch.int32).view(requests, width)
    rows = torch.randperm(total + 3, device="cuda", dtype=torch.int64) if pool else None
    plain = table.tolist()
    want = O.slot_maps(req, ctx, new, plain, total, rows.tolist() if pool else None)
    args = [torch.tensor(x, device="cuda", dtype=t) for x, t in zip((req, ctx, new), types)]
    got = K.build_slot_maps(*args, table, total, rows)
    for g, w in zip(got, want):
        assert g.tolist() == w
    assert table.tolist() == plain
    assert [g.dtype for g in got] == [torch.int32, torch.int64, torch.int32, torch.int32]


@pytest.mark.parametrize("pool", [False, True])
@pytest.mark.parametrize("req,ctx,new,total", [
    ([0], [0], [1], 1), ([2, 0], [3, 0], [1, 5], 6), ([1, 2, 0], [4, 0, 9], [0, 7, 3], 14), ([0, 1], [0, 0], [0, 0], 3), ([0], [2], [6], 4),
    ([1, 1], [0, 5], [5, 2], 7), ([0, 9, -1, 1], [0, 1, 1, 38], [2, 3, 1, 4], 11), ([0, 1], [-3, 2], [2, -5], 4), ([0, 1], [1, 1], [2, 2], 0),
], ids=str)
def test_slot_maps(req, ctx, new, total, pool):
    _maps(req, ctx, new, 40, total, 3, pool)


@pytest.mark.parametrize("pool", [False, True])
@pytest.mark.parametrize("batch,most", [(1, 5000), (300, 40), (1500, 3), (2049, 1), (5, 1025)])
def test_slot_maps_of_many_requests_and_tokens(batch, most, pool):
    gen = torch.Generator().manual_seed(batch)
    req = torch.randperm(batch + 3, generator=gen)[:batch].tolist()
    ctx, new = torch.randint(0, 20, (batch,), generator=gen).tolist(), torch.randint(0, most + 1, (batch,), generator=gen).tolist()
    _maps(req, ctx, new, most + 20, sum(new) + 5, batch + 3, pool, (torch.int64, torch.int32, torch.int64))


def test_slot_maps_of_no_request():
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    rows, pos, start, length = K.build_slot_maps(e, e, e, torch.zeros(2, 4, dtype=torch.int32, device="cuda"), 3)
    assert rows.tolist() == [-1] * 3 and pos.tolist() == [0] * 3 and start.numel() == length.numel() == 0


def test_maps_write_and_decode_as_one_captured_step():
    """The operators as a step uses them, from maps to attention, against the same steps in plain torch; padded to a captured size."""
    heads, hq, d, group, dtype, batch, width = 2, 8, 64, 32, torch.float16, 5, 96
    cache = torch.zeros(batch * width, O.row_bytes(heads, d, group), dtype=torch.uint8, device="cuda")
    table = torch.arange(batch * width, dtype=torch.int32, device="cuda").view(batch, width)
    req = torch.tensor([3, 0, 4], dtype=torch.int32, device="cuda")
    ctx, one = torch.tensor([40, 7, 0], dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    filled = {}
    for r, c in zip(req.tolist(), ctx.tolist()):
        k, v = _normal(c, heads, d, dtype=dtype), _normal(c, heads, d, dtype=dtype)
        K.update_kv_buffer_int4(k, v, table[r, :c].contiguous(), cache, group)
        filled[r] = O.rows_of(k, v, group)
    cos, sin = _rotation(1, width, d, dtype)
    qkv = _normal(4, (hq + 2 * heads) * d, dtype=dtype)          # one padded token

    def step():
        rows, pos, _, lens = K.build_slot_maps(req, ctx, one, table, 4)
        x = qkv.clone().view(4, hq + 2 * heads, d)
        q, k = K.rope_kv_write_int4(x[:, :hq], x[:, hq:hq + heads], x[:, hq + heads:], cos[0, pos].unsqueeze(1), sin[0, pos].unsqueeze(1), rows, cache,
                                    4, 1, group)
        out = K.flash_decoding_int4(q[:3], cache, d**-0.5, table, req, lens, width, heads, group)
        ctx.add_(one)
        return x, out

    kept = ctx.clone(), cache.clone()
    step()
    ctx.copy_(kept[0])
    cache.copy_(kept[1])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        x, out = step()
    for i in range(4):
        qkv.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for b, r in enumerate(req.tolist()):
            new = O.rows_of(x[b:b + 1, hq:hq + heads], x[b:b + 1, hq + heads:], group)
            filled[r] = torch.cat((filled[r], new))
            n = filled[r].shape[0]
            used = _used(heads, d, group)
            assert n == int(kept[0][b]) + i + 1
            assert torch.equal(cache[r * width:r * width + n, :used], filled[r][:, :used])
            want, error = O.attention(x[b:b + 1, :hq], filled[r], heads, group, d**-0.5)
            assert O.within(out[b:b + 1], want, error).all()
    idle = [r for r in range(batch) if r not in filled]
    assert not cache.view(batch, width, -1)[idle].any()
