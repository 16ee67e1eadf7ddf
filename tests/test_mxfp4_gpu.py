"""Microscaled 4-bit operators against their definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

import mxfp4_oracle as O
from lite_llama_b200 import kernels as K

pytestmark = pytest.mark.gpu
HALVES = (torch.float16, torch.bfloat16)


def same_codes(q: K.MXFP4, want) -> None:
    code, byte = want
    got = O.unpack_codes(q.codes)
    assert torch.equal(O.scale_rows(q.scales, q.rows, q.k), byte)
    assert torch.equal(got, code)


# ------------------------------------------------------------------------------------------------- the format
@pytest.mark.parametrize("dtype", (*HALVES, torch.float32))
@pytest.mark.parametrize("rows,k", ((1, 32), (1, 4096), (3, 96), (5, 160), (31, 224), (129, 256), (200, 1056), (7, 18944)))
def test_quantised_like_the_definition(dtype, rows, k):
    x = (torch.randn(rows, k, device="cuda") * torch.randn(rows, 1, device="cuda").exp()).to(dtype)
    x[0, :32] = 0
    q = K.mxfp4_quantize(x)
    same_codes(q, O.quantise(x))
    y = K.mxfp4_dequantize(q, torch.float32)
    assert torch.equal(y.double(), O.rounded(x))


@pytest.mark.parametrize("dtype", HALVES)
def test_every_16_bit_value_in_every_place_of_a_scale(dtype):
    """All 65536 patterns, alone in their block (infinities, NaN, subnormals), beside a block maximum that makes them small, and
    ties between elements."""
    bits = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    alone = torch.zeros(65536, 32, dtype=dtype, device="cuda")
    alone[:, 5] = bits
    same_codes(K.mxfp4_quantize(alone), O.quantise(alone))
    for top in (1.0, 7.5, 2.0 ** -14):
        beside = alone.clone()
        beside[:, 30] = top
        same_codes(K.mxfp4_quantize(beside), O.quantise(beside))


def test_borders_of_32_bit_values():
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], device="cuda")
    near = torch.stack([torch.nextafter(ties, torch.zeros_like(ties)), ties, torch.nextafter(ties, ties + 9)]).flatten()
    x = torch.zeros(64, 64, device="cuda")
    x[:, 0], x[:, 32] = 4.0, -7.9
    x[:, 1:28], x[:, 33:60] = near, -near
    x *= torch.exp2(torch.arange(64, device="cuda") - 32.0)[:, None]
    same_codes(K.mxfp4_quantize(x), O.quantise(x))


def test_smallest_and_largest_scales():
    x = torch.zeros(4, 64, device="cuda")
    x[0, 0], x[0, 33] = 2.0 ** -149, 2.0 ** -127
    x[1, 3], x[1, 40] = 2.0 ** -126, 3 * 2.0 ** -125
    x[2, 3], x[2, 40] = torch.finfo(torch.float32).max, -(2.0 ** 127)
    x[3, 0], x[3, 32] = float("inf"), float("nan")
    q = K.mxfp4_quantize(x)
    same_codes(q, O.quantise(x))
    y = K.mxfp4_dequantize(q, torch.float32)
    assert y[3].isnan().all() and torch.equal(y[:3].double(), O.rounded(x)[:3])


def test_rows_of_any_stride_and_stacks():
    wide = torch.randn(9, 400, device="cuda").half()
    for x in (wide[:, 8:72], wide[:, 3:67], wide[:, ::2][:, :160], wide.t()[:96].t(), wide[::3, 32:64], wide[4:5, 1:33]):
        assert x.shape[1] % 32 == 0
        same_codes(K.mxfp4_quantize(x), O.quantise(x))
    stack = torch.randn(3, 130, 96, device="cuda").bfloat16()
    q = K.mxfp4_quantize(stack)
    same_codes(q, O.quantise(stack))
    assert torch.equal(K.mxfp4_dequantize(q, torch.float32).double(), O.rounded(stack))
    packed = K.mxfp4_pack(q.codes, O.scale_rows(q.scales, 130, 96))
    rows_behind = torch.zeros_like(packed.scales)
    assert torch.equal(O.scale_rows(packed.scales, 130, 96), O.scale_rows(q.scales, 130, 96)) and rows_behind.shape == q.scales.shape
    empty = K.mxfp4_quantize(stack[:, :0])
    assert empty.rows == 0 and K.mxfp4_dequantize(empty).shape == (3, 0, 96)


@pytest.mark.parametrize("dtype", HALVES)
def test_values_come_back_rounded_once(dtype):
    code = torch.randint(0, 16, (40, 96), device="cuda", dtype=torch.uint8)
    byte = torch.randint(100, 140, (40, 3), device="cuda", dtype=torch.uint8)
    byte[0], byte[1, 0] = 255, 0
    y = K.mxfp4_dequantize(K.mxfp4_pack(O.pack_codes(code), byte), dtype)
    want = O.values(code, byte).float().to(dtype)
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y[1:], want[1:])


# ------------------------------------------------------------------------------------------------- the norm
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("rows,n", ((1, 32), (3, 96), (33, 896), (130, 4096), (5, 5120), (2, 16384)))
@pytest.mark.parametrize("with_residual", (True, False))
def test_norm_decides_as_exact_arithmetic(dtype, rows, n, with_residual):
    x = (torch.randn(rows, n, device="cuda") * 2).to(dtype)
    r = (torch.randn(rows, n, device="cuda") * 3).to(dtype) if with_residual else None
    w = (1 + 0.2 * torch.randn(n, device="cuda")).to(dtype)
    y, total = O.norm(x, r, w, 1e-5)
    kept = None if r is None else r.clone()
    q, out = K.skip_rmsnorm_mxfp4(x, r, w, 1e-5)
    same_codes(q, O.quantise(y))
    if with_residual:
        assert out is r and torch.equal(out, (x.float() + kept.float()).to(dtype))
        sums, again = torch.empty_like(kept), kept.clone()
        q2, out2 = K.skip_rmsnorm_mxfp4(x, again, w, 1e-5, out_residual=sums)
        assert out2 is sums and torch.equal(sums, out) and torch.equal(again, kept)
        assert torch.equal(q2.codes, q.codes)
    else:
        assert out is x


def test_norm_of_rows_that_lie_on_borders():
    """All elements alike, so that the norm is just below 1 (a power of two) and the weight puts it on ties; rows of zeros; tiny rows."""
    n = 256
    x = torch.ones(6, n, device="cuda")
    x[1] *= 2.0 ** -8
    x[2] *= 1000
    x[3] = 0
    x[4] *= 1e-7
    x[5, ::2] *= -1
    x = x.half()
    for weights in (1.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0):
        w = torch.full((n,), weights, device="cuda").half()
        w[::32] = 4.0
        q, _ = K.skip_rmsnorm_mxfp4(x, None, w, 1e-6)
        same_codes(q, O.quantise(O.norm(x, None, w, float(torch.tensor(1e-6, dtype=torch.float32)))[0]))


def test_norm_keeps_other_rows_from_a_bad_one():
    x = torch.randn(4, 128, device="cuda").bfloat16()
    good, _ = K.skip_rmsnorm_mxfp4(x, None, torch.ones(128, device="cuda").bfloat16())
    x[2, 7] = float("inf")
    q, _ = K.skip_rmsnorm_mxfp4(x, None, torch.ones(128, device="cuda").bfloat16())
    y, z = K.mxfp4_dequantize(q, torch.float32), K.mxfp4_dequantize(good, torch.float32)
    assert y[2, :32].isnan().all() and torch.equal(y[[0, 1, 3]], z[[0, 1, 3]])


# ------------------------------------------------------------------------------------------------- products
def weights(n, k, spread=0.02):
    w = torch.randn(n, k, device="cuda") * spread
    q = K.mxfp4_quantize_weight(w)
    return q, O.values(O.unpack_codes(q.codes), O.scale_rows(q.scales, n, k))


@pytest.mark.parametrize("t,n,k", ((1, 128, 64), (1, 128, 256), (3, 5, 32), (32, 256, 512), (33, 130, 96), (17, 384, 1120), (64, 200, 2048),
                                   (65, 640, 992), (128, 129, 4096), (100, 1000, 352),
                                   # pairs: one tile, both widths, ragged edges, several tiles to a pair; what they leave (odd n)
                                   (129, 8, 32), (256, 256, 256), (200, 264, 96), (385, 1000, 736), (300, 20488, 256), (1000, 9000, 1312),
                                   (2048, 4096, 512), (140, 131, 256), (300, 33, 1024), (256, 1200, 8192), (150, 40, 4384)))
def test_products_of_whole_numbers_are_exact(t, n, k):
    """Elements and scales whose products add up to whole numbers below 2^11: any order of exact sums gives the same bits, and one
    element, scale, row or block in a wrong place gives others."""
    gen = torch.Generator(device="cuda").manual_seed(t * 7 + n)
    few = lambda rows: torch.where(torch.rand(rows, k, device="cuda", generator=gen) < 16 / k,  # noqa: E731
                                   torch.randint(0, 16, (rows, k), device="cuda", generator=gen), 0).to(torch.uint8)
    xc, wc = few(t), few(n)
    xb, wb = (torch.randint(128, 130, (rows, k // 32), device="cuda", generator=gen, dtype=torch.uint8) for rows in (t, n))
    x, w = K.mxfp4_pack(O.pack_codes(xc), xb), K.mxfp4_pack(O.pack_codes(wc), wb)
    want = O.values(xc, xb) @ O.values(wc, wb).t()
    assert want.abs().max() > 0
    for dtype in HALVES:
        assert torch.equal(K.mxfp4_matmul(x, w, out_dtype=dtype), want.to(dtype))


@pytest.mark.parametrize("k", (512, 1024, 4096, 8192))
@pytest.mark.parametrize("n", (256, 200))
def test_every_number_of_tokens_that_shares_its_sums(n, k):
    """One to eight parts of k, by any number of tokens: which CTA of a cluster adds up a token follows from both."""
    gen = torch.Generator(device="cuda").manual_seed(n + k)
    few = lambda rows: torch.where(torch.rand(rows, k, device="cuda", generator=gen) < 16 / k,  # noqa: E731
                                   torch.randint(0, 16, (rows, k), device="cuda", generator=gen), 0).to(torch.uint8)
    xc, wc = few(130), few(n)
    xb, wb = (torch.randint(128, 130, (rows, k // 32), device="cuda", generator=gen, dtype=torch.uint8) for rows in (130, n))
    w, want = K.mxfp4_pack(O.pack_codes(wc), wb), (O.values(xc, xb) @ O.values(wc, wb).t()).half()
    for t in (*range(1, 34), 63, 64, 65, 96, 127, 128, 129):
        x = K.mxfp4_pack(O.pack_codes(xc[:t]), xb[:t])
        assert torch.equal(K.mxfp4_matmul(x, w), want[:t])
        if n == 256 and t <= 40:
            a = K.mxfp4_matmul(x, w, swiglu=True)
            one = K.mxfp4_matmul(K.mxfp4_pack(O.pack_codes(xc[:130]), xb[:130]), w, swiglu=True)      # all rows at once
            assert torch.equal(a.codes, one.codes[:t])
            assert torch.equal(O.scale_rows(a.scales, t, 128), O.scale_rows(one.scales, 130, 128)[:t])


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,n,k", ((1, 6144, 4096), (2, 896, 4864), (7, 4096, 14336), (31, 77, 3584), (40, 4608, 3584), (128, 1152, 896),
                                   (5, 33, 32), (777, 4608, 3584), (129, 896, 4864), (513, 9728, 896), (200, 77, 1024)))
@pytest.mark.parametrize("with_bias", (False, True))
def test_products_against_64_bits(dtype, t, n, k, with_bias):
    x = torch.randn(t, k, device="cuda").to(dtype)
    w, wv = weights(n, k)
    b = torch.randn(n, device="cuda").to(dtype) if with_bias else None
    y = K.mxfp4_matmul(x, w, bias=b)
    xv = O.rounded(x)
    want = xv @ wv.t()
    bound = O.product_bound(xv, wv, want + (0 if b is None else b.double()), dtype)
    want = want if b is None else want + b.double()
    assert y.dtype == dtype and ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t", (1, 2, 5, 8, 9))
@pytest.mark.parametrize("n,k", ((128, 32), (384, 96), (256, 4096), (6144, 4096), (4096, 14336), (19200, 6144), (19200, 6400), (130, 992)))
def test_activations_in_16_bits_give_the_quantised_ones_bits(dtype, t, n, k):
    """Few rows are quantised inside the product: the codes are those of the quantiser, the sums are in the same order."""
    wide = torch.randn(t, k + 64, device="cuda").to(dtype)
    wide[0, 8] = float("nan")
    w, _ = weights(n, k)
    for x in (wide[:, :k], wide[:, 16:16 + k], wide[:, 3:3 + k]):
        want = K.mxfp4_matmul(K.mxfp4_quantize(x), w, out_dtype=dtype)
        assert torch.equal(K.mxfp4_matmul(x, w).view(torch.int16), want.view(torch.int16))
        if n % 128 == 0:
            a, b = K.mxfp4_matmul(K.mxfp4_quantize(x), w, swiglu=True, out_dtype=dtype), K.mxfp4_matmul(x, w, swiglu=True)
            same_codes(a, (O.unpack_codes(b.codes), O.scale_rows(b.scales, b.rows, b.k)))


# ------------------------------------------------------------------------------------------------- the gated feed-forward
def gated_weights(inner, k, lead=()):
    gate, up = (torch.randn(*lead, inner, k, device="cuda") * 0.05 for _ in range(2))
    q = K.mxfp4_quantize_weight(K.mxfp4_gate_up(gate, up))
    return q, O.rounded(gate), O.rounded(up)


def act_errors(g, u, sums_g, sums_u, k):
    """How far silu(g) u may be off before it is quantised: each product as ``product_bound`` without the rounding, the activation's
    slope in g is at most 1.1, and 2^-20 of it for the exponential and the quotient."""
    e = k * 2.0 ** -23
    act = torch.nn.functional.silu(g) * u
    return act, 1.1 * e * sums_g * u.abs() + e * sums_u * torch.nn.functional.silu(g).abs() + 2.0 ** -20 * act.abs()


def quantised_near(q, act, off):
    """Every value is what some value within `off` of `act` is quantised to: rounding and scales grow with the value, so it lies
    between the quantised ends; a block whose largest magnitude may be on either side of a power of two has either scale."""
    got = K.mxfp4_dequantize(q, torch.float32).double().unflatten(-1, (-1, 32))
    byte = O.scale_rows(q.scales, q.rows, q.k)
    a, o = act.unflatten(-1, (-1, 32)), off.unflatten(-1, (-1, 32))
    high, low = (a.abs() + o).amax(-1), (a.abs() - o).amax(-1).clamp(min=0)
    top = [torch.where(m > 0, (torch.frexp(m)[1] - 3 + 127).clamp(0, 254), 0) for m in (low, high)]
    assert ((byte >= top[0]) & (byte <= top[1])).all()
    scale = torch.exp2(byte.double() - 127)[..., None]

    def grid(v):
        t = (v / scale).abs()
        step = torch.where(t < 2, 0.5, torch.where(t < 4, 1.0, 2.0))
        return torch.sign(v) * (torch.round(t / step) * step).clamp(max=6) * scale
    assert ((got >= grid(a - o)) & (got <= grid(a + o))).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t", (129, 300, 777))
def test_outputs_of_any_number_and_place(dtype, t):
    """Rows that start anywhere have the bits of those that start on 16 bytes, with and without a bias, wherever that lies."""
    x, w = K.mxfp4_quantize(torch.randn(t, 512, device="cuda")), torch.randn(1024, 512, device="cuda") * 0.05
    bias = torch.randn(1025, device="cuda").to(dtype)
    q = K.mxfp4_quantize_weight(w)
    for b in (None, bias[1:]):
        want = K.mxfp4_matmul(x, q, None if b is None else b.clone(), out_dtype=dtype)
        assert torch.equal(K.mxfp4_matmul(x, q, b, out_dtype=dtype), want)
        for n in (1023, 1002, 700, 513, 250, 129):
            part = K.mxfp4_quantize_weight(w[:n])
            assert torch.equal(K.mxfp4_matmul(x, part, None if b is None else b[:n], out_dtype=dtype), want[:, :n])


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,inner,k", ((1, 64, 64), (3, 128, 96), (32, 192, 256), (20, 4864, 896), (50, 320, 1120), (100, 448, 512), (128, 64, 2048),
                                        (129, 64, 64), (300, 320, 256), (260, 4864, 896), (1000, 5056, 352)))
@pytest.mark.parametrize("with_bias", (False, True))
def test_feed_forward_quantises_its_own_sums(dtype, t, inner, k, with_bias):
    x = torch.randn(t, k, device="cuda").to(dtype)
    w, gate, up = gated_weights(inner, k)
    bias = None
    xv = O.rounded(x)
    g, u = xv @ gate.t(), xv @ up.t()
    if with_bias:
        bg, bu = (torch.randn(inner, 1, device="cuda").to(dtype) for _ in range(2))
        bias = K.mxfp4_gate_up(bg, bu).flatten()
        g, u = g + bg.double().t(), u + bu.double().t()
    q = K.mxfp4_matmul(x, w, bias=bias, swiglu=True)
    assert (q.rows, q.k) == (t, inner)
    act, off = act_errors(g, u, xv.abs() @ gate.abs().t() + g.abs(), xv.abs() @ up.abs().t() + u.abs(), k)
    quantised_near(q, act, off)
    behind = q.scales.permute(0, 3, 2, 1, 4).flatten(-2).flatten(0, 2)[:t, inner // 32:]
    assert not behind.any()                                              # blocks behind the end are zero


# ------------------------------------------------------------------------------------------------- routed experts
def experts_reference(x, w1, gate, up, down, weights, ids, dtype):
    """The operator step by step with the framework's own quantised activations in the middle: (out, how far off)."""
    tokens = x.shape[0]
    out, off = torch.zeros(tokens, down.shape[1], dtype=torch.float64, device="cuda"), torch.zeros(tokens, down.shape[1], dtype=torch.float64, device="cuda")
    for e in range(gate.shape[0]):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if not t.numel():
            continue
        q = K.mxfp4_matmul(x[t], K.MXFP4(w1.codes[e], w1.scales[e]), swiglu=True)
        act = O.values(O.unpack_codes(q.codes), O.scale_rows(q.scales, q.rows, q.k))
        y = act @ down[e].t()
        w = weights[t, j].double()[:, None]
        out.index_add_(0, t, w * y)
        off.index_add_(0, t, w.abs() * O.slot_bound(act, down[e], y))
    k = ids.shape[1]
    return out, off * (1 + k * 2.0 ** -23) + k * 2.0 ** -23 * off.new_tensor(1) * out.abs() + out.abs() * torch.finfo(dtype).eps / 2 + 1e-7


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("experts,top_k,hidden,inner,tokens", ((4, 2, 64, 64, 1), (8, 2, 256, 128, 5), (8, 3, 96, 192, 40), (16, 2, 256, 64, 300), (3, 2, 160, 128, 129),
                                                               (4, 4, 128, 320, 200), (5, 2, 160, 576, 700), (3, 2, 160, 576, 700),
                                                               (8, 2, 800, 64, 400), (5, 3, 416, 576, 700)))
def test_experts_step_by_step(dtype, experts, top_k, hidden, inner, tokens):
    x = torch.randn(tokens, hidden, device="cuda").to(dtype)
    w1, gate, up = gated_weights(inner, hidden, (experts,))
    down = torch.randn(experts, hidden, inner, device="cuda") * 0.05
    w2 = K.mxfp4_quantize_weight(down)
    top = torch.softmax(torch.randn(tokens, experts, device="cuda"), -1).topk(top_k, -1)
    for weights, ids in ((top.values.to(dtype), top.indices), (top.values, top.indices.int())):
        want, off = experts_reference(x, w1, gate, up, O.rounded(down), weights, ids, dtype)
        got = K.fused_moe_mxfp4(x, w1, w2, weights, ids)
        assert ((got.double() - want).abs() <= off).all()
        assert torch.equal(got, K.fused_moe_mxfp4(x, w1, w2, weights, ids))


def test_experts_without_tokens_the_same_twice_and_ids_of_none():
    experts, hidden, inner = 8, 128, 64
    x = torch.randn(70, hidden, device="cuda").half()
    w1, gate, up = gated_weights(inner, hidden, (experts,))
    down = torch.randn(experts, hidden, inner, device="cuda") * 0.05
    w2 = K.mxfp4_quantize_weight(down)
    weights = torch.rand(70, 3, device="cuda")
    ids = torch.randint(0, 2, (70, 3), device="cuda")                    # six experts see nobody, some tokens one expert twice
    ids[5], ids[6, 1], ids[7, 2], ids[9, 0] = -1, 8, 2 ** 40, -7
    want, off = experts_reference(x, w1, gate, up, O.rounded(down), weights, ids, torch.float16)
    got = K.fused_moe_mxfp4(x, w1, w2, weights, ids)
    assert ((got.double() - want).abs() <= off).all() and not got[5].any()
    for n in (1, 4, 10, 11, 70):                                         # up to 32 slots in one launch: the same rows
        s = slice(0, n)
        for a in (ids, ids.int()) if n < 8 else (ids,):
            assert torch.equal(K.fused_moe_mxfp4(x[s], w1, w2, weights[s], a[s]), got[s])
        assert not K.fused_moe_mxfp4(x[s], w1, w2, weights[s], torch.full_like(ids[s], -1)).any()
    assert K.fused_moe_mxfp4(x[:0], w1, w2, weights[:0], ids[:0]).shape == (0, hidden)


@pytest.mark.parametrize("tokens,experts", ((3, 4), (70, 4), (700, 5), (700, 3)))      # tiles of 64 (one launch and two), 128 and 256 rows
def test_bad_weights_and_tokens_reach_their_own_outputs_alone(tokens, experts):
    hidden, inner = 160, 576
    x = torch.randn(tokens, hidden, device="cuda").half()
    w1, _, _ = gated_weights(inner, hidden, (experts,))
    down = torch.randn(experts, hidden, inner, device="cuda") * 0.05
    ids = torch.stack([torch.randperm(experts, device="cuda")[:2] for _ in range(tokens)])
    weights = torch.rand(tokens, 2, device="cuda") + 0.1
    ids[0] = torch.tensor([0, 1], device="cuda")
    want = K.fused_moe_mxfp4(x, w1, K.mxfp4_quantize_weight(down), weights, ids)
    down[1, 130, 40], down[1, 7, 3] = float("nan"), float("inf")
    zero = torch.zeros(64, inner, device="cuda")
    down[2, 64:128] = zero
    down[2, 70, 5] = float("nan")                                       # nothing else in its 64 outputs
    got = K.fused_moe_mxfp4(x, w1, K.mxfp4_quantize_weight(down), weights, ids)
    one, two = (ids == 1).any(1), (ids == 2).any(1)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[:, 130] |= one
    bad[:, 7] |= one
    bad[:, 70] |= two
    assert torch.equal(got.isnan(), bad)
    other = ~bad
    other[two, 64:128] = False                                          # those weights are others
    near = (got.double() - want.double()).abs() <= 2.0 ** -9 * want.double().abs().amax()      # without the bad one a block's steps are others
    assert near[other].all()
    x[0, 3] = float("nan")
    got = K.fused_moe_mxfp4(x, w1, K.mxfp4_quantize_weight(down), weights, ids)
    assert got[0].isnan().all() and torch.equal(got[1:].isnan(), bad[1:])
