"""Microscaled 4-bit operators as a program uses them: refusals, streams, graphs, weights just written, large buffers, both forms of the
shims, many slots."""

from __future__ import annotations

import pytest
import torch

import mxfp4_oracle as O
from lite_llama_b200 import kernels as K
from lite_llama_b200.kernels._common import check, lib, stream_handle
from lite_llama_b200.kernels.quantization import mxfp4 as M

pytestmark = pytest.mark.gpu


def randn(*shape, dtype=torch.float16, scale=1.0):
    return (torch.randn(*shape, device="cuda") * scale).to(dtype)


def values(q):
    return O.values(O.unpack_codes(q.codes), O.scale_rows(q.scales, q.rows, q.k))


def same(a, b) -> None:
    """The same bits; of a quantised result the codes and the scales of its rows."""
    if isinstance(a, K.MXFP4):
        assert torch.equal(a.codes, b.codes) and torch.equal(O.scale_rows(a.scales, a.rows, a.k), O.scale_rows(b.scales, b.rows, b.k))
    else:
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------- refusals
def test_refusals():
    x, w = randn(4, 64), K.mxfp4_quantize_weight(randn(128, 64))
    q, ones = K.mxfp4_quantize(x), torch.ones(64, device="cuda").half()
    w1, w2 = K.mxfp4_quantize_weight(randn(4, 128, 64)), K.mxfp4_quantize_weight(randn(4, 64, 64))
    ids, wt = torch.zeros(4, 2, dtype=torch.int64, device="cuda"), torch.ones(4, 2, device="cuda")
    for what, call in (
        ("multiple of 32", lambda: K.mxfp4_quantize(randn(4, 40))),
        ("must have rows", lambda: K.mxfp4_quantize(randn(64))),
        ("float", lambda: K.mxfp4_quantize(torch.zeros(4, 64, dtype=torch.int32, device="cuda"))),
        ("float", lambda: K.mxfp4_dequantize(q, torch.float64)),
        ("contiguous", lambda: K.mxfp4_dequantize(K.MXFP4(q.codes[:, :16].expand(4, 16), q.scales))),
        ("do not belong", lambda: K.mxfp4_dequantize(K.MXFP4(q.codes, w1.scales))),
        ("uint8", lambda: K.mxfp4_dequantize(K.MXFP4(q.codes.view(torch.int8), q.scales))),
        ("CUDA tensors only", lambda: K.mxfp4_dequantize(K.MXFP4(q.codes, q.scales.cpu()))),
        ("CUDA", lambda: K.mxfp4_matmul(x.cpu(), w)),
        ("expects 64", lambda: K.mxfp4_matmul(randn(4, 96), w)),
        ("expects 64", lambda: K.mxfp4_matmul(K.mxfp4_quantize(randn(4, 96)), w)),
        ("float16 or bfloat16", lambda: K.mxfp4_matmul(x.float(), w)),
        ("is torch.float16", lambda: K.mxfp4_matmul(x, w, out_dtype=torch.bfloat16)),
        ("unsupported output", lambda: K.mxfp4_matmul(q, w, out_dtype=torch.float32)),
        ("bias must be", lambda: K.mxfp4_matmul(x, w, torch.zeros(64, device="cuda").half())),
        ("bias must be", lambda: K.mxfp4_matmul(x, w, torch.zeros(128, device="cuda"))),
        ("runs of 64", lambda: K.mxfp4_matmul(x, K.mxfp4_quantize_weight(randn(64, 64)), swiglu=True)),
        ("codes of shape", lambda: K.mxfp4_matmul(x, w1)),
        ("multiple of 32", lambda: K.skip_rmsnorm_mxfp4(randn(4, 40), None, randn(40))),
        ("weight must be", lambda: K.skip_rmsnorm_mxfp4(x, None, ones.float())),
        ("weight must be", lambda: K.skip_rmsnorm_mxfp4(x, None, ones[:32])),
        ("residual must be", lambda: K.skip_rmsnorm_mxfp4(x, x[:2], ones)),
        ("contiguous", lambda: K.skip_rmsnorm_mxfp4(x, randn(4, 128)[:, ::2], ones)),
        ("without a residual", lambda: K.skip_rmsnorm_mxfp4(x, None, ones, out_residual=x)),
        ("do not belong", lambda: K.fused_moe_mxfp4(x, w1, K.mxfp4_quantize_weight(randn(3, 64, 64)), wt, ids)),
        ("hidden_states of shape", lambda: K.fused_moe_mxfp4(randn(4, 96), w1, w2, wt, ids)),
        ("for 4 tokens", lambda: K.fused_moe_mxfp4(x, w1, w2, wt, ids[:3])),
        ("weights must be", lambda: K.fused_moe_mxfp4(x, w1, w2, wt.double(), ids)),
        ("int32 or int64", lambda: K.fused_moe_mxfp4(x, w1, w2, wt, ids.short())),
    ):
        with pytest.raises(ValueError, match=what):
            call()


def test_nothing_in_nothing_out():
    w = K.mxfp4_quantize_weight(randn(128, 64))
    assert K.mxfp4_matmul(randn(0, 64), w).shape == (0, 128) and K.mxfp4_matmul(randn(2, 0, 64), w).shape == (2, 0, 128)
    assert K.mxfp4_matmul(randn(0, 64), w, swiglu=True).codes.shape == (0, 32)
    q, r = K.skip_rmsnorm_mxfp4(randn(0, 64), randn(0, 64), randn(64))
    assert q.rows == 0 and r.shape == (0, 64)


def test_leading_dimensions_and_gradients():
    x, w = randn(2, 3, 64).requires_grad_(), K.mxfp4_quantize_weight(randn(40, 64))
    y = K.mxfp4_matmul(x, w)
    assert y.shape == (2, 3, 40) and not y.requires_grad
    same(y.view(6, 40), K.mxfp4_matmul(x.detach().view(6, 64), w))
    r = randn(2, 3, 64)
    kept = r.clone()
    q, out = K.skip_rmsnorm_mxfp4(x.detach(), r, randn(64))
    assert out is r and q.codes.shape == (6, 32) and torch.equal(out, kept + x.detach())


def test_native_and_python_forms_give_the_same_bits():
    for t in (1, 7, 40, 300):
        x, w, bias = randn(t, 256), K.mxfp4_quantize_weight(randn(384, 256, scale=0.05)), randn(384)
        q = K.mxfp4_quantize(x)
        same(q, M._mxfp4_quantize(x))
        same(K.mxfp4_dequantize(q), M._mxfp4_dequantize(q, torch.float16))
        for b in (None, bias):
            same(K.mxfp4_matmul(x, w, b), M._mxfp4_matmul(x, w, b, False, None))
            same(K.mxfp4_matmul(q, w, b, out_dtype=torch.float16), M._mxfp4_matmul(q, w, b, False, None))
            same(K.mxfp4_matmul(x, w, b, swiglu=True), M._mxfp4_matmul(x, w, b, True, None))
        r, g = randn(t, 256), randn(256)
        sums = [r.clone(), r.clone()]
        same(K.skip_rmsnorm_mxfp4(x, sums[0], g)[0], M._skip_rmsnorm_mxfp4(x, sums[1], g, 1e-5, None)[0])
        assert torch.equal(*sums)
        w1, w2 = K.mxfp4_quantize_weight(randn(8, 256, 256, scale=0.05)), K.mxfp4_quantize_weight(randn(8, 256, 128, scale=0.05))
        top = torch.softmax(randn(t, 8).float(), -1).topk(3, -1)
        same(K.fused_moe_mxfp4(x, w1, w2, top.values, top.indices), M._fused_moe_mxfp4(x, w1, w2, top.values, top.indices))


# ------------------------------------------------------------------------------------------------- weights just written
def test_weights_of_the_kernel_before():
    """A quantiser's result used as a weight right behind it, again and again in the same memory."""
    x = randn(4, 2048)
    codes, scales = torch.empty(8192, 1024, dtype=torch.uint8, device="cuda"), torch.empty(64, 16, 32, 4, 4, dtype=torch.uint8, device="cuda")
    ws = [randn(8192, 2048, scale=s) for s in (0.02, 3.0, 0.5)]
    want = [K.mxfp4_matmul(x, K.mxfp4_quantize_weight(w)) for w in ws]
    for _ in range(20):
        for w, y in zip(ws, want):
            check(lib().b2l_mxfp4_quantize(codes.data_ptr(), scales.data_ptr(), w.data_ptr(), 1, 8192, 2048, 2048, 0, stream_handle()))
            same(K.mxfp4_matmul(x, K.MXFP4(codes, scales, ready=False)), y)


def test_pieces_of_a_stack_just_quantised_and_a_matrix_by_itself():
    for _ in range(5):
        w, x = randn(3, 4096, 1024), randn(4, 1024)
        want = [K.mxfp4_matmul(x, K.mxfp4_quantize_weight(m)) for m in w]
        for e in range(3):
            q = K.mxfp4_quantize(w)
            same(K.mxfp4_matmul(x, K.MXFP4(q.codes[e], q.scales[e], q.ready)), want[e])
    for t in (24, 200):
        m = randn(t, 1024)
        q = K.mxfp4_quantize(m)
        same(K.mxfp4_matmul(q, q), K.mxfp4_matmul(m, K.mxfp4_quantize_weight(m)))


@pytest.mark.parametrize("rows,n", ((3, 4096), (700, 256)))
def test_norm_in_the_place_of_its_inputs(rows, n):
    x, r, w = randn(rows, n), randn(rows, n), randn(n)
    q, total = K.skip_rmsnorm_mxfp4(x, r, w, out_residual=torch.empty_like(r))
    over = x.clone()
    p, s = K.skip_rmsnorm_mxfp4(over, r, w, out_residual=over)
    same(p, q)
    assert s is over and torch.equal(s, total)
    twice = x.clone()
    p, s = K.skip_rmsnorm_mxfp4(twice, twice, w)
    same(p, K.skip_rmsnorm_mxfp4(x, x.clone(), w)[0])
    assert s is twice and torch.equal(s, x + x)


# ------------------------------------------------------------------------------------------------- rows and columns behind the end
@pytest.mark.parametrize("t,n", ((1, 33), (5, 130), (70, 128), (300, 264), (300, 250)))
def test_nothing_is_written_behind_the_outputs(t, n):
    x, w = K.mxfp4_quantize(randn(t, 256)), K.mxfp4_quantize_weight(randn(n, 256, scale=0.05))
    wide = torch.full((t + 3, n + 24), 7.0, device="cuda").half()
    check(lib().b2l_mxfp4_matmul(wide[1:, 8:].data_ptr(), None, x.codes.data_ptr(), x.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(),
                                 None, t, n, 256, 128, 128, n + 24, 0, 1, 0, stream_handle()))
    same(wide[1:t + 1, 8:n + 8], K.mxfp4_matmul(x, w))
    wide[1:t + 1, 8:n + 8] = 7
    assert (wide == 7).all()


# ------------------------------------------------------------------------------------------------- streams and graphs
def chain(x, r, g, w1, w2, e1, e2, weights, ids):
    q, total = K.skip_rmsnorm_mxfp4(x, r, g, out_residual=torch.empty_like(r))
    y = K.mxfp4_matmul(K.mxfp4_matmul(q, w1, swiglu=True), w2, out_dtype=x.dtype)
    z = K.fused_moe_mxfp4(y, e1, e2, weights, ids)
    return total, y, z, K.mxfp4_dequantize(K.mxfp4_quantize(z))


def inputs(t, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, device="cuda", generator=gen).half()  # noqa: E731
    return n(t, 256), n(t, 256), n(256), torch.rand(t, 2, device="cuda", generator=gen), torch.randint(0, 8, (t, 2), device="cuda", generator=gen)


def model():
    gate, up = randn(192, 256, scale=0.1), randn(192, 256, scale=0.1)
    return (K.mxfp4_quantize_weight(K.mxfp4_gate_up(gate, up)), K.mxfp4_quantize_weight(randn(256, 192, scale=0.1)),
            K.mxfp4_quantize_weight(randn(8, 256, 256, scale=0.1)), K.mxfp4_quantize_weight(randn(8, 256, 128, scale=0.1)))


def run(m, i):
    x, r, g, weights, ids = i
    return chain(x, r, g, *m, weights, ids)


@pytest.mark.parametrize("t", (1, 20, 300))
def test_two_streams_at_once(t):
    m, sets = model(), [inputs(t, s) for s in range(4)]
    want = [run(m, i) for i in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for n, i in enumerate(sets):
            with torch.cuda.stream(streams[n % 2]):
                got.append((n, run(m, i)))
    torch.cuda.synchronize()
    for n, out in got:
        for a, b in zip(out, want[n]):
            same(a, b)


@pytest.mark.parametrize("t", (1, 20, 300))
def test_two_captured_graphs_replayed_together(t):
    m = model()
    kept = [inputs(t, 0), inputs(t, 1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in kept:
            run(m, i)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in kept:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(m, i))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for seed in (10, 20, 30):
        fresh = [inputs(t, seed + n) for n in range(2)]
        for old, new in zip(kept, fresh):
            for a, b in zip(old, new):
                a.copy_(b)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for out, i in zip(outs, fresh):
            for a, b in zip(out, run(m, i)):
                same(a, b)


# ------------------------------------------------------------------------------------------------- many slots
@pytest.mark.parametrize("tokens,top_k,experts,skew", ((1, 1, 3, False), (1, 32, 8, False), (4, 8, 128, False), (31, 1, 5, False), (2, 16, 4096, False), (1, 40, 64, False), (700, 8, 16, False), (700, 8, 16, True), (5000, 8, 300, False), (9000, 4, 5, True)))
def test_slots_of_any_number_reach_their_experts(tokens, top_k, experts, skew):
    """Expert e multiplies by e + 1 (its weights are that many times one pattern that sums are exact for), so that a row in a wrong place shows."""
    hidden, inner = 64, 64
    x = torch.zeros(tokens, hidden, device="cuda").half()
    x[:, 0] = torch.arange(tokens, device="cuda") % 4 + 1                # 1 .. 4: exact in the format
    one = torch.zeros(experts, 2 * inner, hidden, device="cuda")
    one[:, 0, 0] = 6 * 2.0 ** 6                                          # gate: large, so that silu is the identity
    one[:, 64, 0] = 2.0 ** -6
    down = torch.zeros(experts, hidden, inner, device="cuda")
    down[:, 1, 0] = 2.0 ** (torch.arange(experts, device="cuda") % 8)
    w1, w2 = K.mxfp4_quantize_weight(one), K.mxfp4_quantize_weight(down)
    ids = torch.randint(0, experts, (tokens, top_k), device="cuda")
    if skew:
        ids[tokens // 10:] = experts - 1
    weights = torch.ones(tokens, top_k, device="cuda")
    out = K.fused_moe_mxfp4(x, w1, w2, weights, ids)
    act = O.rounded((6 * x[:, :1].double() ** 2).repeat(1, 32))[:, 0]    # what the unit is quantised to
    want = (act[:, None] * 2.0 ** (ids % 8).double()).sum(1)
    assert torch.equal(out[:, 1].double(), want.half().double()) and not out[:, 2:].any()


# ------------------------------------------------------------------------------------------------- large buffers
def test_offsets_past_32_bits():
    rows, k = 70000, 32768
    x = torch.zeros(rows, k, device="cuda", dtype=torch.float16)
    x[-40:] = randn(40, k)
    q = K.mxfp4_quantize(x)
    code, byte = O.quantise(x[-40:])
    assert torch.equal(O.unpack_codes(q.codes[-40:]), code)
    assert torch.equal(O.scale_rows(q.scales[-2:].contiguous(), rows - 128 * (q.scales.shape[0] - 2), k)[-40:], byte)
    y = K.mxfp4_dequantize(q)
    assert torch.equal(y[-40:].double(), O.values(code, byte).half().double())
    del y, x, q
    t, n = 150000, 16384                                                 # 2.5e9 outputs
    x, w = randn(t, 64), K.mxfp4_quantize_weight(randn(n, 64))
    y = K.mxfp4_matmul(x, w)
    same(y[-300:], K.mxfp4_matmul(x[-300:].contiguous(), w))
    same(y[70000:70300], K.mxfp4_matmul(x[70000:70300].contiguous(), w))
