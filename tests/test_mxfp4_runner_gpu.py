"""Uniform decoders with weights and activations in microscaled 4-bit floating point: every call of a served model against 64 bits."""

from __future__ import annotations

import pytest
import torch

import mxfp4_oracle as O
from lite_llama_b200 import kernels as K
from lite_llama_b200.engine import Engine
from lite_llama_b200.executor import ModelRunner, decoder
from lite_llama_b200.quantization import methods

pytestmark = pytest.mark.gpu


def values(q):
    return O.values(O.unpack_codes(q.codes), O.scale_rows(q.scales, q.rows, q.k))


def halves(rows):
    """Gate and up rows of weights in runs of 64."""
    g, u = rows.unflatten(-2, (-1, 2, 64)).unbind(-3)
    return g.flatten(-3, -2), u.flatten(-3, -2)


@pytest.fixture
def checked(monkeypatch):
    """Holds every call that the decoder makes of the operators against its definition; counts them."""
    seen = {"matmul": 0, "gated": 0, "norm": 0, "moe": 0}

    def matmul(x, w, bias=None, *, swiglu=False, out_dtype=None):
        y = K.mxfp4_matmul(x, w, bias, swiglu=swiglu, out_dtype=out_dtype)
        xv = values(x) if isinstance(x, K.MXFP4) else O.rounded(x)
        wv = values(w)
        want = xv @ wv.t() + (0 if bias is None else bias.double())
        if swiglu:
            seen["gated"] += 1
            g, u = halves(want.t())
            act = (torch.nn.functional.silu(g) * u).t()
            # a code next to a border may fall on either side: half a step is at most a quarter of the value or of the block's scale
            got, step = values(y), torch.exp2(O.scale_rows(y.scales, y.rows, y.k).double() - 127).repeat_interleave(32, 1)
            off = (got - act).abs()
            cut = act.abs() > 6 * step                                   # the format ends at six scales
            assert (off[~cut] <= torch.maximum(act.abs() / 5, step / 4)[~cut] * (1 + 1e-4)).all()
            assert (got.abs()[cut] == 6 * step[cut]).all()
        else:
            seen["matmul"] += 1
            bound = O.product_bound(xv, wv, want, y.dtype)
            assert ((y.double() - want).abs() <= bound).all()
        return y

    def norm(X, residual, weight, eps=1e-5):
        kept = None if residual is None else residual.clone()
        q, out = K.skip_rmsnorm_mxfp4(X, residual, weight, eps)
        n = X.shape[-1]
        y, _ = O.norm(X.reshape(-1, n), None if kept is None else kept.reshape(-1, n), weight, eps)
        code, byte = O.quantise(y)
        assert torch.equal(O.unpack_codes(q.codes), code) and torch.equal(O.scale_rows(q.scales, q.rows, q.k), byte)
        seen["norm"] += 1
        return q, out

    def moe(x, w1, w2, weights, ids):
        out = K.fused_moe_mxfp4(x, w1, w2, weights, ids)
        want, off = torch.zeros(out.shape, device="cuda", dtype=torch.float64), torch.zeros(out.shape, device="cuda", dtype=torch.float64)
        for e in range(w1.codes.shape[0]):
            t, j = torch.nonzero(ids == e, as_tuple=True)
            if t.numel():
                act = values(K.mxfp4_matmul(x[t], K.MXFP4(w1.codes[e], w1.scales[e]), swiglu=True))
                down = values(K.MXFP4(w2.codes[e], w2.scales[e]))
                y = act @ down.t()
                w = weights[t, j].double()[:, None]
                want.index_add_(0, t, w * y)
                off.index_add_(0, t, w * O.slot_bound(act, down, y))
        eps = torch.finfo(out.dtype).eps
        assert ((out.double() - want).abs() <= off * 1.001 + want.abs() * eps / 2 + 1e-6 * want.abs() + torch.finfo(out.dtype).smallest_normal * eps).all()
        seen["moe"] += 1
        return out

    monkeypatch.setattr(decoder, "mxfp4_matmul", matmul)
    monkeypatch.setattr(methods, "mxfp4_matmul", matmul)
    monkeypatch.setattr(decoder, "skip_rmsnorm_mxfp4", norm)
    monkeypatch.setattr(decoder, "fused_moe_mxfp4", moe)
    return seen


def prefill(runner, batch, prompt):
    ids = torch.randint(0, runner.vocab_size, (batch, prompt), device="cuda")
    pos = torch.arange(prompt, device="cuda").repeat(batch, 1)
    runner.prefill_alloc_kv_cache(prompt, torch.full((batch,), prompt, device="cuda"), torch.arange(batch, device="cuda"))
    return runner.forward(ids, pos)


@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
@pytest.mark.parametrize("name", ("tiny-llama", "tiny-qwen2", "tiny-qwen3", "tiny-qwen3-moe"))
@pytest.mark.parametrize("batch,prompt", ((1, 1), (3, 12), (2, 150)))
def test_every_call_of_a_step(checked, name, dtype, batch, prompt):
    runner = ModelRunner.build(name, max_seq_len=256, max_gpu_num_blocks=1024, quantization="mxfp4", dtype=dtype)
    logits = prefill(runner, batch, prompt)
    assert logits.isfinite().all()
    tok = logits[:, -1].argmax(-1)
    for i in range(2):
        runner.decode_alloc_kv_cache(batch)
        tok = runner.forward(tok.view(batch, 1), torch.full((batch, 1), prompt + i, device="cuda"))[:, -1].argmax(-1)
    moe = name.endswith("moe")
    steps, layers = 3, runner.num_layers
    assert checked["norm"] == steps * layers * (1 if moe else 2)
    assert checked["gated"] == (0 if moe else steps * layers) and checked["moe"] == (steps * layers if moe else 0)
    assert checked["matmul"] == steps * layers * (2 if moe else 3)


@pytest.mark.parametrize("name", ("tiny-llama", "tiny-qwen3-moe"))
def test_a_captured_step_gives_the_eager_steps_bits(name):
    runner = ModelRunner.build(name, max_seq_len=256, max_gpu_num_blocks=1024, quantization="mxfp4")

    def eager_step(tok, pos):
        here = runner.atten_info.max_actual_seq_len
        runner.atten_info.max_actual_seq_len = 256                       # the bucket, so that attention is parted alike
        out = runner.model.forward(tok, pos, runner.atten_info)
        runner.atten_info.max_actual_seq_len = here
        return out

    def run(step):
        torch.manual_seed(3)
        runner.kv_cache_manager.free_all()
        out = [prefill(runner, 4, 20)]
        pos = torch.full((4, 1), 20, device="cuda")
        for _ in range(4):
            runner.decode_alloc_kv_cache(4)
            out.append(step(out[-1][:, -1].argmax(-1).view(4, 1), pos).clone())
            pos = pos + 1
        return out
    eager = run(eager_step)
    runner.kv_cache_manager.free_all()
    runner.enable_cuda_graph((4,), (256,))
    for a, b in zip(eager, run(runner.forward)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name,kw", (("tiny-qwen3", dict(kv_cache_dtype="int4")), ("tiny-qwen3-moe", dict(kv_cache_dtype="int4")), ("tiny-qwen2", {})))
def test_served_by_the_engine(checked, name, kw):
    runner = ModelRunner.build(name, max_seq_len=256, max_gpu_num_blocks=1024, quantization="mxfp4", **kw)
    gen = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, 1000, (n,), generator=gen).tolist() for n in (3, 40, 17)]
    out = Engine(runner).generate(prompts, 5)
    assert [len(o) for o in out] == [5, 5, 5] and checked["matmul"] > 0 and checked["norm"] > 0


def test_weights_take_a_little_more_than_half_a_byte():
    q = methods.make_linear_weights(torch.randn(1024, 2048, device="cuda"), "mxfp4")
    assert q.nbytes() == 1024 * 2048 * 17 // 32
