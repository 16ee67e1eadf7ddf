"""The uniform decoders over a 4-bit pool: every write and every attention call that a model makes is compared with 64 bits."""

from __future__ import annotations

import pytest
import torch

import kv_int4_oracle as O
from lite_llama_b200.engine import Engine
from lite_llama_b200.executor import PRESETS, ModelRunner
from lite_llama_b200.executor import decoder as D
from lite_llama_b200.executor.model_runner import GreedyDecodeLoop

pytestmark = pytest.mark.gpu

MODELS = [("tiny-llama", torch.float16, {}), ("tiny-qwen3", torch.bfloat16, {}), ("tiny-qwen2", torch.float16, dict(quantization="int4")),
          ("tiny-llama", torch.float16, dict(head_dim=128, kv_group_size=32))]


def _build(name, dtype, kw, requests=4, width=64):
    kw = dict(kw)
    cfg = PRESETS[name]
    if "head_dim" in kw:
        cfg = cfg.with_(head_dim=kw.pop("head_dim"))
    return ModelRunner.build(cfg, max_seq_len=width, max_gpu_num_blocks=requests * width, device="cuda", dtype=dtype, seed=0,
                             kv_cache_dtype="int4", **kw)


def _ids(*shape, seed=0):
    return torch.randint(0, 1000, shape, generator=torch.Generator().manual_seed(seed))


@pytest.fixture
def calls(monkeypatch):
    """Checks each call of the decoder's three operators as it is made; counts them."""
    count = dict(write=0, decode=0, portions=0, tokens=None)
    write, decode, portions = D.rope_kv_write_int4, D.flash_decoding_int4, D.flash_attention_int4

    def checked_write(q, k, v, cos, sin, index, pool, batch, seq, group):
        out = write(q, k, v, cos, sin, index, pool, batch, seq, group)
        used = k.shape[1] * (k.shape[2] + 8 * (k.shape[2] // group))
        # a padded prompt's tokens behind its length come from what no kernel wrote: any bits, of which NaN and zeros have several
        real = count["tokens"] if seq > 1 and count["tokens"] is not None else torch.ones(k.shape[0], dtype=torch.bool, device="cuda")
        assert torch.equal(pool[index.long()][real, :used], O.rows_of(k, v, group)[real, :used])
        count["write"] += 1
        return out

    def compare(out, q, pool, scale, table, req, lens, starts, new, heads, group, oracle):
        for r, n, s, m in zip(req.tolist(), lens.tolist(), starts, new):
            want, error = oracle(q[s:s + m], pool[table[r, :n].long()], heads, group, scale)
            assert O.within(out[s:s + m], want, error).all()

    def checked_decode(q, pool, scale, table, req, lens, max_len, heads, group, into=None):
        out = decode(q, pool, scale, table, req, lens, max_len, heads, group, into)
        b = q.shape[0]
        compare(out, q, pool, scale, table, req, lens, range(b), [1] * b, heads, group, O.attention)
        count["decode"] += 1
        return out

    def checked_portions(q, pool, scale, start, new, table, req, lens, max_new, max_len, heads, group, into):
        out = portions(q, pool, scale, start, new, table, req, lens, max_new, max_len, heads, group, into)
        compare(out, q, pool, scale, table, req, lens, start.tolist(), new.tolist(), heads, group, O.prompt_attention)
        count["portions"] += 1
        return out

    monkeypatch.setattr(D, "rope_kv_write_int4", checked_write)
    monkeypatch.setattr(D, "flash_decoding_int4", checked_decode)
    monkeypatch.setattr(D, "flash_attention_int4", checked_portions)
    return count


@pytest.mark.parametrize("name,dtype,kw", MODELS, ids=str)
def test_engine(name, dtype, kw, calls):
    runner = _build(name, dtype, kw)
    heads, d = runner.num_kv_heads, runner.head_dim
    assert all(t.shape[1] == O.row_bytes(heads, d, runner.kv_group_size) for t in runner.kv_cache_manager.gpu_kv_buffer)
    engine = Engine(runner, max_step_tokens=16, max_portion=7)
    prompts = [_ids(n, seed=n).tolist() for n in (1, 13, 40, 5, 7)]          # five requests, three slots
    outs = engine.generate(prompts, 6)
    assert [len(o) for o in outs] == [6] * 5
    assert calls["portions"] > 0 and calls["decode"] > 0 and calls["write"] <= calls["portions"] + calls["decode"]


@pytest.mark.parametrize("name,dtype,kw", MODELS[:2], ids=str)
def test_padded_prompts_then_decode(name, dtype, kw, calls):
    runner = _build(name, dtype, kw)
    lens = torch.tensor([12, 7, 9], device="cuda")
    runner.prefill_alloc_kv_cache(12, lens.clone(), torch.arange(3, device="cuda"))
    calls["tokens"] = (torch.arange(12, device="cuda") < lens[:, None]).flatten()
    logits = runner.forward(_ids(3, 12).cuda(), torch.arange(12, device="cuda").repeat(3, 1))
    assert all(torch.isfinite(logits[b, :n]).all() for b, n in enumerate(lens.tolist()))
    for _ in range(3):
        runner.decode_alloc_kv_cache(3)
        pos = (runner.atten_info.b_seq_len - 1).view(3, 1)
        assert torch.isfinite(runner.forward(_ids(3, 1).cuda(), pos)).all()
    layers = runner.num_layers
    assert (calls["write"], calls["decode"], calls["portions"]) == (4 * layers, 3 * layers, 0)


def test_a_captured_decode_step_is_the_eager_one():
    runner = _build("tiny-llama", torch.float16, {}, requests=3, width=256)
    runner.enable_cuda_graph(batch_sizes=(2,), seq_len_buckets=(256,))
    slots = runner.enable_slot_kv_cache()
    prompt = _ids(1, 150).cuda()
    pos = slots.begin_portions([1, 0], [0, 0], [100, 50])
    assert pos.tolist() == [[*range(100), *range(50)]]
    runner.forward(prompt, pos, last_token_index=torch.tensor([99, 149], device="cuda"))
    at = runner.atten_info
    for step in range(2):
        assert slots.begin_decode([1, 0], [101 + step, 51 + step]) == 2
        token, pos = _ids(2, 1, seed=step).cuda(), torch.tensor([[100 + step], [50 + step]], device="cuda")
        got = runner.forward(token, pos).clone()
        longest, at.max_actual_seq_len = at.max_actual_seq_len, 256                # as captured
        assert torch.equal(got, runner.model.forward(token, pos, at))
        at.max_actual_seq_len = longest


def test_portions_of_one_prompt_and_a_captured_last_token():
    """A portion of one token takes the captured decode step: same pool, same bits as the decode step itself."""
    runner = _build("tiny-llama", torch.float16, {}, requests=3, width=256)
    runner.enable_cuda_graph(batch_sizes=(1,), seq_len_buckets=(256,))
    slots = runner.enable_slot_kv_cache()
    prompt = _ids(1, 41).cuda()
    for at in (0, 20):
        pos = slots.begin_portions([1], [at], [20])
        runner.forward(prompt[:, at:at + 20], pos, last_token_index=torch.tensor([0], device="cuda"))
    pos = slots.begin_portions([1], [40], [1])
    one = runner.forward(prompt[:, 40:], pos, last_token_index=torch.tensor([0], device="cuda")).clone()
    slots.begin_decode([1], [41])
    assert torch.equal(one, runner.forward(prompt[:, 40:], pos))


def test_greedy_loop():
    runner = _build("tiny-qwen3", torch.bfloat16, {}, requests=4, width=64)
    runner.prefill_alloc_kv_cache(10, torch.tensor([10, 10], device="cuda"), torch.arange(2, device="cuda"))
    logits = runner.forward(_ids(2, 10).cuda(), torch.arange(10, device="cuda").repeat(2, 1))
    first, lens = logits[:, -1].argmax(-1), torch.tensor([10, 10], device="cuda")
    loop = GreedyDecodeLoop(runner, 2, 64)
    loop.begin(first, lens, torch.arange(2, device="cuda"), max_steps=5)
    row = loop._reserved[0]
    loop.capture()
    tokens = []
    for _ in range(5):
        loop.step()
        tokens.append(loop.next_tokens.clone())
    loop.begin(first, lens, torch.arange(2, device="cuda"), first_row=row)
    for want in tokens:                                                             # the same steps without the graph
        loop._step_ops()
        assert torch.equal(loop.next_tokens, want)
