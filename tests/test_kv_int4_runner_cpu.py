"""The 4-bit pool of the uniform decoders, on the host: refusals, slot metadata that is refused, the engine's flat steps."""

from __future__ import annotations

import pytest
import torch

from lite_llama_b200.engine import Engine
from lite_llama_b200.executor import ModelRunner
from lite_llama_b200.executor.attention_metadata import AttentionMetadata
from lite_llama_b200.executor.kv_cache_manager import KVCacheManager
from lite_llama_b200.executor.model_config import PRESETS, LayeredConfig
from lite_llama_b200.executor.slot_batch import SlotBatch

CFG = PRESETS["tiny-llama"]


@pytest.mark.parametrize("config,kw", [
    (CFG, dict(kv_cache_dtype="fp8")), (CFG, dict(kv_group_size=32)), (CFG, dict(kv_cache_dtype="int4", kv_group_size=64)),
    (CFG.with_(head_dim=96), dict(kv_cache_dtype="int4")), (object.__new__(LayeredConfig), dict(kv_cache_dtype="int4"))],
    ids=["no such type", "a group without the type", "a group larger than a head", "a head size without rows", "layer lists"])
def test_runner_refuses(config, kw):
    with pytest.raises(ValueError):
        ModelRunner(config, None, 64, device="cpu", **kw)


class _Runner:
    """What a SlotBatch and the engine touch, on the CPU; ``forward`` only records."""

    ragged_steps = False

    def __init__(self, group):
        self.device, self.max_seq_len, self.kv_group_size = "cpu", 16, group
        self.kv_cache_manager = KVCacheManager(1, 1, 32, 64, dtype=torch.uint8, device="cpu", row_widths=[48])
        self.b_req_tokens_table = torch.zeros((4, 16), dtype=torch.int32)
        self.atten_info = AttentionMetadata(b_req_tokens_table=self.b_req_tokens_table)

    def graph_batch_size(self, n):
        return n

    def enable_slot_kv_cache(self):
        return SlotBatch(self)


def test_portions_need_a_4_bit_pool():
    with pytest.raises(RuntimeError):
        SlotBatch(_Runner(0)).begin_portions([0], [0], [1])


@pytest.mark.parametrize("slots,cached,new", [([], [], []), ([0], [0, 1], [1]), ([0, 1], [0, 0], [1, 0]), ([0], [-1], [2]), ([1, 1], [0, 0], [1, 1]),
                                              ([3], [0], [1]), ([-1], [0], [1]), ([0], [10], [7])], ids=str)
def test_portions_that_do_not_fit(slots, cached, new):
    with pytest.raises(ValueError):
        SlotBatch(_Runner(32)).begin_portions(slots, cached, new)


def test_the_engine_reads_prompts_in_portions_beside_decoding_requests():
    """The flat steps' requests, cached lengths and tokens: decoding requests first, portions of at most 4 under a budget of 6."""
    engine = Engine(_Runner(32), max_step_tokens=6, max_portion=4)
    for n in (2, 9, 3):
        engine.add_request(range(100 * n, 100 * n + n), 3)
    steps = []

    def step():
        entries, samplers, want = engine._schedule()
        steps.append([(r.rid, c, t) for r, c, t in entries])
        for r in samplers:
            engine._accept(r, 7, [])
        return want

    engine._admit()
    assert step() == [1]
    assert step() == [0]
    assert step() == [0, 1, 3]                    # 9 = 4 + 4 + 1 and 3 = 1 + 2: both prompts end here
    assert steps == [[(0, 0, [200, 201]), (1, 0, [900, 901, 902, 903])],
                     [(0, 2, [7]), (1, 4, [904, 905, 906, 907]), (2, 0, [300])],
                     [(0, 3, [7]), (1, 8, [908]), (2, 1, [301, 302])]]
    assert 0 in engine.done                       # three tokens: one at the prompt's end, two after
