"""Served prompts that reach the experts' tiles of 128 and 256 rows, every call of the decoder against 64 bits."""

from __future__ import annotations

import pytest
import torch

from lite_llama_b200.executor import ModelRunner
from lite_llama_b200.executor.model_config import PRESETS
from lite_llama_b200.kernels._common import lib
from test_mxfp4_runner_gpu import checked, prefill  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("experts,tile", ((32, 128), (8, 256)))
@pytest.mark.parametrize("dtype", (torch.float16, torch.bfloat16))
def test_a_prompt_over_many_rows_an_expert(checked, experts, tile, dtype):  # noqa: F811
    batch, prompt = 10, 250
    cfg = PRESETS["tiny-qwen3-moe"].with_(num_experts=experts)
    assert lib().b2l_mxfp4_moe_tile_rows(batch * prompt * 2, experts, 2 * cfg.moe_intermediate_size) == tile
    runner = ModelRunner.build(cfg, max_seq_len=256, max_gpu_num_blocks=4096, quantization="mxfp4", dtype=dtype)
    logits = prefill(runner, batch, prompt)
    assert logits.isfinite().all() and checked["moe"] == runner.num_layers
