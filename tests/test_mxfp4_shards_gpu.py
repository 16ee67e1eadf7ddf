"""Routed decoders in microscaled 4-bit floating point whose experts are cut into shards of any size."""

from __future__ import annotations

import pytest
import torch

import mxfp4_oracle as O
from lite_llama_b200 import kernels as K
from lite_llama_b200.executor import decoder
from lite_llama_b200.executor.model_config import PRESETS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inner,ranks", ((768, 8), (192, 4), (144, 3)))
@pytest.mark.parametrize("tokens", (5, 400))
def test_shards_add_up_to_the_layer(inner, ranks, tokens):
    """96, 48 and 48 of a rank: what each gives is its own columns' part, in the format."""
    cfg = PRESETS["tiny-qwen3-moe"].with_(moe_intermediate_size=inner)
    e, h, il = cfg.num_experts, cfg.hidden_size, inner // ranks
    gate, up, down = (torch.randn(e, *s, device="cuda") * 0.05 for s in ((inner, h), (inner, h), (h, inner)))
    router = torch.randn(e, h, device="cuda")
    x = torch.randn(tokens, h, device="cuda").half()
    top = torch.softmax(torch.randn(tokens, e, device="cuda"), -1).topk(2, -1)
    for rank in range(ranks):
        m = decoder.make_moe_weights(cfg, router, gate, up, down, "mxfp4", ranks, rank, torch.float16)
        assert m.num_experts == e
        part = slice(rank * il, (rank + 1) * il)
        g, u = O.rounded(gate[:, part].half()), O.rounded(up[:, part].half())
        d = O.rounded(torch.nn.functional.pad(down[:, :, part].half(), (0, -il % 32)))[..., :il]
        got = K.fused_moe_mxfp4(x, m.w1, m.w2, top.values, top.indices).double()
        xv, want, off = O.rounded(x), torch.zeros(tokens, h, dtype=torch.float64, device="cuda"), torch.zeros(tokens, h, dtype=torch.float64, device="cuda")
        for i in range(e):
            t, j = torch.nonzero(top.indices == i, as_tuple=True)
            act = torch.nn.functional.silu(xv[t] @ g[i].t()) * (xv[t] @ u[i].t())
            act = torch.nn.functional.pad(act, (0, -il % 32))
            q = O.rounded(act)[:, :il]
            # a value whose sums in 32 bits fall on the other side of a border is one step off, two scales at most
            step = torch.exp2(O.quantise(act)[1].double() - 127).repeat_interleave(32, 1)[:, :il]
            w = top.values[t, j].double()[:, None]
            y = q @ d[i].t()
            want.index_add_(0, t, w * y)
            off.index_add_(0, t, w * (2 * step.amax(-1, keepdim=True) * d[i].abs().amax() + il * 2.0 ** -22 * (q.abs() @ d[i].abs().t())))
        far = (got - want).abs()
        assert (far <= off + want.abs() * 2.0 ** -11 + 1e-7).all()
        assert (far <= off / 1000 + want.abs() * 2.0 ** -10 + 1e-7).float().mean() > 0.98      # hardly any is off at all
