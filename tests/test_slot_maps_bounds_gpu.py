"""build_slot_maps with lengths that 32 bits do not hold: nothing outside the table is written, and what fits is as ever."""

from __future__ import annotations

import pytest
import torch

import kv_int4_oracle as O
from lite_llama_b200 import kernels as K

pytestmark = pytest.mark.gpu
MOST = 2**31 - 1


@pytest.mark.parametrize("pool", [False, True])
@pytest.mark.parametrize("ctx,new", [
    ([2**63 - 1, 1, 0], [3, 2, 4]), ([2**63 - 2, 2**31, 5], [1, 4, 2]), ([0, 2, 1], [2, 2**63 - 1, 2**62]), ([4, 0, 2**40], [2**63 - 1, 2**63 - 1, 2**63 - 1]),
    ([-2**63, -1, 0], [3, -2**63, 5]), ([MOST, 0, MOST], [MOST, 2, MOST]),
], ids=str)
def test_lengths_past_32_bits(ctx, new, pool):
    width, total = 16, 12
    around = torch.full((9, width), -5, dtype=torch.int32, device="cuda")
    around[3:6] = torch.arange(3 * width, dtype=torch.int32, device="cuda").view(3, width)
    table = around[3:6]
    plain = table.tolist()
    rows = torch.arange(100, 100 + total, device="cuda") if pool else None
    within = [[min(max(x, 0), MOST) for x in side] for side in (ctx, new)]
    # the oracle walks a request's new tokens one by one: no more of them than the batch holds
    want = O.slot_maps([0, 1, 2], within[0], [min(x, total + 1) for x in within[1]], plain, total, None if rows is None else rows.tolist())
    i64 = dict(dtype=torch.int64, device="cuda")
    got = K.build_slot_maps(torch.tensor([0, 1, 2], **i64), torch.tensor(ctx, **i64), torch.tensor(new, **i64), table, total, rows)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1] and table.tolist() == plain
    assert (around[:3] == -5).all() and (around[6:] == -5).all()
    starts = [min(sum(within[1][:b]), MOST) for b in range(3)]
    assert got[2].tolist() == starts and got[3].tolist() == [min(c + n, MOST) for c, n in zip(*within)]
