"""flash_attention_int4 where ranges of q overlap: nothing is written outside the workspace, and rows hold one of their sequences' results."""

from __future__ import annotations

import pytest
import torch

import kv_int4_oracle as O
from lite_llama_b200 import _lib
from test_kv_int4_gpu import _normal, _step

pytestmark = pytest.mark.gpu


def _call(step, heads, group, scale, max_new, max_len, out):
    """The C entry with a workspace of the stated size inside a larger tensor, whose rest stays as it is."""
    lib = _lib.load()
    q, rows, start, new, table, req, n = step
    tokens, hq, d = q.shape
    batch = req.shape[0]
    nbytes = lib.b2l_flash_attention_int4_workspace_bytes(batch, tokens, hq, heads, d, group, max_len)
    ws = torch.full((nbytes + (1 << 20),), 0x5A, dtype=torch.uint8, device="cuda")
    _lib.check(lib.b2l_flash_attention_int4(
        out.data_ptr(), q.data_ptr(), rows.data_ptr(), rows.stride(0), rows.shape[0], start.data_ptr(), 4, new.data_ptr(), 4, table.data_ptr(),
        *table.stride(), *table.shape, req.data_ptr(), 4, n.data_ptr(), 4, batch, tokens, max_new, hq, heads, d, group, max_len, scale,
        q.stride(0), q.stride(1), out.stride(0), out.stride(1), ws.data_ptr(), nbytes, 0, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert (ws[nbytes:] == 0x5A).all()
    return out


@pytest.mark.parametrize("max_len", [700, 1 << 15])          # operands beside the products, and made ready
@pytest.mark.parametrize("batch,tokens", [(8, 512), (300, 512), (40, 64)])
def test_sequences_on_one_range(batch, tokens, max_len):
    """All sequences are one: every row has one result, whichever sequence gives it."""
    heads, d, group, length = 2, 64, 64, tokens + 88
    rows, table, req, n = _step([length], heads, d, group, torch.float16)
    q = _normal(tokens, 32, d, dtype=torch.float16)
    one = torch.ones(batch, dtype=torch.int32, device="cuda")
    step = (q, rows, 0 * one, tokens * one, table, req[0] * one, n[0] * one)
    # row blocks of 256: 16 to a token, so a sequence of 512 tokens has 32, and 8 of them 256; disjoint ranges 32 + 8
    out = _call(step, heads, group, 0.125, tokens, max_len, torch.full_like(q, 7.0))
    want, error = O.prompt_attention(q, rows[table[int(req[0]), :length].long()], heads, group, 0.125)
    assert O.within(out, want, error).all()


def test_starts_of_an_earlier_step():
    """Longer portions on the starts of shorter ones: a row holds its own sequence's result or that of the one before."""
    heads, d, group = 4, 128, 64
    lens, new, starts = [900, 700, 800, 600], [128] * 4, [0, 8, 16, 24]
    rows, table, req, n = _step(lens, heads, d, group, torch.float16)
    q = _normal(152, 64, d, dtype=torch.float16)
    i32 = dict(dtype=torch.int32, device="cuda")
    step = (q, rows, torch.tensor(starts, **i32), torch.tensor(new, **i32), table, req, n)
    # 128 tokens of 16 heads: 8 row blocks a sequence, 32 in all; disjoint ranges: 10 + 4, so that the first sequence alone fits
    keep = _normal(152, 64, d, dtype=torch.float16)
    out = _call(step, heads, group, 0.088, 128, 1024, keep.clone())
    want, error = O.prompt_attention(q[:128], rows[table[int(req[0]), :900].long()], heads, group, 0.088)
    assert O.within(out[:128], want, error).all() and torch.equal(out[128:], keep[128:])
