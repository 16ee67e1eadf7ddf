"""Slot maps of a ragged step, built on the GPU from the requests' lengths."""

from __future__ import annotations

import torch

from . import _native
from ._common import check, index_width, lib, no_grad, stream_handle
from .kv_int4 import _same_device, _table, _vector


def build_slot_maps(b_req_idx, b_ctx_len, b_new_len, b_req_tokens_table, total_tokens: int, rows=None):
    """Where the new tokens of a flat batch lie: request ``b`` (row ``b_req_idx[b]`` of ``b_req_tokens_table [requests, width]`` int32)
    has ``b_ctx_len[b]`` tokens cached and brings ``b_new_len[b]``, behind those of the requests before it.

    Returns ``(select_index int32 [total], position_ids int64 [total], b_start_loc int32 [B], b_seq_len int32 [B])``: a token's row of the
    pool and its position, each request's first token, and its length with the new tokens.  The rows come from the table (fixed slots),
    or from ``rows`` (at least ``total`` entries, int32 or int64), which are then entered into the table.  ``total_tokens`` may exceed the sum of the
    lengths (a captured size): the tokens behind it get row -1, which ``update_kv_buffer_int4`` skips, and position 0, and take nothing from
    ``rows``.  A position or request outside the table gets row -1; lengths, starts and their sums count up to 2^31 - 1.  Requests are
    different rows of the table: where two tokens with ``rows`` have one request and position, it holds the row of either.  Nothing is
    read by the host, so the call can be captured."""
    maps = _native.slot_maps(b_req_idx, b_ctx_len, b_new_len, b_req_tokens_table, total_tokens, rows)
    return _build_slot_maps(b_req_idx, b_ctx_len, b_new_len, b_req_tokens_table, total_tokens, rows) if maps is None else maps


@no_grad
def _build_slot_maps(b_req_idx, b_ctx_len, b_new_len, b_req_tokens_table, total_tokens: int, rows=None):
    what = "build_slot_maps"
    batch, total = b_req_idx.shape[0], int(total_tokens)
    for t, name in ((b_req_idx, "b_req_idx"), (b_ctx_len, "b_ctx_len"), (b_new_len, "b_new_len")):
        _vector(t, batch, name, what)
    rs, cs, requests, width = _table(b_req_tokens_table, what)
    if total < 0:
        raise ValueError(f"{what}: total_tokens is {total}")
    if rows is not None and (rows.dim() != 1 or rows.shape[0] < total or not rows.is_contiguous()):
        raise ValueError(f"{what}: rows is a contiguous vector with at least total_tokens entries")
    _same_device(what, b_req_idx, b_ctx_len, b_new_len, b_req_tokens_table, rows)
    dev = b_req_tokens_table.device
    select_index = torch.empty(total, dtype=torch.int32, device=dev)
    position_ids = torch.empty(total, dtype=torch.int64, device=dev)
    start, length = torch.empty(2, batch, dtype=torch.int32, device=dev)
    if total or batch:
        check(lib().b2l_slot_maps(
            select_index.data_ptr(), position_ids.data_ptr(), start.data_ptr(), length.data_ptr(),
            b_req_idx.data_ptr(), index_width(b_req_idx, "b_req_idx"), b_ctx_len.data_ptr(), index_width(b_ctx_len, "b_ctx_len"),
            b_new_len.data_ptr(), index_width(b_new_len, "b_new_len"),
            None if rows is None else rows.data_ptr(), 4 if rows is None else index_width(rows, "rows"),
            b_req_tokens_table.data_ptr(), rs, cs, requests, width, batch, total, stream_handle()))
    return select_index, position_ids, start, length
