"""K and V cached in 4 bits: the writer, the reader, decode and prompt attention over it.

The counterparts of ``rope_kv_write``, ``update_kv_buffer_split`` and ``flash_decoding`` for a pool ``[max_tokens, row_bytes]`` of
bytes.  A row holds one token: for every kv head the codes of K, the codes of V (4 bits each, element ``2i`` in the low half of byte
``i``), then K's and V's (scale, minimum) per group of ``group_size`` elements in the activations' type; the row is filled up to a
multiple of 16 bytes (``kv_int4_row_bytes``).  An element is ``minimum + scale * code``: a group's smallest element is kept, its
largest is met up to the rounding of the scale, the others are at most half a step off.  A group with an infinity or a NaN reads as
NaN.  Head sizes 32, 64 and 128; groups of 32, 64 or 128, at most the head size.  A cache is written and read in one activation
type, float16 or bfloat16.
"""

from __future__ import annotations

import torch

from . import _native
from ._common import check, dtype_code, index_width, lib, no_grad, require_cuda, stream_handle, workspace


def kv_int4_row_bytes(num_kv_heads: int, head_dim: int, group_size: int = 64) -> int:
    """Bytes of one token's row."""
    nbytes = lib().b2l_kv_int4_row_bytes(num_kv_heads, head_dim, group_size)
    if nbytes == 0:
        raise ValueError(f"a 4-bit cache has no rows of {num_kv_heads} heads of {head_dim} in groups of {group_size} "
                         "(head_dim 32, 64 or 128; groups of 32, 64 or 128, at most head_dim)")
    return nbytes


def _cache_rows(kv_buffer: torch.Tensor, num_kv_heads: int, head_dim: int, group_size: int, what: str) -> tuple[int, int, int]:
    """Address, row stride and number of rows of a cache that holds such heads."""
    if kv_buffer.dtype != torch.uint8 or kv_buffer.dim() != 2 or kv_buffer.stride(1) != 1:
        raise ValueError(f"{what}: the cache is a uint8 matrix [max_tokens, row_bytes] with contiguous rows")
    need = kv_int4_row_bytes(num_kv_heads, head_dim, group_size)
    rows, width = kv_buffer.shape
    if width < need:
        raise ValueError(f"{what}: a row of {num_kv_heads} heads of {head_dim} in groups of {group_size} takes {need} bytes, "
                         f"the cache has {width}")
    stride = kv_buffer.stride(0) if rows > 1 else (width + 15) // 16 * 16
    if stride < width:
        raise ValueError(f"{what}: the cache's rows overlap")
    return kv_buffer.data_ptr(), stride, rows


def _same_device(what: str, *tensors: torch.Tensor) -> None:
    """All on the current device, whose stream the launch goes to."""
    require_cuda(*tensors)
    current = torch._C._cuda_getDevice()
    for t in tensors:
        if t is not None and t.device.index != current:
            raise ValueError(f"{what}: a tensor is on {t.device}, the current device is cuda:{current}")


def _heads(t: torch.Tensor, what: str) -> tuple[int, int]:
    if t.dim() != 3 or t.stride(2) != 1:
        raise ValueError(f"{what} must be [tokens, heads, head_dim] with a contiguous head_dim")
    return t.stride(0), t.stride(1)


@no_grad
def update_kv_buffer_int4(K_Values, V_Values, Select_Index, KV_Buffer, group_size: int = 64) -> None:
    """Store the rows ``K_Values`` and ``V_Values [tokens, Hkv, D]`` in ``KV_Buffer`` at ``Select_Index`` (int32 or int64).

    An index outside ``[0, max_tokens)`` stores nothing (padded tokens: -1).  Where two tokens name one row, what it holds afterwards
    may come from either of them, element by element."""
    code = dtype_code(K_Values, "K_Values")
    ks, vs = _heads(K_Values, "K_Values"), _heads(V_Values, "V_Values")
    n, hkv, d = K_Values.shape
    if V_Values.shape != K_Values.shape or V_Values.dtype != K_Values.dtype:
        raise ValueError("update_kv_buffer_int4: K_Values and V_Values must have one shape and type")
    if Select_Index.dim() != 1 or Select_Index.shape[0] != n or not Select_Index.is_contiguous():
        raise ValueError("update_kv_buffer_int4: Select_Index is a contiguous vector with one entry per token")
    address, stride, rows = _cache_rows(KV_Buffer, hkv, d, group_size, "update_kv_buffer_int4")
    _same_device("update_kv_buffer_int4", K_Values, V_Values, Select_Index, KV_Buffer)
    if n:
        check(lib().b2l_kv_int4_write(
            None, None, None, K_Values.data_ptr(), V_Values.data_ptr(), None, None, Select_Index.data_ptr(),
            index_width(Select_Index, "Select_Index"), address, stride, rows, n, 1, 0, hkv, d, group_size, 0, 0, *ks, *vs, 0, 0, 0, 0,
            0, 0, code, stream_handle()))


def rope_kv_write_int4(q, k, v, cos, sin, select_index, kv_buffer, batch_size, seq_len, group_size: int = 64, out_q=None, out_k=None):
    """``rope_kv_write`` into a 4-bit cache: rotate ``q [T, Hq, D]`` and ``k [T, Hkv, D]`` by ``cos/sin [batch, seq, D]`` (the first half
    of a row is read) and store the rotated, rounded keys and ``v`` at ``select_index``, in one launch.

    The rotated tensors go to ``out_q`` and ``out_k``, by default to ``q`` and ``k`` themselves; both are returned.  The rotation is done in
    32 bits and rounded once.  Rows as in ``update_kv_buffer_int4``."""
    out = _native.kv4_rope_write(q, k, v, cos, sin, select_index, kv_buffer, batch_size, seq_len, group_size, out_q, out_k)
    return _rope_kv_write_int4(q, k, v, cos, sin, select_index, kv_buffer, batch_size, seq_len, group_size, out_q, out_k) if out is None else out


@no_grad
def _rope_kv_write_int4(q, k, v, cos, sin, select_index, kv_buffer, batch_size, seq_len, group_size: int = 64, out_q=None, out_k=None):
    out_q, out_k = q if out_q is None else out_q, k if out_k is None else out_k
    code = dtype_code(q, "q")
    qs, ks, vs = _heads(q, "q"), _heads(k, "k"), _heads(v, "v")
    qo, ko = _heads(out_q, "out_q"), _heads(out_k, "out_k")
    n, hq, d = q.shape
    hkv = k.shape[1]
    if batch_size * seq_len != n or k.shape[0] != n or v.shape != k.shape or k.shape[2] != d:
        raise ValueError("rope_kv_write_int4: q, k and v hold batch_size * seq_len tokens of one head size")
    if out_q.shape != q.shape or out_k.shape != k.shape:
        raise ValueError("rope_kv_write_int4: out_q and out_k have the shapes of q and k")
    if any(t.dtype != q.dtype for t in (k, v, cos, sin, out_q, out_k)):
        raise ValueError("rope_kv_write_int4: all tensors must be in the activation dtype")
    if cos.dim() == 2:                               # one row per token
        cos, sin = cos.unsqueeze(0) if batch_size == 1 else cos.view(batch_size, seq_len, -1), \
            sin.unsqueeze(0) if batch_size == 1 else sin.view(batch_size, seq_len, -1)
    if cos.shape != sin.shape or cos.stride() != sin.stride() or cos.stride(-1) != 1 or cos.shape[:2] != (batch_size, seq_len) \
            or cos.shape[-1] < d // 2:
        raise ValueError("rope_kv_write_int4: cos and sin must be alike, [batch, seq, at least D / 2], with contiguous rows")
    if select_index.dim() != 1 or select_index.shape[0] != n or not select_index.is_contiguous():
        raise ValueError("rope_kv_write_int4: select_index is a contiguous vector with one entry per token")
    address, stride, rows = _cache_rows(kv_buffer, hkv, d, group_size, "rope_kv_write_int4")
    _same_device("rope_kv_write_int4", q, k, v, cos, sin, select_index, kv_buffer, out_q, out_k)
    if n:
        check(lib().b2l_kv_int4_write(
            out_q.data_ptr(), out_k.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(),
            select_index.data_ptr(), index_width(select_index, "select_index"), address, stride, rows, n, seq_len, hq, hkv, d, group_size,
            *qs, *ks, *vs, cos.stride(0), cos.stride(1), *qo, *ko, code, stream_handle()))
    return out_q, out_k


def read_kv_buffer_int4(KV_Buffer, Select_Index, num_kv_heads: int, head_dim: int, dtype: torch.dtype, group_size: int = 64) -> torch.Tensor:
    """The values of the rows ``Select_Index`` as ``[tokens, 2 * Hkv, D]`` (K heads, then V heads) in ``dtype``, the type the cache was
    written in, at most its largest finite number.  An index outside the cache reads as zeros."""
    out = _native.kv4_read(KV_Buffer, Select_Index, num_kv_heads, head_dim, dtype, group_size)
    return _read_kv_buffer_int4(KV_Buffer, Select_Index, num_kv_heads, head_dim, dtype, group_size) if out is None else out


@no_grad
def _read_kv_buffer_int4(KV_Buffer, Select_Index, num_kv_heads: int, head_dim: int, dtype: torch.dtype, group_size: int = 64) -> torch.Tensor:
    if Select_Index.dim() != 1 or not Select_Index.is_contiguous():
        raise ValueError("read_kv_buffer_int4: Select_Index is a contiguous vector")
    address, stride, rows = _cache_rows(KV_Buffer, num_kv_heads, head_dim, group_size, "read_kv_buffer_int4")
    _same_device("read_kv_buffer_int4", KV_Buffer, Select_Index)
    out = torch.empty((Select_Index.shape[0], 2 * num_kv_heads, head_dim), dtype=dtype, device=KV_Buffer.device)
    code = dtype_code(out, "dtype")
    if out.numel():
        check(lib().b2l_kv_int4_read(out.data_ptr(), address, stride, rows, Select_Index.data_ptr(),
                                     index_width(Select_Index, "Select_Index"), Select_Index.shape[0], num_kv_heads, head_dim, group_size,
                                     code, stream_handle()))
    return out


def _table(b_req_tokens_table, what: str) -> tuple[int, int, int, int]:
    if b_req_tokens_table.dtype != torch.int32 or b_req_tokens_table.dim() != 2:
        raise ValueError(f"{what}: b_req_tokens_table must be an int32 matrix, got {b_req_tokens_table.dtype}")
    return (*b_req_tokens_table.stride(), *b_req_tokens_table.shape)


def _vector(t: torch.Tensor, n: int, name: str, what: str) -> None:
    if t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{what}: {name} is a contiguous vector with one entry per sequence")


def flash_decoding_int4(q, kv_buffer, qk_scale, b_req_tokens_table, b_req_idx, b_seq_len, max_actual_seq_len, num_kv_heads: int,
                        group_size: int = 64, out=None) -> torch.Tensor:
    """``flash_decoding`` over a 4-bit cache: one query ``q [B, Hq, D]`` per sequence against its cached tokens, ``qk_scale = 1/sqrt(D)``;
    into ``out``, by default a new tensor.

    Scores, softmax and sums are held in 32 bits and the cached elements enter as they are, so the result is that of 32-bit attention
    over ``read_kv_buffer_int4``'s values before their rounding, rounded once.  A row of length 0, or of a request outside the table, is
    zero; a table entry outside the cache reads row 0; lengths count up to ``max_actual_seq_len`` and the table's width.  Up to 64 query
    heads share a kv head.

    The same arguments give the same bits.  Where a row's tokens are parted for the sum follows from the lengths of all rows, so a
    sequence's last bits may change with what stands beside it."""
    args = (q, kv_buffer, qk_scale, b_req_tokens_table, b_req_idx, b_seq_len, max_actual_seq_len, num_kv_heads, group_size, out)
    got = _native.kv4_decode(*args)
    return _flash_decoding_int4(*args) if got is None else got


@no_grad
def _flash_decoding_int4(q, kv_buffer, qk_scale, b_req_tokens_table, b_req_idx, b_seq_len, max_actual_seq_len, num_kv_heads: int,
                        group_size: int = 64, out=None) -> torch.Tensor:
    what = "flash_decoding_int4"
    code = dtype_code(q, "q")
    if q.dim() != 3:
        raise ValueError(f"{what}: q must be [batch, heads, head_dim]")
    if q.stride(2) != 1:
        q = q.contiguous()
    batch, hq, d = q.shape
    if num_kv_heads < 1 or hq % num_kv_heads:
        raise ValueError(f"{what}: {hq} query heads are no multiple of {num_kv_heads} kv heads")
    _vector(b_req_idx, batch, "b_req_idx", what)
    _vector(b_seq_len, batch, "b_seq_len", what)
    address, stride, rows = _cache_rows(kv_buffer, num_kv_heads, d, group_size, what)
    table = _table(b_req_tokens_table, what)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1):
        raise ValueError(f"{what}: out has the shape and type of q and a contiguous head_dim")
    _same_device(what, q, kv_buffer, b_req_tokens_table, b_req_idx, b_seq_len, out)
    if out is None:
        out = torch.empty((batch, hq, d), dtype=q.dtype, device=q.device)
    if batch == 0:
        return out
    max_len = int(max_actual_seq_len)
    nbytes = lib().b2l_flash_decoding_int4_workspace_bytes(batch, hq, num_kv_heads, d, group_size, max_len)
    ws = workspace(max(nbytes, 16), q.device)
    check(lib().b2l_flash_decoding_int4(
        out.data_ptr(), q.data_ptr(), address, stride, rows, b_req_tokens_table.data_ptr(), *table,
        b_req_idx.data_ptr(), index_width(b_req_idx, "b_req_idx"), b_seq_len.data_ptr(), index_width(b_seq_len, "b_seq_len"),
        batch, hq, num_kv_heads, d, group_size, max_len, float(qk_scale), q.stride(0), q.stride(1), out.stride(0), out.stride(1),
        ws.data_ptr(), nbytes, code, stream_handle()))
    return out


def flash_attention_int4(q, kv_buffer, qk_scale, b_start_loc, b_new_len, b_req_tokens_table, b_req_idx, b_seq_len, max_new_len,
                         max_actual_seq_len, num_kv_heads: int, group_size: int = 64, out=None) -> torch.Tensor:
    """Portions of prompts over a 4-bit cache that already holds them: sequence ``b`` brings the ``b_new_len[b]`` rows of ``q [T, Hq, D]``
    from ``b_start_loc[b]`` on, its last tokens of ``b_seq_len[b]`` cached ones; each sees the cached tokens up to itself.

    The products are of 16-bit operands: cached elements are rounded to halves, by 2^-11 of themselves or by 2^-25 (for bf16 models too, whose
    elements beyond 65504 count as 65504), and so are the probabilities; sums and the softmax are held in 32 bits.  ``max_new_len`` and ``max_actual_seq_len`` are
    bounds that the host knows: new tokens and keys past them do not count.  A row that sees nothing is zero; rows of ``q`` that belong to no
    sequence are not written (``out``, by default a new tensor, keeps what it held there); a table entry outside the cache reads row 0.
    A row belongs to one sequence: where the ranges overlap (starts of an earlier step), it holds what one of its sequences gives, and
    sequences past the row blocks that disjoint ranges could make are left out, their rows not written.

    The same arguments give the same bits; where a row's keys are parted for the sum follows from all lengths of the step."""
    args = (q, kv_buffer, qk_scale, b_start_loc, b_new_len, b_req_tokens_table, b_req_idx, b_seq_len, max_new_len, max_actual_seq_len,
            num_kv_heads, group_size, out)
    got = _native.kv4_prompt(*args)
    return _flash_attention_int4(*args) if got is None else got


@no_grad
def _flash_attention_int4(q, kv_buffer, qk_scale, b_start_loc, b_new_len, b_req_tokens_table, b_req_idx, b_seq_len, max_new_len,
                         max_actual_seq_len, num_kv_heads: int, group_size: int = 64, out=None) -> torch.Tensor:
    what = "flash_attention_int4"
    code = dtype_code(q, "q")
    if q.dim() != 3:
        raise ValueError(f"{what}: q must be [tokens, heads, head_dim]")
    if q.stride(2) != 1:
        q = q.contiguous()
    tokens, hq, d = q.shape
    if num_kv_heads < 1 or hq % num_kv_heads:
        raise ValueError(f"{what}: {hq} query heads are no multiple of {num_kv_heads} kv heads")
    batch = b_req_idx.shape[0]
    for t, name in ((b_start_loc, "b_start_loc"), (b_new_len, "b_new_len"), (b_req_idx, "b_req_idx"), (b_seq_len, "b_seq_len")):
        _vector(t, batch, name, what)
    address, stride, rows = _cache_rows(kv_buffer, num_kv_heads, d, group_size, what)
    table = _table(b_req_tokens_table, what)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1):
        raise ValueError(f"{what}: out has the shape and type of q and a contiguous head_dim")
    _same_device(what, q, kv_buffer, b_start_loc, b_new_len, b_req_tokens_table, b_req_idx, b_seq_len, out)
    if out is None:
        out = torch.empty((tokens, hq, d), dtype=q.dtype, device=q.device)
    if batch == 0 or tokens == 0:
        return out
    max_len = int(max_actual_seq_len)
    nbytes = lib().b2l_flash_attention_int4_workspace_bytes(batch, tokens, hq, num_kv_heads, d, group_size, max_len)
    ws = workspace(max(nbytes, 16), q.device)
    check(lib().b2l_flash_attention_int4(
        out.data_ptr(), q.data_ptr(), address, stride, rows, b_start_loc.data_ptr(), index_width(b_start_loc, "b_start_loc"),
        b_new_len.data_ptr(), index_width(b_new_len, "b_new_len"), b_req_tokens_table.data_ptr(), *table,
        b_req_idx.data_ptr(), index_width(b_req_idx, "b_req_idx"), b_seq_len.data_ptr(), index_width(b_seq_len, "b_seq_len"),
        batch, tokens, int(max_new_len), hq, num_kv_heads, d, group_size, max_len, float(qk_scale),
        q.stride(0), q.stride(1), out.stride(0), out.stride(1), ws.data_ptr(), nbytes, code, stream_handle()))
    return out
