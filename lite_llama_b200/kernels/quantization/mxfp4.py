"""Microscaled 4-bit floating point (MXFP4): e2m1 elements with a power of two for 32 of them, for weights and activations.

No counterpart in the reference, whose 4-bit weights are integers under 16-bit activations (lite_llama/kernels/quantization/
w4a16.py:152-207); beside the other quantised projections, this one multiplies 4 bits by 4 bits on the tensor cores.  Format, layout and
kernels: csrc/mxfp4.cuh, mxfp4_quant.cu, mxfp4_gemm.cu.
"""

from __future__ import annotations

from contextlib import nullcontext
from typing import NamedTuple

import torch

from .. import _native
from .._common import as_rows, check, current_device, dtype_code, float_code, index_width, lib, no_grad, ptr, require_cuda, stream_handle, weights_written

BLOCK = 32          # elements that share a scale
GATE_RUN = 64       # gate rows, then as many up rows


class MXFP4(NamedTuple):
    """A matrix ``[..., rows, k]`` in the format (or a stack of them).

    ``codes`` uint8 ``[..., rows, k / 2]``, element 2i in the low half of byte i; ``scales`` uint8
    ``[..., ceil(rows / 128), ceil(k / 128), 32, 4, 4]``, indices row % 32, row % 128 / 32, block % 4: the order the tensor cores read
    (``mxfp4_pack`` makes it from scales in rows; blocks behind ``k`` are 0, rows behind the last hold anything).  ``ready``: nothing that is still running on the GPU writes it, so that a product
    may request it as its weight while the kernel before is at work.  What the operators here return is not ready in this sense, nor
    are pieces of it (``MXFP4(q.codes[e], q.scales[e], q.ready)``); ``mxfp4_pack`` and ``mxfp4_quantize_weight`` return weights that
    are, and a pair of tensors that other code wrote is."""

    codes: torch.Tensor
    scales: torch.Tensor
    ready: bool = True

    @property
    def rows(self) -> int:
        return self.codes.shape[-2]

    @property
    def k(self) -> int:
        return 2 * self.codes.shape[-1]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()


def _tiles(rows: int, k: int) -> tuple[int, ...]:
    return (-(-rows // 128), -(-k // 128), 32, 4, 4)


def _on(t: torch.Tensor):
    """The device of ``t`` as the current one."""
    return nullcontext() if t.get_device() == current_device() else torch.cuda.device(t.device)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """The matrix ``t`` with rows that start on 16 bytes."""
    step = t.stride(0) * t.element_size()
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or (step % 16 == 0 and step >= 0)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _row_stride(t: torch.Tensor) -> int:
    """Of a matrix that ``_aligned`` returned: a single row may claim any."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _together(what: str, *tensors: torch.Tensor | None) -> None:
    require_cuda(*tensors)
    if len({t.device for t in tensors if t is not None}) > 1:
        raise ValueError(f"{what}: all tensors must be on one device")


def _check(q: MXFP4, what: str, dims: int | None = None) -> None:
    c, s = q.codes, q.scales
    _together(what, c, s)
    if c.dtype != torch.uint8 or s.dtype != torch.uint8:
        raise ValueError(f"{what}: codes and scales must be uint8, got {c.dtype} and {s.dtype}")
    if c.dim() < 2 or (dims is not None and c.dim() != dims):
        raise ValueError(f"{what}: codes of shape {tuple(c.shape)}")
    if q.k % BLOCK != 0 or q.k == 0:
        raise ValueError(f"{what}: a row holds {q.k} elements, not a multiple of {BLOCK}")
    if tuple(s.shape) != (*c.shape[:-2], *_tiles(q.rows, q.k)):
        raise ValueError(f"{what}: scales of shape {tuple(s.shape)} do not belong to codes of shape {tuple(c.shape)}")
    if not (s.is_contiguous() or s.numel() == 0) or not (c.is_contiguous() or c.numel() == 0) or c.data_ptr() % 16 or s.data_ptr() % 16:
        raise ValueError(f"{what}: codes and scales must be contiguous and start on 16 bytes")


def mxfp4_quantize(x: torch.Tensor) -> MXFP4:
    """``x [..., rows, k]`` (fp16, bf16 or fp32; k a multiple of 32) in the format.  A block's scale is the largest power of two not
    above its largest magnitude, over 4; elements are rounded to the nearest, ties to the even code, and end at 6 scales.  A block
    that holds an infinity or a NaN becomes NaN."""
    out = _native.mx4_quantize(x)
    return _mxfp4_quantize(x) if out is None else out


@no_grad
def _mxfp4_quantize(x: torch.Tensor) -> MXFP4:
    require_cuda(x)
    code = float_code(x, "x")
    if x.dim() < 2:
        raise ValueError(f"mxfp4_quantize: x must have rows, got shape {tuple(x.shape)}")
    *lead, rows, k = x.shape
    if k % BLOCK != 0 or k == 0:
        raise ValueError(f"mxfp4_quantize: a row holds {k} elements, not a multiple of {BLOCK}")
    flat = _aligned(x if x.dim() == 2 else x.reshape(-1, k))
    with _on(x):
        codes = torch.empty((*lead, rows, k // 2), dtype=torch.uint8, device=x.device)
        scales = torch.empty((*lead, *_tiles(rows, k)), dtype=torch.uint8, device=x.device)
        if flat.shape[0]:
            check(lib().b2l_mxfp4_quantize(codes.data_ptr(), scales.data_ptr(), flat.data_ptr(), flat.shape[0] // rows, rows, k,
                                           _row_stride(flat), code, stream_handle()))
    return MXFP4(codes, scales, ready=False)


def mxfp4_dequantize(q: MXFP4, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values that ``q`` stands for, rounded to ``dtype`` (fp16, bf16 or fp32): ``[..., rows, k]``."""
    y = _native.mx4_dequantize(q, dtype) if isinstance(q, MXFP4) else None
    return _mxfp4_dequantize(q, dtype) if y is None else y


@no_grad
def _mxfp4_dequantize(q: MXFP4, dtype: torch.dtype) -> torch.Tensor:
    if not isinstance(q, MXFP4):
        raise ValueError(f"mxfp4_dequantize: q must be MXFP4, got {type(q).__name__}")
    _check(q, "mxfp4_dequantize")
    with _on(q.codes):
        y = torch.empty((*q.codes.shape[:-1], q.k), dtype=dtype, device=q.device)
        code = float_code(y, "dtype")
        if y.numel():
            check(lib().b2l_mxfp4_dequantize(y.data_ptr(), q.codes.data_ptr(), q.scales.data_ptr(), y.numel() // (q.rows * q.k),
                                             q.rows, q.k, q.k // 2, code, stream_handle()))
    return y


@no_grad
def mxfp4_pack(codes: torch.Tensor, scales: torch.Tensor) -> MXFP4:
    """Weights of a checkpoint: ``codes`` uint8 ``[..., rows, k / 2]`` and scale bytes in rows, ``[..., rows, k / 32]``."""
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError(f"mxfp4_pack: codes and scales must be uint8, got {codes.dtype} and {scales.dtype}")
    rows, k = codes.shape[-2], 2 * codes.shape[-1]
    if k % BLOCK != 0 or k == 0 or tuple(scales.shape) != (*codes.shape[:-1], k // BLOCK):
        raise ValueError(f"mxfp4_pack: scales of shape {tuple(scales.shape)} do not belong to codes of shape {tuple(codes.shape)}")
    b = torch.nn.functional.pad(scales, (0, -(k // BLOCK) % 4, 0, -rows % 128))
    b = b.unflatten(-1, (-1, 4)).unflatten(-3, (-1, 4, 32))                # [..., row tile, 4, 32, k tile, 4]
    tiles = b.movedim(-2, -4).transpose(-3, -2).contiguous()
    codes = codes.contiguous()
    return MXFP4(codes if codes.data_ptr() % 16 == 0 else codes.clone(), tiles)


def mxfp4_quantize_weight(w: torch.Tensor) -> MXFP4:
    """:func:`mxfp4_quantize` for weights that many products will read: what follows on the stream may take it as finished."""
    q = mxfp4_quantize(w)
    with _on(w):
        weights_written()
    return MXFP4(q.codes, q.scales)


def mxfp4_gate_up(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """Gate and up rows ``[..., inner, k]`` (or biases ``[inner, 1]``) in the order of ``mxfp4_matmul(..., swiglu=True)``: runs of 64
    gate rows, each followed by its up rows."""
    if gate.shape != up.shape or gate.dim() < 2 or gate.shape[-2] % GATE_RUN != 0:
        raise ValueError(f"mxfp4_gate_up: gate {tuple(gate.shape)} and up {tuple(up.shape)} must be alike, in rows of a multiple of {GATE_RUN}")
    return torch.stack((gate.unflatten(-2, (-1, GATE_RUN)), up.unflatten(-2, (-1, GATE_RUN))), -3).flatten(-4, -2)


def skip_rmsnorm_mxfp4(X: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-5, *,
                       out_residual: torch.Tensor | None = None) -> tuple[MXFP4, torch.Tensor]:
    """``(q, residual)``: ``residual += X`` in place (or into ``out_residual``), ``q`` the RMS norm of it times ``weight`` in the
    format, ``[rows, n]`` with the leading dimensions joined.  ``residual=None``: the norm of ``X``, which comes back as the second value.

    What is written may lie in the place of ``X`` or ``residual``, row by row; another overlap is refused.  The norm is not rounded to 16 bits
    before it is quantised (:func:`~lite_llama_b200.kernels.skip_rmsnorm` rounds twice), and decides borders as exact arithmetic does, with
    ``eps`` in 32 bits.  n: a multiple of 32, at most 16384."""
    out = _native.mx4_norm(X, residual, weight, eps, out_residual)
    if out is None:
        return _skip_rmsnorm_mxfp4(X, residual, weight, eps, out_residual)
    return out, X if residual is None else residual if out_residual is None else out_residual


@no_grad
def _skip_rmsnorm_mxfp4(X, residual, weight, eps, out_residual) -> tuple[MXFP4, torch.Tensor]:
    _together("skip_rmsnorm_mxfp4", X, residual, weight, out_residual)
    n = X.shape[-1]
    code = dtype_code(X, "X")
    if weight.dtype != X.dtype or weight.shape != (n,):
        raise ValueError(f"skip_rmsnorm_mxfp4: weight must be {X.dtype} [{n}], got {weight.dtype} {tuple(weight.shape)}")
    if n % BLOCK != 0 or n == 0 or n > 16384:
        raise ValueError(f"skip_rmsnorm_mxfp4 needs a multiple of {BLOCK} up to 16384, got {n}")
    if out_residual is not None and residual is None:
        raise ValueError("skip_rmsnorm_mxfp4: out_residual without a residual")
    for t in (residual, out_residual):
        if t is not None and (t.dtype != X.dtype or t.shape != X.shape):
            raise ValueError(f"skip_rmsnorm_mxfp4: residual must be {X.dtype} {tuple(X.shape)}, got {t.dtype} {tuple(t.shape)}")
    x2, w = _aligned(as_rows(X)), weight if weight.stride(0) == 1 and weight.data_ptr() % 16 == 0 else weight.clone()
    total = out_residual if out_residual is not None else residual
    if total is not None and not (total.is_contiguous() and total.data_ptr() % 16 == 0):
        raise ValueError("skip_rmsnorm_mxfp4: the residual is written in place and must be contiguous")
    r2 = None if residual is None else _aligned(as_rows(residual))
    rows = x2.shape[0]
    with _on(X):
        codes = torch.empty((rows, n // 2), dtype=torch.uint8, device=X.device)
        scales = torch.empty(_tiles(rows, n), dtype=torch.uint8, device=X.device)
        check(lib().b2l_skip_rmsnorm_mxfp4(codes.data_ptr(), scales.data_ptr(), ptr(total), x2.data_ptr(), ptr(r2), w.data_ptr(),
                                           rows, n, _row_stride(x2), n if r2 is None else _row_stride(r2), n, float(eps), code,
                                           stream_handle()))
    return MXFP4(codes, scales, ready=False), X if total is None else total


def mxfp4_matmul(x: torch.Tensor | MXFP4, w: MXFP4, bias: torch.Tensor | None = None, *, swiglu: bool = False,
                 out_dtype: torch.dtype | None = None) -> torch.Tensor | MXFP4:
    """``x @ w.T (+ bias)`` with both operands in the format, sums in 32 bits.

    ``x``: 16-bit ``[..., k]`` (quantised here) or an :class:`MXFP4` ``[rows, k]``; ``w`` ``[n, k]``; ``bias [n]`` in the output's
    type.  The output is of ``x``'s type, for quantised ``x`` of ``out_dtype`` (default fp16).  ``swiglu``: the rows of ``w`` (and
    ``bias``) alternate as ``mxfp4_gate_up`` orders them, and ``silu(gate) * up`` comes back in the format, ``[rows, n / 2]``,
    quantised from the sums themselves: the codes of exact arithmetic on them."""
    if isinstance(w, MXFP4) and isinstance(x, (torch.Tensor, MXFP4)):
        y = _native.mx4_matmul(x, w, bias, swiglu, out_dtype)
        if y is not None:
            return y
    return _mxfp4_matmul(x, w, bias, swiglu, out_dtype)


@no_grad
def _mxfp4_matmul(x, w, bias, swiglu, out_dtype) -> torch.Tensor | MXFP4:
    if not isinstance(w, MXFP4):
        raise ValueError(f"mxfp4_matmul: w must be MXFP4, got {type(w).__name__}")
    _check(w, "mxfp4_matmul: w", 2)
    lead = None
    if isinstance(x, MXFP4):
        _check(x, "mxfp4_matmul: x", 2)
        dtype = out_dtype or (torch.float16 if bias is None else bias.dtype)
    else:
        if not isinstance(x, torch.Tensor):
            raise ValueError(f"mxfp4_matmul: x must be a tensor or MXFP4, got {type(x).__name__}")
        require_cuda(x)
        dtype_code(x, "x")
        if out_dtype not in (None, x.dtype):
            raise ValueError(f"mxfp4_matmul: the output of {x.dtype} activations is {x.dtype}, not {out_dtype}")
        dtype, lead = x.dtype, x.shape[:-1]
        if x.shape[-1] != w.k:
            raise ValueError(f"x has {x.shape[-1]} cols but weight expects {w.k}")
        x = _aligned(as_rows(x))
        if not lib().b2l_mxfp4_matmul_takes_16bit(x.shape[0], w.rows, w.k):
            x = mxfp4_quantize(x)
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"mxfp4_matmul: unsupported output dtype {dtype}")
    if isinstance(x, MXFP4):
        if x.k != w.k:
            raise ValueError(f"x has {x.k} cols but weight expects {w.k}")
        xc, xs, t, stride = x.codes, x.scales, x.rows, w.k // 2
    else:                                                 # few rows: the product quantises them itself
        xc, xs, t, stride = x, None, x.shape[0], _row_stride(x)
    _together("mxfp4_matmul", xc, w.codes, bias)
    n = w.rows
    if swiglu and n % (2 * GATE_RUN) != 0:
        raise ValueError(f"mxfp4_matmul: gate and up rows come in runs of {GATE_RUN}, got {n} rows")
    if bias is not None:
        if bias.shape != (n,) or bias.dtype != dtype:
            raise ValueError(f"mxfp4_matmul: bias must be {dtype} [{n}], got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.contiguous()
    with _on(w.codes):
        if not w.ready:
            weights_written()
        if swiglu:
            y = torch.empty((t, n // 4), dtype=torch.uint8, device=w.device)
            ys = torch.empty(_tiles(t, n // 2), dtype=torch.uint8, device=w.device)
        else:
            y, ys = torch.empty((t, n), dtype=dtype, device=w.device), None
        code = {torch.float16: 0, torch.bfloat16: 1}[dtype]
        check(lib().b2l_mxfp4_matmul(y.data_ptr(), ptr(ys), xc.data_ptr(), ptr(xs), w.codes.data_ptr(), w.scales.data_ptr(), ptr(bias), t, n,
                                     w.k, stride, w.k // 2, y.shape[1], int(swiglu), 1, code, stream_handle()))
    if swiglu:
        return MXFP4(y, ys, ready=False)
    return y if lead is None or len(lead) == 1 else y.view(*lead, n)


def fused_moe_mxfp4(hidden_states: torch.Tensor, w1: MXFP4, w2: MXFP4, topk_weights: torch.Tensor, topk_ids: torch.Tensor) -> torch.Tensor:
    """``sum_k w_k * (silu(x @ W1g.T) * (x @ W1u.T)) @ W2.T`` over the routed experts, both products with 4-bit operands.

    ``hidden_states`` 16-bit ``[tokens, h]``; ``w1`` ``[experts, 2 inner, h]`` with rows as ``mxfp4_gate_up`` orders them, ``w2``
    ``[experts, h, inner]``; ``topk_weights`` (fp32 or the activations' type) and ``topk_ids`` (int32 or int64) ``[tokens, k]``.  Tokens are
    quantised once and sorted by expert, the activation is quantised from the first product's sums, and a slot's output and the weighted sum
    are held in 32 bits.  Ids that name no expert add nothing."""
    if isinstance(w1, MXFP4) and isinstance(w2, MXFP4):
        out = _native.mx4_moe(hidden_states, w1, w2, topk_weights, topk_ids)
        if out is not None:
            return out
    return _fused_moe_mxfp4(hidden_states, w1, w2, topk_weights, topk_ids)


@no_grad
def _fused_moe_mxfp4(hidden_states, w1, w2, topk_weights, topk_ids) -> torch.Tensor:
    for w, what in ((w1, "w1"), (w2, "w2")):
        if not isinstance(w, MXFP4):
            raise ValueError(f"fused_moe_mxfp4: {what} must be MXFP4, got {type(w).__name__}")
        _check(w, f"fused_moe_mxfp4: {what}", 3)
    x, dtype = hidden_states, hidden_states.dtype
    _together("fused_moe_mxfp4", x, w1.codes, w2.codes, topk_weights, topk_ids)
    code = dtype_code(x, "hidden_states")
    experts, rows1, hidden, inner = w1.codes.shape[0], w1.rows, w1.k, w2.k
    if x.dim() != 2 or x.shape[1] != hidden:
        raise ValueError(f"fused_moe_mxfp4: hidden_states of shape {tuple(x.shape)} under experts of {hidden} inputs")
    if w2.codes.shape[0] != experts or w2.rows != hidden or rows1 != 2 * inner or inner % GATE_RUN != 0:
        raise ValueError(f"fused_moe_mxfp4: w1 [{experts}, {rows1}, {hidden}] and w2 {[*w2.codes.shape[:2], inner]} do not belong together")
    tokens = x.shape[0]
    if topk_ids.dim() != 2 or topk_ids.shape[0] != tokens or topk_ids.shape != topk_weights.shape or topk_ids.shape[1] == 0:
        raise ValueError(f"fused_moe_mxfp4: ids {tuple(topk_ids.shape)} and weights {tuple(topk_weights.shape)} for {tokens} tokens")
    if topk_weights.dtype not in (torch.float32, dtype):
        raise ValueError(f"fused_moe_mxfp4: weights must be float32 or {dtype}, got {topk_weights.dtype}")
    width = index_width(topk_ids, "topk_ids")
    top_k = topk_ids.shape[1]
    slots = tokens * top_k
    out = torch.empty((tokens, hidden), dtype=dtype, device=x.device)
    if tokens == 0:
        return out
    x, ids, weights = _aligned(x), topk_ids.contiguous(), topk_weights.contiguous()
    with _on(x):
        L, dev, st = lib(), x.device, stream_handle()
        tile = L.b2l_mxfp4_moe_tile_rows(slots, experts, rows1)
        tiles = L.b2l_mxfp4_moe_max_tiles(slots, tile, experts)
        def buffer(*shape):
            return torch.empty(shape, dtype=torch.uint8, device=dev)

        plan = torch.empty(slots + 1 + 2 * tiles, dtype=torch.int32, device=dev)
        place, table = plan.data_ptr(), plan.data_ptr() + 4 * slots
        xq, xs = buffer(tiles * tile, hidden // 2), buffer(*_tiles(max(tile, 128) * tiles, hidden))
        check(L.b2l_mxfp4_moe_scatter(place, table, xq.data_ptr(), xs.data_ptr(), x.data_ptr(), ids.data_ptr(), width, tokens, top_k, tile, experts,
                                      hidden, _row_stride(x), code, st))
        aq, as_ = buffer(tiles * tile, inner // 2), buffer(*_tiles(max(tile, 128) * tiles, inner))
        check(L.b2l_mxfp4_grouped_matmul(aq.data_ptr(), as_.data_ptr(), xq.data_ptr(), xs.data_ptr(), w1.codes.data_ptr(),
                                         w1.scales.data_ptr(), table, tiles, tile, experts, rows1, hidden, 1, st))
        # 32 bits a sum; in tiles of 128 rows or more the upper and the lower halves by themselves
        y = torch.empty((tiles * tile, hidden), dtype=torch.float32 if tile == 64 else torch.int16, device=dev)
        low = None if tile == 64 else torch.empty_like(y)
        check(L.b2l_mxfp4_grouped_matmul(y.data_ptr(), ptr(low), aq.data_ptr(), as_.data_ptr(), w2.codes.data_ptr(), w2.scales.data_ptr(),
                                         table, tiles, tile, experts, hidden, inner, 0, st))
        check(L.b2l_mxfp4_moe_combine(out.data_ptr(), y.data_ptr(), ptr(low), place, weights.data_ptr(), int(weights.dtype == torch.float32),
                                      tokens, top_k, hidden, code, st))
    return out
