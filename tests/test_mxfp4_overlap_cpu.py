"""The norm with quantised output where its buffers overlap: row by row in place, otherwise refused before any launch."""

from __future__ import annotations

import ctypes

import pytest

from lite_llama_b200 import _lib

ROWS, N = 4, 64
ROW = 2 * N      # bytes


def call(total, x, residual, weight, x_stride=N, r_stride=N, dtype=0):
    lib = _lib.load()
    buf = ctypes.create_string_buffer(1 << 14)
    base = (ctypes.addressof(buf) + 127) // 128 * 128
    codes, scales = base + 8192, base + 12288
    rc = lib.b2l_skip_rmsnorm_mxfp4(codes, scales, base + total, base + x, base + residual, base + weight, ROWS, N, x_stride, r_stride, N,
                                    ctypes.c_float(1e-5), dtype, None)
    return rc, lib.b2l_last_error().decode()


FAR, OTHER, LAST = 2048, 4096, 6144      # bytes apart


@pytest.mark.parametrize("args,strides", (
    ((ROW, 0, FAR, LAST), {}),                                  # the sums lie a row behind x
    ((0, ROW, FAR, LAST), {}),
    ((0, FAR, 16, LAST), {}),                                   # within a row of the residual
    ((0, 0, FAR, LAST), {"x_stride": 0}),                       # every row of x is the sums' first
    ((0, 0, FAR, LAST), {"x_stride": 2 * N}),
    ((FAR, 0, FAR - 2 * ROW, LAST), {"r_stride": 2 * N}),       # the residual's second row is the sums' first
    ((0, FAR, OTHER, ROW), {}),                                 # the weight is one of the sums' rows
    ((0, FAR, OTHER, 4 * ROW - 16), {}),
))
def test_sums_over_what_is_still_read(args, strides):
    rc, why = call(*args, **strides)
    assert rc < 0 and "overlap" in why, why


@pytest.mark.parametrize("args,strides", (
    ((0, 0, FAR, LAST), {}), ((0, FAR, 0, LAST), {}), ((0, 0, 0, LAST), {}),      # in place
    ((0, FAR, OTHER, LAST), {}),
    ((4 * ROW, 0, FAR, LAST), {}),                                                # side by side
    ((ROW, 0, FAR, LAST), {"x_stride": 0}),                                       # behind the row that all rows of x are
    ((ROW, 0, FAR, LAST), {"x_stride": 5 * N}),                                   # between two rows of x
))
def test_in_place_or_apart(args, strides):
    """Refused for its type alone, which is looked at behind the rows: nothing is launched."""
    rc, why = call(*args, **strides, dtype=2)
    assert rc < 0 and "dtype" in why, why
