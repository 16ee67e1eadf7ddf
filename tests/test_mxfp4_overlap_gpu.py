"""The norm with quantised output refuses sums that lie over rows which other rows still read."""

from __future__ import annotations

import pytest
import torch

from lite_llama_b200 import kernels as K

pytestmark = pytest.mark.gpu


def test_overlaps_are_refused_and_leave_the_buffers_alone():
    rows, n = 300, 256
    buf, other, w = (torch.randn(rows + 1, n, device="cuda").half() for _ in range(3))
    w, kept = w[0].contiguous(), buf.clone()
    for x, residual, weight, out in ((buf[:-1], buf[1:], w, None), (buf[1:], buf[:-1], w, None), (buf[:1].expand(rows, n), buf[:-1], w, None),
                                     (other[1:], buf[:-1], w, buf[1:]), (other[1:], buf[:-1], buf[7], None)):
        with pytest.raises(ValueError, match="overlap"):
            K.skip_rmsnorm_mxfp4(x, residual, weight, 1e-5, out_residual=out)
    assert torch.equal(buf, kept)
    K.skip_rmsnorm_mxfp4(other[:1].expand(rows, n), buf[1:], w)          # one row read by all, the sums elsewhere
    assert torch.equal(buf[1:], kept[1:] + other[:1])
