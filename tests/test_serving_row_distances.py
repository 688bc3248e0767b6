"""Rows of an output that would share memory, and too many of them, are refused by the C entries before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest

from cuda_b200 import _lib


@pytest.mark.parametrize("out_ld", [0, 7, -7])
def test_adjusted_rows(out_ld):
    a = _lib.AdjustArgs(logits=16, out=4096, dtype=_lib.F32, rows=2, vocab=8, ld=8, out_ld=out_ld)
    with pytest.raises(_lib.KernelError, match="share memory"):
        _lib.call("cb_adjust_logits", ctypes.byref(a), None)


@pytest.mark.parametrize("out_ld", [0, 31, -31])
def test_products(out_ld):
    w = _lib.Weights4Args(codes=16, scales=16, scale_dtype=_lib.BF16, group=64, outputs=32, inputs=128)
    a = _lib.Linear4Args(weights=w, x=16, out=16, dtype=_lib.BF16, rows=2, ld=128, out_ld=out_ld)
    with pytest.raises(_lib.KernelError, match="share memory"):
        _lib.call("cb_linear4", ctypes.byref(a), None, None)


@pytest.mark.parametrize("dtype, most", [(_lib.BF16, 2097120), (_lib.F16, 2097120), (_lib.F32, 655350)])
def test_most_rows(dtype, most):
    """The documented limit; at the limit the call is taken (and here ends for want of the workspace of off-lying rows)."""
    w = _lib.Weights4Args(codes=16, scales=16, scale_dtype=_lib.BF16, group=64, outputs=32, inputs=128)
    for rows, message in ((most + 1, "at most"), (most, "scratch")):
        a = _lib.Linear4Args(weights=w, x=20, out=16, dtype=dtype, rows=rows, ld=128, out_ld=32)
        with pytest.raises(_lib.KernelError, match=message):
            _lib.call("cb_linear4", ctypes.byref(a), None, None)
