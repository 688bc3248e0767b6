"""Rows of an output that would share memory are refused by the C entries, before any CUDA call."""

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
