"""Logit adjustments and 4-bit weights without a GPU: structure layout, refusals of the C entries
(each returns before any CUDA call) and of the Python argument checks."""

from __future__ import annotations

import ctypes

import pytest
import torch

import test_abi
from cuda_b200 import _lib, logits, quantized
from cuda_b200.paged import overlap


def test_structures_match_the_header(tmp_path, monkeypatch):
    monkeypatch.setattr(test_abi, "STRUCTS", {"cb_adjust_args": _lib.AdjustArgs, "cb_weights4": _lib.Weights4Args,
                                              "cb_linear4_args": _lib.Linear4Args})
    test_abi.test_ctypes_structures_match_the_header(tmp_path)


def adjust(**changes):
    a = _lib.AdjustArgs(logits=16, out=16, dtype=_lib.F32, rows=1, vocab=8, ld=8, out_ld=8)
    for name, value in changes.items():
        setattr(a, name, value)
    _lib.call("cb_adjust_logits", ctypes.byref(a), None)


@pytest.mark.parametrize("change", [dict(dtype=_lib.I32), dict(rows=-1), dict(vocab=2 ** 30), dict(logits=None),
                                    dict(out=None), dict(out=18), dict(tokens=16, token_dtype=_lib.F32, history=2),
                                    dict(history=2), dict(tokens=16, token_dtype=_lib.I32, history=2 ** 20), dict(biases=1024), dict(biases=1), dict(history=-1),
                                    dict(biases=2, bias=16, bias_tokens=16, bias_token_dtype=_lib.BF16),
                                    dict(rows=2 ** 31 - 1, vocab=2 ** 30 - 1)])
def test_adjust_refusals(change):
    with pytest.raises(_lib.KernelError):
        adjust(**change)


def test_empty_calls_do_nothing():
    adjust(rows=0)
    adjust(vocab=0, logits=None)
    linear(rows=0)


def weights(**changes):
    w = _lib.Weights4Args(codes=16, scales=16, scale_dtype=_lib.BF16, group=64, outputs=32, inputs=128)
    for name, value in changes.items():
        setattr(w, name, value)
    return w


def linear(w=None, **changes):
    a = _lib.Linear4Args(weights=w or weights(), x=16, out=16, dtype=_lib.BF16, rows=1, ld=128, out_ld=32)
    for name, value in changes.items():
        setattr(a, name, value)
    _lib.call("cb_linear4", ctypes.byref(a), None, None)


@pytest.mark.parametrize("change", [dict(group=48), dict(group=16), dict(inputs=96), dict(inputs=0), dict(outputs=0),
                                    dict(scale_dtype=_lib.F32), dict(outputs=2 ** 31), dict(codes=None),
                                    dict(scales=8), dict(outputs=2 ** 30, inputs=2 ** 20)])
def test_weights_refusals(change):
    w = weights(**change)
    with pytest.raises(_lib.KernelError):
        linear(w)
    with pytest.raises(_lib.KernelError):
        _lib.call("cb_weights4_pack", ctypes.byref(w), 16, 16, None)
    with pytest.raises(_lib.KernelError):
        _lib.call("cb_weights4_dequantise", ctypes.byref(w), 16, _lib.BF16, 2 ** 21, None)


@pytest.mark.parametrize("change", [dict(dtype=_lib.I32), dict(rows=-1), dict(x=None), dict(out=None),
                                    dict(rows=2 ** 24), dict(x=2), dict(dtype=_lib.F32), dict(rows=2, ld=129)])
def test_linear_refusals(change):
    """(The last three need a workspace, and none is given.)"""
    with pytest.raises(_lib.KernelError):
        linear(**change)


def test_more_refusals():
    w, ref = weights(), ctypes.byref
    for name, args in (("cb_weights4_quantise", (16, _lib.I32, 128, 16, 16)),
                       ("cb_weights4_quantise", (None, _lib.F32, 128, 16, 16)),
                       ("cb_weights4_pack", (None, 16)), ("cb_weights4_dequantise", (None, _lib.F32, 128)),
                       ("cb_weights4_dequantise", (16, _lib.I8, 128)), ("cb_weights4_dequantise", (16, _lib.F32, 127))):
        with pytest.raises(_lib.KernelError):
            _lib.call(name, ref(w), *args, None)


def test_sizes():
    """Codes: 512 bytes to 16 outputs x 64 inputs; scales: 32, 64 or 128 inputs to one of 16 rows."""
    lib, ref = _lib.load(), ctypes.byref
    for group, inputs, outputs, codes, scales in ((32, 96, 17, 2 * 2 * 512, 2 * 4 * 32), (64, 192, 16, 3 * 512, 3 * 32),
                                                  (128, 384, 1, 6 * 512, 3 * 32)):
        w = weights(group=group, inputs=inputs, outputs=outputs, codes=None, scales=None)
        assert lib.cb_weights4_code_bytes(ref(w)) == codes
        assert lib.cb_weights4_scale_bytes(ref(w)) == scales
    a = _lib.Linear4Args(weights=weights(), x=16, out=16, dtype=_lib.F32, rows=5, ld=128, out_ld=32)
    assert lib.cb_linear4_scratch(ref(a)) == 5 * 3 * 128 * 2
    a.dtype = _lib.F16
    assert lib.cb_linear4_scratch(ref(a)) == 0


def test_python_refusals():
    with pytest.raises(ValueError, match="CUDA"):
        logits.adjust(torch.zeros(2, 8))
    with pytest.raises(TypeError):
        logits.adjust([1.0])
    with pytest.raises(ValueError, match="CUDA"):
        quantized.quantise(torch.zeros(16, 128))
    with pytest.raises(ValueError, match="CUDA"):
        quantized.Weights4.pack(torch.zeros(16, 64, dtype=torch.uint8), torch.zeros(16, 1, dtype=torch.bfloat16))
    for group, scales, error in ((48, torch.bfloat16, ValueError), (64, torch.float32, TypeError)):
        with pytest.raises(error):
            quantized._args(16, 192, group, scales)
    with pytest.raises(ValueError):
        quantized._args(16, 96, 64, torch.float16)


def test_rows():
    """Rows of any leading dimensions that lie at one distance."""
    x = torch.zeros(6, 4, 32)
    assert quantized._rows(x) == (24, 32)
    assert quantized._rows(x[:, 1]) == (6, 128)
    assert quantized._rows(x[0, 0]) == (1, 32)
    assert quantized._rows(x[:0]) == (0, 32)
    assert quantized._rows(x[:1, ::2]) == (2, 64)
    assert quantized._rows(x[0, :1].expand(5, 32)) == (5, 0)
    with pytest.raises(ValueError):
        quantized._rows(x[:, :3])


def cache(**changes):
    c = _lib.PagedCacheArgs(k_pages=16, v_pages=16, k_scale=16, v_scale=16, storage=_lib.I8, kv_heads=2, page=16,
                            head_size=64, pages=8, table=16, lengths=16, slots=2, columns=4)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


def shared(c, scratch=16, counters=16, **changes):
    a = _lib.PagedAttentionArgs(cache=c, q=16, out=16, dtype=_lib.F32, batch=1, tokens=1, heads=2, scale=1.0)
    for name, value in changes.items():
        setattr(a, name, value)
    return _lib.call("cb_paged_attention_shared", ctypes.byref(a), 0, scratch, counters, None)


@pytest.mark.parametrize("change", [dict(storage=_lib.BF16), dict(head_size=48), dict(page=24), dict(kv_heads=0),
                                    dict(columns=2 ** 31 // 16), dict(k_pages=None), dict(v_pages=8)])
def test_shared_cache_refusals(change):
    with pytest.raises(_lib.KernelError):
        shared(cache(**change))


@pytest.mark.parametrize("change", [dict(dtype=_lib.I64), dict(heads=3), dict(heads=0), dict(out=None), dict(q=None),
                                    dict(batch=65536), dict(tokens=-1), dict(out=8), dict(scratch=None),
                                    dict(scratch=8), dict(counters=None)])
def test_shared_call_refusals(change):
    with pytest.raises(_lib.KernelError):
        shared(cache(), **change)


def test_shared_calls_with_too_much_work():
    """Rows and keys whose division would pass 32 bits, and empty calls, which do nothing."""
    with pytest.raises(_lib.KernelError, match="too many"):
        shared(cache(columns=2 ** 26), batch=65535, tokens=64)
    shared(cache(), batch=0)
    shared(cache(), tokens=0)


def test_alignment():
    """Values that do not lie on multiples of their type."""
    ref, w = ctypes.byref, weights()
    for change in (dict(x=17), dict(out=17), dict(out=18, dtype=_lib.F32)):
        with pytest.raises(_lib.KernelError, match="aligned"):
            linear(**change)
    for name, args in (("cb_weights4_quantise", (18, _lib.F32, 128, 16, 16)),
                       ("cb_weights4_quantise", (16, _lib.F32, 128, 16, 17)), ("cb_weights4_pack", (16, 17)),
                       ("cb_weights4_dequantise", (18, _lib.F32, 128))):
        with pytest.raises(_lib.KernelError, match="aligned"):
            _lib.call(name, ref(w), *args, None)


def test_overlap():
    room = torch.zeros(4, 64)
    assert overlap(room, room[3, 63:]) and overlap(room[:2], room[1:])
    assert not overlap(room[:2], room[2:]) and not overlap(room, room[:0])
    assert overlap(room[:, :8], room[:, 8:])  # (spans, not elements)
