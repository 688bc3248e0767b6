"""Linear layers with 4-bit weights and group scales.

The graphs' Linear is ``inputs @ weight.T`` with float32 or bfloat16 weights
(``_linear``, chomikgrad/llama.py:275-277; here ``cb_gemv`` and
``cb_gemm_rows``).  ``Weights4`` holds such a weight in 4 bits, a quarter of the
bytes that a decode step reads::

    weights = Weights4.quantise(weight, group=128)      # (outputs, inputs)
    y = weights.linear(x)                               # (..., inputs) -> (..., outputs)
    dense = weights.dequantise(torch.bfloat16)          # for a prompt's large products

Values are CUDA ``torch.Tensor`` or ``DeviceArray``; every call runs on the
current stream, reads nothing back and can be captured in a CUDA graph.  There
is no backward pass.
"""

from __future__ import annotations

import ctypes
from typing import Any, Optional

import torch

from . import _lib
from .paged import (_VALUES, Prepared, aligned, current_stream, meet, no_grad_needed, reach, require, signature,
                    tensor_of)

GROUPS = (32, 64, 128)
_SCALES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


class Weights4:
    """A weight (outputs, inputs) as codes -8 .. 7 and a scale for each ``group`` neighbouring inputs.

    Made by ``quantise`` or ``pack``; ``codes`` and ``scales`` are in the order in
    which the kernels read them.
    """

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, *, outputs: int, inputs: int, group: int) -> None:
        args = _args(outputs, inputs, group, scales.dtype)
        self.outputs, self.inputs, self.group, self.device = int(outputs), int(inputs), int(group), codes.device
        if codes.device.type != "cuda":
            raise ValueError(f"weights have to be on a CUDA device, got {codes.device}")
        self._lib = _lib.load()
        size = self._lib.cb_weights4_code_bytes(ctypes.byref(args))
        require(codes, "codes", self.device, (torch.uint8,), (size,), 1)
        size = self._lib.cb_weights4_scale_bytes(ctypes.byref(args)) // 2
        require(scales, "scales", self.device, tuple(_SCALES), (size,), 1)
        aligned(codes, "codes")
        aligned(scales, "scales")
        self.codes, self.scales = codes, scales
        self._spans = [("codes", codes.data_ptr(), codes.nbytes), ("scales", scales.data_ptr(), scales.nbytes)]
        args.codes, args.scales = codes.data_ptr(), scales.data_ptr()
        self._args = args
        self._linear_args = Prepared()

    @classmethod
    def pack(cls, codes: Any, scales: Any) -> "Weights4":
        """Weights from their plain form.

        ``codes`` (outputs, inputs / 2) uint8 holds input 2 i in the low half of byte
        i and 2 i + 1 in the high one, each plus 8; ``scales`` (outputs, inputs /
        group) bfloat16 or float16, with groups of 32, 64 or 128 inputs.
        """
        codes, scales = tensor_of(codes), tensor_of(scales)
        if codes.ndim != 2 or scales.ndim != 2:
            raise ValueError("codes and scales have to be (outputs, inputs / 2) and (outputs, inputs / group)")
        device, (outputs, inputs) = codes.device, (codes.shape[0], 2 * codes.shape[1])
        if device.type != "cuda":
            raise ValueError(f"codes are on {device}, expected a CUDA device")
        require(codes, "codes", device, (torch.uint8,), (None, None), 2)
        require(scales, "scales", device, tuple(_SCALES), (outputs, None), 2)
        no_grad_needed(scales)
        if scales.shape[1] == 0 or inputs % scales.shape[1]:
            raise ValueError(f"{scales.shape[1]} scales for {inputs} inputs")
        weights = cls._empty(outputs, inputs, inputs // scales.shape[1], scales.dtype, device)
        _lib.check(weights._lib.cb_weights4_pack(ctypes.byref(weights._args), codes.data_ptr(), scales.data_ptr(),
                                                 current_stream(device)), "cb_weights4_pack")
        return weights

    @classmethod
    def quantise(cls, weight: Any, *, group: int = 128, scales: torch.dtype = torch.bfloat16) -> "Weights4":
        """The nearest 4-bit weights of ``weight`` (outputs, inputs), float32, bfloat16 or float16.

        A group's scale is its largest magnitude / 7, rounded to the type
        ``scales``; codes are rounded to the nearest.  The products of a group that
        holds an infinity or a NaN, or whose scale is beyond the type, are NaN.
        """
        return cls.pack(*quantise(weight, group=group, scales=scales))

    @classmethod
    def _empty(cls, outputs: int, inputs: int, group: int, dtype: torch.dtype, device: torch.device) -> "Weights4":
        args, lib = _args(outputs, inputs, group, dtype), _lib.load()
        codes = torch.empty(lib.cb_weights4_code_bytes(ctypes.byref(args)), dtype=torch.uint8, device=device)
        scales = torch.empty(lib.cb_weights4_scale_bytes(ctypes.byref(args)) // 2, dtype=dtype, device=device)
        return cls(codes, scales, outputs=outputs, inputs=inputs, group=group)

    def linear(self, x: Any, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``x @ weight.T`` for x (..., inputs) in float32, bfloat16 or float16: (..., outputs) of x's type.

        Products are exact and sums float32 (those of a group's codes and x, before its
        scale, have to be within it).  Up to 8 rows (2 of float32) cost about what one
        costs; every 32 rows (10 of float32) read the weights again, so a prompt's rows
        are better multiplied with ``dequantise``'s.  float32 rows, and 16-bit rows
        that do not begin on 16 bytes, are first copied to a workspace.  At most
        2,097,120 rows are taken (655,350 of float32).  ``out`` is contiguous and
        shares no memory with x or the weights.
        """
        x = tensor_of(x)
        no_grad_needed(x)
        key = signature(x)
        known = self._linear_args.get(key)
        if known is None:
            known = self._linear_args[key] = self._prepare_linear(x)
        shape = (*x.shape[:-1], self.outputs)
        if out is None:
            out = x.new_empty(shape)
        else:
            require(out, "out", self.device, (x.dtype,), shape, len(shape))
            self._apart(out, x)
            no_grad_needed(out)
            if not out.is_inference():  # a backward pass that kept what it held notices
                torch.autograd.graph.increment_version(out)
        a = _lib.Linear4Args.from_buffer_copy(known[0])
        a.x, a.out = x.data_ptr(), out.data_ptr()
        stream = current_stream(self.device)
        scratch = None
        if known[1] or x.data_ptr() % 16:
            scratch = x.new_empty(self._lib.cb_linear4_scratch(ctypes.byref(a)), dtype=torch.uint8)
        _lib.check(self._lib.cb_linear4(ctypes.byref(a), None if scratch is None else scratch.data_ptr(), stream),
                   "cb_linear4")
        return out

    def _apart(self, out: torch.Tensor, x: Optional[torch.Tensor] = None) -> None:
        """Refuse an ``out`` over x or the weights: other blocks read those while it is written."""
        at, size = out.data_ptr(), reach(out)
        for name, start, held in self._spans:
            if meet(at, size, start, held):
                raise ValueError(f"out shares memory with {name}")
        if x is not None and meet(at, size, x.data_ptr(), reach(x)):
            raise ValueError("out shares memory with x")

    def _prepare_linear(self, x: torch.Tensor):
        if x.ndim < 1:
            raise ValueError(f"x has shape (), expected (..., {self.inputs})")
        require(x, "x", self.device, tuple(_VALUES), (*(None,) * (x.ndim - 1), self.inputs), 1)
        a = _lib.Linear4Args()
        a.weights, a.dtype = self._args, _VALUES[x.dtype]
        a.rows, a.ld = _rows(x)
        a.out_ld = self.outputs
        a.x = 16
        return a, self._lib.cb_linear4_scratch(ctypes.byref(a)) > 0

    def dequantise(self, dtype: torch.dtype = torch.bfloat16, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The weights as (outputs, inputs) numbers of ``dtype`` (of ``out``'s with one), each rounded once."""
        if out is None:
            if dtype not in _VALUES:
                raise TypeError(f"dtype {dtype}, expected one of {', '.join(map(str, _VALUES))}")
            out = torch.empty(self.outputs, self.inputs, dtype=dtype, device=self.device)
        else:
            require(out, "out", self.device, tuple(_VALUES), (self.outputs, self.inputs), 1)
            if self.outputs > 1 and out.stride(0) < self.inputs:
                raise ValueError("the rows of out share memory")
            self._apart(out)
            no_grad_needed(out)
            if not out.is_inference():
                torch.autograd.graph.increment_version(out)
        ld = out.stride(0) if self.outputs > 1 else self.inputs
        _lib.check(self._lib.cb_weights4_dequantise(ctypes.byref(self._args), out.data_ptr(), _VALUES[out.dtype], ld,
                                                    current_stream(self.device)), "cb_weights4_dequantise")
        return out


def quantise(weight: Any, *, group: int = 128, scales: torch.dtype = torch.bfloat16):
    """The plain form of ``Weights4.quantise``: codes and scales as ``Weights4.pack`` takes them."""
    weight = tensor_of(weight)
    no_grad_needed(weight)
    device = weight.device
    if device.type != "cuda":
        raise ValueError(f"weight is on {device}, expected a CUDA device")
    require(weight, "weight", device, tuple(_VALUES), (None, None), 1)
    outputs, inputs = weight.shape
    args = _args(outputs, inputs, group, scales)
    codes = torch.empty(outputs, inputs // 2, dtype=torch.uint8, device=device)
    scale = torch.empty(outputs, inputs // group, dtype=scales, device=device)
    _lib.check(_lib.load().cb_weights4_quantise(ctypes.byref(args), weight.data_ptr(), _VALUES[weight.dtype],
                                                weight.stride(0), codes.data_ptr(), scale.data_ptr(),
                                                current_stream(device)), "cb_weights4_quantise")
    return codes, scale


def _args(outputs: int, inputs: int, group: int, scales: torch.dtype) -> _lib.Weights4Args:
    if scales not in _SCALES:
        raise TypeError(f"scales of {scales}, expected bfloat16 or float16")
    if group not in GROUPS:
        raise ValueError(f"groups of {group} inputs, expected one of {GROUPS}")
    if outputs < 1 or inputs < group or inputs % group:
        raise ValueError(f"{outputs} outputs of {inputs} inputs in groups of {group}")
    if max(outputs, inputs) >= 2 ** 31 or -(-outputs // 16) * -(-inputs // 64) >= 2 ** 31:
        raise ValueError(f"{outputs} outputs of {inputs} inputs are too many")
    return _lib.Weights4Args(scale_dtype=_SCALES[scales], group=group, outputs=outputs, inputs=inputs)


def _rows(x: torch.Tensor):
    """Number of rows of (..., inputs) and the one stride between them."""
    rows, ld = 1, None
    for size, stride in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
        if size != 1:
            if ld is None:
                ld = stride
            elif rows and stride != rows * ld:
                raise ValueError("the rows of x have to lie at one distance from each other")
            rows *= size
    return rows, x.shape[-1] if ld is None else ld
