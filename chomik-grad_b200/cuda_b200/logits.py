"""Penalties, biases and grammar masks on logits, before a token is chosen.

The reference samples from its model's logits as they are, with temperature and
top-k (``sample_token``, examples/generate_tinyllama.py:124-143; here
``CudaB200Device.sample_rows``).  ``adjust`` is the step before that::

    logits = adjust(logits, tokens=history, lengths=lengths, prompts=prompts, repetition=1.1, presence=0.5,
                    bias_tokens=ids, bias=values, allowed=bits)

It takes CUDA ``torch.Tensor`` or ``DeviceArray`` values and runs on the current
stream; nothing is read back, so a step can be captured in a CUDA graph.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any, Dict, Optional, Tuple, Union

import torch

from . import _lib
from .paged import _VALUES, Prepared, current_stream, meet, no_grad_needed, reach, require, signature, tensor_of

_INDICES = {torch.int32: _lib.I32, torch.int64: _lib.I64}
MAX_BIASES, MAX_HISTORY = 1023, 2 ** 20 - 1
_ADJUST_ARGS = Prepared()


def adjust(logits: Any, *, tokens: Any = None, lengths: Any = None, prompts: Any = None,
           repetition: Union[float, Any] = 1.0, frequency: Union[float, Any] = 0.0,
           presence: Union[float, Any] = 0.0, bias_tokens: Any = None, bias: Any = None, allowed: Any = None,
           out: Optional[torch.Tensor] = None, error_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The rows of ``logits`` (rows, vocab) with penalties, biases and a mask applied, in that order.

    ``tokens`` (rows, n) int32 or int64, n < 2**20, is each row's history, of which
    ``lengths[row]`` tokens count (all without) and the first ``prompts[row]``
    were given rather than made (none without); both int32.  With c the times
    that a token is among them and d those from ``prompts[row]`` on, its logit is
    divided by ``repetition`` where c > 0 and it is positive, multiplied where it is
    not, and loses ``frequency * d``, and ``presence`` where d > 0.  Each of the
    three is a number or a float32 tensor (rows).

    ``bias`` (rows, m) float32 is added to the logits of ``bias_tokens`` (rows,
    m) int32 or int64, at most 1023 to a row; a token that is listed twice gets
    both.  Tokens outside the vocabulary are passed over in both lists, so a -1
    pads them.  ``allowed`` (rows, ceil(vocab / 32)) int32 holds a bit for each
    token, the lowest first: a token whose bit is clear becomes -inf, and a row
    without any set is -inf throughout.

    float32, bfloat16 or float16 with rows of any stride (a history, bias or mask
    that all rows share can be expanded).  The sums are float32 and rounded once.
    ``out`` may be ``logits`` itself; it shares no memory with another argument.
    Lengths outside the history are taken as its ends and set ``error_flag`` (an
    int32 of the caller's, read with ``speculative.check``).
    """
    if type(logits) is not torch.Tensor:
        logits = tensor_of(logits)
    numbers, pointers, values, key = [], [], {}, [signature(logits), signature(error_flag)]
    for name, value in (("repetition", repetition), ("frequency", frequency), ("presence", presence),
                        ("bias", bias), ("tokens", tokens), ("lengths", lengths), ("prompts", prompts),
                        ("bias_tokens", bias_tokens), ("allowed", allowed)):
        if name in _FIELDS and isinstance(value, (int, float)):
            numbers.append(float(value))
            continue
        if value is None and name not in _FIELDS:
            continue
        if type(value) is not torch.Tensor:
            value = tensor_of(value)
        if name in _FIELDS:
            numbers.append(None)
        values[name] = value
        key.append(name)
        key.append(signature(value))
        pointers.append((_FIELDS.get(name, name), value.data_ptr()))
    no_grad_needed(logits, *(values[name] for name in _FLOATS if name in values))
    fresh = out is None
    if fresh:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    else:
        no_grad_needed(out)
        key.append(signature(out))
    key.extend(numbers)
    key = tuple(key)
    known = _ADJUST_ARGS.get(key)
    if known is None:
        known = _ADJUST_ARGS[key] = _prepare(logits, out, values, numbers, error_flag)
    stream = current_stream(logits.device)
    a, spans = known
    if not fresh:
        apart(logits, out, spans, pointers, error_flag)
        if not out.is_inference():  # a backward pass that kept what it held notices
            torch.autograd.graph.increment_version(out)
    a = _lib.AdjustArgs.from_buffer_copy(a)
    a.logits, a.out = logits.data_ptr(), out.data_ptr()
    for name, pointer in pointers:
        setattr(a, name, pointer)
    if error_flag is not None:
        a.error_flag = error_flag.data_ptr()
    _lib.check(_lib.load().cb_adjust_logits(ctypes.byref(a), stream), "cb_adjust_logits")
    return out


_FLOATS = ("repetition", "frequency", "presence", "bias")
_FIELDS = {"repetition": "repetitions", "frequency": "frequencies", "presence": "presences"}


def apart(logits: torch.Tensor, out: torch.Tensor, spans, pointers, error_flag: Optional[torch.Tensor]) -> None:
    """Refuse an ``out`` that shares memory with an argument, but for ``logits``' own rows: blocks write it while
    others read.  ``spans``: the bytes that each argument reaches over, by its name."""
    at, size = out.data_ptr(), spans["out"]
    same = logits.data_ptr() == at and (logits.stride(0) == out.stride(0) or logits.shape[0] <= 1)
    if not same and meet(at, size, logits.data_ptr(), spans["logits"]):
        raise ValueError("out has to be logits itself, or memory of its own")
    for name, pointer in pointers:
        if meet(at, size, pointer, spans[name]):
            raise ValueError(f"out shares memory with {name}")
    if error_flag is not None and meet(at, size, error_flag.data_ptr(), 4):
        raise ValueError("out shares memory with error_flag")


def _prepare(logits: torch.Tensor, out: torch.Tensor, values, numbers,
             error_flag: Optional[torch.Tensor]) -> Tuple[_lib.AdjustArgs, Dict[str, int]]:
    device = logits.device
    if device.type != "cuda":
        raise ValueError(f"logits are on {device}, expected a CUDA device")
    require(logits, "logits", device, tuple(_VALUES), (None, None), 1)
    rows, vocab = logits.shape
    if vocab >= 2 ** 30:
        raise ValueError(f"a vocabulary of {vocab} tokens, fewer than 2**30 are taken")
    require(out, "out", device, (logits.dtype,), (rows, vocab), 1)
    if rows > 1 and vocab and abs(out.stride(0)) < vocab:
        raise ValueError("the rows of out share memory")
    a = _lib.AdjustArgs()
    a.dtype, a.rows, a.vocab, a.ld, a.out_ld = _VALUES[logits.dtype], rows, vocab, logits.stride(0), out.stride(0)
    if "tokens" in values:
        tokens = values["tokens"]
        require(tokens, "tokens", device, tuple(_INDICES), (rows, None), 1)
        if tokens.shape[1] > MAX_HISTORY:
            raise ValueError(f"a history of {tokens.shape[1]} tokens, at most {MAX_HISTORY} are taken")
        a.token_dtype, a.history, a.token_ld = _INDICES[tokens.dtype], tokens.shape[1], tokens.stride(0)
    for name, number, neutral in zip(_FIELDS, numbers, (1.0, 0.0, 0.0)):
        if name in values:
            require(values[name], name, device, (torch.float32,), (rows,), 1)
        else:
            single = ctypes.c_float(number).value  # as the kernel has it
            if not math.isfinite(single) or (name == "repetition" and single <= 0.0):
                raise ValueError(f"{name} is {number}, expected a finite float32"
                                 + (" above 0" if name == "repetition" else ""))
        if "tokens" not in values and (name in values or number != neutral):
            raise ValueError(f"{name} needs the tokens of a history")
    a.repetition, a.frequency, a.presence = (0.0 if n is None else n for n in numbers)
    for name in ("lengths", "prompts"):
        if name in values:
            if "tokens" not in values:
                raise ValueError(f"{name} need the tokens of a history")
            require(values[name], name, device, (torch.int32,), (rows,), 1)
    if ("bias" in values) != ("bias_tokens" in values):
        raise ValueError("bias and bias_tokens belong together")
    if "bias" in values:
        ids, bias = values["bias_tokens"], values["bias"]
        require(ids, "bias_tokens", device, tuple(_INDICES), (rows, None), 1)
        require(bias, "bias", device, (torch.float32,), tuple(ids.shape), 1)
        if ids.shape[1] > MAX_BIASES:
            raise ValueError(f"{ids.shape[1]} biases to a row, at most {MAX_BIASES} are taken")
        a.bias_token_dtype, a.biases = _INDICES[ids.dtype], ids.shape[1]
        a.bias_token_ld, a.bias_ld = ids.stride(0), bias.stride(0)
    if "allowed" in values:
        require(values["allowed"], "allowed", device, (torch.int32,), (rows, -(-vocab // 32)), 1)
        a.allowed_ld = values["allowed"].stride(0)
    if error_flag is not None:
        require(error_flag, "error_flag", device, (torch.int32,), (1,), 1)
    return a, {_FIELDS.get(name, name): reach(value)
               for name, value in (("logits", logits), ("out", out), *values.items())}
