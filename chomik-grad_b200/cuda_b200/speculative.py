"""Verification of drafted tokens against the target model's probabilities.

The reference verifies greedy drafts (``verify_greedy_candidates``,
chomikgrad/generation.py:15-28: the longest prefix that the target's argmax
repeats).  ``verify`` is its counterpart for sampled decoding: the tokens that
it emits are distributed as the target's own samples, for the uniform numbers
that the caller draws (as ``CudaB200Device.sample`` takes them from the
caller's generator).
"""

from __future__ import annotations

import ctypes
from typing import Any, Optional, Tuple

import torch

from . import _lib
from .paged import _VALUES, require, tensor_of


def verify(target: Any, draft: Any, tokens: Any, uniforms: Any, *, counts: Any = None,
           error_flag: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Accepted drafts of each row and the tokens that the row goes on with.

    ``draft`` (batch, n, vocab) holds the probabilities that ``tokens``
    (batch, n) int64 were drawn from, ``target`` (batch, n + 1, vocab) the
    target model's, ``uniforms`` (batch, n + 1) float64 numbers in [0, 1);
    ``counts`` (batch) int32 gives fewer drafts for some rows.  Token t is
    accepted while ``u[t] * q < p``; the first refused one is replaced by a draw
    from ``max(p - q, 0)``, and after n accepted ones a token is drawn from the
    last target row, both with ``u[n]``.

    Returns ``accepted`` (batch) int32 and ``emitted`` (batch, n + 1) int64: the
    accepted tokens, the drawn one, then -1.  Rows whose probabilities hold a
    NaN or are all zero emit -1 in the drawn token's place and set
    ``error_flag`` (an int32 of the caller's, read with ``check``).  Sums are
    exact, so equal inputs give equal tokens on any launch.
    """
    target, draft, tokens, uniforms = (tensor_of(v) for v in (target, draft, tokens, uniforms))
    if target.device.type != "cuda":
        raise ValueError(f"target is on {target.device}, expected a CUDA device")
    if target.ndim != 3 or target.shape[1] < 1 or target.shape[2] < 1:
        raise ValueError(f"target has shape {tuple(target.shape)}, expected (batch, n + 1, vocab)")
    batch, n, vocab = target.shape[0], target.shape[1] - 1, target.shape[2]
    require(target, "target", target.device, tuple(_VALUES), (batch, n + 1, vocab), 1)
    require(draft, "draft", target.device, (target.dtype,), (batch, n, vocab), 1)
    require(tokens, "tokens", target.device, (torch.int64,), (batch, n), 2)
    require(uniforms, "uniforms", target.device, (torch.float64,), (batch, n + 1), 2)
    if counts is not None:
        counts = tensor_of(counts)
        require(counts, "counts", target.device, (torch.int32,), (batch,), 1)
    if error_flag is not None:
        require(error_flag, "error_flag", target.device, (torch.int32,), (1,), 1)
    if torch.cuda.current_device() != target.device.index:
        raise ValueError(f"target is on {target.device}, the current device is cuda:{torch.cuda.current_device()}")
    accepted = torch.empty(batch, dtype=torch.int32, device=target.device)
    emitted = torch.empty(batch, n + 1, dtype=torch.int64, device=target.device)
    a = _lib.VerifyArgs()
    a.target, a.draft, a.dtype = target.data_ptr(), draft.data_ptr(), _VALUES[target.dtype]
    a.batch, a.tokens, a.vocab = batch, n, vocab
    a.target_strides[:], a.draft_strides[:] = target.stride()[:2], draft.stride()[:2]
    a.drafted, a.uniforms = tokens.data_ptr(), uniforms.data_ptr()
    a.counts = None if counts is None else counts.data_ptr()
    a.accepted, a.out = accepted.data_ptr(), emitted.data_ptr()
    a.error_flag = None if error_flag is None else error_flag.data_ptr()
    _lib.call("cb_verify_draft", ctypes.byref(a), torch.cuda.current_stream().cuda_stream)
    return accepted, emitted


def check(error_flag: torch.Tensor) -> None:
    """Raise what ``verify`` found (reads one number back)."""
    value = int(error_flag.item())
    if value:
        error_flag.zero_()
        raise _lib.flag_error(value)
