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
from .paged import _VALUES, Prepared, current_stream, no_grad_needed, require, signature, tensor_of

_VERIFY_ARGS = Prepared()


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
    target, draft, tokens, uniforms = tensor_of(target), tensor_of(draft), tensor_of(tokens), tensor_of(uniforms)
    counts = None if counts is None else tensor_of(counts)
    no_grad_needed(target, draft)
    key = (signature(target), signature(draft), signature(tokens), signature(uniforms), signature(counts),
           signature(error_flag))
    known = _VERIFY_ARGS.get(key)
    if known is None:
        known = _VERIFY_ARGS[key] = _prepare(target, draft, tokens, uniforms, counts, error_flag)
    stream = current_stream(target.device)
    emitted = torch.empty_like(uniforms, dtype=torch.int64)
    accepted = torch.empty(target.shape[0], dtype=torch.int32, device=target.device)
    a = _lib.VerifyArgs.from_buffer_copy(known)
    a.target, a.draft, a.drafted, a.uniforms = (target.data_ptr(), draft.data_ptr(), tokens.data_ptr(),
                                                uniforms.data_ptr())
    a.accepted, a.out = accepted.data_ptr(), emitted.data_ptr()
    if counts is not None:
        a.counts = counts.data_ptr()
    if error_flag is not None:
        a.error_flag = error_flag.data_ptr()
    _lib.check(_lib.load().cb_verify_draft(ctypes.byref(a), stream), "cb_verify_draft")
    return accepted, emitted


def _prepare(target: torch.Tensor, draft: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor,
             counts: Optional[torch.Tensor], error_flag: Optional[torch.Tensor]) -> _lib.VerifyArgs:
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
        require(counts, "counts", target.device, (torch.int32,), (batch,), 1)
    if error_flag is not None:
        require(error_flag, "error_flag", target.device, (torch.int32,), (1,), 1)
    a = _lib.VerifyArgs()
    a.dtype, a.batch, a.tokens, a.vocab = _VALUES[target.dtype], batch, n, vocab
    a.target_strides[:], a.draft_strides[:] = target.stride()[:2], draft.stride()[:2]
    return a


def check(error_flag: torch.Tensor) -> None:
    """Raise what ``verify`` found (reads one number back)."""
    value = int(error_flag.item())
    if value:
        error_flag.zero_()
        raise _lib.flag_error(value)
