"""Penalties, biases and masks on one logit row in float64 (``cuda_b200.logits.adjust``)."""

from __future__ import annotations

import numpy as np


def adjust(logits, tokens=(), length=None, prompt=0, repetition=1.0, frequency=0.0, presence=0.0, bias_tokens=(),
           bias=(), allowed=None):
    """The adjusted row, and for each value the largest magnitude that its sum went through."""
    x = np.array(logits, np.float64)
    vocab = len(x)
    length = len(tokens) if length is None else min(max(int(length), 0), len(tokens))
    prompt = min(max(int(prompt), 0), length)
    size = np.abs(x)
    held = [t for t in np.asarray(tokens)[:length].tolist() if 0 <= t < vocab]
    made = [t for t in np.asarray(tokens)[prompt:length].tolist() if 0 <= t < vocab]
    with np.errstate(invalid="ignore"):
        for t in set(held):
            x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
            size[t] = max(size[t], abs(x[t]))
        for t in set(made):
            x[t] -= frequency * made.count(t) + presence
            size[t] += abs(frequency) * made.count(t) + abs(presence)
        total = {}
        for t, b in zip(np.asarray(bias_tokens).tolist(), np.asarray(bias, np.float64).tolist()):
            if 0 <= t < vocab:
                total[t] = total.get(t, 0.0) + b
                size[t] += abs(b)
        for t, b in total.items():
            x[t] += b
    if allowed is not None:
        words = np.asarray(allowed).astype(np.int64) & 0xFFFFFFFF
        token = np.arange(vocab)
        x[(words[token // 32] >> (token % 32)) & 1 == 0] = -np.inf
    return x, size
