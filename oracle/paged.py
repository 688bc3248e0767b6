"""Plain forms of the paged-cache operators: 64-bit attention, and page, quantising and
verification rules written one slot, page and token at a time (NumPy and Python integers)."""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import ml_dtypes
import numpy as np

E4M3 = np.dtype(ml_dtypes.float8_e4m3fn)
TOP = {np.dtype(np.int8): np.float32(127), E4M3: np.float32(448)}


class Cache:
    """Pools and book in host memory; the operations are the rules, applied slot after slot."""

    def __init__(self, layers: int, pages: int, kv_heads: int, page: int, head_size: int, slots: int, columns: int,
                 storage=np.int8) -> None:
        shape = (layers, pages, kv_heads, page, head_size)
        self.page = page
        self.pools = [np.zeros(shape, storage) for _ in range(2)]
        self.scales = [np.zeros(shape[:3], np.float32) for _ in range(2)]
        self.table = np.full((slots, columns), -1, np.int32)
        self.lengths = np.zeros(slots, np.int32)
        self.refs = np.zeros(pages, np.int32)
        self.free: List[int] = list(range(pages - 1, -1, -1))

    def held(self, tokens: int) -> int:
        return -(-tokens // self.page)

    def copy_page(self, source: int, target: int) -> None:
        for array in (*self.pools, *self.scales):
            array[:, target] = array[:, source]

    def extend(self, counts: Sequence[int], sequences: Optional[Sequence[int]] = None) -> None:
        for i, count in enumerate(counts):
            slot = i if sequences is None else sequences[i]
            length = int(self.lengths[slot])
            have, need = self.held(length), self.held(length + count)
            if count and length % self.page:
                tail = int(self.table[slot, have - 1])
                if self.refs[tail] > 1:
                    page = self.free.pop()
                    self.copy_page(tail, page)
                    self.refs[tail] -= 1
                    self.refs[page] = 1
                    self.table[slot, have - 1] = page
            for column in range(have, need):
                page = self.free.pop()
                self.refs[page] = 1
                self.table[slot, column] = page
            self.lengths[slot] += count

    def fork(self, parents: Sequence[int], children: Sequence[int]) -> None:
        for parent, child in zip(parents, children):
            self.table[child] = self.table[parent]
            self.lengths[child] = self.lengths[parent]
            for page in self.table[child, :self.held(int(self.lengths[child]))]:
                self.refs[page] += 1

    def truncate(self, counts: Optional[Sequence[int]], sequences: Sequence[int]) -> None:
        dropped = []
        for i, slot in enumerate(sequences):
            length = int(self.lengths[slot])
            rest = 0 if counts is None else length - counts[i]
            for column in range(self.held(rest), self.held(length)):
                dropped.append(int(self.table[slot, column]))
                self.table[slot, column] = -1
            self.lengths[slot] = rest
        for page in dropped:
            self.refs[page] -= 1
        for at in range(len(dropped) - 1, -1, -1):  # the last entry of a page pushes it
            if self.refs[dropped[at]] == 0 and dropped[at] not in dropped[at + 1:]:
                self.free.append(dropped[at])

    def compact(self) -> None:
        held = int((self.refs > 0).sum())
        holes = [p for p in range(held) if self.refs[p] == 0]
        for source, target in zip([p for p in range(held, len(self.refs)) if self.refs[p] > 0], holes):
            self.copy_page(source, target)
            self.refs[target], self.refs[source] = self.refs[source], 0
            self.table[self.table == source] = target
        self.free = list(range(len(self.refs) - 1, held - 1, -1))

    def append(self, layer: int, which: int, rows: np.ndarray, slot: int, count: int) -> None:
        """``rows[:count]`` (tokens, kv_heads, head_size) float32 as the last tokens of ``slot``; float32 arithmetic."""
        end = int(self.lengths[slot])
        start = end - count
        for column in range(start // self.page, self.held(end)) if count else ():
            page, first = int(self.table[slot, column]), column * self.page
            lo, hi = max(start, first), min(end, first + self.page)
            for head in range(rows.shape[1]):
                self.scales[which][layer, page, head] = append_block(
                    self.pools[which][layer, page, head], self.scales[which][layer, page, head],
                    rows[lo - start:hi - start, head], lo - first)

    def read(self, layer: int, which: int, slot: int) -> np.ndarray:
        """(tokens, kv_heads, head_size) float64 values of a slot."""
        length = int(self.lengths[slot])
        used = self.table[slot, :self.held(length)]
        values = (self.pools[which][layer, used].astype(np.float64)
                  * self.scales[which][layer, used].astype(np.float64)[..., None, None])
        return values.transpose(0, 2, 1, 3).reshape(-1, values.shape[1], values.shape[3])[:length]


def append_block(codes: np.ndarray, scale: np.float32, rows: np.ndarray, older: int) -> np.float32:
    """Quantise ``rows`` behind the first ``older`` rows of one page and head, in place; the new scale."""
    top = TOP[codes.dtype]
    before = np.float32(scale) if older else np.float32(0)
    finite = np.abs(rows[np.isfinite(rows)])
    grown = np.float32(finite.max() if finite.size else 0) * (np.float32(1) / top)
    after = max(before, grown if grown >= np.float32(2.0 ** -110) else np.float32(0))
    inverse = np.float32(1) / after if after > 0 else np.float32(0)

    def code(x):
        x = np.where(np.isnan(x) | (inverse == 0), np.float32(0), x)
        x = np.clip(x, -top, top)
        return (np.rint(x) if codes.dtype == np.int8 else x).astype(codes.dtype)

    with np.errstate(invalid="ignore", over="ignore"):
        if older and after > before:
            codes[:older] = code(codes[:older].astype(np.float32) * (before * inverse))
        codes[older:older + len(rows)] = code(rows * inverse)
    return after


def attend(q: np.ndarray, keys: np.ndarray, values: np.ndarray, scale: float) -> np.ndarray:
    """q (tokens, heads, size), the last tokens of ``keys`` and ``values`` (length, kv_heads, size); float64."""
    out = np.zeros(q.shape)
    group = q.shape[1] // keys.shape[1]
    for t in range(q.shape[0]):
        end = keys.shape[0] - q.shape[0] + t + 1
        for h in range(q.shape[1]):
            score = keys[:end, h // group] @ q[t, h].astype(np.float64) * scale
            weight = np.exp(score - score.max())
            out[t, h] = weight @ values[:end, h // group] / weight.sum()
    return out


def verify(target: np.ndarray, draft: np.ndarray, tokens: np.ndarray, uniforms: np.ndarray,
           count: int) -> Tuple[int, List[int]]:
    """One row: accepted drafts and the emitted tokens (padded with -1); exact integer sums."""
    accepted = 0
    while accepted < count and (float(uniforms[accepted]) * float(draft[accepted, tokens[accepted]])
                                < float(target[accepted, tokens[accepted]])):
        accepted += 1
    p = target[accepted].astype(np.float32)
    q = draft[accepted].astype(np.float32) if accepted < count else np.zeros_like(p)

    def fixed(x):
        return [int(w) for w in np.trunc(np.clip(np.where(x > 0, x, 0), 0, 1).astype(np.float64) * 2.0 ** 40)]

    token = -1
    if not (np.isnan(p).any() or np.isnan(q).any()):
        weights = fixed(p - q)
        weights = weights if sum(weights) else fixed(p)
        total = sum(weights)
        if total:
            bar = min(int(float(uniforms[len(tokens)]) * float(total)), total - 1)
            running = 0
            for token, w in enumerate(weights):
                running += w
                if running > bar:
                    break
    return accepted, [int(x) for x in tokens[:accepted]] + [token] + [-1] * (len(tokens) - accepted)
