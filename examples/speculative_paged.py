"""Speculative serving over paged 8-bit caches: a batch of prompts of unlike
lengths, a draft model and a target model, on the library's kernels.

    python examples/speculative_paged.py [--storage e4m3] [--drafts 4] [--tokens 64]

Each step the draft model proposes ``--drafts`` tokens one at a time, the target
model scores them and the token before them as one block, ``speculative.verify``
accepts a prefix and draws the next token, and both caches drop what was
refused.  One more sequence is forked from a running one, shares its pages and
goes on by itself; at the end a slot is released and the cache compacted.

The models are Llama decoders (RMSNorm, rotate-half RoPE, grouped heads, SwiGLU)
with random bfloat16 weights, so the text means nothing: what the example shows
is the calls and their order.  Linear layers run as ``cb_gemm_rows`` (up to 256
rows a call), the probabilities as ``cb_softmax_rows``.
"""

from __future__ import annotations

import argparse
import ctypes
from dataclasses import dataclass
from pathlib import Path
import sys
from typing import Dict, List, Optional

import torch

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "chomik-grad_b200"))

from cuda_b200 import _lib, speculative
from cuda_b200.paged import PagedCache


@dataclass(frozen=True)
class Shape:
    layers: int = 4
    hidden: int = 256
    heads: int = 8
    kv_heads: int = 2
    head_size: int = 64
    intermediate: int = 688
    vocab: int = 4096
    theta: float = 10_000.0
    eps: float = 1e-5


class Linear:
    """Rows times up to three bfloat16 weights: cb_gemm_rows with its prologues and residual."""

    def __init__(self, device: torch.device) -> None:
        self.device, self.lib = device, _lib.load()
        self.counters = torch.zeros(0, dtype=torch.int32, device=device)
        self.flag = torch.zeros(1, dtype=torch.int32, device=device)

    def __call__(self, x: torch.Tensor, *weights: torch.Tensor, norm: Optional[torch.Tensor] = None, eps: float = 0.0,
                 gate: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None) -> List[torch.Tensor]:
        source = x if gate is None else gate  # SwiGLU: silu(gate) * x
        rows, k = source.shape
        out = [torch.empty(rows, w.shape[0], device=self.device) for w in weights]
        a = _lib.GemmRowsArgs()
        a.x, a.x_dtype, a.ldx, a.rows, a.k, a.n_w = source.data_ptr(), _lib.F32, k, rows, k, len(weights)
        for i, (w, o) in enumerate(zip(weights, out)):
            a.w[i], a.w_rows[i], a.out[i], a.ldo[i] = w.data_ptr(), w.shape[0], o.data_ptr(), w.shape[0]
        if norm is not None:
            a.x_mode, a.norm_w, a.norm_w_dtype, a.divisor, a.eps = (_lib.ROWS_X_RMS, norm.data_ptr(), _lib.BF16,
                                                                   float(k), eps)
        if gate is not None:
            a.x_mode, a.x2, a.x2_dtype, a.ldx2 = _lib.ROWS_X_SWIGLU, x.data_ptr(), _lib.F32, k
        if residual is not None:
            a.residual, a.ldr = residual.data_ptr(), residual.shape[1]
        need = self.lib.cb_gemm_rows_counters(ctypes.byref(a))
        if self.counters.numel() < need:
            self.counters = torch.zeros(need, dtype=torch.int32, device=self.device)
        scratch = torch.empty(self.lib.cb_gemm_rows_scratch(ctypes.byref(a)), dtype=torch.uint8, device=self.device)
        a.scratch, a.counters, a.error_flag = scratch.data_ptr(), self.counters.data_ptr(), self.flag.data_ptr()
        _lib.call("cb_gemm_rows", ctypes.byref(a), torch.cuda.current_stream().cuda_stream)
        return out


class Decoder:
    """A Llama decoder whose keys and values live in a ``PagedCache``."""

    def __init__(self, shape: Shape, weights: Dict[str, torch.Tensor], cache: PagedCache) -> None:
        self.shape, self.weights, self.cache = shape, weights, cache
        self.linear = Linear(cache.device)
        step = torch.arange(0, shape.head_size, 2, device=cache.device, dtype=torch.float32) / shape.head_size
        self.frequency = shape.theta ** -step

    def rope(self, x: torch.Tensor, position: torch.Tensor) -> torch.Tensor:
        angle = position[..., None, None].float() * self.frequency
        cos, sin = angle.cos(), angle.sin()
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    def __call__(self, tokens: torch.Tensor, counts: torch.Tensor) -> torch.Tensor:
        """Probabilities (batch, n, vocab) after each of row b's first counts[b] tokens, for which it makes room."""
        s, w, cache = self.shape, self.weights, self.cache
        batch, n = tokens.shape
        cache.extend(counts)
        start = (cache.lengths[:batch] - counts)[:, None]
        position = start + torch.arange(n, device=tokens.device)
        hidden = w["embed"][tokens.reshape(-1)].float()
        for layer in range(s.layers):
            def part(name):
                return w[f"{layer}.{name}"]

            q, k, v = self.linear(hidden, part("q"), part("k"), part("v"), norm=part("norm1"), eps=s.eps)
            q = self.rope(q.view(batch, n, s.heads, s.head_size), position)
            k = self.rope(k.view(batch, n, s.kv_heads, s.head_size), position)
            cache.append(layer, k, v.view(batch, n, s.kv_heads, s.head_size), counts=counts)
            heads = cache.attend(layer, q, counts=counts).view(batch * n, -1)
            hidden, = self.linear(heads, part("o"), residual=hidden)
            gate, up = self.linear(hidden, part("gate"), part("up"), norm=part("norm2"), eps=s.eps)
            hidden, = self.linear(up, part("down"), gate=gate, residual=hidden)
        logits, = self.linear(hidden, w["head"], norm=w["norm"], eps=s.eps)
        out = torch.empty_like(logits)
        _lib.call("cb_softmax_rows", logits.data_ptr(), logits.shape[0], s.vocab, 0, out.data_ptr(),
                  torch.cuda.current_stream().cuda_stream)
        return out.view(batch, n, s.vocab)


def random_weights(shape: Shape, seed: int, device: torch.device, spread: float = 0.08) -> Dict[str, torch.Tensor]:
    gen = torch.Generator(device=device).manual_seed(seed)

    def matrix(rows, columns):
        return (spread * torch.randn(rows, columns, device=device, generator=gen)).bfloat16()

    q, kv = shape.heads * shape.head_size, shape.kv_heads * shape.head_size
    w = {"embed": matrix(shape.vocab, shape.hidden), "head": matrix(shape.vocab, shape.hidden),
         "norm": torch.ones(shape.hidden, device=device, dtype=torch.bfloat16)}
    for layer in range(shape.layers):
        w |= {f"{layer}.q": matrix(q, shape.hidden), f"{layer}.k": matrix(kv, shape.hidden),
              f"{layer}.v": matrix(kv, shape.hidden), f"{layer}.o": matrix(shape.hidden, q),
              f"{layer}.gate": matrix(shape.intermediate, shape.hidden),
              f"{layer}.up": matrix(shape.intermediate, shape.hidden),
              f"{layer}.down": matrix(shape.hidden, shape.intermediate)}
        for name in ("norm1", "norm2"):
            w[f"{layer}.{name}"] = torch.ones(shape.hidden, device=device, dtype=torch.bfloat16)
    return w


def draw(probabilities: torch.Tensor, gen: torch.Generator) -> torch.Tensor:
    return torch.multinomial(probabilities, 1, generator=gen)


def serve(target: Decoder, draft: Decoder, prompts: List[List[int]], tokens: int, drafts: int, seed: int) -> dict:
    """At least ``tokens`` tokens of every prompt; slot len(prompts) - 1 (an empty prompt) continues slot 0."""
    device = target.cache.device
    gen = torch.Generator(device=device).manual_seed(seed)
    batch = len(prompts)
    longest = max(map(len, prompts))
    counts = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=device)
    padded = torch.tensor([p + [0] * (longest - len(p)) for p in prompts], device=device)
    first = target(padded, counts)[torch.arange(batch, device=device), (counts.long() - 1).clamp(min=0)]
    draft(padded, counts)
    for cache in (target.cache, draft.cache):  # the last slot is another sample of the first prompt
        cache.fork([0], [batch - 1])
    first[batch - 1] = first[0]
    last = draw(first, gen)  # (batch, 1)
    emitted: List[List[int]] = [[int(t)] for t in last[:, 0].tolist()]
    one = torch.ones(batch, dtype=torch.int32, device=device)
    proposed = accepted_total = 0
    while min(map(len, emitted)) < tokens:
        block, rows = [last], []
        for _ in range(drafts):
            rows.append(draft(block[-1], one))
            block.append(draw(rows[-1][:, 0], gen))
        draft(block[-1], one)  # its cache holds the block too
        block = torch.cat(block, 1)
        scores = target(block, one * (drafts + 1))
        uniforms = torch.rand(batch, drafts + 1, dtype=torch.float64, device=device, generator=gen)
        accepted, out = speculative.verify(scores, torch.cat(rows, 1), block[:, 1:].contiguous(), uniforms)
        refused = drafts - accepted
        target.cache.truncate(refused)
        draft.cache.truncate(refused)
        last = out.gather(1, accepted.long()[:, None])
        for sequence, row, n in zip(emitted, out.tolist(), accepted.tolist()):
            sequence.extend(row[:n + 1])
            accepted_total += n
        proposed += batch * drafts
    for decoder in (target, draft):
        decoder.cache.check_errors()
    target.cache.release([batch - 1])
    target.cache.compact()
    target.cache.check_errors()
    return {"emitted": emitted, "accepted": accepted_total / proposed}


def build(storage: str, seed: int, slots: int, same: bool, device: torch.device):
    """A target and a draft model of half its layers (``same``: twice the target), with caches of their own."""
    shape = Shape()
    small = shape if same else Shape(layers=2)
    dtype = torch.int8 if storage == "int8" else torch.float8_e4m3fn

    def decoder(s, weights):
        return Decoder(s, weights, PagedCache.allocate(
            layers=s.layers, pages=slots * 16, kv_heads=s.kv_heads, page_size=16, head_size=s.head_size,
            sequences=slots, pages_per_sequence=16, storage=dtype, device=device))

    weights = random_weights(shape, seed, device)
    return decoder(shape, weights), decoder(small, weights)


def main(argv: Optional[List[str]] = None) -> dict:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--storage", choices=["int8", "e4m3"], default="int8")
    parser.add_argument("--drafts", type=int, default=4)
    parser.add_argument("--tokens", type=int, default=64)
    parser.add_argument("--seed", type=int, default=0)
    parser.add_argument("--same", action="store_true", help="draft with the target model itself")
    args = parser.parse_args(argv)
    device = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator().manual_seed(args.seed + 1)
    prompts = [torch.randint(0, 4096, (n,), generator=gen).tolist() for n in (23, 40, 7)] + [[]]
    target, draft = build(args.storage, args.seed, len(prompts), args.same, device)
    result = serve(target, draft, prompts, args.tokens, args.drafts, args.seed)
    print(f"{sum(map(len, result['emitted']))} tokens of {len(prompts)} sequences, "
          f"{100 * result['accepted']:.0f}% of the drafts accepted; "
          f"{int((target.cache.refs > 0).sum())} pages held after a release and compaction")
    return result


if __name__ == "__main__":
    main()
