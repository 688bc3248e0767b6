"""Many samples of one prompt, as the operators are used together: 4-bit projections, a
prompt in a paged cache, forks of it, and for each step append, attention over the
shared pages, 4-bit logits, penalties and a grammar's mask, and the chosen tokens.

Every stage is compared with the same stage in float64 on what the one before gave, within
the bounds of the operators' own tests.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from cuda_b200 import logits as operators
from cuda_b200.paged import PagedCache
from cuda_b200.quantized import Weights4
from oracle import logits as plain_logits
from oracle import paged as plain
from paged_helpers import DTYPE, wide
from test_gpu_logits import words_of
from test_gpu_paged_attention import ROUNDING, WEIGHTS
from test_gpu_quantized import close

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV_HEADS, SIZE, VOCAB, SAMPLES, STEPS = 256, 8, 2, 64, 1000, 5, 4


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("storage", [torch.int8, torch.float8_e4m3fn])
def test_samples_of_one_prompt(name, storage):
    dtype = DTYPE[name]
    rng = np.random.default_rng(17)

    def weights(outputs, inputs):
        w = torch.from_numpy(rng.normal(0, 1 / math.sqrt(inputs), (outputs, inputs)).astype(np.float32)).cuda()
        return Weights4.quantise(w, group=64)

    width = (HEADS + 2 * KV_HEADS) * SIZE
    qkv, o, head = weights(width, HIDDEN), weights(HIDDEN, HEADS * SIZE), weights(VOCAB, HIDDEN)
    exact = {w: wide(w.dequantise(torch.float32)) for w in (qkv, o, head)}
    embedding = torch.from_numpy(rng.normal(0, 1, (VOCAB, HIDDEN)).astype(np.float32)).cuda().to(dtype)
    cache = PagedCache.allocate(layers=1, pages=120, kv_heads=KV_HEADS, page_size=16, head_size=SIZE,
                                sequences=SAMPLES, pages_per_sequence=40, storage=storage)

    def linear(w, x):
        y = w.linear(x)
        close(y.view(-1, y.shape[-1]), x.reshape(-1, x.shape[-1]), exact[w], 64)
        return y

    def split(rows):
        batch, tokens = rows.shape[:2]
        q = rows[..., :HEADS * SIZE].view(batch, tokens, HEADS, SIZE)
        k = rows[..., HEADS * SIZE:(HEADS + KV_HEADS) * SIZE].view(batch, tokens, KV_HEADS, SIZE)
        return q, k, rows[..., (HEADS + KV_HEADS) * SIZE:].view(batch, tokens, KV_HEADS, SIZE)

    def held(slot):
        """Keys and values of a slot in float64, (tokens, kv_heads, size)."""
        length = int(cache.lengths[slot])
        pages = cache.table[slot, :-(-length // 16)].long()
        out = []
        for pool, scale in ((cache.k_pages, cache.k_scale), (cache.v_pages, cache.v_scale)):
            x = wide(pool[0, pages].float()) * wide(scale[0, pages])[..., None, None]
            out.append(x.transpose(0, 2, 1, 3).reshape(-1, KV_HEADS, SIZE)[:length])
        return out

    # the prompt, then four more samples of it
    prompt = torch.from_numpy(rng.integers(0, VOCAB, (1, 333))).cuda()
    cache.extend([333], sequences=[0])
    _, k, v = split(linear(qkv, embedding[prompt]))
    cache.append(0, k, v, sequences=[0])
    cache.fork([0] * (SAMPLES - 1), list(range(1, SAMPLES)))
    history = torch.full((SAMPLES, 333 + STEPS + 1), -1, dtype=torch.int32, device="cuda")
    history[:, :333] = prompt.int()
    history[:, 333] = torch.from_numpy(rng.integers(0, VOCAB, SAMPLES)).cuda()
    prompts = torch.full((SAMPLES,), 333, dtype=torch.int32, device="cuda")
    ones = torch.ones(SAMPLES, dtype=torch.int32, device="cuda")
    for step in range(STEPS):
        lengths = prompts + step + 1
        x = embedding[history[torch.arange(SAMPLES), 333 + step].long()].view(SAMPLES, 1, HIDDEN)
        q, k, v = split(linear(qkv, x))
        cache.extend(ones)
        cache.append(0, k, v)
        attended = cache.attend_shared(0, q, least_bytes=0)
        cache.check_errors()
        for b in range(SAMPLES):
            keys, values = held(b)
            want = plain.attend(wide(q[b]), keys, values, 1 / math.sqrt(SIZE))
            largest = float(np.abs(values).max())
            assert np.all(np.abs(wide(attended[b]) - want)
                          <= 2 * WEIGHTS[name] * largest + ROUNDING[name] * np.abs(want) + 1e-7 * largest)
        y = x.view(SAMPLES, HIDDEN) + linear(o, attended.view(SAMPLES, HEADS * SIZE))
        rows = linear(head, y)
        bits = rng.random((SAMPLES, VOCAB)) < 0.3
        allowed = torch.from_numpy(words_of(bits)).cuda()
        adjusted = operators.adjust(rows, tokens=history, lengths=lengths, prompts=prompts, repetition=1.3,
                                    frequency=0.2, presence=0.5, allowed=allowed)
        half = torch.finfo(dtype).eps / 2
        for b in range(SAMPLES):
            want, size = plain_logits.adjust(wide(rows[b]), history[b].cpu().numpy(), int(lengths[b]), 333, 1.3, 0.2,
                                             0.5, allowed=words_of(bits)[b])
            have, fine = wide(adjusted[b]), np.isfinite(want)
            assert np.array_equal(np.isfinite(have), fine) and np.array_equal(fine, bits[b])
            error = 6 * 2.0 ** -24 * size[fine]
            assert np.all(np.abs(have[fine] - want[fine]) <= error + half * (np.abs(want[fine]) + error))
        token = adjusted.float().argmax(-1)
        assert all(bits[b, int(t)] for b, t in enumerate(token))
        history[:, 333 + step + 1] = token.int()
    assert len({tuple(h) for h in history.tolist()}) == SAMPLES  # the samples went their own ways
    cache.release(list(range(SAMPLES)))
    cache.check_errors()
    assert int(cache.height) == 120
