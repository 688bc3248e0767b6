"""Shared pages, logit adjustments and 4-bit products at their largest: pools, weights and vocabularies
beyond 32 bits, thousands of sequences, the largest pages, blocks of hundreds of tokens."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from cuda_b200 import logits
from cuda_b200.paged import PagedCache
from cuda_b200.quantized import Weights4, quantise
from paged_helpers import DTYPE, to_device, wide
from test_gpu_paged_attention import ROUNDING, WEIGHTS, expected, queries
from test_gpu_paged_shared import check, family

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("storage", [torch.int8, torch.float8_e4m3fn])
def test_shared_pages_beyond_32_bits(storage):
    """Pages at the end of a pool of more than 2^32 bytes give the bits that they give in a small one."""
    pages, kv_heads, page, size = 16_500, 8, 256, 128
    assert pages * kv_heads * page * size > 2 ** 32
    generator = torch.Generator("cuda").manual_seed(5)
    k, v = (torch.randn(1, 700, kv_heads, size, device="cuda", generator=generator) for _ in range(2))
    outputs = []
    for count in (12, pages):
        cache = PagedCache.allocate(layers=1, pages=count, kv_heads=kv_heads, page_size=page, head_size=size, sequences=3,
                                    pages_per_sequence=4, storage=storage)
        cache.free.copy_(torch.arange(count, dtype=torch.int32, device="cuda"))  # handed out from the end
        cache.extend([700], sequences=[0])
        cache.append(0, k, v, sequences=[0])
        cache.fork([0, 0], [1, 2])
        cache.extend([1, 1, 1])
        cache.append(0, k[:, :1].expand(3, 1, kv_heads, size), v[:, :1].expand(3, 1, kv_heads, size))
        held = cache.table[cache.table >= 0]
        assert int(held.min()) >= count - 7
        out = []
        for dtype in DTYPE.values():
            q = torch.randn(3, 1, 2 * kv_heads, size, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
            out.append(cache.attend_shared(0, q.to(dtype), least_bytes=0))
        cache.check_errors()
        outputs.append(out)
    for small, large in zip(*outputs):
        assert torch.equal(small, large) and bool(torch.isfinite(small).all()) and float(small.abs().max()) > 0


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("storage", ["int8", "e4m3"])
@pytest.mark.parametrize("prefix", [255, 256, 1000])
def test_largest_pages(dtype, storage, prefix):
    rng = np.random.default_rng(prefix)
    host = family(rng, prefix, [1, 300, 2, 513], page=256, head_size=128, storage=storage)
    check(host, queries(rng, 4, 1, 8, 128, dtype), [1] * 4, None, dtype)


@pytest.mark.parametrize("dtype", list(DTYPE))
def test_blocks_of_hundreds_of_tokens(dtype):
    """300 tokens and 4 heads to a kv head: rows of one sequence fill several blocks of the shared keys."""
    rng = np.random.default_rng(300)
    host = family(rng, 800, [300, 301, 400], kv_heads=1, head_size=32)
    check(host, queries(rng, 3, 300, 4, 32, dtype), [300, 7, 299], None, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_thousands_of_rows_of_few_slots(dtype):
    """3000 rows of a call on five slots: more than the threads that look for common pages, and far more than slots."""
    rng = np.random.default_rng(3)
    host = family(rng, 500, [1, 9, 33, 2, 70], head_size=32)
    cache = to_device(host)
    few = queries(rng, 5, 1, 4, 32, dtype)
    slots = torch.from_numpy(rng.integers(0, 5, 3000).astype(np.int32)).cuda()
    got = cache.attend_shared(0, few[slots.long()], sequences=slots, least_bytes=0)
    cache.check_errors()
    want = expected(host, few, [1] * 5, range(5), 1 / math.sqrt(32))[slots.cpu().numpy()]
    values = max(float(np.abs(host.read(0, 1, s)).max()) for s in range(5))
    assert (np.abs(wide(got) - want) <= 2 * WEIGHTS[dtype] * values + ROUNDING[dtype] * np.abs(want) + 1e-7 * values).all()


def test_largest_vocabulary():
    """2^30 - 1 tokens, in place: the first and last, a masked one, a bias, and no other changes."""
    vocab = 2 ** 30 - 1
    x = torch.ones(1, vocab, dtype=torch.bfloat16, device="cuda")
    tokens = torch.tensor([[0, vocab - 1, vocab, 7, -1, 2 ** 31 + 5, 2 ** 40]], device="cuda")
    allowed = torch.full((1, 2 ** 25), -1, dtype=torch.int32, device="cuda")
    allowed[0, -1] &= ~(1 << 29)  # token vocab - 2
    logits.adjust(x, tokens=tokens, repetition=2.0, bias_tokens=torch.tensor([[vocab - 1, 5, vocab + 4]], device="cuda"),
                  bias=torch.tensor([[4.0, 8.0, 1.0]], device="cuda"), allowed=allowed, out=x)
    assert [float(x[0, at]) for at in (0, 5, 7, vocab - 2, vocab - 1)] == [0.5, 9.0, 0.5, -math.inf, 4.5]
    assert int((x == 1).sum()) == vocab - 5


def test_many_rows_of_few_tokens():
    """A million rows of three tokens, each with a token of its own to lose."""
    rows = 2 ** 20
    x = torch.arange(3, device="cuda", dtype=torch.float32).repeat(rows, 1)
    tokens = (torch.arange(rows, device="cuda") % 4).int()[:, None]  # (token 3 is none)
    got = logits.adjust(x, tokens=tokens, presence=10.0)
    assert torch.equal(got, x - 10 * (torch.arange(3, device="cuda") == tokens))


@pytest.mark.parametrize("dtype", list(DTYPE))
def test_weights_beyond_32_bits(dtype):
    """2^32 weights and more: their codes, and the numbers that they are made of, pass 32 bits."""
    outputs, inputs = 131_136, 32_768
    gen = torch.Generator("cuda").manual_seed(2)
    codes = torch.randint(0, 256, (outputs, inputs // 2), device="cuda", generator=gen, dtype=torch.uint8)
    scales = torch.ones(outputs, inputs // 128, dtype=torch.bfloat16, device="cuda")
    weights = Weights4.pack(codes, scales)
    x = torch.randint(-2, 3, (2, inputs), device="cuda", generator=gen).to(DTYPE[dtype])
    got = weights.linear(x)
    dense = weights.dequantise(torch.bfloat16)  # whole numbers -8 .. 7
    for rows in (slice(0, 500), slice(65_300, 65_700), slice(outputs - 500, outputs)):
        byte = codes[rows].short()
        want = torch.stack([byte & 15, byte >> 4], -1).flatten(1) - 8
        assert torch.equal(dense[rows].short(), want)
        assert torch.equal(got[:, rows], (x.double() @ want.double().T).to(DTYPE[dtype]))  # sums below 2^20: exact
    del codes, weights
    again, scale = quantise(dense)
    assert torch.equal(scale[-64:].cpu(), (dense[-64:].view(64, -1, 128).abs().amax(-1).float().cpu() / 7).bfloat16())
    ratio = dense[-64:].float().cpu().view(64, -1, 128) / scale[-64:].float().cpu()[..., None]
    byte = again[-64:].cpu().short()
    assert torch.equal(torch.stack([byte & 15, byte >> 4], -1).flatten(1) - 8, ratio.round().clamp(-8, 7).flatten(1).short())
