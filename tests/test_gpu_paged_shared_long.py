"""cb_paged_attention_shared where a block walks many tiles of shared keys, or several items one
after the other: what the blocks of a large call do, made small by many kv heads of 32.

An item is a kv head and a block of rows.  With more items than half the SMs each is one
block's, so its tiles of 64 keys are not cut; with more than the SMs some blocks take two or
three items.  The bound is the one derived in test_gpu_paged_attention.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from paged_helpers import DTYPE, to_device, wide
from test_gpu_paged_attention import ROUNDING, WEIGHTS, queries
from test_gpu_paged_shared import family

pytestmark = pytest.mark.gpu

SIZE = 32


def sms() -> int:
    return torch.cuda.get_device_properties(0).multi_processor_count


def exact(cache, q, counts, slots=None):
    """float64 attention over the cache's dequantised layer 0, on the device."""
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b in range(q.shape[0]):
        slot, n = b if slots is None else slots[b], counts[b]
        length = int(cache.lengths[slot])
        if n == 0:
            continue
        held = cache.table[slot, :-(-length // cache.page_size)].long()
        keys, values = ((pool[0, held].double() * scale[0, held].double()[..., None, None]).transpose(0, 1).flatten(1, 2)
                        [:, :length] for pool, scale in ((cache.k_pages, cache.k_scale), (cache.v_pages, cache.v_scale)))
        rows = q[b, :n].double().view(n, cache.kv_heads, -1, q.shape[-1]).permute(1, 0, 2, 3)  # (kv_heads, n, group, size)
        score = torch.einsum("hngd,hkd->hngk", rows, keys) / math.sqrt(q.shape[-1])
        limit = length - n + 1 + torch.arange(n, device="cuda")
        score.masked_fill_(torch.arange(length, device="cuda") >= limit[:, None, None], -math.inf)
        got = torch.einsum("hngk,hkd->hngd", torch.softmax(score, -1), values)
        out[b, :n] = got.permute(1, 0, 2, 3).reshape(n, -1, q.shape[-1])
    return out.cpu().numpy()


def run(rng, dtype, storage, prefix, tails, kv_heads, group, tokens=1, page=16, counts=None):
    host = family(rng, prefix, tails, kv_heads=kv_heads, head_size=SIZE, storage=storage, page=page)
    cache = to_device(host)
    counts = [min(tokens, t) for t in tails] if counts is None else counts
    q = queries(rng, len(tails), tokens, kv_heads * group, SIZE, dtype)
    given = torch.tensor(counts, dtype=torch.int32, device="cuda")
    got = cache.attend_shared(0, q, counts=given, least_bytes=0)
    cache.check_errors()
    want = exact(cache, q, counts)
    values = float(np.nanmax(np.abs(host.pools[1].astype(np.float32) * host.scales[1][..., None, None])))
    bound = 2 * WEIGHTS[dtype] * values + ROUNDING[dtype] * np.abs(want) + 1e-7 * values
    have = wide(got)
    assert np.isfinite(have).all()
    assert (np.abs(have - want) <= bound).all(), float(np.max(np.abs(have - want) / bound))
    for _ in range(3):
        assert torch.equal(got, cache.attend_shared(0, q, counts=given, least_bytes=0))
    cache.check_errors()


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("storage", ["int8", "e4m3"])
@pytest.mark.parametrize("keys", [1700, 1536, 3300])
def test_many_tiles_of_few_rows(dtype, storage, keys):
    """27, 24 and 52 tiles to a block, both sets the same rows: the pages and scales that are looked up
    eight tiles at a time take the place of those of tiles before."""
    run(np.random.default_rng(keys), dtype, storage, keys, [1, 30], sms() // 2 + 6, 1)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("storage", ["int8", "e4m3"])
@pytest.mark.parametrize("keys", [1700, 3300])
def test_many_tiles_of_many_rows(dtype, storage, keys):
    """The same with two sets of rows, the second with a few."""
    run(np.random.default_rng(keys + 1), dtype, storage, keys, [1 + b % 5 for b in range(17)], sms() // 2 + 6, 8)


def several(more):
    """``more`` kv heads than there are SMs (a few blocks take two items), or fewer than twice as many (a few take one)."""
    return more + sms() * (2 if more < 0 else 1)


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("storage", ["int8", "e4m3"])
@pytest.mark.parametrize("keys", [64, 130, 208, 320, 900])
@pytest.mark.parametrize("more", [13, -9])
def test_several_items_of_few_rows(dtype, storage, keys, more):
    """1, 2, 4 (the last of 16 keys), 5 and 14 tiles of each item: one set has fewer tiles than the other or none, and
    tiles that are looked up together belong to two or more items."""
    run(np.random.default_rng(keys + more), dtype, storage, keys, [1, 7, 18], several(more), 1)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("storage", ["int8", "e4m3"])
@pytest.mark.parametrize("keys", [64, 130, 320, 900])
def test_several_items_of_many_rows(dtype, storage, keys):
    run(np.random.default_rng(keys), dtype, storage, keys, [1 + b % 4 for b in range(18)], several(13), 8)


@pytest.mark.parametrize("dtype", list(DTYPE))
def test_several_items_of_blocks(dtype):
    """Items that are blocks of rows as well as heads: 90 sequences of 5 tokens (fewer in some, none in one) on 80 kv
    heads; 450 rows a head are four blocks of 128, or two of 256."""
    rng = np.random.default_rng(90)
    tails = [0 if b == 7 else 5 + b % 3 for b in range(90)]
    counts = [0 if b == 7 else 5 - b % 4 for b in range(90)]
    run(rng, dtype, "int8", 700, tails, sms() // 2 + 6, 1, tokens=5, counts=counts)


@pytest.mark.parametrize("dtype", list(DTYPE))
def test_three_items_and_more(dtype):
    """Five items to a block, of 7 and 25 tiles."""
    rng = np.random.default_rng(5)
    for keys in (440, 1600):
        run(rng, dtype, "e4m3", keys, [1, 3], 4 * sms() + 5, 1)
