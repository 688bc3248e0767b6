"""cb_paged_attention_shared: NaN codes, rows that share a warp with others, keys that a heavy one
outweighs, and the bits that weights keep."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from paged_helpers import DTYPE, to_device, wide
from test_gpu_paged_attention import expected, queries
from test_gpu_paged_attention_range import WEIGHTS
from test_gpu_paged_shared import family

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("sequences", [3, 40])
@pytest.mark.parametrize("larger", [1, 512])
def test_nan_codes(dtype, sequences, larger):
    """A NaN in a shared key makes all NaN, wherever it stands among its neighbours; one in a value its element."""
    rng = np.random.default_rng(1)
    host = family(rng, 256, [1 + b % 5 for b in range(sequences)], kv_heads=1, head_size=64, storage="e4m3")
    host.scales[1] *= np.float32(larger)
    q = queries(rng, sequences, 1, 4, 64, dtype)
    clean = to_device(host).attend_shared(0, q, least_bytes=0)
    assert torch.isfinite(clean).all()
    for row in range(16):
        page = int(host.table[0, row])
        for which in range(2):
            cache = to_device(host)
            pool = (cache.k_pages, cache.v_pages)[which].view(torch.uint8)
            pool[0, page, 0, row, 7] = 0x7F
            got = cache.attend_shared(0, q, least_bytes=0)
            cache.check_errors()
            if which == 0:
                assert torch.isnan(got).all(), row
            else:
                assert torch.isnan(got[..., 7]).all(), row
                assert torch.equal(got[..., :7], clean[..., :7]) and torch.equal(got[..., 8:], clean[..., 8:])


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("storage", ["int8", "e4m3"])
@pytest.mark.parametrize("sequences", [3, 40])
def test_rows_by_themselves(dtype, storage, sequences):
    """What the queries past a count hold, and those of other sequences, does not move a bit of a row."""
    rng = np.random.default_rng(2)
    tails = [5 + b % 3 for b in range(sequences)]
    counts = [5 - b % 4 for b in range(sequences)]
    host = family(rng, 1000, tails, kv_heads=2, head_size=64, storage=storage)
    cache = to_device(host)
    given = torch.tensor(counts, dtype=torch.int32, device="cuda")
    q = queries(rng, sequences, 5, 8, 64, dtype)
    for b, n in enumerate(counts):
        q[b, n:] = 0
    want = cache.attend_shared(0, q, counts=given, least_bytes=0)
    for size in (3.0, 100.0, 3000.0, math.inf, math.nan):
        other = q.clone()
        for b, n in enumerate(counts):
            other[b, n:] = (size * torch.from_numpy(rng.normal(0, 1, (5 - n, 8, 64)).astype(np.float32))).to(q.dtype).cuda()
        assert torch.equal(cache.attend_shared(0, other, counts=given, least_bytes=0), want), size
        other = q.clone()
        other[1] *= size
        got = cache.attend_shared(0, other, counts=given, least_bytes=0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[2:], want[2:]), size
    cache.check_errors()


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("sequences", [3, 40])
@pytest.mark.parametrize("above", [5, 12, 20, 40, 60, 90])
@pytest.mark.parametrize("where", [0, 700, 1279])
def test_what_a_heavy_key_leaves(dtype, sequences, above, where):
    """One key outweighs each of the others by 2^above and has a value of zero: the others are the result, all tiles
    but its own to their full bits.

    With s the others' share of the weights, largest the largest value: an error e of the weights moves an output
    by 2 e s largest; a tile's weights are rounded to 2^-25 (in two parts of float32: 2^-23 of the largest at worst) of
    what its own largest is above, 2^-8 (2^-2), and the heavy key's tile to 2^-27 of the heavy weight, where no key
    loses more than itself.
    """
    rng = np.random.default_rng(above + where)
    size, prefix = 64, 1280
    host = family(rng, prefix, [1 + 4 * b % 9 for b in range(sequences)], kv_heads=1, head_size=size, page=64)
    host.scales[0][np.isfinite(host.scales[0])] = 0.25
    host.scales[1][np.isfinite(host.scales[1])] = 2.0 ** -6
    for slot in range(sequences):
        for at in range(host.held(int(host.lengths[slot]))):
            page = int(host.table[slot, at])
            rows = min(64, int(host.lengths[slot]) - 64 * at)
            if at < prefix // 64 and slot > 0:
                continue
            host.pools[0][0, page, 0, :rows] = 0
            host.pools[0][0, page, 0, :rows, 0] = rng.integers(-4, 5, rows)
            host.pools[1][0, page, 0, :rows] = rng.integers(64, 128, (rows, size))  # one sign: nothing cancels
    page, row = int(host.table[0, where // 64]), where % 64
    host.pools[0][0, page, 0, row, 0] = 127
    host.pools[1][0, page, 0, row] = 0
    q = torch.zeros(sequences, 1, 4, size, device="cuda", dtype=DTYPE[dtype])
    q[..., 0] = above * math.log(2.0) / (0.25 * 127)
    cache = to_device(host)
    got = wide(cache.attend_shared(0, q, scale=1.0, least_bytes=0))
    cache.check_errors()
    want = expected(host, q, [1] * sequences, range(sequences), 1.0)
    info, largest = torch.finfo(DTYPE[dtype]), 127 * 2.0 ** -6
    score = 0.25 * float(q[0, 0, 0, 0])
    tile = slice(where // 64 * 64, where // 64 * 64 + 64)
    for b in range(sequences):
        weight = np.exp(score * (host.read(0, 0, b)[:, 0, 0] / 0.25 - 127))  # of the heavy one
        total = weight.sum()
        others = np.delete(weight, where) / total
        share, mine = others.sum(), np.delete(weight[tile], where % 64) / total
        part = 2.0 ** -23 if dtype == "f32" else 2.0 ** -17
        bound = (2 * (WEIGHTS[dtype] + part * math.exp(8 * score)) * share + np.minimum(mine, 2.0 ** -27).sum()) * largest
        bound = bound + info.eps / 2 * np.abs(want[b]) + info.tiny * info.eps / 2
        if np.abs(want[b]).min() > 4 * info.tiny * info.eps:  # (what the type holds)
            assert (np.abs(want[b]) > bound).all()  # zeros would not do
        assert (np.abs(got[b] - want[b]) <= bound).all(), float(np.max(np.abs(got[b] - want[b]) / bound))


@pytest.mark.parametrize("storage", ["int8", "e4m3"])
@pytest.mark.parametrize("sequences, tokens, size", [(3, 1, 64), (40, 1, 128), (9, 5, 32)])
def test_float16_keeps_its_bits(storage, sequences, tokens, size):
    """float16 outputs are as near as their own rounding: weights and queries are held to more than its 11 bits.

    In the 2-norm, over the result's: rounding to 11 bits moves float16 numbers by 1.9e-4 to 2.4e-4 (what `floor` is
    here); weights held to 2^-16 (scores below 64 in base 2 of 22 bits, exponentials to 2.5e-6, two parts) move the
    result by 3.1e-5 before that at most, 0.15 of it.
    """
    rng = np.random.default_rng(size)
    tails = [tokens + b % 3 for b in range(sequences)]
    host = family(rng, 1280, tails, kv_heads=1, head_size=size, storage=storage)
    q = queries(rng, sequences, tokens, 4, size, "f16")
    cache = to_device(host)
    got = wide(cache.attend_shared(0, q, least_bytes=0))
    cache.check_errors()
    want = expected(host, q, [tokens] * sequences, range(sequences), 1 / math.sqrt(size))
    floor = np.linalg.norm(want.astype(np.float16).astype(np.float64) - want)
    assert np.linalg.norm(got - want) <= 1.15 * floor, float(np.linalg.norm(got - want) / floor)


@pytest.mark.parametrize("dtype, sequences, pages", [("f32", 2, 290), ("bf16", 2, 290), ("f16", 2, 290), ("bf16", 150, 145),
                                                    ("f16", 150, 145)])
def test_long_runs_of_zero_values(dtype, sequences, pages):
    """Thousands of shared keys with values of zero, whose scores rise by 12.9 (in base 2) behind the first page: they
    take nearly all of the weight, and what is left of each sequence's own keys is the result."""
    rng = np.random.default_rng(sequences)
    kv_heads, size, page = torch.cuda.get_device_properties(0).multi_processor_count // 2 + 6, 32, 64
    prefix, tails = 64 * pages, [2 + b % 4 for b in range(sequences)]
    host = family(rng, prefix, tails, kv_heads=kv_heads, head_size=size, page=page)
    host.scales[0][np.isfinite(host.scales[0])] = 0.25
    shared, own = host.table[0, :pages], host.table[:, pages]
    host.pools[0][0, shared] = 0
    host.pools[0][0, shared[1:], :, :, 0] = 56
    host.scales[1][0, shared] = 0
    host.pools[1][0, shared] = 0
    for slot, n in enumerate(tails):
        host.pools[0][0, own[slot], :, :n] = 0
        host.pools[0][0, own[slot], :, :n, 0] = 56
    q = torch.zeros(sequences, 1, kv_heads, size, device="cuda", dtype=DTYPE[dtype])
    q[..., 0] = 12.9 * math.log(2.0) / (0.25 * 56)
    cache = to_device(host)
    got = wide(cache.attend_shared(0, q, scale=1.0, least_bytes=0))
    cache.check_errors()
    score, info = float(q[0, 0, 0, 0]) * 0.25 * 56, torch.finfo(DTYPE[dtype])
    for slot, n in enumerate(tails):
        values = host.pools[1][0, own[slot], :, :n].astype(np.float64) * host.scales[1][0, own[slot], :, None, None]
        total = (prefix - 64 + n) + 64 * math.exp(-score)
        want, share = values.sum(1) / total, n / total  # (kv_heads, size)
        bound = 2 * WEIGHTS[dtype] * share * np.abs(values).max() + info.eps / 2 * np.abs(want) + info.tiny * info.eps
        assert (np.abs(want) > bound).any() and (np.abs(got[slot, 0] - want) <= bound).all()
