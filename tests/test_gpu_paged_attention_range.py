"""cb_paged_attention where value scales or weights lie far apart, against a float64 softmax.

Bound, from the formula: an output is sum w v / sum w.  An error e of the
weights (relative) moves it by at most 2 e max|v|, and where keys whose values
are zero hold most of the weight, by at most 2 e max|v| times the share f of
the others.  e is that of the other tests of this entry point: scores below 64
in base 2 of numbers held to 22 bits or more give 2^-16, weights rounded to 11
bits (16-bit types) 2^-11 more.  Weights are rounded against the largest of
their step of 2048 / head_size keys, whose low parts end 2^-30 below it, so the
keys of the step that holds a dominant one may be off by that each.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import paged as plain
from paged_helpers import DTYPE, filled, to_device, wide

pytestmark = pytest.mark.gpu

WEIGHTS = {"f32": 2.0 ** -16, "bf16": 2.0 ** -16 + 2.0 ** -11, "f16": 2.0 ** -16 + 2.0 ** -11}


def compare(got, want, largest, dtype, share=1.0, lost=0.0):
    """``largest``: of the values; ``share``: of the weights that count (broadcasts); ``lost``: absolute, of largest."""
    info = torch.finfo(DTYPE[dtype])
    bound = (2 * WEIGHTS[dtype] * share + lost) * largest + info.eps / 2 * np.abs(want) + info.tiny * info.eps / 2
    got = wide(got)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), float(np.max(np.abs(got - want) / bound))


def expected(host, q, slots, scale):
    return np.stack([plain.attend(wide(q[b]), host.read(0, 0, slot), host.read(0, 1, slot), scale)
                     for b, slot in enumerate(slots)])


def magnitude(host):
    return max(float(np.abs(host.read(0, 1, s)).max()) for s in range(len(host.lengths)))


# (tokens, heads, kv_heads): rows of a kv head in one set of eight, two, three, four, and two blocks of three
ROWS = [(1, 4, 1), (3, 8, 2), (5, 4, 1), (7, 4, 1), (10, 4, 1)]


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("storage, size, page", [("int8", 128, 64), ("e4m3", 64, 16), ("int8", 32, 32)])
@pytest.mark.parametrize("tokens, heads, kv_heads", ROWS)
@pytest.mark.parametrize("exponent", [-5, -12, -20, -26, -100])
def test_pages_of_zero_values(dtype, storage, size, page, tokens, heads, kv_heads, exponent):
    """Zero value scales first, between, last, all but one and everywhere: their keys count, their values do not."""
    rng = np.random.default_rng(tokens - exponent)
    # the first page of every warp, some between, the last pages, all but one, and all
    kinds = [lambda n: np.arange(n) < n - 1 - n // 3, lambda n: np.arange(n) % 3 == 1, lambda n: np.arange(n) >= n // 2,
             lambda n: np.arange(n) != n // 2, lambda n: np.arange(n) >= 0]
    lengths = [12 * page - 3] * len(kinds)
    host = filled(rng, lengths, kv_heads=kv_heads, head_size=size, storage=storage, page=page)
    host.scales[1] = (rng.uniform(1, 2, host.scales[1].shape) * 2.0 ** exponent).astype(np.float32)
    for slot, kind in enumerate(kinds):
        pages = host.table[slot, :12][kind(12)]
        host.scales[1][0, pages] = 0
        host.pools[1][0, pages] = 0
    q = torch.from_numpy(rng.normal(0, 1, (len(kinds), tokens, heads, size)).astype(np.float32)).cuda().to(DTYPE[dtype])
    cache = to_device(host)
    got = cache.attend(0, q)
    cache.check_errors()
    compare(got, expected(host, q, range(len(kinds)), 1 / math.sqrt(size)), magnitude(host), dtype)


def test_appended_zeros_before_small_values():
    """The cache's own append stores a scale of zero for rows of zeros; small values follow."""
    from cuda_b200.paged import PagedCache

    cache = PagedCache.allocate(layers=1, pages=8, kv_heads=1, page_size=64, head_size=128, sequences=1,
                                pages_per_sequence=8)
    rng = np.random.default_rng(0)
    k = torch.from_numpy(rng.normal(0, 1, (1, 384, 1, 128)).astype(np.float32)).cuda()
    v = 2.0 ** -20 * k.flip(1)
    v[:, :64] = 0
    cache.extend([384])
    cache.append(0, k, v)
    q = torch.from_numpy(rng.normal(0, 1, (1, 1, 4, 128)).astype(np.float32)).cuda()
    host = filled(rng, [384], kv_heads=1, head_size=128, page=64, spare=2, garbage=False)
    host.table = cache.table.cpu().numpy()
    host.pools = [p.cpu().numpy() for p in (cache.k_pages, cache.v_pages)]
    host.scales = [s.cpu().numpy() for s in (cache.k_scale, cache.v_scale)]
    assert host.scales[1][0, host.table[0, 0], 0] == 0
    got = cache.attend(0, q)
    cache.check_errors()
    compare(got, expected(host, q, [0], 1 / math.sqrt(128)), magnitude(host), "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("exponents", [[-108], [118], [-100, 20], [20, -100], [-109, -109, 110], [-60, 60, 0, -60],
                                       [0, -80], [-126, -3]])
@pytest.mark.parametrize("tokens, heads", [(1, 4), (5, 4)])
def test_scales_of_the_whole_range(dtype, exponents, tokens, heads):
    """Pages whose value scales are at the ends of the range, or change by up to 2^219 from one to the next."""
    rng = np.random.default_rng(len(exponents))
    host = filled(rng, [6000, 77], kv_heads=1, head_size=128, page=64)
    for slot in range(2):
        held = host.table[slot, :host.held(int(host.lengths[slot]))]
        host.scales[1][0, held, 0] = 2.0 ** np.array([exponents[i // 8 % len(exponents)] for i in range(len(held))])
    q = torch.from_numpy(rng.normal(0, 1, (2, tokens, heads, 128)).astype(np.float32)).cuda().to(DTYPE[dtype])
    cache = to_device(host)
    got = cache.attend(0, q)
    cache.check_errors()
    want = expected(host, q, range(2), 1 / math.sqrt(128))
    for b in range(2):
        compare(got[b], want[b], float(np.abs(host.read(0, 1, b)).max()), dtype)


def test_a_large_scale_that_earlier_rows_do_not_see():
    """The last page's values are 2^127 times the others'; the first tokens of the block end before it."""
    rng = np.random.default_rng(1)
    host = filled(rng, [131], kv_heads=1, head_size=128, page=16)
    host.scales[1][0, host.table[0, :8], 0] = 2.0 ** -100
    host.scales[1][0, host.table[0, 8], 0] = 2.0 ** 27
    q = torch.from_numpy(rng.normal(0, 1, (1, 5, 4, 128)).astype(np.float32)).cuda()
    want, got = expected(host, q, [0], 0.1)[0], to_device(host).attend(0, q, scale=0.1)[0]
    compare(got[:2], want[:2], 127 * 2.0 ** -100, "f32")
    compare(got[2:], want[2:], 127 * 2.0 ** 27, "f32")


def scored(rng, lengths, codes, size, page, dtype, tokens, heads, scale_exponent=-6):
    """A cache and queries whose scores are codes / 4 (natural logarithm); sinks (codes above 16) have zero values."""
    host = filled(rng, lengths, kv_heads=1, head_size=size, page=page, spare=0, garbage=False)
    host.scales[0][:] = 0.25
    host.scales[1][:] = 2.0 ** scale_exponent
    host.pools[0][:] = 0
    for slot, length in enumerate(lengths):
        at = np.arange(length)
        pages, rows = host.table[slot, at // page], at % page
        host.pools[0][0, pages, 0, rows, 0] = codes[slot]
        values = rng.integers(64, 128, (length, size)).astype(np.int8)  # one sign: nothing cancels
        values[codes[slot] > 16] = 0
        host.pools[1][0, pages, 0, rows] = values
    q = torch.zeros(len(lengths), tokens, heads, size, device="cuda", dtype=DTYPE[dtype])
    q[..., 0] = 1.0
    return host, q


def shares(codes, tokens):
    """The weights' share that is not the sinks', for each token of a block."""
    out = []
    for t in range(tokens):
        seen = codes[:len(codes) - tokens + t + 1].astype(np.float64) / 4
        w = np.exp(seen - seen.max())
        out.append(w[codes[:len(seen)] <= 16].sum() / w.sum())
    return np.array(out)[:, None, None]


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("size, page, tokens, heads", [(128, 64, 1, 4), (64, 16, 1, 8), (32, 32, 1, 1), (128, 32, 3, 4),
                                                       (64, 64, 5, 4), (128, 16, 8, 4), (32, 128, 8, 4)])
@pytest.mark.parametrize("gap", [40, 56, 64, 68, 80, 100])
def test_one_key_takes_the_weight(dtype, size, page, tokens, heads, gap):
    """A dominant key of zero values, 10 to 25 nats above 8,192 others that carry the result: first, amid them, last."""
    rng = np.random.default_rng(gap)
    n = 8192
    codes = [rng.integers(-2, 3, n) for _ in range(4)]
    codes[0][:] = 0                       # equal weights: their roundings add up
    for slot, place in enumerate([0, 5, n // 2, n - tokens]):
        codes[slot][place] = gap
    host, q = scored(rng, [n] * 4, codes, size, page, dtype, tokens, heads)
    cache = to_device(host)
    got = cache.attend(0, q, scale=1.0)
    cache.check_errors()
    want = expected(host, q, range(4), 1.0)
    for b in range(4):
        compare(got[b], want[b], 127 * 2.0 ** -6, dtype, shares(codes[b], tokens), 2.0 ** -30 * 2048 / size)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("size, tokens, heads", [(128, 1, 4), (64, 3, 4), (32, 5, 4)])
def test_scores_that_swing(dtype, size, tokens, heads):
    """Runs of keys whose scores jump up and down by up to 20 nats, in runs around a step's keys."""
    rng = np.random.default_rng(size)
    codes = []
    for run in (7, 16, 64, 300):
        codes.append(np.repeat(rng.integers(-64, 17, 5000 // run + 1), run)[:5000])
    host, q = scored(rng, [5000] * 4, codes, size, 64, dtype, tokens, heads)
    cache = to_device(host)
    got = cache.attend(0, q, scale=1.0)
    cache.check_errors()
    compare(got, expected(host, q, range(4), 1.0), 127 * 2.0 ** -6, dtype)


def test_zero_values_hold_the_weight():
    """Whole pages of zero values, up to 40 nats above the pages that carry the result, before and behind them."""
    rng = np.random.default_rng(3)
    for gap in (20, 60, 100, 127):
        codes = [rng.integers(-1, 2, 2048) for _ in range(3)]
        codes[0][:256] = gap
        codes[1][1024:1280] = gap
        codes[2][-256:] = gap
        host, q = scored(rng, [2048] * 3, codes, 128, 64, "f32", 1, 4)
        for slot in range(3):
            for column in range(32):
                page = host.table[slot, column]
                if not host.pools[1][0, page].any():
                    host.scales[1][0, page] = 0
        got, want = to_device(host).attend(0, q, scale=1.0), expected(host, q, range(3), 1.0)
        for b in range(3):
            compare(got[b], want[b], 127 * 2.0 ** -6, "f32", shares(codes[b], 1))
