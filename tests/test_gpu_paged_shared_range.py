"""cb_paged_attention_shared where value scales or weights lie far apart, against a float64 softmax.

The bounds are those of test_gpu_paged_attention_range: an error e of the weights
moves an output by at most 2 e max|v|, and by at most 2 e max|v| times the share f
of the others where keys whose values are zero hold most of the weight.  In shared
keys a weight is rounded to 2^-25 of what the largest of its tile of 64 keys is at
least: 2^-8 with one part (16-bit types), 2^-2 with two (float32), where another
tile's weight is the reference, and 2^2 where its own is; so e gains 2^-17 or 2^-23
of the tile's largest weight.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from paged_helpers import DTYPE, to_device, wide
from test_gpu_paged_attention_range import WEIGHTS, compare, expected, magnitude
from test_gpu_paged_shared import family, queries

pytestmark = pytest.mark.gpu


def run(host, q, scale=None):
    cache = to_device(host)
    got = cache.attend_shared(0, q, scale=scale, least_bytes=0)
    cache.check_errors()
    return got


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("storage, size, page", [("int8", 128, 64), ("e4m3", 64, 16), ("int8", 32, 32)])
@pytest.mark.parametrize("heads, kv_heads, sequences", [(4, 1, 2), (8, 2, 3), (8, 1, 40)])
@pytest.mark.parametrize("exponent", [-5, -26, -100, 60])
def test_pages_of_zero_values(dtype, storage, size, page, heads, kv_heads, sequences, exponent):
    """Zero value scales first, between, last, all but one and everywhere: their keys count, their values do not."""
    if exponent > 4 and dtype == "f16":
        exponent = 4  # (what float16 outputs hold)
    rng = np.random.default_rng(sequences + abs(exponent))
    n = 12
    for kind in (np.arange(n) < 7, np.arange(n) % 3 == 1, np.arange(n) >= 5, np.arange(n) != 6, np.arange(n) >= 0):
        host = family(rng, n * page, [3 + b % 5 for b in range(sequences)], kv_heads=kv_heads, head_size=size,
                      page=page, storage=storage)
        held = np.isfinite(host.scales[1])
        host.scales[1] = np.where(held, rng.uniform(1, 2, held.shape) * 2.0 ** exponent, np.nan).astype(np.float32)
        pages = host.table[0, :n][kind]
        host.scales[1][0, pages] = 0
        host.pools[1][0, pages] = 0
        q = queries(rng, sequences, 1, heads, size, dtype) * 0.5
        compare(run(host, q), expected(host, q, range(sequences), 1 / math.sqrt(size)), magnitude(host), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("exponents", [[-108], [118], [-100, 20], [20, -100], [-109, -109, 110], [-60, 60, 0, -60],
                                       [0, -80], [-126, -3], [90, -20, -20, -20]])
@pytest.mark.parametrize("sequences", [2, 40])
def test_scales_of_the_whole_range(dtype, exponents, sequences):
    """Pages whose value scales are at the ends of the range, or change by up to 2^219 from one to the next."""
    rng = np.random.default_rng(len(exponents))
    host = family(rng, 6016, [3 + b % 7 for b in range(sequences)], kv_heads=1, head_size=128, page=64)
    for slot in range(sequences):
        held = host.table[slot, :host.held(int(host.lengths[slot]))]
        host.scales[1][0, held, 0] = 2.0 ** np.array([float(exponents[i // 8 % len(exponents)])
                                                      for i in range(len(held))])
    q = queries(rng, sequences, 1, 8, 128, dtype) * 0.5
    got, want = run(host, q), expected(host, q, range(sequences), 1 / math.sqrt(128))
    compare(got, want, magnitude(host), dtype)


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("above", [5, 12, 20, 40, 90])
@pytest.mark.parametrize("where", [0, 700, 1279])
def test_a_heavy_key_without_a_value(dtype, above, where):
    """One key outweighs each of the others by 2^above and has a value of zero: the others are the result."""
    rng = np.random.default_rng(above + where)
    sequences, size, prefix = 3, 64, 1280
    host = family(rng, prefix, [1, 5, 9], kv_heads=1, head_size=size, page=64)
    host.scales[0][np.isfinite(host.scales[0])] = 0.25
    host.scales[1][np.isfinite(host.scales[1])] = 2.0 ** -6
    for slot in range(sequences):
        for at in range(host.held(int(host.lengths[slot]))):
            page = int(host.table[slot, at])
            rows = min(64, int(host.lengths[slot]) - 64 * at)
            host.pools[0][0, page, 0, :rows] = 0
            host.pools[0][0, page, 0, :rows, 0] = rng.integers(-4, 5, rows)
            host.pools[1][0, page, 0, :rows] = rng.integers(64, 128, (rows, size))  # one sign: nothing cancels
    page, row = int(host.table[0, where // 64]), where % 64
    host.pools[0][0, page, 0, row, 0] = 127
    host.pools[1][0, page, 0, row] = 0
    q = torch.zeros(sequences, 1, 4, size, device="cuda", dtype=DTYPE[dtype])
    q[..., 0] = above * math.log(2.0) / (0.25 * 127)
    got, want = run(host, q, scale=1.0), expected(host, q, range(sequences), 1.0)
    score = 0.25 * float(q[0, 0, 0, 0])
    weight = math.exp(127 * score)
    share = prefix * math.exp(4 * score) / (weight + prefix * math.exp(-4 * score))  # of the others, at most
    # its own tile: 64 keys, each off by 2^-25 of 2^-2 of the heavy one; the others as the module's text says
    part = 2.0 ** -23 if dtype == "f32" else 2.0 ** -17
    lost = 64 * 2.0 ** -27 + 2 * part * min(share, 1.0) * math.exp(8 * score)
    compare(got, want, magnitude(host), dtype, min(share, 1.0), lost)
    assert WEIGHTS["bf16"] > WEIGHTS["f32"] and np.isfinite(wide(got)).all()
