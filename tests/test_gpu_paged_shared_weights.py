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
