"""cb_paged_attention at the ends of its integers: the division of the work, positions near 2^31."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from cuda_b200 import _lib
from cuda_b200.paged import PagedCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("units, fits", [(2 ** 31 - 400, False), (2 ** 31 - 32768, True), (2 ** 31 + 32767, False)])
def test_work_near_the_limit(units, fits):
    """Sizes alone (no launch): units of work whose rounding up to the blocks would pass 2^31 have no scratch."""
    # one row of one kv head of 128: a slot has columns / 4 tiles and 4 units more
    for batch in range(65535, 1, -1):
        if units % batch == 0:
            break
    per = units // batch
    cache = _lib.PagedCacheArgs(k_pages=16, v_pages=16, k_scale=16, v_scale=16, storage=_lib.I8, kv_heads=1, page=16,
                                head_size=128, pages=8, table=16, lengths=16, slots=batch, columns=4 * (per - 4))
    a = _lib.PagedAttentionArgs(cache=cache, q=16, out=16, dtype=_lib.F32, batch=batch, tokens=1, heads=1, scale=1.0)
    sms = ctypes.c_int()
    _lib.call("cb_sm_count", ctypes.byref(sms))
    assert batch * per == units and 3 * sms.value < 32768
    assert (_lib.load().cb_paged_attention_scratch(ctypes.byref(a)) > 0) == fits


def test_a_sequence_that_ends_at_the_last_position():
    """2^31 - 19 keys on four pages: the new tokens land in the last columns, and an earlier one does not see a later.

    Column i holds page 0 but for the last three.  The last token's key is 20
    nats above the others and the one before it 10, so that its weight in the
    earlier tokens' rows, or the tail missing, would show.  A lane adds up some
    80,000 weights and a product 20,000 steps in float32, each rounded to 2^-25
    (2^-24) of the sum: 2.4e-3 + 1.2e-3, of values below 2.
    """
    columns, page, size = 2 ** 27 - 1, 16, 32
    cache = PagedCache.allocate(layers=1, pages=4, kv_heads=1, page_size=page, head_size=size, sequences=1,
                                pages_per_sequence=columns)
    length, tokens = columns * page - 3, 5
    cache.table[0] = 0
    cache.table[0, -3:] = torch.tensor([1, 2, 3], dtype=torch.int32)
    cache.lengths[0] = length
    rng = np.random.default_rng(0)
    cache.k_pages[0, :, 0, :, 0] = 0
    codes = torch.from_numpy(rng.integers(-127, 128, (4, page, size)).astype(np.int8)).cuda()
    cache.v_pages[0, :, 0] = codes
    cache.k_scale.fill_(1 / 4)
    cache.v_scale.fill_(1 / 64)
    before = cache.book[-16:].clone()
    k = torch.zeros(1, 300, 1, size, device="cuda")
    k[0, 3, 0, 0], k[0, 4, 0, 0] = 10.0, 127 / 4
    v = torch.from_numpy(rng.integers(-127, 128, (1, 300, 1, size)).astype(np.float32)).cuda() / 64
    v[0, :, 0, 0] = 127 / 64  # the scale of both pages stays as it is
    cache.append(0, k, v, counts=[tokens])  # 300 rows would reach past the last column
    cache.check_errors()
    assert torch.equal(cache.book[-16:], before)
    q = torch.zeros(1, tokens, 1, size, device="cuda")
    q[..., 0] = 20 / (127 / 4)
    got = cache.attend(0, q, scale=1.0)[0, :, 0].double().cpu().numpy()
    cache.check_errors()
    # page 0 `columns - 3` times, then the rows of pages 1 to 3
    pools = [x[0, :, 0].double().cpu().numpy() * s[0, :, 0].double().cpu().numpy()[:, None, None]
             for x, s in ((cache.k_pages, cache.k_scale), (cache.v_pages, cache.v_scale))]
    keys, values = (p.reshape(64, size) for p in pools)
    times = np.r_[np.full(16, columns - 3.0), np.ones(48)]
    for t in range(tokens):
        seen = 16 + 48 - 3 - tokens + t + 1
        w = times[:seen] * np.exp(keys[:seen, 0] * (20 / (127 / 4)))
        want = w @ values[:seen] / w.sum()
        assert np.abs(got[t] - want).max() <= 2.0 ** -7, t
    assert np.abs(got[4] - got[2]).max() > 0.1  # (the last key does carry weight)
