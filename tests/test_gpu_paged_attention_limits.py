"""cb_paged_attention at the ends of its integers: the division of the work, positions near 2^31."""

from __future__ import annotations

import ctypes

import pytest

from cuda_b200 import _lib

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
