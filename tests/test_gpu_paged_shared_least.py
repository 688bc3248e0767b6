"""attend_shared where the device decides whether shared keys are computed apart: from ``least_bytes``
of repeated reads on, counted over the sequences that take part and the whole pages that all of
them hold, in caches whose tables have room for more."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from cuda_b200 import _lib
from cuda_b200.paged import PagedCache
from paged_helpers import DTYPE, to_device
from test_gpu_paged_attention import compare, expected, queries
from test_gpu_paged_shared import family

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("storage, page, kv_heads, size, tokens", [("int8", 16, 2, 64, 1), ("e4m3", 64, 1, 128, 3),
                                                                  ("int8", 32, 3, 32, 5)])
@pytest.mark.parametrize("idle", [(), (0,), (2, 5)])
def test_the_border(dtype, storage, page, kv_heads, size, tokens, idle):
    rng = np.random.default_rng(page + len(idle))
    prefix, tails = 10 * page + 3, [tokens, tokens + 9, 2 * page, 40, tokens + 1, 70, tokens]
    host = family(rng, prefix, tails, kv_heads=kv_heads, head_size=size, page=page, storage=storage, room=50)
    cache = to_device(host)
    counts = [0 if b in idle else tokens for b in range(len(tails))]
    given = torch.tensor(counts, dtype=torch.int32, device="cuda")
    q = queries(rng, len(tails), tokens, 4 * kv_heads, size, dtype)

    def call(least_bytes):
        got = cache.attend_shared(0, q, counts=given, least_bytes=least_bytes)
        cache.check_errors()
        return got

    # ten whole pages are common to all; the first rows of a block see keys of their own from there on
    border = (len(tails) - len(idle) - 1) * 10 * page * kv_heads * size * 2
    apart, whole = call(0), cache.attend(0, q, counts=given)
    want = expected(host, q, counts, range(len(tails)), 1 / math.sqrt(size))
    compare(apart, want, host, dtype)
    compare(whole, want, host, dtype)
    if dtype == "f32":  # (so that equal bits say which way a call went)
        assert not torch.equal(apart, whole)
    assert torch.equal(call(border - 1), apart) and torch.equal(call(border), apart)
    assert torch.equal(call(border + 1), whole)
    assert torch.equal(call(border + page * kv_heads * size * 2), whole)


def test_the_border_follows_the_tables():
    """The same call before and after a sequence leaves the family, and while one that never belonged takes part."""
    rng = np.random.default_rng(8)
    host = family(rng, 320, [1, 1, 1, 1], kv_heads=2, head_size=64, page=16, room=30)
    q = queries(rng, 4, 1, 8, 64, "f32")
    cache = to_device(host)
    unit = 20 * 16 * 2 * 64 * 2  # a repeated read of the twenty pages
    ones = torch.ones(4, dtype=torch.int32, device="cuda")
    apart, whole = cache.attend_shared(0, q, least_bytes=0), cache.attend(0, q)
    assert not torch.equal(apart, whole)
    assert torch.equal(cache.attend_shared(0, q, least_bytes=3 * unit), apart)
    ones[3] = 0  # three are left: two repeated reads
    three = cache.attend_shared(0, q, counts=ones, least_bytes=2 * unit)
    assert torch.equal(three, cache.attend_shared(0, q, counts=ones, least_bytes=0))
    assert torch.equal(cache.attend_shared(0, q, counts=ones, least_bytes=2 * unit + 1), cache.attend(0, q, counts=ones))
    cache.release([3])
    cache.extend([0, 0, 0, 40])
    zeros = torch.zeros(1, 40, 2, 64, device="cuda")
    cache.append(0, zeros, zeros, sequences=[3])
    cache.check_errors()
    assert torch.equal(cache.attend_shared(0, q, least_bytes=1), cache.attend(0, q))  # nothing is common to all four
    assert torch.equal(cache.attend_shared(0, q, counts=ones, least_bytes=2 * unit), three)
    cache.check_errors()


def test_too_many_for_one_call():
    """What the kernel of the sequences' own keys cannot divide is refused before a kernel of the call runs."""
    cache = PagedCache.allocate(layers=1, pages=8, kv_heads=8, page_size=16, head_size=32, sequences=2,
                                pages_per_sequence=2 ** 16)
    slots = torch.zeros(65535, dtype=torch.int32, device="cuda")
    q = torch.zeros(65535, 1, 8, 32, device="cuda")
    for call in (dict(least_bytes=0), dict()):
        with pytest.raises(_lib.KernelError, match="too many"):
            cache.attend_shared(0, q, sequences=slots, **call)
    cache.check_errors()  # (a kernel would have found that slot 0 holds no token)


# heads and kv heads of 128, sequences, tokens, dtype; keys in common from which they are computed apart by
# themselves (None: at no length that is tried)
RULE = [(32, 8, 64, 1, "bf16", 1664), (32, 8, 64, 1, "f32", 1664), (32, 8, 16, 5, "f16", 7616), (32, 8, 8, 1, "bf16", 19712),
        (32, 8, 4, 1, "bf16", 98304), (32, 8, 3, 1, "bf16", None), (32, 8, 2, 1, "f32", None), (32, 1, 16, 1, "bf16", None),
        (32, 1, 64, 1, "bf16", 12928)]


@pytest.mark.parametrize("heads, kv_heads, batch, tokens, dtype, keys", RULE)
def test_the_rule_by_itself(heads, kv_heads, batch, tokens, dtype, keys):
    """Without least_bytes: 192 MB that all but three of the sequences would read, items for a 32nd of the SMs, and one
    page less is attend's, bit for bit."""
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the borders are those of 148 SMs")
    page, size = 64, 128
    most = (200_000 if keys is None else keys) // page * page
    cache = PagedCache.allocate(layers=1, pages=most // page + 2 * batch, kv_heads=kv_heads, page_size=page, head_size=size,
                                sequences=batch, pages_per_sequence=most // page + 3)
    gen = torch.Generator(device="cuda").manual_seed(keys or 1)
    cache.k_pages.copy_(torch.randint(-90, 91, cache.k_pages.shape, device="cuda", generator=gen, dtype=torch.int8))
    cache.v_pages.copy_(torch.randint(-90, 91, cache.v_pages.shape, device="cuda", generator=gen, dtype=torch.int8))
    cache.k_scale.fill_(0.01), cache.v_scale.fill_(0.02)
    q = torch.randn(batch, tokens, heads, size, device="cuda", generator=gen).to(DTYPE[dtype])
    for length in ([most] if keys is None else [most - page, most]):
        cache.release(list(range(batch)))
        cache.extend([length], sequences=[0])
        cache.fork([0] * (batch - 1), list(range(1, batch)))
        cache.extend([tokens] * batch)
        got, whole = cache.attend_shared(0, q), cache.attend(0, q)
        apart = cache.attend_shared(0, q, least_bytes=0)
        cache.check_errors()
        assert not torch.equal(apart, whole)  # (so that equal bits say which way a call went)
        assert torch.equal(got, apart if length == keys else whole)
