"""Pools of more than 2^32 bytes: pages at their end give the bits that the same
pages at the front of a small pool give, through append, attend, copies on
write and compaction."""

from __future__ import annotations

import pytest
import torch

from cuda_b200.paged import PagedCache

pytestmark = pytest.mark.gpu

PAGES, KV_HEADS, PAGE, SIZE = 16_500, 8, 256, 128  # 4.3e9 bytes of K, as many of V


def cache_of(pages: int, storage: torch.dtype) -> PagedCache:
    return PagedCache.allocate(layers=1, pages=pages, kv_heads=KV_HEADS, page_size=PAGE, head_size=SIZE, sequences=3,
                               pages_per_sequence=4, storage=storage, device=torch.device("cuda", 0))


@pytest.mark.parametrize("storage", [torch.int8, torch.float8_e4m3fn])
def test_pages_beyond_32_bits(storage):
    assert PAGES * KV_HEADS * PAGE * SIZE > 2 ** 32
    generator = torch.Generator("cuda").manual_seed(5)
    caches = [cache_of(12, storage), cache_of(PAGES, storage)]
    small, large = caches
    # both hand out pages from the end of their pools, in the same order
    for cache in caches:
        free, height = cache.split(cache.book)[3:]
        assert int(height) == cache.pages
        free.copy_(torch.arange(cache.pages, dtype=torch.int32, device="cuda"))
    lengths = torch.tensor([700, 300], dtype=torch.int32, device="cuda")
    slots = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(2, 700, KV_HEADS, SIZE, device="cuda", generator=generator) for _ in range(2))
    q = torch.randn(3, 1, 2 * KV_HEADS, SIZE, device="cuda", generator=generator)
    outputs = []
    for cache in caches:
        cache.extend(lengths, sequences=slots)
        cache.append(0, k, v, counts=lengths, sequences=slots)
        cache.fork(slots[:1], slots[:1] + 2)
        cache.extend(torch.ones(3, dtype=torch.int32, device="cuda"))  # slot 0's last page is copied first
        cache.append(0, k[:1, :1].expand(3, 1, KV_HEADS, SIZE), v[:1, :1].expand(3, 1, KV_HEADS, SIZE))
        before = cache.attend(0, q)
        table = cache.split(cache.book)[0]
        lowest = int(table[table >= 0].min())
        cache.compact()
        assert int(cache.split(cache.book)[0].max()) == 5 and cache.pages - lowest <= 7
        after = cache.attend(0, q)
        cache.check_errors()
        assert torch.equal(before, after)
        outputs.append(after)
    assert torch.equal(*outputs) and bool(torch.isfinite(outputs[0]).all()) and float(outputs[0].abs().max()) > 0
