"""cb_pages_*: book and pools equal the rules applied slot after slot (whole numbers and moved bytes)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as plain
from paged_helpers import filled, same_book, same_pools, to_device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(6))
def test_random_programs(seed):
    """Random steps of a scheduler; every page is held or free after each."""
    rng = np.random.default_rng(seed)
    page = int(rng.choice([16, 32]))
    host = plain.Cache(2, 200, 2, page, 32, 24, 9)
    for array in host.pools:
        array[:] = rng.integers(-127, 128, array.shape)
    for array in host.scales:
        array[:] = rng.uniform(0.1, 1, array.shape)
    cache = to_device(host)
    for _ in range(40):
        busy = [s for s in range(24) if host.lengths[s]]
        empty = [s for s in range(24) if not host.lengths[s]]
        what = rng.choice(["extend", "extend", "fork", "truncate", "release", "compact", "copy"])
        if what == "extend":
            slots = rng.permutation(24)[:rng.integers(1, 25)].tolist()
            counts = [int(min(rng.integers(0, 40), 9 * page - host.lengths[s])) for s in slots]
            if sum(-(-c // page) + 1 for c in counts) > len(host.free):
                continue
            cache.extend(counts, sequences=slots)
            host.extend(counts, slots)
        elif what == "fork" and busy and empty:
            children = rng.permutation(empty)[:rng.integers(1, len(empty) + 1)].tolist()
            parents = rng.choice(busy, len(children)).tolist()
            cache.fork(parents, children)
            host.fork(parents, children)
        elif what == "truncate" and busy:
            counts = [int(rng.integers(0, host.lengths[s] + 1)) for s in busy]
            cache.truncate(counts, sequences=busy)
            host.truncate(counts, busy)
        elif what == "release" and busy:
            slots = rng.permutation(busy)[:rng.integers(1, len(busy) + 1)].tolist()
            cache.release(slots)
            host.truncate(None, slots)
        elif what == "compact":
            cache.compact()
            host.compact()
        elif what == "copy":
            pair = rng.permutation(200)[:6]
            cache.copy_pages(pair[:3].tolist(), pair[3:].tolist())
            for source, target in zip(pair[:3], pair[3:]):
                host.copy_page(int(source), int(target))
        cache.check_errors()
        same_book(cache, host)
        same_pools(cache, host)
        assert (host.refs > 0).sum() + len(host.free) == 200
        assert all(host.refs[p] == (host.table == p).sum() for p in range(200))


def test_many_entries():
    """More entries and pages than one block has threads; shared prefixes dropped in one call."""
    rng = np.random.default_rng(1)
    host = filled(rng, [1600, 1595] + [0] * 60, kv_heads=1, head_size=32, page=16, spare=5000, columns=110,
                  garbage=False)
    cache = to_device(host)
    children = list(range(2, 62))
    parents = [s % 2 for s in children]
    counts = [int(rng.integers(0, 100)) for _ in range(62)]
    for target, n in ((cache, None), (host, None)):
        target.fork(parents, children)
        target.extend(counts)
    cache.check_errors()
    same_book(cache, host)
    same_pools(cache, host)
    gone = rng.permutation(62)[:45].tolist()
    cache.release(gone)
    host.truncate(None, gone)
    same_book(cache, host)
    cache.compact()
    host.compact()
    cache.check_errors()
    same_book(cache, host)
    same_pools(cache, host)


def test_extend_is_undone_by_release():
    host = filled(np.random.default_rng(2), [33, 0, 0, 0], spare=20, columns=8)
    cache = to_device(host)
    before = cache.book.clone()
    cache.fork([0, 0, 0], [1, 2, 3])
    cache.extend([0, 5, 40, 1], sequences=[0, 1, 2, 3])
    cache.release([1, 2, 3])
    cache.check_errors()
    assert torch.equal(cache.book, before)


def test_room_is_all_or_nothing():
    host = filled(np.random.default_rng(3), [30, 30, 0], spare=2, columns=4)
    cache = to_device(host)
    before = cache.book.clone()
    for counts in ([3, 3, 1], [40, 0, 0], [0, 0, 2 ** 31 - 1]):  # pages; columns; far beyond both
        cache.extend(counts)
        with pytest.raises(MemoryError):
            cache.check_errors()
        assert torch.equal(cache.book, before)
    cache.extend([3, 2, 1])  # the last two pages
    host.extend([3, 2, 1])
    cache.check_errors()
    same_book(cache, host)


def test_calls_that_contradict_the_book():
    """Nothing changes, and the flag is set."""
    host = filled(np.random.default_rng(4), [30, 30, 0, 0], spare=8)
    cache = to_device(host)
    before = cache.book.clone()
    calls = [lambda: cache.extend([-1]), lambda: cache.extend([1], sequences=[4]),
             lambda: cache.extend([1, 1], sequences=[1, 1]), lambda: cache.truncate([31]),
             lambda: cache.truncate([-1]), lambda: cache.release([0, 0]), lambda: cache.release([-1]),
             lambda: cache.fork([0], [1]), lambda: cache.fork([0], [0]), lambda: cache.fork([0, 1], [2, 2]),
             lambda: cache.fork([4], [2])]
    for call in calls:
        call()
        with pytest.raises(IndexError):
            cache.check_errors()
        assert torch.equal(cache.book, before)
    pools = cache.k_pages.clone()
    cache.copy_pages([0, 1], [cache.pages, -1])
    with pytest.raises(IndexError):
        cache.check_errors()
    assert torch.equal(cache.k_pages, pools)
    cache.release([2, 3])  # empty slots are fine
    cache.extend([0, 0, 0, 0])
    cache.check_errors()
    assert torch.equal(cache.book, before)
    for arguments in (dict(parents=[0], children=[1, 2]), dict(parents=[0] * 5, children=[1] * 5)):
        with pytest.raises(ValueError):
            cache.fork(**arguments)
    with pytest.raises(ValueError):
        cache.extend([1] * 5)
    with pytest.raises(TypeError):
        cache.extend(torch.ones(2, device="cuda"))


def test_allocated_cache_is_empty():
    from cuda_b200.paged import PagedCache

    for storage in (torch.int8, torch.float8_e4m3fn):
        cache = PagedCache.allocate(layers=2, pages=5, kv_heads=1, page_size=32, head_size=64, sequences=3,
                                    pages_per_sequence=2, storage=storage)
        assert cache.k_pages.dtype == storage and int(cache.height) == 5 and not cache.refs.any()
        cache.extend([33, 1])
        cache.check_errors()
        assert cache.table.tolist() == [[0, 1], [2, -1], [-1, -1]]
    with pytest.raises(ValueError):
        PagedCache.allocate(layers=1, pages=5, kv_heads=1, page_size=24, head_size=64, sequences=3,
                            pages_per_sequence=2)
    with pytest.raises(ValueError):
        PagedCache.allocate(layers=1, pages=5, kv_heads=1, page_size=16, head_size=96, sequences=3,
                            pages_per_sequence=2)
