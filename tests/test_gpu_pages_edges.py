"""Page operations at sizes and books where their kernels' loops and checks could go wrong."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from paged_helpers import filled, same_book, same_pools, to_device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots, columns", [(31, 33), (32, 33), (33, 47), (45, 129), (64, 128), (65, 127), (7, 1171)])
def test_entries_that_end_inside_a_warp(slots, columns):
    """Clusters of 1 to 8 blocks over entry counts that leave lanes of a warp with unlike numbers of them."""
    rng = np.random.default_rng(slots)
    lengths = [int(n) for n in rng.integers(0, 16 * columns + 1, slots)]
    host = filled(rng, lengths, kv_heads=1, head_size=32, page=16, spare=columns, columns=columns, garbage=False)
    cache = to_device(host)
    counts = [int(rng.integers(0, n + 1)) for n in lengths]
    cache.truncate(counts)
    host.truncate(counts, range(slots))
    cache.check_errors()
    same_book(cache, host)
    gone = rng.permutation(slots)[:slots // 2 + 1].tolist()
    cache.release(gone)
    host.truncate(None, gone)
    cache.check_errors()
    same_book(cache, host)
    cache.compact()
    host.compact()
    cache.check_errors()
    same_book(cache, host)
    same_pools(cache, host)


def refused(cache, call):
    """``call`` raises IndexError at the check and leaves book and pools as they are."""
    whole = (cache.book, cache.k_pages, cache.k_scale.view(torch.int32))  # (bits: what no slot holds is NaN)
    before = [t.clone() for t in whole]
    call()
    with pytest.raises(IndexError):
        cache.check_errors()
    for now, was in zip(whole, before):
        assert torch.equal(now, was)


@pytest.mark.parametrize("bad", ["beyond", "negative", "held", "twice"])
@pytest.mark.parametrize("depth", [0, 2])
def test_extend_checks_the_free_stack_first(bad, depth):
    """An id on the stack that is no free page: as a slot's next page, and as the target of a copy on write."""
    host = filled(np.random.default_rng(5), [20, 33, 0, 0], spare=8, columns=4)
    cache = to_device(host)
    cache.fork([0], [3])  # slot 0's and 3's open page is shared: the first of them to grow copies it
    height = int(cache.height)
    cache.free[height - 1 - depth] = {"beyond": cache.pages, "negative": -1, "held": int(cache.table[1, 0]),
                                      "twice": int(cache.free[height - 2])}[bad]
    refused(cache, lambda: cache.extend([1, 20, 5, 1]))
    cache.extend([1, 0, 0, 0][:1 + depth // 2] if depth else [0])  # what takes no page from there goes on
    cache.check_errors()


@pytest.mark.parametrize("height", [-1, -7, "beyond"])
def test_heights_outside_the_stack(height):
    host = filled(np.random.default_rng(6), [40, 33, 0, 0], spare=8, columns=4)
    cache = to_device(host)
    cache.height.fill_(cache.pages + 1 if height == "beyond" else height)
    refused(cache, lambda: cache.extend([30, 1]))
    refused(cache, lambda: cache.truncate([17, 3]))
    refused(cache, lambda: cache.release([0, 1]))


@pytest.mark.parametrize("page", ["beyond", -1, -5])
def test_fork_checks_the_parents_pages_first(page):
    """A row that names a page outside the pool: neither the child's row nor a count changes."""
    host = filled(np.random.default_rng(7), [40, 33, 0, 0], spare=8, columns=4)
    cache = to_device(host)
    cache.table[0, 2] = cache.pages if page == "beyond" else page
    refused(cache, lambda: cache.fork([0], [2]))


def test_fork_decides_for_each_pair():
    """A pair that is refused leaves the others of the call as they are."""
    host = filled(np.random.default_rng(8), [40, 33, 0, 0, 0], spare=8, columns=4)
    for parents, children in (([0, 1], [1, 3]), ([9, 1], [2, 3]), ([1, 0], [3, -1])):
        cache = to_device(host)
        cache.fork(parents, children)
        with pytest.raises(IndexError):
            cache.check_errors()
        want = to_device(host)
        want.fork([1], [3])
        want.check_errors()
        assert torch.equal(cache.book, want.book)
