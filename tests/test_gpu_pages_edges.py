"""Page operations at sizes and books where their kernels' loops and checks could go wrong."""

from __future__ import annotations

import numpy as np
import pytest

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
