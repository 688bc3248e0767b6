"""Checks of the paged cache's host side on the device."""

from __future__ import annotations

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from cuda_b200 import _lib, speculative
from cuda_b200.paged import PagedCache
from paged_helpers import filled, to_device

pytestmark = pytest.mark.gpu


def test_derivatives_are_refused():
    cache = to_device(filled(np.random.default_rng(0), [20, 20]))
    q, rows = torch.randn(2, 1, 4, 64, device="cuda"), torch.randn(2, 1, 2, 64, device="cuda")
    p = torch.full((1, 2, 4), 0.25, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(ValueError):
            cache.attend(0, dual)
        with pytest.raises(ValueError):
            cache.append(0, rows, forward_ad.make_dual(rows, rows))
        with pytest.raises(ValueError):
            tokens, uniforms = (torch.zeros(1, n, dtype=t, device="cuda") for n, t in ((1, torch.int64),
                                                                                     (2, torch.float64)))
            speculative.verify(forward_ad.make_dual(p, p), p[:, :1], tokens, uniforms)
    out = torch.zeros_like(q)
    for bad in (out.clone().requires_grad_(), out.clone().requires_grad_() * 1):
        with pytest.raises(ValueError):
            cache.attend(0, q, out=bad)
    with torch.no_grad():
        cache.attend(0, q, out=out.clone().requires_grad_())


def test_a_kept_activation_that_is_overwritten_is_noticed():
    """``out`` counts as written in place for a backward pass that kept it."""
    cache = to_device(filled(np.random.default_rng(0), [20, 20]))
    q = torch.randn(2, 1, 4, 64, device="cuda")
    out, weight = cache.attend(0, q), torch.ones(64, device="cuda", requires_grad=True)
    loss = (out * weight).sum()  # keeps out
    cache.attend(0, 2 * q, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        cache.attend(0, q, out=torch.empty_like(q))


def test_lists_are_refused_in_a_capture():
    """A host list would be copied by the host; the same step with tensors is captured and replayed."""
    cache = to_device(filled(np.random.default_rng(0), [20, 20], spare=8))
    rows, q = torch.randn(2, 1, 2, 64, device="cuda"), torch.randn(2, 1, 4, 64, device="cuda")
    ones, slots = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([1, 1], [0, 1]))
    out, graph = torch.empty_like(q), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: cache.extend([1, 1]), lambda: cache.append(0, rows, rows, counts=(1, 1)),
                     lambda: cache.attend(0, q, sequences=[0, 1]), lambda: cache.truncate([1, 1]),
                     lambda: cache.release([0]), lambda: cache.fork([0], [1]), lambda: cache.copy_pages([0], [1])):
            with pytest.raises(ValueError, match="captured"):
                call()
        cache.extend(ones, sequences=slots)
        cache.append(0, rows, rows, sequences=slots)
        cache.attend(0, q, sequences=slots, out=out)
        cache.truncate(ones, sequences=slots)
    for _ in range(2):
        graph.replay()
    cache.check_errors()
    assert cache.lengths.tolist() == [20, 20]
    cache.extend([1, 1])
    cache.append(0, rows, rows)
    assert torch.equal(out, cache.attend(0, q))


def test_addresses_off_16_bytes_are_value_errors():
    cache = to_device(filled(np.random.default_rng(0), [20, 20]))
    q = torch.randn(2, 1, 4, 64, device="cuda")
    store = torch.zeros(2 * 4 * 64 + 1, device="cuda")
    with pytest.raises(ValueError, match="16 bytes"):
        cache.attend(0, q, out=store[1:].view(2, 1, 4, 64))
    pools = [torch.zeros(cache.k_pages.numel() + 8, dtype=torch.int8, device="cuda")[8:].view(cache.k_pages.shape)
             for _ in range(2)]
    for k, v in ((pools[0], cache.v_pages), (cache.k_pages, pools[1])):
        with pytest.raises(ValueError, match="16 bytes"):
            PagedCache(k, v, cache.k_scale, cache.v_scale, cache.book, sequences=cache.sequences,
                       pages_per_sequence=cache.pages_per_sequence)


def test_too_much_work_for_one_call_says_so():
    """Lengths that a table of this many columns could hold, for this many rows: refused before any launch."""
    cache = PagedCache.allocate(layers=1, pages=1, kv_heads=1, page_size=16, head_size=128, sequences=1,
                                pages_per_sequence=131_072)
    q = torch.zeros(65_535, 1, 1, 128, device="cuda")
    with pytest.raises(_lib.KernelError, match="too many for one call"):
        cache.attend(0, q, sequences=torch.zeros(65_535, dtype=torch.int32, device="cuda"))
