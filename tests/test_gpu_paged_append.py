"""cb_paged_append: codes and scales equal the rule in float32 bit for bit, and the
stored values are within half a step of the given ones."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as plain
from paged_helpers import DTYPE, filled, same_pools, to_device, wide

pytestmark = pytest.mark.gpu


def appended(host, rows, counts, slots):
    for which in range(2):
        for b, slot in enumerate(slots):
            host.append(0, which, wide(rows[which][b]).astype(np.float32), slot, counts[b])


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("storage", ["int8", "e4m3"])
@pytest.mark.parametrize("page, size, kv_heads, tokens", [(16, 32, 3, 1), (16, 64, 2, 40), (32, 128, 1, 33),
                                                          (64, 64, 2, 64), (128, 128, 2, 150), (256, 128, 1, 300)])
def test_codes_and_scales(dtype, storage, page, size, kv_heads, tokens):
    """Starts inside pages, at their ends and at zero; counts from none to all; slots in another order."""
    rng = np.random.default_rng(page + tokens)
    slots, counts = [2, 0, 3, 1, 4], [tokens, max(0, tokens - 1), 0, tokens, 1]
    before = [7, page, 3 * page - 1, 0, page + 1]  # by slot
    lengths = [before[s] + counts[slots.index(s)] for s in range(5)]
    host = filled(rng, lengths, kv_heads=kv_heads, page=page, head_size=size, storage=storage)
    cache = to_device(host)
    shape = (5, tokens, kv_heads, size)
    rows = [torch.from_numpy((rng.normal(0, 1, shape) * rng.choice([0.1, 1, 8], (5, 1, 1, 1))).astype(np.float32))
            .cuda().to(DTYPE[dtype]) for _ in range(2)]
    cache.append(0, *rows, counts=counts, sequences=slots)
    cache.check_errors()
    appended(host, rows, counts, slots)
    same_pools(cache, host)
    for which in range(2):
        for b, slot in enumerate(slots):
            n = counts[b]
            if not n:
                continue
            given, stored = wide(rows[which][b, :n]), host.read(0, which, slot)[lengths[slot] - n:]
            used = host.table[slot, (lengths[slot] - n + np.arange(n)) // page]
            step = host.scales[which][0, used].astype(np.float64)[..., None]
            # int8: half a step; e4m3 (4 significant bits): 2^-4 of the value, or half of its smallest step 2^-9
            off = 0.5 * step if storage == "int8" else np.maximum(np.abs(given) * 2.0 ** -4, step * 2.0 ** -10)
            assert (np.abs(stored - given) <= off * (1 + 1e-5)).all()


@pytest.mark.parametrize("storage", ["int8", "e4m3"])
def test_one_token_at_a_time(storage):
    """A growing sequence whose values grow too: scales follow, older rows are requantised."""
    rng = np.random.default_rng(3)
    host = plain.Cache(1, 6, 2, 16, 64, 2, 3, np.int8 if storage == "int8" else plain.E4M3)
    cache = to_device(host)
    for step in range(40):
        host.extend([1, 1])
        cache.extend([1, 1])
        rows = [torch.from_numpy(rng.normal(0, 1.1 ** step, (2, 1, 2, 64)).astype(np.float32)).cuda()
                for _ in range(2)]
        cache.append(0, *rows)
        appended(host, rows, [1, 1], [0, 1])
        same_pools(cache, host)
    cache.append(0, *rows)  # the same rows once more change nothing
    same_pools(cache, host)
    cache.check_errors()


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("storage", ["int8", "e4m3"])
def test_values_at_the_ends(dtype, storage):
    """Zeros, the smallest and largest numbers, ties, infinities and NaN."""
    rng = np.random.default_rng(8)
    host = filled(rng, [16] * 8, kv_heads=1, page=16, head_size=32, storage=storage)
    cache = to_device(host)
    rows = torch.from_numpy(rng.normal(0, 1, (8, 16, 1, 32)).astype(np.float32)).cuda().to(DTYPE[dtype])
    rows[0] = 0.0
    rows[1] = -0.0
    rows[2] *= 1e-4 if dtype == "f16" else 1e-38
    rows[3] = torch.finfo(DTYPE[dtype]).max
    rows[4, 3, 0, 5], rows[4, 4, 0, 6] = float("inf"), float("-inf")
    rows[5, 0, 0, 0], rows[5, 15, 0, 31] = float("nan"), float("nan")
    rows[6, :, 0, :] = float("inf")
    rows[7] = torch.arange(-256, 256, device="cuda").view(16, 1, 32) / 2.0  # halves: ties where the scale is one
    cache.append(0, rows, rows.clone())
    cache.check_errors()
    appended(host, [rows, rows], [16] * 8, range(8))
    same_pools(cache, host)


@pytest.mark.parametrize("dtype", list(DTYPE))
def test_strides(dtype):
    """Slices of a fused projection at odd offsets, heads outermost, an expanded head."""
    rng = np.random.default_rng(6)
    host = filled(rng, [40, 25], kv_heads=2, page=16, head_size=32)
    wide_rows = torch.from_numpy(rng.normal(0, 1, (2, 20, 135)).astype(np.float32)).cuda().to(DTYPE[dtype])
    sliced = wide_rows[..., 3:67].view(2, 20, 2, 32)
    turned = sliced.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    shared = sliced[:, :, :1].expand(2, 20, 2, 32)
    for rows in ((sliced, turned), (turned, shared), (shared, sliced)):
        cache = to_device(host)
        cache.append(0, *rows)
        want = filled(np.random.default_rng(6), [40, 25], kv_heads=2, page=16, head_size=32)
        appended(want, rows, [20, 20], [0, 1])
        same_pools(cache, want)


def test_layers_and_errors():
    rng = np.random.default_rng(7)
    host = filled(rng, [20, 9], layers=3)
    cache = to_device(host)
    rows = [torch.from_numpy(rng.normal(0, 1, (2, 4, 2, 64)).astype(np.float32)).cuda() for _ in range(2)]
    cache.append(1, *rows)
    for which in range(2):
        for b in range(2):
            host.append(1, which, wide(rows[which][b]).astype(np.float32), b, 4)
    same_pools(cache, host)
    for counts, slots in (([5, 1], [0, 1]), ([-1, 1], [0, 1]), ([1, 1], [0, 2]), ([4, 1], [-1, 0])):
        cache.append(0, *[r[:, :0] for r in rows], counts=[0, 0])
        cache.check_errors()
        cache.append(0, *rows, counts=counts, sequences=slots)
        with pytest.raises(IndexError):
            cache.check_errors()
    cache.lengths[0] = 2
    cache.append(0, *rows, counts=[4, 0])
    with pytest.raises(IndexError):
        cache.check_errors()
    for k, v in ((rows[0], rows[1].half()), (rows[0], rows[1][:, :3]), (rows[0][:, :, :1], rows[1]),
                 (rows[0].transpose(2, 3), rows[1]), (rows[0].cpu(), rows[1]), (rows[0].long(), rows[1].long())):
        with pytest.raises((TypeError, ValueError)):
            cache.append(0, k, v)
    with pytest.raises(ValueError):
        cache.append(3, *rows)
