"""Host caches of the oracle and their copies on the device."""

from __future__ import annotations

import ml_dtypes
import numpy as np
import torch

from cuda_b200.paged import PagedCache
from oracle import paged as plain

STORAGE = {"int8": np.dtype(np.int8), "e4m3": plain.E4M3}
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {plain.E4M3: torch.float8_e4m3fn, np.dtype(np.int8): torch.int8}


def book_of(host: plain.Cache) -> np.ndarray:
    free = np.zeros(len(host.refs), np.int32)
    free[:len(host.free)] = host.free
    return np.concatenate([host.table.ravel(), host.lengths, host.refs, free,
                           np.array([len(host.free)])]).astype(np.int32)


def to_device(host: plain.Cache) -> PagedCache:
    pools = [torch.from_numpy(p.view(np.int8).copy()).cuda().view(CODE[p.dtype]) for p in host.pools]
    scales = [torch.from_numpy(s.copy()).cuda() for s in host.scales]
    return PagedCache(*pools, *scales, torch.from_numpy(book_of(host)).cuda(), sequences=host.table.shape[0],
                      pages_per_sequence=host.table.shape[1])


def same_book(cache: PagedCache, host: plain.Cache) -> None:
    table, lengths, refs, free, height = (t.cpu().numpy() for t in cache.split(cache.book))
    assert np.array_equal(table, host.table)
    assert np.array_equal(lengths, host.lengths)
    assert np.array_equal(refs, host.refs)
    assert free[:int(height[0])].tolist() == host.free


def same_pools(cache: PagedCache, host: plain.Cache) -> None:
    for got, want in zip((cache.k_pages, cache.v_pages), host.pools):
        assert np.array_equal(got.view(torch.int8).cpu().numpy(), want.view(np.int8))
    for got, want in zip((cache.k_scale, cache.v_scale), host.scales):
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True)


def filled(rng, lengths, *, kv_heads=2, page=16, head_size=64, storage="int8", layers=1, spare=3, columns=None,
           garbage=True) -> plain.Cache:
    """Slots of these lengths on pages scattered over the pool; rows and pages that nobody holds are garbage."""
    need = [-(-n // page) for n in lengths]
    host = plain.Cache(layers, sum(need) + spare, kv_heads, page, head_size, len(lengths),
                       columns or max(1, *need), STORAGE[storage])
    host.free = [int(p) for p in rng.permutation(len(host.refs))]
    host.extend(lengths)
    for which in range(2):
        shape = host.pools[which].shape
        if storage == "int8":
            codes = np.clip(np.rint(rng.normal(0, 36, shape)), -127, 127).astype(np.int8)
        else:
            codes = np.clip(rng.normal(0, 128, shape), -448, 448).astype(ml_dtypes.float8_e4m3fn)
        scales = (rng.uniform(0.5, 2.0, shape[:3]) * 3.5 / float(plain.TOP[STORAGE[storage]])).astype(np.float32)
        if garbage:  # what no slot holds: NaN codes and NaN scales
            rest = codes.view(np.uint8)
            for slot, length in enumerate(lengths):
                if length % page:
                    rest[:, host.table[slot, length // page], :, length % page:] = 0x7F
            rest[:, host.refs == 0] = 0x7F
            scales[:, host.refs == 0] = np.nan
        host.pools[which], host.scales[which] = codes, scales
    return host


def wide(x: torch.Tensor) -> np.ndarray:
    return x.double().cpu().numpy()
