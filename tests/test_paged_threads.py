"""Calls of one cache from several host threads, without a GPU: attend and attend_shared keep a workspace for each
stream, and the launches of one call use it one after the other, so no other call's may come between."""

from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor
import threading
import time

import pytest
import torch

from cuda_b200 import _lib, paged


class Library:
    """Stands for the C library: notes how many calls are inside at the same time."""

    def __init__(self):
        self.inside, self.most, self.guard = 0, 0, threading.Lock()

    def cb_paged_attention_scratch(self, args):
        return 64

    def cb_paged_attention_shared_scratch(self, args, least_bytes):
        return 64 * (1 + least_bytes)

    def cb_paged_attention_counters(self, args):
        return 8

    def call(self):
        with self.guard:
            self.inside += 1
            self.most = max(self.most, self.inside)
        time.sleep(0.002)  # (as ctypes does, this lets other threads run)
        with self.guard:
            self.inside -= 1
        return 0

    def cb_paged_attention(self, args, scratch, counters, stream):
        return self.call()

    def cb_paged_attention_shared(self, args, least_bytes, scratch, counters, stream):
        return self.call()


@pytest.fixture
def cache(monkeypatch):
    library = Library()
    monkeypatch.setattr(_lib, "load", lambda: library)
    monkeypatch.setattr(paged, "current_stream", lambda device: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    made = paged.PagedCache.__new__(paged.PagedCache)  # (the constructor asks for a CUDA device)
    made.device, made.layers, made.kv_heads, made.head_size, made.sequences = torch.device("cpu"), 1, 2, 64, 2
    made._layer_args, made._lib, made._flag = [_lib.PagedCacheArgs()], library, torch.zeros(1, dtype=torch.int32)
    made._attend_args, made._workspaces, made._lists = paged.Prepared(), paged.Prepared(), paged.Prepared()
    made._calls = threading.Lock()
    return made, library


@pytest.mark.parametrize("name", ["attend", "attend_shared"])
def test_calls_of_threads_do_not_meet(cache, name):
    cache, library = cache
    q = torch.zeros(2, 1, 4, 64)

    def work(i):
        more = {"least_bytes": i} if name == "attend_shared" else {}
        for _ in range(5):
            getattr(cache, name)(0, q, **more)

    with ThreadPoolExecutor(6) as pool:
        list(pool.map(work, range(6)))
    assert library.most == 1 and library.inside == 0


def test_a_call_that_fails_lets_others_in(cache):
    cache, library = cache
    q = torch.zeros(2, 1, 4, 64)
    library.cb_paged_attention = lambda *args: 1
    library.cb_last_error = lambda: b"refused"
    with pytest.raises(_lib.KernelError, match="refused"):
        cache.attend(0, q)
    cache.attend_shared(0, q)
    assert library.most == 1


@pytest.mark.gpu
@pytest.mark.parametrize("streams", [1, 2])
def test_threads_on_the_device(streams):
    """Threads of one stream, or of two, with calls of other sizes and sequences: each gets its own results."""
    cache = paged.PagedCache.allocate(layers=1, pages=300, kv_heads=2, page_size=16, head_size=64, sequences=12,
                                      pages_per_sequence=60)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for parent, length in ((0, 500), (4, 700), (8, 90)):
        cache.extend([length], sequences=[parent])
        k, v = (torch.randn(1, length, 2, 64, device="cuda", generator=gen) for _ in range(2))
        cache.append(0, k, v, sequences=[parent])
        cache.fork([parent] * 3, [parent + i for i in (1, 2, 3)])
    calls = []
    for i in range(6):
        slots = torch.arange(i % 3 * 4, i % 3 * 4 + 4 - i % 2, device="cuda").int()
        q = torch.randn(len(slots), 1 + i, 8, 64, device="cuda", generator=gen)
        calls.append((q, slots, cache.attend_shared(0, q, sequences=slots, least_bytes=0)))
    cache.check_errors()
    torch.cuda.synchronize()
    used = [torch.cuda.Stream() for _ in range(streams)]

    def work(i):
        q, slots, want = calls[i]
        with torch.cuda.stream(used[i % streams]):
            got = [cache.attend_shared(0, q, sequences=slots, least_bytes=0) for _ in range(40)]
        torch.cuda.synchronize()
        return all(torch.equal(g, want) for g in got)

    with ThreadPoolExecutor(6) as pool:
        assert all(pool.map(work, range(6)))
    cache.check_errors()
