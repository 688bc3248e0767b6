"""cb_paged_attention_shared against a float64 softmax over the dequantised cache: forked
sequences of all lengths, and calls whose sequences share little, nothing or everything.

The bound is the one derived in test_gpu_paged_attention.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from paged_helpers import DTYPE, filled, to_device, wide
from test_gpu_paged_attention import compare, expected, queries

pytestmark = pytest.mark.gpu


def spoil(host):
    """NaN codes and scales in all that no slot holds."""
    held = {}
    for slot, length in enumerate(host.lengths):
        for at in range(-(-int(length) // host.pools[0].shape[3])):
            page = int(host.table[slot, at])
            rows = min(host.pools[0].shape[3], int(length) - at * host.pools[0].shape[3])
            held[page] = max(held.get(page, 0), rows)
    for which in range(2):
        raw = host.pools[which].view(np.uint8)
        for page in range(raw.shape[1]):
            raw[:, page, :, held.get(page, 0):] = 0x7F
            if page not in held:
                host.scales[which][:, page] = np.nan
    return host


def family(rng, prefix, tails, *, kv_heads=2, page=16, head_size=64, storage="int8", room=0):
    """Slot 0 holds ``prefix`` tokens, the others are forked from it, and slot b goes on by ``tails[b]`` of its own."""
    n = len(tails)
    longest = -(-(prefix + max(tails)) // page)
    spare = sum(-(-t // page) + 1 for t in tails) + 2
    host = filled(rng, [prefix] + [0] * (n - 1), kv_heads=kv_heads, page=page, head_size=head_size, storage=storage,
                  spare=spare, columns=longest + room, garbage=False)
    if n > 1:
        host.fork([0] * (n - 1), list(range(1, n)))
    host.extend(list(tails))
    return spoil(host)


def check(host, q, counts, slots, dtype, scale=None, **call):
    cache = to_device(host)
    given = {"counts": torch.tensor(counts, dtype=torch.int32, device="cuda")}
    if slots is not None:
        given["sequences"] = torch.tensor(slots, dtype=torch.int32, device="cuda")
    got = cache.attend_shared(0, q, least_bytes=0, scale=scale, **given, **call)
    cache.check_errors()
    size = q.shape[-1]
    want = expected(host, q, counts, range(q.shape[0]) if slots is None else slots,
                    1 / math.sqrt(size) if scale is None else scale)
    compare(got, want, host, dtype)
    return cache, got


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("storage", ["int8", "e4m3"])
@pytest.mark.parametrize("heads, kv_heads, size, page", [(8, 2, 32, 32), (32, 4, 64, 16), (32, 8, 128, 64), (3, 3, 64, 16),
                                                         (16, 1, 128, 16), (48, 1, 32, 16), (5, 1, 64, 128)])
@pytest.mark.parametrize("prefix", [16, 100, 1039])
def test_forks(dtype, storage, heads, kv_heads, size, page, prefix):
    """Tails of one token and more, a slot without a row."""
    rng = np.random.default_rng(heads + size + prefix)
    tails = [1, 2, 17, 0, 40, 130, 1]
    host = family(rng, prefix, tails, kv_heads=kv_heads, head_size=size, page=page, storage=storage)
    q = queries(rng, len(tails), 1, heads, size, dtype)
    check(host, q, [int(t > 0) for t in tails], None, dtype)


@pytest.mark.parametrize("prefix", [0, 1, 15, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 640, 641, 5000])
def test_prefixes(prefix):
    rng = np.random.default_rng(prefix)
    for dtype in DTYPE:
        host = family(rng, prefix, [5, 1, 9, 70], head_size=128)
        check(host, queries(rng, 4, 1, 8, 128, dtype), [1] * 4, None, dtype)


@pytest.mark.parametrize("dtype, storage", [("f32", "e4m3"), ("bf16", "int8"), ("f16", "e4m3"), ("f32", "int8")])
@pytest.mark.parametrize("tokens", [2, 5, 8, 33])
@pytest.mark.parametrize("heads, kv_heads, size, page", [(8, 2, 32, 32), (32, 4, 64, 16), (8, 2, 128, 64), (28, 4, 64, 128)])
def test_blocks_of_tokens(dtype, storage, tokens, heads, kv_heads, size, page):
    """Drafted blocks, fewer counts than tokens in some, blocks that reach back into the shared pages."""
    rng = np.random.default_rng(tokens)
    tails = [tokens, tokens + 1, 100 + tokens, 3, tokens]
    counts = [tokens, tokens, tokens, min(tokens, 10), tokens - 1]
    host = family(rng, 300, tails, kv_heads=kv_heads, head_size=size, storage=storage, page=page)
    check(host, queries(rng, len(tails), tokens, heads, size, dtype), counts, None, dtype)


@pytest.mark.parametrize("batch, prefix", [(2, 40001), (64, 2000), (150, 333), (300, 64)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows_and_long_prefixes(batch, prefix, dtype):
    """More rows than a block takes, prefixes that many blocks divide; equal calls give equal bits."""
    rng = np.random.default_rng(batch)
    host = family(rng, prefix, [1 + 7 * b % 50 for b in range(batch)], page=64)
    q = queries(rng, batch, 1, 8, 64, dtype)
    cache, got = check(host, q, [1] * batch, None, dtype)
    for _ in range(3):
        assert torch.equal(got, cache.attend_shared(0, q, least_bytes=0))


def test_whole_sequences_shared():
    """Forks that have not gone on: all pages but the last key's are common, page ends included."""
    rng = np.random.default_rng(2)
    for length in (1, 16, 17, 64, 65, 200):
        host = family(rng, length, [0, 0, 0])
        for dtype in DTYPE:
            check(host, queries(rng, 3, 1, 4, 64, dtype), [1, 1, 1], None, dtype)


def test_little_or_nothing_shared():
    """Sequences of their own, two families in one call, one sequence alone, none."""
    rng = np.random.default_rng(3)
    host = filled(rng, [40, 0, 333, 1], kv_heads=2, head_size=64)
    for dtype in DTYPE:
        check(host, queries(rng, 4, 1, 8, 64, dtype), [1, 0, 1, 1], None, dtype)
        check(host, queries(rng, 1, 1, 8, 64, dtype), [1], [2], dtype)
        check(host, queries(rng, 2, 1, 8, 64, dtype), [0, 0], None, dtype)
    two = filled(rng, [100, 0, 90, 0, 0], kv_heads=2, head_size=64, spare=20, columns=10, garbage=False)
    two.fork([0, 2, 2], [1, 3, 4])
    two.extend([1, 30, 2, 3, 4])
    spoil(two)
    for dtype in DTYPE:
        check(two, queries(rng, 5, 1, 8, 64, dtype), [1] * 5, None, dtype)
        check(two, queries(rng, 3, 1, 8, 64, dtype), [1] * 3, [4, 2, 3], dtype)
        check(two, queries(rng, 4, 1, 8, 64, dtype), [0, 0, 1, 1], [0, 4, 3, 2], dtype)
    assert check(two, queries(rng, 0, 1, 8, 64, "f32"), [], [], "f32")[1].shape == (0, 1, 8, 64)


def test_strides_slots_scale_and_out():
    rng = np.random.default_rng(5)
    host = family(rng, 400, [3, 50, 20, 81], room=7)
    rows = torch.from_numpy(rng.normal(0, 1, (2, 3, 8 * 64 + 7)).astype(np.float32)).cuda().to(torch.bfloat16)
    q = rows[:, :, 3:3 + 512].view(2, 3, 8, 64)  # odd offset and row length
    out = torch.full((2, 3, 8, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    assert check(host, q, [3, 3], [3, 2], "bf16", scale=-0.3, out=out)[1] is out
    swapped = queries(rng, 8, 3, 2, 64, "f32").permute(2, 1, 0, 3)  # heads outermost
    check(host, swapped, [3, 3], [1, 3], "f32")
    check(host, queries(rng, 1, 3, 8, 64, "f16").expand(4, 3, 8, 64), [3, 3, 3, 3], None, "f16", scale=0.0)


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("size", [2.0 ** -14, 1e-3, 300.0])
def test_queries_of_any_size(size, dtype):
    """Rows whose queries are tiny (all weights alike) or so large that one key takes all."""
    rng = np.random.default_rng(9)
    host = family(rng, 700, [8, 200], kv_heads=1, head_size=128)
    q = queries(rng, 2, 1, 4, 128, dtype) * size
    cache = to_device(host)
    want = expected(host, q, [1, 1], range(2), 1 / math.sqrt(128))
    got = wide(cache.attend_shared(0, q, least_bytes=0))
    cache.check_errors()
    values = max(float(np.abs(host.read(0, 1, s)).max()) for s in range(2))
    # scores of thousands in base 2 move by their own float32 rounding: 2^-22 of them
    largest = float(np.abs(wide(q)).max()) * 128 * 16 / math.sqrt(128) * 1.45
    allowed = 2 * (max(64.0, largest) * 2.0 ** -22 + (0 if dtype == "f32" else 2.0 ** -11)) * values
    assert (np.abs(got - want) <= allowed + torch.finfo(q.dtype).eps / 2 * np.abs(want) + 1e-7 * values).all()


@pytest.mark.parametrize("dtype", list(DTYPE))
def test_scales_far_apart(dtype):
    """Value scales that differ by powers of two from page to page, zero pages among them, first, between and last."""
    rng = np.random.default_rng(7)
    host = family(rng, 640, [5, 33, 12], head_size=128)
    for which, spread in ((0, 3), (1, 30)):
        for column in range(40):
            page = int(host.table[0, column])
            host.scales[which][:, page] *= np.float32(2.0 ** int(rng.integers(-spread, 1)))
            if which == 1 and column % 7 == 0:
                host.scales[which][:, page] = 0.0
    check(host, queries(rng, 3, 1, 8, 128, dtype), [1] * 3, None, dtype)


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("where", [0, 300, 639])
def test_one_key_takes_nearly_all(dtype, where):
    """A key whose score is far above the others', with a value of zero: what is left is the others' weighted values."""
    rng = np.random.default_rng(where)
    host = family(rng, 640, [5, 12], kv_heads=1, head_size=64)
    q = queries(rng, 2, 1, 4, 64, dtype)
    page, row = int(host.table[0, where // 16]), where % 16
    q[...] = 0.25 * q + 1.0
    host.pools[0][0, page, 0, row] = 127
    host.scales[0][0, page, 0] = 16 * host.scales[0][0, page, 0]
    host.pools[0][0, page, 0, :row] //= 16
    host.pools[0][0, page, 0, row + 1:] //= 16
    host.pools[1][0, page, 0, row] = 0
    check(host, q, [1, 1], None, dtype)


def test_captured_on_other_streams():
    """Two captured calls, replayed on two streams at once, with other lengths than they were captured with."""
    rng = np.random.default_rng(11)
    host = family(rng, 2000, [5, 40, 9], page=64)
    cache = to_device(host)
    q = queries(rng, 3, 1, 8, 64, "bf16")
    counts = torch.ones(3, dtype=torch.int32, device="cuda")
    cache.attend_shared(0, q, least_bytes=0, counts=counts)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(cache.attend_shared(0, q, least_bytes=0, counts=counts))
        graphs.append(graph)
    host.truncate([3, 30, 8], [0, 1, 2])
    cache.truncate([3, 30, 8])
    q.copy_(queries(rng, 3, 1, 8, 64, "bf16"))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    cache.check_errors()
    for out in outs:
        compare(out, expected(host, q, [1] * 3, range(3), 0.125), host, "bf16")
    with torch.cuda.stream(streams[0]):
        assert torch.equal(cache.attend_shared(0, q, least_bytes=0, counts=counts), outs[0])
    torch.cuda.synchronize()


def test_bad_books_are_flagged():
    """A page outside the pool in a column that all name, a slot and a count outside their ranges: IndexError."""
    rng = np.random.default_rng(13)
    host = family(rng, 100, [5, 9, 20])
    q = queries(rng, 3, 1, 4, 64, "f32")
    for bad in (len(host.refs), -1, 2 ** 31 - 1):
        cache = to_device(host)
        cache.table[:, 2] = bad
        cache.attend_shared(0, q, least_bytes=0)
        with pytest.raises(IndexError):
            cache.check_errors()
    cache = to_device(host)
    ones = torch.ones(3, dtype=torch.int32, device="cuda")
    for call in (dict(sequences=2 * ones), dict(counts=3 * ones), dict(counts=-ones),
                 dict(sequences=torch.tensor([3, 0, 1], dtype=torch.int32, device="cuda"))):
        got = cache.attend_shared(0, q, least_bytes=0, **call)
        if "sequences" in call and int(call["sequences"][0]) == 2:
            cache.check_errors()  # (one slot three times is a call of its own)
            continue
        with pytest.raises(IndexError):
            cache.check_errors()
        assert torch.isfinite(got).all()
    compare(cache.attend_shared(0, q, least_bytes=0), expected(host, q, [1] * 3, range(3), 0.125), host, "f32")
    cache.check_errors()


def test_refusals():
    host = family(np.random.default_rng(1), 40, [1, 2])
    cache = to_device(host)
    q = torch.zeros(2, 1, 4, 64, device="cuda")
    for call in (dict(q=q[..., :32]), dict(q=q[:, :, :3]), dict(q=q, counts=torch.ones(3, dtype=torch.int32, device="cuda")),
                 dict(q=q.cpu()), dict(q=q, out=torch.zeros(2, 1, 4, 32, device="cuda")), dict(q=q, layer=1)):
        with pytest.raises(ValueError):
            cache.attend_shared(**{"layer": 0, **call})
    with pytest.raises(TypeError):
        cache.attend_shared(0, q.double())
    with pytest.raises(ValueError):
        cache.attend_shared(0, q, least_bytes=-1)
    with pytest.raises(ValueError):
        cache.attend_shared(0, q.requires_grad_())
