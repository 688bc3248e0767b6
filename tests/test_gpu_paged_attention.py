"""cb_paged_attention against a float64 softmax over the dequantised cache.

Bound, from the formula: an output is a mean of values, so an error e of its
weights (relative) moves it by at most 2 e max|v|, and rounding to the output's
type adds half its last place.  float32: the scores are sums of head_size
products of numbers held to 22 bits or more and the largest score here is below
64 in base 2, so e < 64 * 2^-22 = 2^-16; 16-bit types: weights are rounded to
11 bits, e < 2^-11 more.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from cuda_b200 import _lib
from oracle import paged as plain
from paged_helpers import DTYPE, filled, to_device, wide

pytestmark = pytest.mark.gpu

WEIGHTS = {"f32": 2.0 ** -16, "bf16": 2.0 ** -16 + 2.0 ** -11, "f16": 2.0 ** -16 + 2.0 ** -11}
ROUNDING = {name: torch.finfo(dtype).eps / 2 for name, dtype in DTYPE.items()}


def expected(host, q, counts, slots, scale):
    out = np.zeros(q.shape)
    for b, slot in enumerate(slots):
        n = counts[b]
        if n:
            out[b, :n] = plain.attend(wide(q[b, :n]), host.read(0, 0, slot), host.read(0, 1, slot), scale)
    return out


def compare(got, want, host, dtype):
    values = max(float(np.nanmax(np.abs(host.read(0, 1, s)), initial=0.0)) for s in range(len(host.lengths)))
    bound = 2 * WEIGHTS[dtype] * values + ROUNDING[dtype] * np.abs(want) + 1e-7 * values
    got = wide(got)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), float(np.max(np.abs(got - want) / bound))


def queries(rng, batch, tokens, heads, size, dtype):
    return torch.from_numpy(rng.normal(0, 2, (batch, tokens, heads, size)).astype(np.float32)).cuda().to(DTYPE[dtype])


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("storage", ["int8", "e4m3"])
@pytest.mark.parametrize("heads, kv_heads, size", [(8, 2, 32), (32, 4, 64), (32, 8, 128), (3, 3, 64), (16, 1, 128),
                                                   (48, 1, 32), (5, 1, 64)])
def test_ragged_single_tokens(dtype, storage, heads, kv_heads, size):
    """Lengths of zero, one, around tiles and pages, and some thousand; one row of counts zero."""
    rng = np.random.default_rng(heads + size)
    lengths = [0, 1, 15, 16, 17, 63, 64, 65, 129, 700, 2047, 33]
    counts = [0] + [1] * 10 + [0]
    host = filled(rng, lengths, kv_heads=kv_heads, head_size=size, storage=storage)
    cache = to_device(host)
    q = queries(rng, len(lengths), 1, heads, size, dtype)
    got = cache.attend(0, q, counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
    cache.check_errors()
    compare(got, expected(host, q, counts, range(len(lengths)), 1 / math.sqrt(size)), host, dtype)


@pytest.mark.parametrize("dtype, storage", [("f32", "e4m3"), ("bf16", "int8"), ("f16", "e4m3"), ("f32", "int8")])
@pytest.mark.parametrize("tokens", [2, 4, 5, 8, 17, 70])
@pytest.mark.parametrize("heads, kv_heads, size, page", [(8, 2, 32, 32), (32, 4, 64, 16), (8, 2, 128, 64),
                                                         (6, 6, 128, 256), (28, 4, 64, 128)])
def test_blocks_of_tokens(dtype, storage, tokens, heads, kv_heads, size, page):
    """Drafted blocks and short chunks: every token sees its own past, fewer counts than tokens, block at the start."""
    rng = np.random.default_rng(tokens)
    lengths = [tokens, tokens + 1, 100 + tokens, 513, 5]
    counts = [tokens, tokens, tokens, tokens - 1, min(5, tokens)]
    host = filled(rng, lengths, kv_heads=kv_heads, head_size=size, storage=storage, page=page)
    cache = to_device(host)
    q = queries(rng, len(lengths), tokens, heads, size, dtype)
    got = cache.attend(0, q, counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
    cache.check_errors()
    compare(got, expected(host, q, counts, range(len(lengths)), 1 / math.sqrt(size)), host, dtype)


@pytest.mark.parametrize("batch, length", [(1, 40001), (3, 9000), (150, 300)])
def test_split_keys(batch, length):
    """Long rows that several blocks share and many short ones; equal calls give equal bits."""
    rng = np.random.default_rng(batch)
    lengths = [max(1, length - 97 * b) for b in range(batch)]
    host = filled(rng, lengths, kv_heads=2, head_size=64, page=64)
    cache = to_device(host)
    q = queries(rng, batch, 1, 8, 64, "f32")
    got = cache.attend(0, q)
    compare(got, expected(host, q, [1] * batch, range(batch), 0.125), host, "f32")
    for _ in range(3):
        assert torch.equal(got, cache.attend(0, q))
    cache.check_errors()


def test_strides_slots_scale_and_out():
    """q as a slice of a projection's rows, slots in another order, another scale, the caller's output."""
    rng = np.random.default_rng(5)
    lengths = [50, 0, 333, 81]
    host = filled(rng, lengths, kv_heads=2, head_size=64, columns=40)
    cache = to_device(host)
    rows = torch.from_numpy(rng.normal(0, 1, (2, 3, 8 * 64 + 7)).astype(np.float32)).cuda().to(torch.bfloat16)
    q = rows[:, :, 3:3 + 512].view(2, 3, 8, 64)  # odd offset and row length
    slots = [3, 2]
    out = torch.full((2, 3, 8, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    assert cache.attend(0, q, sequences=slots, scale=0.3, out=out) is out
    compare(out, expected(host, q, [3, 3], slots, 0.3), host, "bf16")
    swapped = queries(rng, 8, 3, 2, 64, "f32").permute(2, 1, 0, 3)  # heads outermost
    compare(cache.attend(0, swapped, sequences=slots), expected(host, swapped, [3, 3], slots, 0.125), host, "f32")


@pytest.mark.parametrize("size", [2.0 ** -60, 1e-3, 300.0, 2.0 ** 40])
def test_queries_of_any_size(size):
    """Rows whose queries are tiny (all weights alike) or so large that one key takes all."""
    rng = np.random.default_rng(9)
    host = filled(rng, [77, 200], kv_heads=1, head_size=128)
    q = queries(rng, 2, 1, 4, 128, "f32") * size
    q[0, 0, 1] = 0.0
    got, want = wide(to_device(host).attend(0, q)), expected(host, q, [1, 1], range(2), 1 / math.sqrt(128))
    # a score s has an error of |s| 2^-22: keys nearer than that to the best one are a tie
    score = np.abs(want).max() * 4 * 2.0 ** -16 if size <= 1 else 0.0
    if size <= 1:
        assert np.abs(got - want).max() <= score + 1e-6
    else:
        best = [host.read(0, 1, b)[int(np.argmax(host.read(0, 0, b)[:, 0] @ wide(q)[b, 0, h])), 0]
                for b in range(2) for h in (0, 2, 3)]
        if size >= 2.0 ** 40:
            assert np.allclose(got[:, 0, [0, 2, 3]].reshape(6, -1), np.array(best), rtol=1e-6)
        else:
            assert np.abs(got - want).max() <= 300 * 64 * 2.0 ** -22 * 8 * 2


def test_scales_far_apart():
    """Pages whose value scales differ by many powers of ten each keep their part of the sum."""
    rng = np.random.default_rng(2)
    host = filled(rng, [160], kv_heads=1, head_size=64, spare=0)
    order = host.table[0]
    host.scales[1][0, order, 0] = np.float32(10.0) ** np.arange(-30, 20, 5, dtype=np.float32)
    q = torch.zeros(1, 1, 2, 64, device="cuda")
    for j, page in enumerate(order):  # the larger a page's values, the smaller its weight
        host.pools[0][0, page, 0] = 0
        host.pools[0][0, page, 0, :, 0] = 50 - 5 * j
    host.scales[0][0, :, 0] = np.float32(math.log(10) * 8)  # scale 1/8: weights 10^(50 - 5 j)
    q[..., 0] = 1.0
    got, want = wide(to_device(host).attend(0, q)), expected(host, q, [1], [0], 0.125)
    assert np.abs(got - want).max() <= 2e-3 * np.abs(want).max()  # scores up to 115: weights to 115 * 2^-17


def test_errors_of_the_book_are_flagged():
    rng = np.random.default_rng(1)
    host = filled(rng, [40, 20, 30])
    for change in ("page", "length", "slot", "count"):
        cache = to_device(host)
        counts, slots = [1, 1, 1], [0, 1, 2]
        if change == "page":
            cache.table[1, 0] = cache.pages
        elif change == "length":
            cache.lengths[1] = cache.pages_per_sequence * cache.page_size + 1
        elif change == "slot":
            slots[1] = 3
        else:
            counts[1] = 2
        q = queries(rng, 3, 1, 4, 64, "f32")
        got = cache.attend(0, q, counts=counts, sequences=slots)
        with pytest.raises(IndexError):
            cache.check_errors()
        cache.check_errors()  # read once
        want = expected(host, q, [1, 0, 1], range(3), 0.125)
        compare(got[[0, 2]], want[[0, 2]], host, "f32")


def test_another_stream_and_a_graph():
    """The current stream carries the call; a captured step follows lengths that grow."""
    rng = np.random.default_rng(4)
    host = filled(rng, [100, 260], kv_heads=2, head_size=128)
    cache = to_device(host)
    q = queries(rng, 2, 1, 8, 128, "bf16")
    want = cache.attend(0, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.attend(0, q)
    side.synchronize()
    assert torch.equal(got, want)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
    with torch.cuda.graph(graph):
        cache.attend(0, q, out=out)
    for lengths in ([100, 260], [3, 17], [96, 1]):
        cache.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, cache.attend(0, q))
    cache.check_errors()


def test_refusals():
    cache = to_device(filled(np.random.default_rng(0), [20, 20]))
    q = torch.zeros(2, 1, 4, 64, device="cuda")
    for bad in (q[..., :32], q[:, :, :3], q.double(), q.cpu(), torch.zeros(3, 1, 4, 64, device="cuda"),
                q.transpose(2, 3), q[0]):
        with pytest.raises((TypeError, ValueError)):
            cache.attend(0, bad)
    for arguments in (dict(counts=[1]), dict(sequences=[0]), dict(counts=torch.ones(2, device="cuda")),
                      dict(out=torch.zeros(2, 1, 4, 64, device="cuda").half())):
        with pytest.raises((TypeError, ValueError)):
            cache.attend(0, q, **arguments)
    with pytest.raises(ValueError):
        cache.attend(1, q)
    with pytest.raises(ValueError):
        cache.attend(0, q.clone().requires_grad_())
    with pytest.raises(TypeError):
        cache.attend(0, [1.0])
    assert cache.attend(0, q[:0]).shape == (0, 1, 4, 64)
    assert _lib.load() is not None
