"""Logit adjustments and 4-bit products: calls at the ends of what they take."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cuda_b200 import logits, quantized, speculative
from cuda_b200.paged import PagedCache
from paged_helpers import DTYPE, wide

pytestmark = pytest.mark.gpu


def test_lengths_of_an_empty_history():
    """A history without columns holds no token: any other length sets the flag, and the rows stay."""
    x = torch.randn(3, 40, device="cuda")
    tokens = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    zeros = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert torch.equal(logits.adjust(x, tokens=tokens, lengths=zeros, prompts=zeros, repetition=2.0, error_flag=flag), x)
    speculative.check(flag)
    assert torch.equal(logits.adjust(x, tokens=tokens, lengths=zeros + 1, repetition=2.0, error_flag=flag), x)
    with pytest.raises(Exception, match="history"):
        speculative.check(flag)


@pytest.mark.parametrize("call", [dict(repetition=1e-60), dict(repetition=1e60), dict(frequency=1e60), dict(presence=-1e60)])
def test_numbers_beyond_float32(call):
    x = torch.zeros(1, 8, device="cuda")
    with pytest.raises(ValueError):
        logits.adjust(x, tokens=torch.zeros(1, 1, dtype=torch.int32, device="cuda"), **call)


def test_largest_history():
    """2**20 - 1 times one token: the count does not reach its neighbours in a token's word."""
    n = 2 ** 20 - 1
    tokens = torch.full((1, n), 5, dtype=torch.int64, device="cuda")
    x = torch.zeros(1, 100, device="cuda")
    got = logits.adjust(x, tokens=tokens, frequency=1.0, bias_tokens=torch.tensor([[6, 5]], device="cuda"),
                        bias=torch.tensor([[2.0, 0.5]], device="cuda"))
    want = torch.zeros(1, 100, device="cuda")
    want[0, 5], want[0, 6] = 0.5 - n, 2.0
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", list(DTYPE.values()))
def test_neighbouring_rows_stay(dtype):
    """What is beside `out` in memory keeps its values, at every alignment of a row."""
    room = torch.full((4, 700), 7.0, device="cuda", dtype=dtype)
    x = torch.zeros(4, 651, device="cuda", dtype=dtype)
    for at in range(9):
        room.fill_(7.0)
        logits.adjust(x, allowed=torch.zeros(4, 21, dtype=torch.int32, device="cuda"), out=room[:, at:at + 651])
        assert (room[:, at:at + 651] == float("-inf")).all()
        assert (room[:, :at] == 7.0).all() and (room[:, at + 651:] == 7.0).all()
    weights = quantized.Weights4.quantise(torch.ones(37, 96, device="cuda"), group=32)
    for at in range(9):
        room.fill_(7.0)
        flat = room.view(-1)
        out = flat[at:at + 5 * 37].view(5, 37)
        weights.linear(torch.ones(5, 96, device="cuda", dtype=dtype), out=out)
        assert (flat[:at] == 7.0).all() and (flat[at + 5 * 37:] == 7.0).all() and torch.isfinite(out).all()
    wider = torch.full((40, 130), 7.0, device="cuda", dtype=dtype)
    for at in range(9):
        wider.fill_(7.0)
        weights.dequantise(out=wider[1:38, at:at + 96])
        assert torch.equal(wider[1:38, at:at + 96], weights.dequantise(dtype))
        assert (wider[0] == 7.0).all() and (wider[38:] == 7.0).all()
        assert (wider[:, :at] == 7.0).all() and (wider[:, at + 96:] == 7.0).all()


def test_out_that_overlaps_x():
    weights = quantized.Weights4.quantise(torch.ones(128, 128, device="cuda"))
    x = torch.ones(4, 128, device="cuda")
    with pytest.raises(ValueError, match="shares"):
        weights.linear(x, out=x)


def test_no_rows():
    weights = quantized.Weights4.quantise(torch.ones(48, 128, device="cuda"))
    assert weights.linear(torch.ones(0, 128, device="cuda")).shape == (0, 48)
    assert weights.linear(torch.ones(3, 0, 128, device="cuda")).shape == (3, 0, 48)
    assert logits.adjust(torch.ones(0, 50, device="cuda")).shape == (0, 50)
    assert logits.adjust(torch.ones(3, 0, device="cuda")).shape == (3, 0)


@pytest.mark.parametrize("dtype", list(DTYPE.values()))
def test_many_rows(dtype):
    """More rows than a launch's block takes, each as when it is alone."""
    torch.manual_seed(0)
    weights = quantized.Weights4.quantise(torch.randn(100, 192, device="cuda"), group=64)
    x = torch.randn(301, 192, device="cuda", dtype=dtype)
    got = wide(weights.linear(x))
    want = wide(x) @ wide(weights.dequantise(torch.float32)).T
    size = np.abs(wide(x)) @ np.abs(wide(weights.dequantise(torch.float32))).T
    # 4 products to a group (three parts of float32), 3 groups, 8 warps and 3 parts: as in the products' own test
    error = (4 * 3 * 2.0 ** -22 + 15 * 2.0 ** -24) * size
    assert np.all(np.abs(got - want) <= error + torch.finfo(dtype).eps / 2 * (np.abs(want) + error))


def test_little_shared_is_attend():
    """Below least_bytes, as always in a cache this small, attend_shared is attend, bit for bit."""
    cache = PagedCache.allocate(layers=1, pages=64, kv_heads=2, page_size=16, head_size=64, sequences=4,
                                pages_per_sequence=16, storage=torch.int8)
    cache.extend([100], sequences=[0])
    kv = torch.randn(2, 1, 100, 2, 64, device="cuda")
    cache.append(0, kv[0], kv[1], sequences=[0])
    cache.fork([0, 0, 0], [1, 2, 3])
    q = torch.randn(4, 1, 8, 64, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(cache.attend_shared(0, q), cache.attend(0, q))
    large = 4 * 100 * 2 * 64 * 4
    assert torch.equal(cache.attend_shared(0, q, least_bytes=large), cache.attend(0, q))
    assert torch.equal(cache.attend_shared(0, q[:1], sequences=[2], least_bytes=0), cache.attend_shared(0, q[:1], sequences=[3],
                                                                                                     least_bytes=0))
    cache.check_errors()


@pytest.mark.parametrize("dtype", list(DTYPE.values()))
@pytest.mark.parametrize("outputs", [2367, 2370, 4750, 7150, 9500, 11900, 16600, 18900, 37900])
@pytest.mark.parametrize("group, inputs", [(32, 96), (64, 704), (128, 1152)])
def test_many_outputs(dtype, outputs, group, inputs):
    """As many tiles of 16 outputs as change a block's form: warps, tiles and blocks an SM.

    A group's products are added within 2^-22 of what its terms add up to for each product of 16 inputs (of three parts
    for float32); then a warp of at least four adds its groups, and up to 16 warps are joined, each float32.
    """
    torch.manual_seed(outputs)
    weights = quantized.Weights4.quantise(torch.randn(outputs, inputs, device="cuda"), group=group)
    w = weights.dequantise(torch.float32).double()
    for rows in (1, 5, 9, 16, 27):
        x = torch.randn(rows, inputs, device="cuda", dtype=dtype)
        got = weights.linear(x).double()
        want, size = x.double() @ w.T, x.double().abs() @ w.abs().T
        steps = group / 16 * (3 if dtype == torch.float32 else 1)
        error = (steps * 2.0 ** -22 + (inputs / group / 4 + 20) * 2.0 ** -24) * size
        assert ((got - want).abs() <= error + torch.finfo(dtype).eps / 2 * (want.abs() + error)).all()
