"""4-bit weights: codes and scales equal the rule, products lie within the roundings of their own sums."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cuda_b200 import quantized
from paged_helpers import DTYPE, wide

pytestmark = pytest.mark.gpu

SCALES = {"bf16": torch.bfloat16, "f16": torch.float16}


def plain_form(rng, outputs, inputs, group, scales="bf16"):
    codes = rng.integers(0, 256, (outputs, inputs // 2)).astype(np.uint8)
    scale = torch.from_numpy(rng.uniform(0.01, 0.1, (outputs, inputs // group)).astype(np.float32)).cuda()
    return torch.from_numpy(codes).cuda(), scale.to(SCALES[scales])


def numbers(codes, scale):
    """The weights in float64."""
    byte = codes.cpu().numpy().astype(np.int64)
    q = np.stack([byte & 15, byte >> 4], -1).reshape(byte.shape[0], -1) - 8
    return q * np.repeat(wide(scale), q.shape[1] // scale.shape[1], 1)


def close(got, x, w, group):
    """A group's products of 16 inputs are added in float32 one after the other (within 2^-22 of what the sum's
    terms add up to), then the groups, eight warps and three parts; last comes the output's own rounding."""
    x, got_dtype, got = wide(x), got.dtype, wide(got)
    want, size = x @ w.T, np.abs(x) @ np.abs(w).T
    groups = w.shape[1] // group
    steps = group / 16 * (3 if got_dtype == torch.float32 else 1)
    bound = (steps * 2.0 ** -22 + (groups / 8 + 14) * 2.0 ** -24) * size
    half = torch.finfo(got_dtype).eps / 2
    assert got.shape == want.shape
    assert np.all(np.abs(got - want) <= bound + half * (np.abs(want) + bound))


def inputs_of(rng, rows, inputs, dtype):
    return torch.from_numpy(rng.normal(0, 1, (rows, inputs)).astype(np.float32)).cuda().to(DTYPE[dtype])


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("group, inputs", [(32, 32), (32, 96), (32, 2048), (64, 64), (64, 320), (64, 5632), (128, 128),
                                           (128, 384), (128, 4096), (128, 1152)])
@pytest.mark.parametrize("outputs", [1, 15, 16, 33, 260])
def test_linear(dtype, group, inputs, outputs):
    rng = np.random.default_rng(inputs + outputs)
    codes, scale = plain_form(rng, outputs, inputs, group, "f16" if outputs % 2 else "bf16")
    weights = quantized.Weights4.pack(codes, scale)
    w = numbers(codes, scale)
    for rows in (1, 5):
        x = inputs_of(rng, rows, inputs, dtype)
        close(weights.linear(x), x, w, group)


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("rows", [0, 2, 7, 8, 9, 16, 17, 24, 31, 32, 33, 65, 100])
def test_rows(dtype, rows):
    rng = np.random.default_rng(rows)
    for group in (32, 64, 128):
        codes, scale = plain_form(rng, 80, 640, group)
        weights = quantized.Weights4.pack(codes, scale)
        x = inputs_of(rng, rows, 640, dtype)
        y = weights.linear(x)
        assert y.shape == (rows, 80) and y.dtype == x.dtype
        if rows:
            close(y, x, numbers(codes, scale), group)


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("outputs, inputs, group", [(1, 32, 32), (16, 64, 64), (37, 672, 32), (100, 192, 64),
                                                    (65, 1280, 128)])
def test_dequantise(dtype, outputs, inputs, group):
    rng = np.random.default_rng(outputs)
    codes, scale = plain_form(rng, outputs, inputs, group, "f16")
    weights = quantized.Weights4.pack(codes, scale)
    want = torch.from_numpy(numbers(codes, scale)).to(DTYPE[dtype])
    assert torch.equal(weights.dequantise(DTYPE[dtype]).cpu(), want)
    room = torch.full((outputs, inputs + 5), 3.0, dtype=DTYPE[dtype], device="cuda")
    weights.dequantise(out=room[:, 2:2 + inputs])
    assert torch.equal(room[:, 2:2 + inputs].cpu(), want)
    assert (room[:, :2] == 3).all() and (room[:, 2 + inputs:] == 3).all()


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("scales", list(SCALES))
@pytest.mark.parametrize("group", quantized.GROUPS)
def test_quantise(dtype, scales, group):
    """Scales and codes equal the rule in float32, also of groups of zeros and of tiny numbers."""
    rng = np.random.default_rng(group)
    room = torch.from_numpy(rng.normal(0, 0.02, (19, group * 3 + 1)).astype(np.float32)).cuda().to(DTYPE[dtype])
    weight = room[:, 1:]
    weight[3, :group] = 0.0
    weight[4] *= 2.0 ** -12
    weight[5, 0] = 3.0
    codes, scale = quantized.quantise(weight, group=group, scales=SCALES[scales])
    parts = weight.float().cpu().reshape(19, -1, group)
    s = (parts.abs().amax(-1) / 7.0).to(SCALES[scales])
    assert torch.equal(scale.cpu(), s)
    q = torch.where(s[..., None] > 0, parts / s.float()[..., None], 0.0).round().clamp(-8, 7).reshape(19, -1)
    byte = codes.cpu().int()
    got = torch.stack([byte & 15, byte >> 4], -1).reshape(19, -1) - 8
    assert torch.equal(got, q.int())
    weights = quantized.Weights4.quantise(weight, group=group, scales=SCALES[scales])
    want = (got.reshape(19, -1, group) * s.float()[..., None]).reshape(19, -1)
    assert torch.equal(weights.dequantise(torch.float32).cpu(), want)


def test_not_finite():
    """A group with an infinity or NaN makes its output NaN and no other; so do such rows of x theirs."""
    weight = torch.ones(40, 256, device="cuda")
    weight[3, 7], weight[20, 200] = float("inf"), float("nan")
    weights = quantized.Weights4.quantise(weight, group=64)
    for dtype in DTYPE.values():
        x = torch.ones(3, 256, device="cuda", dtype=dtype)
        y = weights.linear(x)
        assert torch.isnan(y[:, 3]).all() and torch.isnan(y[:, 20]).all()
        assert int(torch.isfinite(y).sum()) == 3 * 38
        x[1, 5] = float("nan")
        x[2, 6] = float("inf")
        y = quantized.Weights4.quantise(torch.ones(40, 256, device="cuda")).linear(x)
        assert torch.isfinite(y[0]).all() and torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()


@pytest.mark.parametrize("dtype", list(DTYPE))
def test_strides(dtype):
    """Rows within wider ones, off 16 bytes, of three dimensions, turned round; a vector."""
    rng = np.random.default_rng(3)
    codes, scale = plain_form(rng, 48, 256, 64)
    weights, w = quantized.Weights4.pack(codes, scale), numbers(codes, scale)
    room = inputs_of(rng, 12, 301, dtype)
    for at in (0, 1, 8):
        close(weights.linear(room[:, at:at + 256]), room[:, at:at + 256], w, 64)
    x = inputs_of(rng, 12, 256, dtype)
    assert torch.equal(weights.linear(x.view(3, 4, 256)).view(12, 48), weights.linear(x))
    assert torch.equal(weights.linear(x[5]), weights.linear(x[5:6])[0])
    assert torch.equal(weights.linear(x[:1].expand(4, 256)), weights.linear(x[:1].repeat(4, 1)))
    assert torch.equal(weights.linear(x[::2]), weights.linear(x[::2].contiguous()))
    out = torch.empty(12, 48, dtype=x.dtype, device="cuda")
    assert weights.linear(x, out=out).data_ptr() == out.data_ptr()


@pytest.mark.parametrize("dtype", list(DTYPE))
def test_captured(dtype):
    rng = np.random.default_rng(8)
    codes, scale = plain_form(rng, 512, 1024, 128)
    weights = quantized.Weights4.pack(codes, scale)
    x = inputs_of(rng, 3, 1024, dtype)
    weights.linear(x)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(weights.linear(x))
        graphs.append(graph)
    x.copy_(inputs_of(rng, 3, 1024, dtype))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for graph, stream in zip(graphs, streams):
        with torch.cuda.stream(stream):
            graph.replay()
    torch.cuda.synchronize()
    want = weights.linear(x)
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_refusals():
    codes, scale = torch.zeros(16, 64, dtype=torch.uint8, device="cuda"), torch.zeros(16, 2, device="cuda")
    with pytest.raises(TypeError):
        quantized.Weights4.pack(codes, scale)
    scale = scale.bfloat16()
    for bad in ((codes.cpu(), scale), (codes, scale[:8]), (codes, scale[:, :0]), (codes[:, ::2], scale),
                (codes, torch.zeros(16, 8, device="cuda").bfloat16()), (codes[0], scale)):
        with pytest.raises(ValueError):
            quantized.Weights4.pack(*bad)
    weights = quantized.Weights4.pack(codes, scale)
    x = torch.zeros(4, 128, device="cuda")
    for bad in (x[:, :64], x[0, 0], x.T, torch.zeros(2, 3, 256, device="cuda")[:, :2, :128].transpose(0, 1)[:, :, ::2]):
        with pytest.raises(ValueError):
            weights.linear(bad)
    with pytest.raises(TypeError):
        weights.linear(x.double())
    with pytest.raises(ValueError):
        weights.linear(x, out=torch.zeros(4, 15, device="cuda"))
    with pytest.raises(ValueError):
        weights.linear(x.requires_grad_())
    with pytest.raises(TypeError):
        weights.dequantise(torch.int32)
    with pytest.raises(ValueError):
        quantized.quantise(torch.zeros(4, 100, device="cuda"))
    with pytest.raises(ValueError):
        quantized.quantise(torch.zeros(4, 128, device="cuda"), group=48)
