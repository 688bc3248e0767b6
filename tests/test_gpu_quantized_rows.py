"""4-bit products of as many rows as a call takes: whole numbers, so that every sum is exact."""

from __future__ import annotations

import pytest
import torch

from cuda_b200 import _lib
from cuda_b200.quantized import Weights4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, most", [(torch.bfloat16, 2097120), (torch.float16, 2097120), (torch.float32, 655350)])
@pytest.mark.parametrize("off", [0, 1])
def test_most_rows(dtype, most, off):
    gen = torch.Generator(device="cuda").manual_seed(most + off)
    codes = torch.randint(0, 256, (20, 32), device="cuda", generator=gen, dtype=torch.uint8)
    weights = Weights4.pack(codes, torch.ones(20, 1, dtype=torch.bfloat16, device="cuda"))
    room = torch.randint(-4, 5, (most + 1, 64 + off), device="cuda", generator=gen, dtype=torch.int8).to(dtype)
    x = room[:most, off:]
    got = weights.linear(x)
    want = (x.float() @ weights.dequantise(torch.float32).T).to(dtype)  # sums below 2^12
    assert torch.equal(got, want)
    with pytest.raises(_lib.KernelError, match="at most"):
        weights.linear(room[:, off:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("outputs", [100, 5920, 10650, 40250])
@pytest.mark.parametrize("group, inputs", [(32, 2048), (64, 5632), (128, 4096), (128, 1152)])
def test_roundings_of_every_form(dtype, outputs, group, inputs):
    """Blocks of 16, 8 and 4 warps, one tile and two: as many roundings as the most that any of them makes.

    Of what the terms of a sum add up to: each product of 16 inputs adds within 2^-22 (of float32's second and third
    parts, 2^-8 and 2^-16 of the first, as many more); a warp of at least four adds its units of 128 inputs group by
    group; then up to 16 warps are added, and of float32 its three parts as well; last comes the output's rounding.
    """
    gen = torch.Generator(device="cuda").manual_seed(outputs + inputs)
    weights = Weights4.quantise(torch.randn(outputs, inputs, device="cuda", generator=gen), group=group)
    w = weights.dequantise(torch.float32).double()
    adds = -(-inputs // 128 // 4) * (128 // group) + group // 128 + 15 + (32 if dtype == torch.float32 else 0)
    products = group / 16 * (1 + 2.0 ** -7 if dtype == torch.float32 else 1)
    for rows in (1, 3, 9, 16, 24, 40):
        x = torch.randn(rows, inputs, device="cuda", generator=gen).to(dtype)
        got = weights.linear(x).double()
        want, size = x.double() @ w.T, x.double().abs() @ w.abs().T
        error = (products * 2.0 ** -22 + adds * 2.0 ** -24) * size
        assert ((got - want).abs() <= error + torch.finfo(dtype).eps / 2 * (want.abs() + error)).all()
