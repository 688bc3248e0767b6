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
