"""The serving example: the operators in the order that a program calls them."""

from __future__ import annotations

import importlib.util
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("speculative_paged", ROOT / "examples" / "speculative_paged.py")
    module = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = module
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("storage", ["int8", "e4m3"])
def test_serving(example, storage):
    result = example.main(["--storage", storage, "--tokens", "40"])
    again = example.main(["--storage", storage, "--tokens", "40"])
    assert result["emitted"] == again["emitted"]
    assert all(len(s) >= 40 and min(s) >= 0 and max(s) < 4096 for s in result["emitted"])
    # drafts of the target itself: its probabilities come from a block instead of single tokens
    assert example.main(["--storage", storage, "--tokens", "40", "--same"])["accepted"] >= 0.9


def test_a_block_equals_single_tokens(example):
    """The same tokens as one block, one at a time, and after a truncation give the same probabilities.

    The caches differ in when a page's scale grew (older rows are requantised,
    half a step of 1/127 each time), so this is a bound on that: 5% of the
    total variation would be a broken cache, not a rounding.
    """
    device = torch.device("cuda", 0)
    tokens = torch.from_numpy(np.random.default_rng(0).integers(0, 4096, (2, 37))).to(device)
    counts = torch.tensor([37, 20], dtype=torch.int32, device=device)
    block, single = example.build("int8", 3, 2, True, device)
    want = block(tokens, counts)
    steps = [single(tokens[:, i:i + 1], (counts > i).int()) for i in range(37)]
    got = torch.cat(steps, 1)
    for b, n in enumerate(counts.tolist()):
        assert float((got[b, :n] - want[b, :n]).abs().sum(-1).max()) / 2 < 0.05
    single.cache.truncate([5, 0])
    again = single(tokens[:, 32:37], torch.tensor([5, 0], dtype=torch.int32, device=device))
    assert float((again[0] - want[0, 32:]).abs().sum(-1).max()) / 2 < 0.05
    for decoder in (block, single):
        decoder.cache.check_errors()
        assert decoder.cache.lengths.tolist() == [37, 20]
