"""attend_shared right behind the calls that wrote what it reads, without a wait between: pages, scales and
tables that change from one step to the next."""

from __future__ import annotations

import pytest
import torch

from cuda_b200.paged import PagedCache
from paged_helpers import DTYPE

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("storage", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("captured", [False, True])
def test_fresh_pages(dtype, storage, captured):
    """Prompts of other magnitudes take the same pages in other orders; results equal those after everything is done."""
    samples, prompt, heads, size = 40, 2000, 8, 64
    cache = PagedCache.allocate(layers=2, pages=400, kv_heads=heads, page_size=16, head_size=size, sequences=samples,
                                pages_per_sequence=140, storage=storage)
    gen = torch.Generator(device="cuda").manual_seed(3)

    def ints(*values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    first, length, ones = ints(0), ints(prompt), torch.ones(samples, dtype=torch.int32, device="cuda")
    parents, children = torch.zeros(samples - 1, dtype=torch.int32, device="cuda"), torch.arange(1, samples, device="cuda").int()
    k, v = (torch.empty(1, prompt, heads, size, dtype=DTYPE[dtype], device="cuda") for _ in range(2))
    q = torch.empty(samples, 1, 4 * heads, size, dtype=DTYPE[dtype], device="cuda")
    everyone = torch.arange(samples, device="cuda").int()

    def step():
        cache.release(everyone)
        cache.extend(length, sequences=first)
        for layer in range(2):
            cache.append(layer, k, v, sequences=first)
        cache.fork(parents, children)
        cache.extend(ones)
        outs = []
        for layer in range(2):
            cache.append(layer, k[:, :1].expand(samples, 1, heads, size), v[:, 5:6].expand(samples, 1, heads, size))
            outs.append(cache.attend_shared(layer, q, least_bytes=0))
        return outs

    def fill(i):
        for x, scale in ((k, 0.5 + i % 3), (v, 2.0 ** (i % 5 - 2)), (q, 1.0)):
            x.copy_(scale * torch.randn(x.shape, device="cuda", generator=gen))

    fill(0)
    step()
    graph = torch.cuda.CUDAGraph()
    if captured:
        with torch.cuda.graph(graph):
            outs = step()
    for i in range(12):
        fill(i)
        torch.cuda.synchronize()
        if captured:
            graph.replay()
        else:
            outs = step()
        torch.cuda.synchronize()
        cache.check_errors()
        for layer in range(2):
            assert torch.equal(outs[layer], cache.attend_shared(layer, q, least_bytes=0))
            whole = cache.attend(layer, q).float()
            assert torch.isfinite(whole).all() and (outs[layer].float() - whole).abs().max() < 0.05 * whole.abs().max()
