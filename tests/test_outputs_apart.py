"""An ``out`` that lies over an argument is refused: other blocks read that while it is written."""

from __future__ import annotations

import pytest
import torch

from cuda_b200 import logits
from cuda_b200.paged import PagedCache, meet, reach
from cuda_b200.quantized import Weights4


def test_spans():
    room = torch.zeros(4, 64)
    assert reach(room) == 1024 and reach(room[:, :8]) == 3 * 256 + 32 and reach(room[:0]) == 0
    assert reach(room[0].expand(9, 64)) == 256 and reach(room.bfloat16()[1:, ::2]) == 2 * 128 + 63 * 2
    assert meet(100, 10, 109, 1) and not meet(100, 10, 110, 5) and not meet(110, 5, 100, 10)
    assert not meet(100, 10, 100, 0) and not meet(100, 0, 90, 100)


def test_adjust_apart():
    """The check by itself, on host memory: which arguments an out may lie over."""
    room = torch.zeros(3, 64)
    rows, flag = room[:, :40], torch.zeros(1, dtype=torch.int32)
    tokens, allowed = room.view(torch.int32)[:, 48:], torch.zeros(3, 2, dtype=torch.int32)

    def check(out, source=rows, **more):
        spans = {"logits": reach(source), "out": reach(out)} | {name: reach(t) for name, t in more.items()}
        logits.apart(source, out, spans, [(name, t.data_ptr()) for name, t in more.items()], flag)

    check(rows)
    check(torch.zeros(3, 40), tokens=tokens, allowed=allowed)
    check(rows, allowed=allowed)
    for out, more in ((room[:, 1:41], {}), (rows, {"tokens": tokens}), (allowed.view(torch.float32), {"allowed": allowed}),
                      (flag.view(torch.float32).expand(1, 1), {})):
        with pytest.raises(ValueError, match="out "):
            check(out, **more)


@pytest.mark.gpu
def test_adjust_refuses():
    room = torch.zeros(8, 64, device="cuda")
    words = room.view(torch.int32)
    x = torch.zeros(4, 64, device="cuda")
    for name, more in (("tokens", dict(tokens=words[3:7, :9])), ("bias", dict(bias_tokens=words[4:, :9].clone(), bias=room[3:7, :9])),
                       ("bias_tokens", dict(bias_tokens=words[3:7, :9], bias=room[4:, :9].clone())),
                       ("allowed", dict(allowed=words[3:7, :2])), ("lengths", dict(tokens=words[4:], lengths=words[0, :4])),
                       ("presences", dict(tokens=words[4:], presence=room[1, 3:7])), ("error_flag", dict(error_flag=words[3, 63:]))):
        with pytest.raises(ValueError, match=name):
            logits.adjust(x, out=room[:4], **more)
    rows = torch.randn(4, 64, device="cuda")
    words.zero_()
    want = logits.adjust(rows, tokens=words[4:], presence=0.5)
    assert logits.adjust(rows, tokens=words[4:], presence=0.5, out=room[:4]) is not want
    assert torch.equal(room[:4], want)
    assert torch.equal(logits.adjust(rows, tokens=words[4:], presence=0.5, out=rows), want)


@pytest.mark.gpu
def test_weights_refuse():
    weights = Weights4.quantise(torch.randn(64, 128, device="cuda"), group=32)
    x = torch.randn(2, 128, device="cuda")
    codes, scales = weights.codes.clone(), weights.scales.clone()
    for name, out in (("codes", weights.codes[:512].view(torch.float32).view(2, 64)),
                      ("scales", weights.scales.view(torch.float32)[:128].view(2, 64)), ("x", x.view(-1)[64:192].view(2, 64))):
        with pytest.raises(ValueError, match=name):
            weights.linear(x, out=out)
    room = torch.zeros(64 * 64 * 2 + 64 * 128 * 2, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="codes"):  # the last of the codes, in a buffer that holds both
        over = Weights4(room[:weights.codes.numel()], weights.scales, outputs=64, inputs=128, group=32)
        over.dequantise(out=room[weights.codes.numel() - 16:][:64 * 128 * 2].view(torch.bfloat16).view(64, 128))
    assert torch.equal(weights.codes, codes) and torch.equal(weights.scales, scales)
    over = Weights4(room[:weights.codes.numel()], weights.scales, outputs=64, inputs=128, group=32)
    over.codes.copy_(codes)
    behind = room[weights.codes.numel():][:64 * 128 * 2].view(torch.bfloat16).view(64, 128)
    assert torch.equal(over.dequantise(out=behind), weights.dequantise(torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["attend", "attend_shared"])
def test_attention_refuses(name):
    """Pools, scales and book in one buffer with the output, queries that it partly covers; the queries' own place."""
    q = torch.randn(2, 3, 4, 64, device="cuda")
    sizes = [1 * 8 * 2 * 16 * 64] * 2 + [4 * 16] * 2 + [4 * (2 * 4 + 2 + 16 + 1)]
    room = torch.zeros(sum(sizes) + 16 * 1024, dtype=torch.uint8, device="cuda")
    starts = [0, sizes[0], sum(sizes[:2]), sum(sizes[:3]), sum(sizes[:4])]
    parts = [room[a:a + n] for a, n in zip(starts, sizes)]
    pools = [p.view(torch.int8).view(1, 8, 2, 16, 64) for p in parts[:2]]
    scales = [p.view(torch.float32).view(1, 8, 2) for p in parts[2:4]]
    book = parts[4].view(torch.int32)
    book[:8].fill_(-1)
    book[10 + 8:10 + 16] = torch.arange(8, device="cuda")
    book[-1] = 8
    cache = PagedCache(*pools, *scales, book, sequences=2, pages_per_sequence=4)
    cache.extend([20, 30])
    for at, what in ((0, "k_pages"), (sizes[0] + 16, "v_pages"), (starts[2], "k_scale"), (starts[3], "v_scale"),
                     (starts[4] // 16 * 16 + 16, "the book")):
        out = room[at:at + 2 * 3 * 4 * 64 * 4].view(torch.float32).view(2, 3, 4, 64)
        with pytest.raises(ValueError, match=what):
            getattr(cache, name)(0, q, out=out)
    wide = torch.randn(3, 3, 4, 64, device="cuda")
    with pytest.raises(ValueError, match="q"):
        getattr(cache, name)(0, wide[:2], out=wide[1:])
    words = torch.ones(3 * 3 * 4 * 64, dtype=torch.int32, device="cuda")
    for more in ("counts", "sequences"):
        with pytest.raises(ValueError, match=more):
            getattr(cache, name)(0, q, out=words[4:].view(torch.float32)[:2 * 3 * 4 * 64].view(2, 3, 4, 64),
                                 **{more: words[8:10]})
    rows = torch.randn(2, 50, 2, 64, device="cuda")
    cache.append(0, rows[:, :20], rows[:, 20:40], counts=[20, 20])
    more = {"least_bytes": 0} if name == "attend_shared" else {}
    want = getattr(cache, name)(0, q, **more)
    assert getattr(cache, name)(0, q, out=q, **more) is q and torch.equal(q, want)
    cache.check_errors()
