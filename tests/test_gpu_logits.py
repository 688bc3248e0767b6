"""cb_adjust_logits against the rule in float64: penalties, biases and masks on logit rows."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cuda_b200 import logits as operators
from cuda_b200 import speculative
from oracle import logits as plain
from paged_helpers import DTYPE, wide

pytestmark = pytest.mark.gpu


def tensor(x, dtype=None):
    return None if x is None else torch.as_tensor(np.asarray(x), device="cuda", dtype=dtype)


def close(got, rows, given):
    """Each value within the roundings of its own sum, and one of the type; infinities and NaN in their places."""
    half = torch.finfo(got.dtype).eps / 2
    for b, row in enumerate(rows):
        want, size = plain.adjust(row, **{k: (v[b] if isinstance(v, (np.ndarray, list)) else v)
                                          for k, v in given.items()})
        have, want = wide(got[b]), torch.from_numpy(want).to(got.dtype).double().numpy() if got.dtype != torch.float32 \
            else want
        assert np.array_equal(np.isnan(have), np.isnan(want))
        fine = np.isfinite(want)
        assert np.array_equal(have[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
        # six float32 roundings and one for each further bias of a token, then one of the type (two where the exact
        # value was rounded here as well)
        steps = 6 + len(np.atleast_1d(given.get("bias", [[]])[b] if "bias" in given else []))
        have, want, size = have[fine], want[fine], size[fine]
        assert np.all(np.abs(have - want) <= steps * 2.0 ** -24 * size + 2 * half * np.abs(want))


def words_of(bits):
    """One bit a token as int32 words, what is past the vocabulary set."""
    rows, vocab = bits.shape
    padded = np.ones((rows, -(-vocab // 32) * 32), bool)
    padded[:, :vocab] = bits
    value = (padded.reshape(rows, -1, 32).astype(np.uint64) << np.arange(32, dtype=np.uint64)).sum(-1)
    return value.astype(np.uint32).view(np.int32)


def case(rng, rows, vocab, history=0, biases=0, grammar=False, index=np.int32, scalars=False):
    given, call = {}, {}
    if history:
        tokens = rng.integers(-2, max(2, vocab // 3) + 2, (rows, history)).astype(index)  # some of them no tokens
        lengths = rng.integers(0, history + 1, rows).astype(np.int32)
        prompts = (lengths * rng.random(rows)).astype(np.int32)
        given |= {"tokens": tokens, "length": lengths, "prompt": prompts}
        call |= {"tokens": tensor(tokens), "lengths": tensor(lengths), "prompts": tensor(prompts)}
        for name, top in (("repetition", 1.5), ("frequency", 0.7), ("presence", 1.0)):
            value = rng.uniform(0.5, top, rows).astype(np.float32)
            if scalars:
                given[name] = call[name] = float(value[0])
            else:
                given[name], call[name] = value, tensor(value)
    if biases:
        ids = rng.integers(-1, vocab + 1, (rows, biases)).astype(index)
        bias = rng.normal(0, 3, (rows, biases)).astype(np.float32)
        given |= {"bias_tokens": ids, "bias": bias}
        call |= {"bias_tokens": tensor(ids), "bias": tensor(bias)}
    if grammar:
        bits = rng.random((rows, vocab)) < rng.random((rows, 1))
        bits[rows // 2] = False  # nothing is left of this row
        given["allowed"] = words_of(bits)
        call["allowed"] = tensor(given["allowed"])
    return given, call


def rows_of(rng, rows, vocab, dtype):
    return torch.from_numpy(rng.normal(0, 4, (rows, vocab)).astype(np.float32)).cuda().to(DTYPE[dtype])


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("vocab", [1, 7, 8, 31, 32, 33, 1000, 4095, 4097, 8192, 32003])
def test_everything_together(dtype, vocab):
    rng = np.random.default_rng(vocab)
    x = rows_of(rng, 3, vocab, dtype)
    given, call = case(rng, 3, vocab, 77, 9, True, scalars=vocab % 2 == 0)
    close(operators.adjust(x, **call), wide(x), given)


@pytest.mark.parametrize("what", [{}, {"history": 1}, {"history": 1500}, {"biases": 1}, {"biases": 1023},
                                  {"grammar": True}, {"history": 40, "grammar": True}, {"history": 9, "biases": 700}])
def test_one_at_a_time(what):
    rng = np.random.default_rng(len(str(what)))
    x = rows_of(rng, 5, 9000, "f32")
    given, call = case(rng, 5, 9000, index=np.int64, **what)
    close(operators.adjust(x, **call), wide(x), given)


def test_tokens_listed_many_times():
    """One token in all of a history, and biases of one token that are added in the list's order: equal bits."""
    rng = np.random.default_rng(1)
    x = rows_of(rng, 2, 500, "f32")
    tokens = np.full((2, 3000), 17, np.int32)
    ids, bias = np.full((2, 600), 17, np.int32), rng.normal(0, 1, (2, 600)).astype(np.float32)
    call = dict(tokens=tensor(tokens), frequency=0.25, presence=0.5, repetition=1.25, bias_tokens=tensor(ids),
                bias=tensor(bias))
    got = operators.adjust(x, **call)
    close(got, wide(x), dict(tokens=tokens, frequency=0.25, presence=0.5, repetition=1.25, bias_tokens=ids, bias=bias))
    want = np.float32(bias[0, 0])
    for b in bias[0, 1:]:
        want = np.float32(want + b)
    assert all(torch.equal(operators.adjust(x, **call), got) for _ in range(3))
    alone = operators.adjust(torch.zeros_like(x), bias_tokens=tensor(ids), bias=tensor(bias))
    assert float(alone[0, 17]) == float(want)


def test_infinities_and_nan():
    x = torch.tensor([[np.inf, -np.inf, np.nan, 1.0, -1.0, 0.0, -0.0, np.nan]], device="cuda")
    tokens = np.arange(8, dtype=np.int32)[None]
    bias, ids = np.array([[-np.inf, np.inf]], np.float32), np.array([[3, 4]], np.int32)
    allowed = np.array([[0x7F]], np.int32)
    got = operators.adjust(x, tokens=tensor(tokens), repetition=2.0, presence=1.0, bias_tokens=tensor(ids),
                           bias=tensor(bias), allowed=tensor(allowed))
    close(got, wide(x), dict(tokens=tokens, repetition=2.0, presence=1.0, bias_tokens=ids, bias=bias, allowed=allowed))
    low = torch.full((2, 100), torch.finfo(torch.float16).min, dtype=torch.float16, device="cuda")
    got = operators.adjust(low, tokens=tensor(np.zeros((2, 3), np.int32)), repetition=1.5)
    assert torch.isinf(got[:, 0]).all() and torch.equal(got[:, 1:], low[:, 1:])


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("at, out_at", [(0, 0), (1, 1), (3, 3), (1, 2), (8, 0)])
def test_strides_and_in_place(dtype, at, out_at):
    """Rows within wider ones, that begin off 16 bytes alike or not; out apart or the logits themselves."""
    rng = np.random.default_rng(at)
    given, call = case(rng, 4, 4100, 60, 12, True)
    room = torch.full((4, 4133), 5.0, device="cuda", dtype=DTYPE[dtype])
    x = room[:, at:at + 4100]
    x.copy_(rows_of(rng, 4, 4100, dtype))
    before = wide(x)
    target = torch.full((4, 4117), 7.0, device="cuda", dtype=DTYPE[dtype])
    out = target[:, out_at:out_at + 4100]
    got = operators.adjust(x, **call, out=out)
    assert got.data_ptr() == out.data_ptr()
    close(got, before, given)
    assert (target[:, :out_at] == 7).all() and (target[:, out_at + 4100:] == 7).all()
    same = operators.adjust(x, **call, out=x)
    assert torch.equal(same.nan_to_num(), got.nan_to_num())
    assert (room[:, :at] == 5).all() and (room[:, at + 4100:] == 5).all()


def test_shared_rows():
    """One history, bias list and mask that all rows share, by expanding them; one row of logits for all."""
    rng = np.random.default_rng(9)
    given, call = case(rng, 1, 3001, 30, 5, True, scalars=True)
    call["allowed"] |= torch.tensor(0x55555555, dtype=torch.int32, device="cuda")
    given["allowed"] = call["allowed"].cpu().numpy()
    x = rows_of(rng, 1, 3001, "bf16").expand(6, 3001)
    for name in ("tokens", "bias_tokens", "bias", "allowed"):
        call[name] = call[name].expand(6, call[name].shape[1])
    for name in ("lengths", "prompts"):
        call[name] = call[name].repeat(6)
    close(operators.adjust(x, **call), wide(x), {k: (np.repeat(v, 6, 0) if isinstance(v, np.ndarray) else v)
                                                 for k, v in given.items()})


def test_lengths_outside_the_history():
    rng = np.random.default_rng(4)
    x = rows_of(rng, 4, 64, "f32")
    tokens = rng.integers(0, 64, (4, 20)).astype(np.int32)
    lengths, prompts = np.array([-1, 21, 5, 5], np.int32), np.array([0, 0, -3, 9], np.int32)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = operators.adjust(x, tokens=tensor(tokens), lengths=tensor(lengths), prompts=tensor(prompts), presence=1.0,
                           repetition=1.5, error_flag=flag)
    close(got, wide(x), dict(tokens=tokens, length=lengths, prompt=prompts, presence=1.0, repetition=1.5))
    with pytest.raises(IndexError):
        speculative.check(flag)
    speculative.check(flag)


def test_empty_and_captured():
    assert operators.adjust(torch.zeros(0, 50, device="cuda")).shape == (0, 50)
    assert operators.adjust(torch.zeros(3, 0, device="cuda")).shape == (3, 0)
    rng = np.random.default_rng(6)
    given, call = case(rng, 8, 32000, 200, 16, True)
    x = rows_of(rng, 8, 32000, "bf16")
    want = operators.adjust(x, **call)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    out = torch.empty_like(x)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        operators.adjust(x, **call, out=out)
    other = rows_of(rng, 8, 32000, "bf16")
    x.copy_(other)
    graph.replay()
    assert torch.equal(out, operators.adjust(other, **call))
    x.copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    close(out, wide(other), given)
    assert want.shape == out.shape


def test_refusals():
    x = torch.zeros(4, 64, device="cuda")
    tokens = torch.zeros(4, 3, dtype=torch.int32, device="cuda")
    bias = torch.zeros(4, 3, device="cuda")
    bad = [dict(tokens=tokens[:2]), dict(tokens=tokens, repetition=0.0), dict(tokens=tokens, presence=float("nan")),
           dict(presence=1.0), dict(lengths=torch.zeros(4, dtype=torch.int32, device="cuda")), dict(bias=bias),
           dict(bias_tokens=tokens), dict(bias_tokens=tokens, bias=bias[:, :2]),
           dict(allowed=torch.zeros(4, 3, dtype=torch.int32, device="cuda")), dict(out=x[:, 1:]),
           dict(out=torch.zeros(64, device="cuda").expand(4, 64)), dict(tokens=tokens.cpu()),
           dict(bias_tokens=torch.zeros(4, 1024, dtype=torch.int32, device="cuda"),
                bias=torch.zeros(4, 1024, device="cuda"))]
    for call in bad:
        with pytest.raises(ValueError):
            operators.adjust(x, **call)
    for call in (dict(tokens=tokens.float()), dict(tokens=tokens, frequency=torch.zeros(4, dtype=torch.float64,
                                                                                        device="cuda")),
                 dict(allowed=torch.zeros(4, 2, dtype=torch.int64, device="cuda"))):
        with pytest.raises(TypeError):
            operators.adjust(x, **call)
    with pytest.raises(TypeError):
        operators.adjust(x.double())
    room = torch.zeros(5, 64, device="cuda")
    with pytest.raises(ValueError):
        operators.adjust(room[:4], out=room[1:])
    with pytest.raises(ValueError):
        operators.adjust(x.requires_grad_())
