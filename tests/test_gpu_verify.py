"""cb_verify_draft: the emitted tokens equal the rule in exact integers, and are distributed as the target's."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cuda_b200 import speculative
from oracle import paged as plain
from paged_helpers import DTYPE

pytestmark = pytest.mark.gpu


def inputs(rng, batch, n, vocab, dtype):
    logits = rng.normal(0, 2, (batch, n + 1, vocab))
    other = logits[:, :n] + rng.normal(0, 0.7, (batch, n, vocab))

    def probabilities(x):
        x = np.exp(x - x.max(-1, keepdims=True)) if x.size else x
        return torch.from_numpy((x / x.sum(-1, keepdims=True)).astype(np.float32)).cuda().to(DTYPE[dtype])

    target, draft = probabilities(logits), probabilities(other)
    tokens = torch.from_numpy(rng.integers(0, min(vocab, 5), (batch, n))).cuda()
    uniforms = torch.from_numpy(rng.random((batch, n + 1))).cuda()
    return target, draft, tokens, uniforms


def rule(target, draft, tokens, uniforms, counts=None):
    host = [t.float().cpu().numpy() if t.is_floating_point() and t.dtype != torch.float64 else t.cpu().numpy()
            for t in (target, draft, tokens, uniforms)]
    rows = [plain.verify(*(h[b] for h in host), tokens.shape[1] if counts is None else counts[b])
            for b in range(tokens.shape[0])]
    return [r[0] for r in rows], [r[1] for r in rows]


def check_rows(args, counts=None):
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    accepted, emitted = speculative.verify(*args, counts=None if counts is None else torch.tensor(
        counts, dtype=torch.int32, device="cuda"), error_flag=flag)
    want = rule(*args, counts)
    assert accepted.tolist() == want[0]
    assert emitted.tolist() == want[1]
    return flag


@pytest.mark.parametrize("dtype", list(DTYPE))
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 32000, 150001])
def test_tokens(dtype, vocab):
    rng = np.random.default_rng(vocab)
    for n in (0, 1, 4):
        speculative.check(check_rows(inputs(rng, 5, n, vocab, dtype)))


def test_counts_and_strides():
    """Fewer drafts in some rows; probabilities as slices of wider rows at odd offsets."""
    rng = np.random.default_rng(3)
    target, draft, tokens, uniforms = inputs(rng, 6, 5, 777, "f32")
    wide = torch.zeros(6, 6, 801, device="cuda")
    wide[..., 5:782] = target
    turned = draft.transpose(0, 1).contiguous().transpose(0, 1)
    check_rows((wide[..., 5:782], turned, tokens, uniforms), [0, 1, 5, 3, 2, 4])


def test_degenerate_rows():
    """Equal models with u near one, a draft that covers the target, unnormalised and zero weights, u at its ends."""
    target = torch.zeros(7, 2, 40, device="cuda")
    draft = torch.zeros(7, 1, 40, device="cuda")
    tokens = torch.zeros(7, 1, dtype=torch.int64, device="cuda")
    uniforms = torch.full((7, 2), 0.5, dtype=torch.float64, device="cuda")
    target[:, :, 3], target[:, :, 7] = 0.25, 0.75
    draft[0, 0, :2] = 0.5                       # refused: the target gives token 0 nothing
    draft[1, 0] = target[1, 0]
    tokens[1, 0] = 9                            # 0 < 0 refuses, and nothing is left over: drawn from the target
    draft[2, 0, 0], target[2, 0] = 1.0, 0.0     # no weight anywhere: -1 and the flag
    target[3, 0, 5], uniforms[3] = 3.0, 0.999   # weights above one are one
    uniforms[4, 1] = 0.0
    uniforms[5, 1] = 1.0 - 2.0 ** -53
    draft[3:, 0, 0] = 1.0
    target[6, 0, 39] = float("nan")
    flag = check_rows((target, draft, tokens, uniforms))
    with pytest.raises(ValueError):
        speculative.check(flag)
    speculative.check(flag)


def test_draft_outside_the_vocabulary_is_refused():
    rng = np.random.default_rng(5)
    args = inputs(rng, 2, 2, 50, "f32")
    args[2][0, 0], args[2][1, 1] = -1, 50
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    accepted, emitted = speculative.verify(*args, error_flag=flag)
    assert accepted[0] == 0 and accepted[1] <= 1
    with pytest.raises(IndexError):
        speculative.check(flag)


def test_emitted_tokens_follow_the_target():
    """First emitted tokens of many rows: their counts within 5 deviations of the target's probabilities."""
    rng = np.random.default_rng(11)
    rows, vocab = 40000, 12
    target, draft, _, _ = inputs(rng, 1, 1, vocab, "f32")
    q = draft[0, 0].double().cpu().numpy()
    tokens = torch.from_numpy(rng.choice(vocab, rows, p=q / q.sum())).cuda().view(rows, 1)
    uniforms = torch.from_numpy(rng.random((rows, 2))).cuda()
    _, emitted = speculative.verify(target.expand(rows, 2, vocab), draft.expand(rows, 1, vocab), tokens, uniforms)
    counts = np.bincount(emitted[:, 0].cpu().numpy(), minlength=vocab)
    p = target[0, 0].double().cpu().numpy()
    p /= p.sum()
    assert (np.abs(counts - rows * p) <= 5 * np.sqrt(rows * p * (1 - p)) + 1).all()


def test_refusals():
    target, draft, tokens, uniforms = inputs(np.random.default_rng(0), 2, 3, 20, "f32")
    bad = [(target[:, :3], draft, tokens, uniforms), (target, draft.half(), tokens, uniforms),
           (target, draft, tokens.int(), uniforms), (target, draft, tokens, uniforms.float()),
           (target, draft, tokens, uniforms[:, :3]), (target.cpu(), draft, tokens, uniforms),
           (target.transpose(1, 2), draft, tokens, uniforms), (target.double(), draft.double(), tokens, uniforms)]
    for args in bad:
        with pytest.raises((TypeError, ValueError)):
            speculative.verify(*args)
    with pytest.raises(ValueError):
        speculative.verify(target, draft, tokens, uniforms, counts=torch.zeros(3, dtype=torch.int32, device="cuda"))
    accepted, emitted = speculative.verify(target[:0], draft[:0], tokens[:0], uniforms[:0])
    assert accepted.shape == (0,) and emitted.shape == (0, 4)
