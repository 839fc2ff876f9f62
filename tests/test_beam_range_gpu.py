"""Beam search's selection (fk_beam_select) over the whole range of bf16 logits and fp32 scores: masks of the type's lowest value, logits and scores of its
largest, against a statement in 64 bits that subtracts a row's largest logit first.

Beams and tokens are compared exactly: by the total, then the beam, inside it by the logits, then the token.  A score is a sum of the row's score, a logit
and the logarithm of a sum of exponentials that are each off by at most 2^-21 of themselves, and is rounded to fp32 once: 2^-21 + 2^-24 |score|."""
import numpy as np
import pytest

import oracle
from helpers import normal_bf16, rng
from paged_reference import wide
from test_beam_gpu import select

pytestmark = pytest.mark.gpu
LOWEST, LARGEST = 0xFF7F, 0x7F7F


def plain(logits, scores, finished, pad, groups, n_beams, k):
    x = wide(logits)
    m = x.max(-1, keepdims=True)
    total = scores.astype(np.float64)[:, None] + ((x - m) - np.log(np.exp(x - m).sum(-1, keepdims=True)))
    if finished is not None:
        over = finished != 0
        total[over] = -np.inf
        total[over, pad] = scores[over]
    vocab = x.shape[1]
    out = []
    for g in range(groups):
        rows = slice(g * n_beams, (g + 1) * n_beams)
        beam, token = (i.ravel() for i in np.indices((n_beams, vocab)))
        t = total[rows].ravel()
        order = np.lexsort((token, -x[rows].ravel(), beam, -t))
        alive = order[t[order] > -np.inf][:k]
        rest = np.setdiff1d(np.arange(min(t.size, 2 * k)), alive)[:k - len(alive)]     # (the lowest places that are left)
        order = np.concatenate([alive, rest])
        out.append((np.where(np.arange(k) < len(alive), t[order], -np.inf), beam[order], token[order]))
    return [np.stack(a) for a in zip(*out)]


def check(fk, logits, scores, groups, n_beams, k, finished=None, pad=0):
    scores = np.asarray(scores, np.float32)
    got = select(fk, logits, scores, groups, n_beams, k, finished, pad)
    ref = plain(logits, scores, finished, pad, groups, n_beams, k)
    assert bool((got[1] == ref[1]).all() and (got[2] == ref[2]).all())
    with np.errstate(over="ignore"):
        far = np.isinf(ref[0].astype(np.float32))
    assert bool(np.isneginf(got[0][far]).all())
    assert bool((np.abs(got[0][~far] - ref[0][~far]) <= 2.0 ** -21 + 2.0 ** -24 * np.abs(ref[0][~far])).all())


def make(seed, rows, vocab):
    return normal_bf16(seed, (rows, vocab), std=3.0), (-20 * rng(seed + 1).random(rows) - 1).astype(np.float32)


# 4 x 3 rows in pieces of 2048 tokens, 40 x 4 of more than 8192 in pieces of 8192
@pytest.mark.parametrize("groups,n_beams,vocab,k", [(4, 3, 300, 6), (4, 3, 5000, 6), (4, 3, 40001, 8), (40, 4, 40001, 8), (1, 4, 151851, 40)])
def test_masks_of_the_lowest_value(fk, groups, n_beams, vocab, k):
    x, s = make(vocab + k, groups * n_beams, vocab)
    allowed = rng(k).integers(0, vocab, (groups * n_beams, 5))       # a few tokens of every beam
    for r, t in enumerate(allowed):
        keep = x[r, t].copy()
        x[r] = LOWEST
        x[r, t] = keep
    check(fk, x, s, groups, n_beams, k)
    y, s = make(vocab + k + 1, groups * n_beams, vocab)
    y[::2, vocab // 3:] = LOWEST                                     # a run of tokens, as long as a wave's or a piece's and longer
    y[1::2, :vocab // 2] = LOWEST
    check(fk, y, s, groups, n_beams, k)


@pytest.mark.parametrize("groups,n_beams,vocab", [(2, 4, 700), (2, 4, 9000), (40, 4, 40001)])
def test_rows_without_a_choice(fk, groups, n_beams, vocab):
    """Every logit the lowest: the row is uniform, and its tokens follow one another."""
    x, s = make(vocab, groups * n_beams, vocab)
    x[1::2] = LOWEST
    check(fk, x, s, groups, n_beams, 12)
    s[1::2] = -0.5                                                   # (a uniform row ahead of the others by its score, not by a sum that was lost)
    check(fk, x, s, groups, n_beams, 12)
    x[:] = LOWEST
    check(fk, x, np.arange(groups * n_beams) * -0.25, groups, n_beams, 12)


@pytest.mark.parametrize("groups,n_beams,vocab", [(2, 4, 700), (2, 4, 9000), (40, 4, 40001)])
def test_logits_of_the_largest_value(fk, groups, n_beams, vocab):
    x, s = make(vocab + 1, groups * n_beams, vocab)
    x[0, 5] = LARGEST
    x[1, [7, vocab - 1]] = LARGEST
    x[2] = LARGEST
    x[3, vocab // 2] = LARGEST
    x[3, vocab // 2 + 1:] = LOWEST                                   # (twice the type's range apart)
    check(fk, x, s, groups, n_beams, 9)


@pytest.mark.parametrize("offset", [1e3, 1e6, 3e7, 1e9, 1e20, 1e35, 2.6e38])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_logits(fk, offset, sign):
    for groups, n_beams, vocab in ((2, 3, 5001), (40, 4, 40001)):
        g = rng(int(np.log10(offset)))
        x = oracle.f32_to_bf16((sign * offset * (1 + 0.02 * g.standard_normal((groups * n_beams, vocab)))).astype(np.float32))
        check(fk, x, -g.random(groups * n_beams), groups, n_beams, 7)


@pytest.mark.parametrize("score", [-1e10, -1e17, -1e30, -1e37, -3.3895314e38, -3.4028235e38])
def test_scores_that_logits_are_lost_in(fk, score):
    """A beam that took a masked token: its continuations are still in the order of its logits, and behind the other beams'."""
    x, _ = make(9, 6, 3000)
    lost = score * (1 - np.arange(6) / 16)                           # (far apart, so that beams do not meet)
    check(fk, x, np.where([1, 0, 1, 0, 1, 1], lost, [0, -1, 0, -2, 0, 0]), 2, 3, 10)
    check(fk, np.repeat(x[:1], 6, 0), np.full(6, score), 2, 3, 10)    # equal beams: the lower first
    x[:, 4:] = LOWEST                                                # totals beyond fp32: listed as -inf, in their order
    check(fk, x, np.where([1, 0, 1, 0, 1, 1], lost, [0, -1, 0, -2, 0, 0]), 2, 3, 20)
    check(fk, x, np.where([1, 0, 1, 0, 0, 1], lost, -np.inf), 2, 3, 20)


def test_masks_and_finished_beams(fk):
    x, s = make(12, 8, 6000)
    x[:, 3:] = LOWEST
    f = np.array([0, 1, 0, 0, 1, 1, 0, 0])
    check(fk, x, s, 2, 4, 16, finished=f, pad=5999)
    s[1] = -3e38
    check(fk, x, s, 2, 4, 16, finished=f, pad=2)


def test_steps_under_a_mask(fk):
    """The scores of one step are those of the next, as a search that may take one token a step has them."""
    s = np.zeros(4, np.float32)
    s[1:] = -np.inf
    for step in range(5):
        x, _ = make(40 + step, 4, 5000)
        keep = x[:, 17 + step].copy()
        x[:] = LOWEST
        x[:, 17 + step] = keep
        check(fk, x, s, 1, 4, 4)
        s = select(fk, x, s, 1, 4, 4)[0][0]
        assert s[0] == 0.0


def test_scores_in_place(fk):
    """What a search without host steps does: the new scores where the old ones were."""
    groups, n_beams, vocab = 9, 5, 5003
    x, s = make(50, groups * n_beams, vocab)
    s = s.astype(np.float32)
    d, scores = fk.DeviceBuffer.from_numpy(x), fk.DeviceBuffer.from_numpy(s)
    outs = [fk.zeros(4 * groups * n_beams) for _ in range(2)]
    ws = fk.zeros(fk.beam_select_workspace_bytes(groups, n_beams, vocab, n_beams))
    for _ in range(3):
        ref = plain(x, s, None, 0, groups, n_beams, n_beams)
        fk.beam_select(d, vocab, scores, None, 0, groups, n_beams, vocab, n_beams, scores, *outs, ws, ws.nbytes)
        fk.sync()
        got = [b.to_numpy(t, (groups, n_beams)) for b, t in zip((scores, *outs), (np.float32, np.uint32, np.uint32))]
        assert bool((got[1] == ref[1]).all() and (got[2] == ref[2]).all())
        assert bool((np.abs(got[0] - ref[0]) <= 2.0 ** -21 + 2.0 ** -24 * np.abs(ref[0])).all())
        s = got[0].ravel()
