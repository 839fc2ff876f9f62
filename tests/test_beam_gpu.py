"""Beam search's selection (fk_beam_select) and the rows of state that follow it (fk_beam_reorder) against plain statements in 64 bits.

Beams and tokens are compared exactly; a score is a sum of the row's score, a logit and the logarithm of a sum of exponentials
that are each off by at most 2^-21 of themselves, and is rounded to fp32 once: 2^-21 + 2^-24 |score|."""
import numpy as np
import pytest

import oracle
from helpers import normal_bf16, rng
from paged_reference import beams as plain
from paged_reference import wide

pytestmark = pytest.mark.gpu


def select(fk, logits, scores, groups, n_beams, k, finished=None, pad=0, stride=None, shift=0, workspace=None):
    vocab = logits.shape[1]
    stride = stride or vocab
    raw = np.full((logits.shape[0], stride), 0x7F80, np.uint16)       # between the rows: never read
    raw[:, :vocab] = logits
    d = fk.DeviceBuffer.from_numpy(np.concatenate([np.full(shift, 0x7F80, np.uint16), raw.reshape(-1)]))
    outs = [fk.DeviceBuffer.from_numpy(np.full((groups, k), 0x55555555, np.uint32)) for _ in range(3)]
    ws = workspace or fk.zeros(fk.beam_select_workspace_bytes(groups, n_beams, vocab, k))
    fin = None if finished is None else fk.DeviceBuffer.from_numpy(finished.astype(np.uint32))
    fk.beam_select(d.ptr + 2 * shift, stride, fk.DeviceBuffer.from_numpy(scores.astype(np.float32)), fin, pad, groups, n_beams, vocab, k, *outs, ws, ws.nbytes)
    fk.sync()
    return tuple(o.to_numpy(t, (groups, k)) for o, t in zip(outs, (np.float32, np.uint32, np.uint32)))


def check(fk, logits, scores, groups, n_beams, k, finished=None, pad=0, **more):
    got = select(fk, logits, scores, groups, n_beams, k, finished, pad, **more)
    ref = plain(wide(logits), scores.astype(np.float32), finished, pad, groups, n_beams, k)
    assert bool((got[1] == ref[1]).all() and (got[2] == ref[2]).all())
    far = np.isinf(ref[0])
    assert bool((got[0][far] == ref[0][far]).all())
    assert bool((np.abs(got[0][~far] - ref[0][~far]) <= 2.0 ** -21 + 2.0 ** -24 * np.abs(ref[0][~far])).all())


def make(seed, groups, n_beams, vocab, std=3.0):
    return normal_bf16(seed, (groups * n_beams, vocab), std=std), (-20 * rng(seed + 1).random(groups * n_beams) - 1).astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 63, 64, 65, 255, 256, 257, 1000, 2047, 2048, 2049, 8191, 8193, 32000, 70001])
@pytest.mark.parametrize("groups,n_beams,k", [(1, 1, 1), (2, 4, 8), (3, 5, 5)])
def test_sizes(fk, vocab, groups, n_beams, k):
    k = min(k, n_beams * vocab)
    check(fk, *make(vocab, groups, n_beams, vocab), groups, n_beams, k)


@pytest.mark.parametrize("groups,n_beams,k", [(1, 64, 64), (7, 1, 64), (2, 3, 64), (40, 8, 16), (1, 16, 32), (300, 2, 3)])
def test_beams_and_k(fk, groups, n_beams, k):
    check(fk, *make(k, groups, n_beams, 3001), groups, n_beams, k)


def test_more_lists_than_are_held_at_once(fk):
    check(fk, *make(4, 2, 64, 70001), 2, 64, 64)
    check(fk, *make(4, 1, 64, 70001, std=0.05), 1, 64, 64)    # ties, too


def test_large_vocabulary(fk):
    check(fk, *make(5, 2, 8, 260003), 2, 8, 16)
    check(fk, *make(6, 1, 1, 151936), 1, 1, 1)


@pytest.mark.parametrize("shift,stride", [(0, 1003), (1, 1001), (3, 1008), (5, 1001)])
def test_rows_at_any_address(fk, shift, stride):
    check(fk, *make(7, 3, 4, 1001), 3, 4, 8, shift=shift, stride=stride)


def test_ties_go_to_the_lowest_place(fk):
    for vocab in (50, 5000, 40000):
        x = np.zeros((4, vocab), np.uint16)                       # everything equal: beams are equal too
        check(fk, x, np.full(4, -2.0), 1, 4, 9)
        x[:, vocab // 2] = 0x8000                                  # -0 is 0
        check(fk, x, np.full(4, -2.0), 1, 4, 9)
        x, s = make(8, 1, 4, vocab, std=0.5)
        x[1], x[3] = x[0], x[2]                                    # the same rows and scores twice
        s[1], s[3] = s[0], s[2]
        check(fk, x, s, 1, 4, 16)
        x = oracle.f32_to_bf16(rng(9).integers(0, 3, (4, vocab)).astype(np.float32))
        check(fk, x, np.array([-1.0, -1.0, -3.0, -1.0]), 1, 4, 40)


def test_rows_alike_at_unlike_addresses(fk):
    """A row's sum does not depend on where it lies: equal beams stay equal where rows are an odd number of values apart."""
    x, _ = make(10, 1, 1, 50001)
    x = np.repeat(x, 6, 0)
    check(fk, x, np.full(6, -3.0), 1, 6, 12)
    check(fk, x, np.full(6, -3.0), 2, 3, 6, shift=3, stride=50003)


def test_infinities_and_nan(fk):
    x, s = make(11, 2, 4, 900)
    x[0, 100:] = 0xFF80                # masked tokens
    x[1] = 0xFF80                      # nothing left in a beam
    x[2, 5] = 0x7FC0                   # NaN counts as -inf
    x[3, :] = 0x7FC0
    x[4, 7] = 0x7F80                   # +inf: the row's log softmax is not a number
    s[5] = -np.inf
    s[6] = np.nan
    check(fk, x, s, 2, 4, 16)
    check(fk, np.full((4, 300), 0xFF80, np.uint16), np.zeros(4), 1, 4, 8)


def test_fewer_continuations_than_k(fk):
    x = np.full((3, 40), 0xFF80, np.uint16)
    x[0, 3], x[0, 1], x[2, 0] = 0x3F80, 0x4000, 0x3F80
    check(fk, x, np.array([-1.0, -1.0, -2.0]), 1, 3, 12)
    check(fk, x[:, :4], np.array([-1.0, -1.0, -2.0]), 1, 3, 12)
    check(fk, x, np.array([-1.0, -1.0, -2.0]), 1, 3, 5, finished=np.array([1, 1, 1]), pad=7)


def test_finished_beams(fk):
    x, s = make(12, 3, 4, 2000)
    f = np.array([0, 1, 0, 0, 1, 1, 1, 1, 0, 0, 0, 7])
    s[1] = -0.5
    s[6] = -np.inf
    check(fk, x, s, 3, 4, 8, finished=f, pad=1999)
    check(fk, x, s, 3, 4, 4, finished=np.zeros(12), pad=0)


def test_first_step(fk):
    x, s = make(13, 2, 5, 3000)
    s = np.where(np.arange(10) % 5, -np.inf, 0.0)
    check(fk, np.repeat(x[::5], 5, 0), s, 2, 5, 10)


def test_a_workspace_serves_one_call_after_another(fk):
    """Whatever its shape: also many groups behind one, whose counters lie where sums might have lain."""
    ws = fk.zeros(fk.beam_select_workspace_bytes(40, 8, 20000, 16))
    for i in range(3):
        check(fk, *make(20 + i, 4, 8, 20000), 4, 8, 16, workspace=ws)
        check(fk, *make(30 + i, 1, 3, 500), 1, 3, 4, workspace=ws)
        check(fk, *make(40 + i, 40, 2, 700), 40, 2, 4, workspace=ws)


@pytest.mark.parametrize("row_bytes", [1, 3, 4, 16, 20, 1000, 4096, 65552])
@pytest.mark.parametrize("groups,n_beams,n_out", [(1, 4, 4), (3, 5, 5), (2, 4, 9), (2, 9, 4), (1, 64, 64), (5, 1, 1)])
def test_reorder(fk, row_bytes, groups, n_beams, n_out):
    src = rng(row_bytes).integers(0, 256, (groups, n_beams, row_bytes), dtype=np.uint8)
    parents = rng(n_out).integers(0, n_beams, (groups, n_out)).astype(np.uint32)
    ref = np.take_along_axis(src, parents[:, :, None].astype(np.int64), 1)
    s, p = fk.DeviceBuffer.from_numpy(src), fk.DeviceBuffer.from_numpy(parents)
    dst = fk.DeviceBuffer(ref.nbytes)
    fk.beam_reorder(s, dst, row_bytes, p, groups, n_beams, n_out)
    fk.sync()
    assert bool((dst.to_numpy(np.uint8, ref.shape) == ref).all() and (s.to_numpy(np.uint8, src.shape) == src).all())
    if n_out == n_beams:
        fk.beam_reorder(s, s, row_bytes, p, groups, n_beams, n_out)
        fk.sync()
        assert bool((s.to_numpy(np.uint8, ref.shape) == ref).all())


def test_reorder_takes_the_last_beam_for_an_index_beyond(fk):
    src = np.arange(4 * 32, dtype=np.uint32).reshape(1, 4, 32)
    s, p = fk.DeviceBuffer.from_numpy(src), fk.DeviceBuffer.from_numpy(np.array([3, 4, 0xFFFFFFFF, 0], np.uint32))
    fk.beam_reorder(s, s, 128, p, 1, 4, 4)
    fk.sync()
    assert bool((s.to_numpy(np.uint32, src.shape) == src[:, [3, 3, 3, 0]]).all())


@pytest.mark.parametrize("row,src_stride,dst_stride", [(4, 4, 400), (4, 36, 4), (16, 48, 160), (7, 9, 30), (64, 128, 64)])
@pytest.mark.parametrize("groups,n_beams,n_out", [(1, 4, 4), (3, 5, 5), (2, 3, 20)])
def test_reorder_rows_that_lie_apart(fk, row, src_stride, dst_stride, groups, n_beams, n_out):
    src = rng(row).integers(0, 256, (groups, n_beams, src_stride), dtype=np.uint8)
    old = rng(row + 1).integers(0, 256, (groups, n_out, dst_stride), dtype=np.uint8)
    parents = rng(n_out).integers(0, n_beams, (groups, n_out)).astype(np.uint32)
    s, d, p = fk.DeviceBuffer.from_numpy(src), fk.DeviceBuffer.from_numpy(old), fk.DeviceBuffer.from_numpy(parents)
    fk.beam_reorder(s, d, row, p, groups, n_beams, n_out, src_stride=src_stride, dst_stride=dst_stride)
    fk.sync()
    ref = old.copy()
    ref[:, :, :row] = np.take_along_axis(src, parents[:, :, None].astype(np.int64), 1)[:, :, :row]
    assert bool((d.to_numpy(np.uint8, old.shape) == ref).all())
    if n_out == n_beams:                       # in place, what lies between the rows stays
        fk.beam_reorder(s, s, row, p, groups, n_beams, n_out, src_stride=src_stride, dst_stride=src_stride)
        fk.sync()
        ref = src.copy()
        ref[:, :, :row] = np.take_along_axis(src, parents[:, :, None].astype(np.int64), 1)[:, :, :row]
        assert bool((s.to_numpy(np.uint8, src.shape) == ref).all())
