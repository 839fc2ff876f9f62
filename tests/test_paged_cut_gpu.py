"""Attention over a paged cache (fk_sdpa_paged) where tiles are cut along their positions and joined: what the parts are, what they leave in the workspace, against
the statement in 64 bits.  Tolerances: those of test_paged_gpu.py."""
import numpy as np
import pytest

import oracle
from helpers import normal_bf16, rng
from paged_reference import Paged, attention, wide
from test_paged_gpu import attend, check_attention
from test_paged_graph_gpu import Graph, stream  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def test_a_falling_row_start_leaves_the_workspace_ready(fk):
    """More tiles than rows account for, the last of them long: what such a batch writes is undefined, what the next one does is not."""
    n_heads, n_kv, dim, rows = 64, 8, 64, 30
    starts = [0]
    while len(starts) < 131:                                  # ten sequences of three rows, then back to the first row
        starts.append(starts[-1] + 3 if starts[-1] < 30 else 0)
    lens = np.full(130, 3, np.uint32)
    lens[[i for i in range(120, 130) if starts[i + 1] > starts[i]][-3:]] = 60000
    fault = fk.zeros(4)
    up = fk.DeviceBuffer.from_numpy
    pages = [up(normal_bf16(i, (4, n_kv, 64, dim))) for i in (1, 2)]
    d = [up(np.array(starts, np.uint32)), up(lens), up(np.zeros((130, 938), np.uint32))]
    q, out = up(normal_bf16(3, (rows, n_heads * dim))), fk.zeros(2 * rows * n_heads * dim)
    ws = fk.zeros(fk.SDPA_PAGED_WORKSPACE_MOST)
    fk.sdpa_paged(q, n_heads * dim, out, n_heads * dim, n_heads, 0.125, 0.0, 0, fk.PagedBatch(*d, 938, 130, rows, 4, 60000, fault),
                  fk.PagePool(*pages, 4, 64, n_kv, dim), ws, ws.nbytes)
    with pytest.raises(fk.InvalidArgument, match="row_start"):
        fk.paged_check(fault)
    assert not ws.to_numpy(np.uint8)[:16384].any()
    check_attention(fk, Paged([1], [9000], n_kv, dim, 64, seed=1), n_heads, workspace=ws)


def test_a_falling_row_start_with_chunks_leaves_the_workspace_ready(fk):
    n_heads, n_kv, dim = 64, 64, 64
    starts = [0, 400, 401, 0, 400, 401, 402]                  # two chunks over the same rows, long tokens behind both
    lens = np.array([400, 60000, 500, 400, 60000, 60000], np.uint32)
    fault = fk.zeros(4)
    up = fk.DeviceBuffer.from_numpy
    pages = [up(normal_bf16(i, (4, n_kv, 64, dim))) for i in (1, 2)]
    d = [up(np.array(starts, np.uint32)), up(lens), up(np.zeros((6, 938), np.uint32))]
    q, out = up(normal_bf16(3, (402, n_heads * dim))), fk.zeros(2 * 402 * n_heads * dim)
    ws = fk.zeros(fk.SDPA_PAGED_WORKSPACE_MOST)
    fk.sdpa_paged(q, n_heads * dim, out, n_heads * dim, n_heads, 0.125, 0.0, 0, fk.PagedBatch(*d, 938, 6, 402, 400, 60000, fault),
                  fk.PagePool(*pages, 4, 64, n_kv, dim), ws, ws.nbytes)
    with pytest.raises(fk.InvalidArgument, match="row_start"):
        fk.paged_check(fault)
    assert not ws.to_numpy(np.uint8)[:16384].any()
    check_attention(fk, Paged([1], [9000], 8, dim, 64, seed=1), n_heads, workspace=ws)


def attention_of_chunks(p, q, n_heads, scale, softcap=0.0, window=0):
    """paged_reference.attention, a head's rows together."""
    out, size, at = np.zeros((sum(p.rows), n_heads, p.dim)), np.zeros((sum(p.rows), n_heads, p.dim)), 0
    for i, (r, n) in enumerate(zip(p.rows, p.lens)):
        k, v = (np.ascontiguousarray(p.gathered(i, a).transpose(1, 0, 2)) for a in (p.k, p.v))
        pos = np.arange(n - r, n)[:, None] - np.arange(n)
        seen = (pos >= 0) & (pos < window if window else True)
        bad = ~np.isfinite(k).all(-1) | ~np.isfinite(v).all(-1)                 # (only where rows that see none of them are looked at)
        for h in range(n_heads):
            g = h // (n_heads // p.n_kv)
            kk, vv = (np.where(bad[g][:, None], 0.0, a[g]) for a in (k, v))
            x = wide(q[at:at + r, h]) @ kk.T * scale
            if softcap:
                x = softcap * np.tanh(x / softcap)
            x = np.where(seen, x, -np.inf)
            w = np.exp(x - x.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            out[at:at + r, h], size[at:at + r, h] = w @ vv, w @ np.abs(vv)
        at += r
    return out, size


def parts_left(ws, slot_columns, dim):
    """Slots of a workspace, zero before, that a launch has written into."""
    slot = slot_columns * (dim + 2) * 4
    held = ws.to_numpy(np.uint8)[16384:]
    return int(held[:len(held) // slot * slot].reshape(-1, slot).any(-1).sum())


def within(got, ref, size):
    return bool((np.abs(wide(got) - ref) <= 2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -11) * size).all())


def check_cut(fk, p, n_heads, softcap=0.0, window=0, chunks=(0,), fine=slice(None)):
    ws = fk.zeros(fk.sdpa_paged_workspace_bytes(n_heads, p.n_kv, p.dim, len(p.rows), sum(p.rows), max(p.lens)))
    q, got, _ = attend(fk, p, n_heads, softcap=softcap, window=window, workspace=ws)
    tiles = sum(-(-p.rows[i] * n_heads // p.n_kv // 128) for i in chunks) * p.n_kv
    assert parts_left(ws, 128, p.dim) >= 2 * tiles            # every tile of the chunks was cut
    assert not ws.to_numpy(np.uint8)[:16384].any()
    ref, size = attention_of_chunks(p, q, n_heads, p.dim ** -0.5, softcap, window)
    assert np.isfinite(wide(got[fine])).all() and within(got[fine], ref[fine], size[fine])
    assert bool((attend(fk, p, n_heads, softcap=softcap, window=window, workspace=ws)[1] == got).all())   # again, on what the first left
    return got


@pytest.mark.parametrize("rows,length", [(64, 1500), (130, 3000), (300, 3100), (33, 9001), (9, 12000)])
@pytest.mark.parametrize("n_heads,n_kv,dim,page_rows", [(8, 2, 128, 64), (14, 2, 64, 16), (5, 1, 128, 256), (4, 4, 64, 32)])
def test_cut_chunks(fk, rows, length, n_heads, n_kv, dim, page_rows):
    rows = max(rows, 32 // (n_heads // n_kv) + 1)              # (fewer columns are tiles of 16)
    p = Paged([rows], [length], n_kv, dim, page_rows, seed=rows)
    check_cut(fk, p, n_heads)


@pytest.mark.parametrize("window,softcap", [(900, 0.0), (0, 20.0), (2111, 30.0)])
@pytest.mark.parametrize("n_heads,n_kv,dim", [(8, 2, 128), (7, 1, 64)])
def test_cut_chunks_with_window_and_cap(fk, window, softcap, n_heads, n_kv, dim):
    check_cut(fk, Paged([130], [4000], n_kv, dim, 32, seed=window), n_heads, softcap, window)
    check_cut(fk, Paged([64, 40], [3000, 2500], n_kv, dim, 16, seed=window + 1), n_heads, softcap, window, chunks=(0, 1))


@pytest.mark.parametrize("rows,lens,chunks", [([130, 1, 1], [3130, 5000, 70], (0,)), ([1, 70, 0, 2, 100], [9000, 2000, 300, 2500, 2600], (1, 4)),
                                              ([200, 1], [2500, 2300], (0,))])
@pytest.mark.parametrize("n_heads,n_kv,dim,window", [(8, 2, 128, 0), (14, 2, 64, 1500)])
def test_cut_chunks_among_long_tokens(fk, rows, lens, chunks, n_heads, n_kv, dim, window):
    check_cut(fk, Paged(rows, lens, n_kv, dim, 64, seed=len(rows)), n_heads, window=window, chunks=chunks)


@pytest.mark.parametrize("bad_bits", [0x7F80, 0xFF80, 0x7FC0])
@pytest.mark.parametrize("dim", [64, 128])
def test_infinities_and_nan_in_masked_places_of_cut_chunks(fk, bad_bits, dim):
    p = Paged([100, 1], [3100, 4000], 2, dim, 32, seed=5)
    for i, at in ((0, np.r_[3095:3100]), (1, np.r_[0:500]), (0, np.r_[0:900])):   # the chunk's last rows; before the windows
        page, slot = p.where(i, at)
        p.k[page, :, slot] = bad_bits
        p.v[page, :, slot] = bad_bits
    fine = np.r_[0:95, 100]
    got = attend(fk, p, 8, window=2000)[1]
    if bad_bits == 0x7FC0:
        assert np.isnan(wide(got[95:100])).all()
        check_nan = got[fine]
        ws = fk.zeros(fk.sdpa_paged_workspace_bytes(8, 2, dim, 2, 101, 4000))
        assert bool((attend(fk, p, 8, window=2000, workspace=ws)[1][fine] == check_nan).all())
    q = normal_bf16(3, (101, 8, dim), std=2.0)
    ref, size = attention_of_chunks(p, q, 8, dim ** -0.5, 0.0, 2000)
    assert np.isfinite(wide(got[fine])).all() and within(got[fine], ref[fine], size[fine])


def test_a_bad_page_in_a_cut_chunk(fk):
    fault = fk.zeros(4)
    p = Paged([70, 60], [2300, 3100], 2, 128, 16, seed=6)
    p.table[0, 100] = p.n_pages + 3
    q, got, _ = attend(fk, p, 8, fault=fault)
    p.table[0, 100] = 0
    ref, size = attention_of_chunks(p, q, 8, 128 ** -0.5)
    assert within(got[70:], ref[70:], size[70:])
    with pytest.raises(fk.InvalidArgument, match="page id"):
        fk.paged_check(fault)


# ---------------------------------------------------------------- the probabilities of few columns: 16 bits

@pytest.mark.parametrize("rows,lens,n_heads,n_kv", [([1], [2], 4, 2), ([1] * 5, [2, 3, 17, 40, 150], 8, 1), ([1], [5000], 8, 1),          # 8 columns, whole and cut
                                                    ([1, 1], [2, 9], 16, 1), ([3, 2], [3, 33], 10, 1), ([1], [4000], 24, 1),             # 16
                                                    ([60, 1, 2, 1], [60, 2, 31, 700], 8, 1), ([100, 1], [2500, 3000], 8, 2)])            # among chunks
@pytest.mark.parametrize("dim", [64, 128])
def test_probabilities_of_few_columns_have_16_bits(fk, rows, lens, n_heads, n_kv, dim):
    """Exact scores (one dim differs from 0) and values that nearly cancel, so that the output's own rounding does not hide a probability's.  It is the sum of two
    bf16 values: off by 2^-8 2^-8 of itself; exponentials and sums in fp32 2^-20 A, A = sum p |v| / sum p; the output's rounding 2^-8 of it."""
    few = [i for i, r in enumerate(rows) if r * n_heads // n_kv <= 32]
    p = Paged(rows, lens, n_kv, dim, 16, seed=7)
    g = rng(dim + sum(lens))
    for i, n in enumerate(lens):
        page, slot = p.where(i, np.arange(n))
        k = np.zeros((n, n_kv, dim), np.float32)
        k[..., 0] = -g.random((n, n_kv)) * (0.5 if n < 100 else 8)
        sign = np.where((np.arange(n)[:, None, None] + g.integers(0, 2, (1, n_kv, dim))) % 2, 1, -1)
        v = sign * (1 + 0.05 * g.random((n, n_kv, dim)))

        p.k[page, :, slot], p.v[page, :, slot] = oracle.f32_to_bf16(k), oracle.f32_to_bf16(v.astype(np.float32))
    q = np.zeros((sum(rows), n_heads, dim), np.uint16)
    q[..., 0] = oracle.f32_to_bf16((0.5 + g.random((sum(rows), n_heads))).astype(np.float32))
    _, got, _ = attend(fk, p, n_heads, scale=1.0, q=q)
    ref, a = attention(p, q, n_heads, 1.0)
    start = np.cumsum([0] + rows)
    at = np.concatenate([np.arange(start[i], start[i + 1]) for i in few])
    off = np.abs(wide(got[at]) - ref[at]) - (2.0 ** -8 * np.abs(ref[at]) + (2.0 ** -16 + 2.0 ** -20) * a[at])
    assert off.max() <= 0, off.max()
    # probabilities of one bf16 value would not pass (over thousands of positions their roundings may average out)
    lost = 0
    for i in few:
        k, v = p.gathered(i, p.k), p.gathered(i, p.v)
        for j in range(rows[i]):
            for h in range(n_heads):
                end, kvh = lens[i] - rows[i] + j + 1, h // (n_heads // n_kv)
                x = k[:end, kvh] @ wide(q[start[i] + j, h])
                w = np.exp(x - x.max())
                coarse = wide(oracle.f32_to_bf16(w.astype(np.float32))) @ v[:end, kvh] / w.sum()
                r = start[i] + j
                lost += (np.abs(coarse - ref[r, h]) > 2.0 ** -8 * np.abs(ref[r, h]) + (2.0 ** -16 + 2.0 ** -20) * a[r, h]).sum()
    assert lost > 0 or min(lens[i] for i in few) > 1000


# ---------------------------------------------------------------- captured, and on several streams

class Planned:
    """A call planned for up to `longest` positions, whose lengths are device values."""

    def __init__(self, fk, rows, longest, n_heads, n_kv, dim, seed, page_rows=32):
        self.fk, up = fk, fk.DeviceBuffer.from_numpy
        n, self.rows, self.width = len(rows), sum(rows), n_heads * dim
        per = -(-longest // page_rows)
        table = rng(seed).permutation(n * per).astype(np.uint32)
        self.lens = fk.zeros(4 * n)
        self.d = [up(np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32)), up(table)]
        self.pages = [up(normal_bf16(seed + i, (n * per, n_kv, page_rows, dim))) for i in (1, 2)]
        self.q, self.out = up(normal_bf16(seed + 3, (self.rows, self.width), std=2.0)), fk.zeros(2 * self.rows * self.width)
        self.batch = fk.PagedBatch(self.d[0], self.lens, self.d[1], per, n, self.rows, max(rows), longest)
        self.pool = fk.PagePool(*self.pages, n * per, page_rows, n_kv, dim)
        self.ws, self.shape = fk.zeros(fk.sdpa_paged_workspace_bytes(n_heads, n_kv, dim, n, self.rows, longest)), (n_heads, dim)

    def run(self, stream=None, out=None, workspace=None):
        n_heads, dim = self.shape
        ws = workspace or self.ws
        self.fk.sdpa_paged(self.q, self.width, out or self.out, self.width, n_heads, dim ** -0.5, 0.0, 0, self.batch, self.pool, ws, ws.nbytes, stream)


@pytest.mark.parametrize("rows", [[70, 1], [1, 100, 2], [40]])
@pytest.mark.parametrize("n_heads,n_kv,dim", [(8, 2, 128), (14, 2, 64)])
def test_cut_chunks_in_a_graph_whose_lengths_change(fk, stream, rows, n_heads, n_kv, dim):  # noqa: F811
    st = stream()
    a = Planned(fk, rows, 6000, n_heads, n_kv, dim, seed=20 + len(rows))
    plain, ws = fk.zeros(a.out.nbytes), fk.zeros(a.ws.nbytes)
    a.lens.upload(np.array([5000] * len(rows), np.uint32))
    a.run(st)
    fk.sync(st)
    g = Graph(fk, st, lambda: a.run(st))
    for i, length in enumerate((6000, 700, 3001, 5999, 150, 6000)):
        a.lens.upload(np.array([max(r, length - 37 * j) for j, r in enumerate(rows)], np.uint32))
        g.replay()
        fk.sync(st)
        a.run(st, plain, ws)
        fk.sync(st)
        assert np.array_equal(a.out.to_numpy(np.uint16), plain.to_numpy(np.uint16)), i
        assert not a.ws.to_numpy(np.uint8)[:16384].any()
    g.free()


def test_cut_chunks_on_two_streams_at_once(fk, stream):  # noqa: F811
    one, two = stream(), stream()
    a, b = (Planned(fk, r, 5000, 8, 2, 128, seed=s) for r, s in (([90, 1], 31), ([1, 60, 1], 41)))
    for p in (a, b):
        p.lens.upload(np.array([5000 - 400 * i for i in range(p.batch.n_seqs)], np.uint32))
    want = []
    for p in (a, b):
        p.run()
        fk.sync()
        want.append(p.out.to_numpy(np.uint16))
        p.out.upload(np.zeros(p.rows * p.width, np.uint16))
    for _ in range(8):
        a.run(one)
        b.run(two)
    for st, p, w in ((one, a, want[0]), (two, b, want[1])):
        fk.sync(st)
        assert np.array_equal(p.out.to_numpy(np.uint16), w)
