"""Attention over a paged cache through a window with the first positions visible besides (fk_sdpa_paged_sinks), against a plain statement in 64 bits.

Tolerances: those of attention over a paged cache -- the probabilities as bf16, 2^-8 of A = sum p |v| / sum p; one rounding of the output, 2^-8 of it; fp32
scores, 2^-11 of A."""
import numpy as np
import pytest

from decode_loop_reference import attention
from helpers import normal_bf16, rng
from paged_reference import Paged, wide
from test_paged_graph_gpu import Graph, stream  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def attend(fk, p, n_heads, window, sinks, seed=3, softcap=0.0, q=None, rows=None, pad=0, plain=False, **sizes):
    n = sum(p.rows)
    q = normal_bf16(seed, (n, n_heads, p.dim), std=2.0) if q is None else q
    rows, stride = rows or max(1, n), n_heads * p.dim + pad
    qb = np.full((rows, stride), 0x7FC0, np.uint16)
    qb[:n, :n_heads * p.dim] = q.reshape(n, -1)
    batch, pool = p.device(fk, rows=rows, **sizes)
    out = fk.DeviceBuffer.from_numpy(np.full((rows, stride), 0x4242, np.uint16))
    ws = fk.zeros(fk.sdpa_paged_workspace_bytes(n_heads, p.n_kv, p.dim, len(p.rows), rows, batch.max_len))
    args = (fk.DeviceBuffer.from_numpy(qb), stride, out, stride, n_heads, p.dim ** -0.5, softcap, window)
    if plain:
        fk.sdpa_paged(*args, batch, pool, ws, ws.nbytes)
    else:
        fk.sdpa_paged_sinks(*args, sinks, batch, pool, ws, ws.nbytes)
    fk.sync()
    whole = out.to_numpy(np.uint16, (rows, stride))
    assert bool((whole[n:] == 0x4242).all() and (whole[:, n_heads * p.dim:] == 0x4242).all())   # nothing else is written
    return q, whole[:n, :n_heads * p.dim].reshape(n, n_heads, p.dim)


def check(fk, p, n_heads, window, sinks, softcap=0.0, **more):
    q, got = attend(fk, p, n_heads, window, sinks, softcap=softcap, **more)
    with np.errstate(all="ignore"):
        ref, size = attention(p, q, n_heads, p.dim ** -0.5, window, sinks, softcap)
    got = wide(got)
    assert np.isfinite(got).all()
    off = np.abs(got - ref) - (2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -11) * size)
    assert off.max() <= 0, (off.max(), np.unravel_index(off.argmax(), off.shape))


@pytest.mark.parametrize("sinks", [1, 4, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 5000])
@pytest.mark.parametrize("window", [1, 16, 100, 129])
@pytest.mark.parametrize("n_heads,n_kv,dim", [(8, 2, 128), (14, 2, 64)])
def test_one_token(fk, window, sinks, n_heads, n_kv, dim):
    check(fk, Paged([1, 1, 1, 1], [700, 333, 64, 1], n_kv, dim, 16, seed=sinks), n_heads, window, sinks)


@pytest.mark.parametrize("sinks", [1, 5, 63, 64, 65, 130, 400])
@pytest.mark.parametrize("window", [1, 40, 64, 200])
@pytest.mark.parametrize("n_heads,n_kv,dim,page_rows", [(8, 2, 128, 16), (7, 1, 64, 32), (4, 2, 64, 256)])
def test_chunks_and_tokens(fk, window, sinks, n_heads, n_kv, dim, page_rows):
    check(fk, Paged([150, 1, 7, 0, 1], [430, 600, 90, 12, 1], n_kv, dim, page_rows, seed=window), n_heads, window, sinks)
    check(fk, Paged([70], [70], n_kv, dim, page_rows, seed=window), n_heads, window, sinks)


@pytest.mark.parametrize("window,sinks,softcap", [(0, 9, 0.0), (200, 17, 30.0), (0, 3, 5.0), (90, 0, 0.0)])
def test_without_a_window_and_with_a_cap(fk, window, sinks, softcap):
    check(fk, Paged([40, 1, 1], [300, 700, 20], 2, 128, 32, seed=5), 8, window, sinks, softcap=softcap)
    check(fk, Paged([1, 2], [500, 260], 2, 64, 16, seed=6), 4, window, sinks, softcap=softcap)


@pytest.mark.parametrize("n_heads,n_kv", [(1, 1), (16, 1), (40, 1), (33, 3), (130, 1)])
def test_head_layouts(fk, n_heads, n_kv):
    check(fk, Paged([3, 1], [400, 260], n_kv, 64, 16, seed=4), n_heads, 100, 70)
    check(fk, Paged([1], [660], n_kv, 128, 16, seed=5), n_heads, 200, 33)


def test_long_contexts_cut_along_their_positions(fk):
    """Items of one tile on both sides of the gap, and a gap of many pages."""
    check(fk, Paged([1], [9985], 1, 128, 64, seed=7), 4, 3000, 700)
    check(fk, Paged([1, 1, 2], [6145, 3, 2000], 2, 64, 16, seed=8), 14, 1500, 300)
    check(fk, Paged([130, 1], [5000, 4000], 1, 128, 32, seed=9), 4, 1500, 900)
    check(fk, Paged([64], [8000], 2, 64, 16, seed=10), 4, 2000, 1000)


def test_many_sequences(fk):
    lens = [int(n) for n in rng(1).integers(1, 400, 150)]
    check(fk, Paged([1] * 150, lens, 2, 64, 16, seed=6), 4, 90, 40)


def test_strides_and_plans_for_longer_contexts(fk):
    check(fk, Paged([4, 0, 1], [500, 7, 300], 2, 64, 16, seed=9, spare_table=300), 4, 120, 10, rows=11, pad=24, max_rows=9, max_len=4000)


@pytest.mark.parametrize("bad", [0x7F80, 0xFF80, 0x7FC0])
@pytest.mark.parametrize("dim,page_rows", [(64, 16), (128, 64)])
def test_what_lies_between_sinks_and_window_reaches_no_row(fk, dim, page_rows, bad):
    """Infinities and NaN in the positions that no row sees."""
    p = Paged([20, 1, 1], [500, 900, 150], 2, dim, page_rows, seed=11)
    for i, (lo, hi) in enumerate(((5, 380), (5, 799), (5, 49))):     # sinks 5, window 100: the first row of the chunk sees 381 on
        page, slot = p.where(i, np.arange(lo, hi))
        p.k[page, :, slot] = bad
        p.v[page, :, slot] = bad
    check(fk, p, 4, 100, 5)


def test_infinities_that_some_rows_see(fk):
    p = Paged([20, 1], [300, 200], 2, 64, 16, seed=12)
    page, slot = p.where(0, np.arange(295, 300))                    # the last five rows of the chunk
    p.k[page, :, slot] = p.v[page, :, slot] = 0x7FC0
    page, slot = p.where(1, np.arange(3, 4))                        # a sink of the second
    p.k[page, :, slot] = p.v[page, :, slot] = 0x7FC0
    q, got = attend(fk, p, 4, 50, 4)
    assert np.isnan(wide(got[15:])).all()
    with np.errstate(all="ignore"):
        ref, size = attention(p, q, 4, 0.125, 50, 4)
    off = np.abs(wide(got[:15]) - ref[:15]) - (2.0 ** -8 * np.abs(ref[:15]) + (2.0 ** -8 + 2.0 ** -11) * size[:15])
    assert off.max() <= 0


def test_scores_beyond_what_fp32_s_exponents_tell_apart(fk):
    """Scores of 1e10: rows that are done again, position by position, on both sides of the gap."""
    p = Paged([1, 40], [400, 300], 1, 64, 16, seed=13)
    q = normal_bf16(14, (41, 2, 64), std=2.0e9)
    _, got = attend(fk, p, 2, 60, 20, q=q)
    ref, size = attention(p, q, 2, 0.125, 60, 20)
    # one key takes everything but where two scores are nearly the same: fp32's rounding of them decides there
    near = np.abs(wide(got) - ref).max(-1) <= 2.0 ** -7 * np.abs(ref).max(-1) + 2.0 ** -9
    assert np.isfinite(wide(got)).all() and near.mean() > 0.95


def test_rows_that_see_nothing(fk):
    """A length below the new rows."""
    p = Paged([3, 1], [400, 260], 2, 64, 16, seed=14)
    p.kv_len[0] = 2
    _, got = attend(fk, p, 4, 50, 4)
    assert not got[0].any() and got[1:].any(-1).all()


@pytest.mark.parametrize("window", [0, 1, 70, 300])
@pytest.mark.parametrize("rows,lens", [([1, 1], [500, 40]), ([200, 1], [700, 90])])
def test_no_sinks_is_the_window_alone_bit_for_bit(fk, window, rows, lens):
    p = Paged(rows, lens, 2, 128, 16, seed=15)
    assert np.array_equal(attend(fk, p, 8, window, 0)[1], attend(fk, p, 8, window, 0, plain=True)[1])
    assert np.array_equal(attend(fk, p, 8, 0, 77)[1], attend(fk, p, 8, 0, 0, plain=True)[1])


def test_replays_while_lengths_grow(fk, stream):  # noqa: F811
    st = stream()
    p = Paged([1, 30, 1], [900, 700, 500], 2, 64, 16, seed=16)
    batch, pool = p.device(fk)
    q = normal_bf16(17, (32, 4, 64), std=2.0)
    d_q, out, ws = fk.DeviceBuffer.from_numpy(q), fk.zeros(2 * q.size), fk.zeros(fk.SDPA_PAGED_WORKSPACE_MOST)
    call = lambda: fk.sdpa_paged_sinks(d_q, 256, out, 256, 4, 0.125, 0.0, 200, 20, batch, pool, ws, ws.nbytes, st)
    call()
    fk.sync(st)
    g = Graph(fk, st, call)
    for lens in ([300, 400, 5], [900, 30, 500], [221, 700, 220], [1, 250, 499]):
        p.d[1].upload(np.array(lens, np.uint32))
        g.replay()
        fk.sync(st)
        r = Paged(p.rows, lens, 2, 64, 16)
        r.table, r.k, r.v, r.lens = p.table, p.k, p.v, lens
        ref, size = attention(r, q, 4, 0.125, 200, 20)
        off = np.abs(wide(out.to_numpy(np.uint16, q.shape)) - ref) - (2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -11) * size)
        assert off.max() <= 0, lens
    g.free()


@pytest.mark.parametrize("window,sinks", [(2 ** 32 - 1, 2 ** 32 - 1), (2 ** 32 - 1, 7), (1, 2 ** 32 - 1), (1, 2 ** 31), (599, 1), (600, 1), (2 ** 31, 2 ** 31 + 1)])
def test_windows_and_sinks_of_any_size(fk, window, sinks):
    check(fk, Paged([1, 1, 0], [600, 1, 5], 2, 64, 16, seed=8), 8, window, sinks)
    check(fk, Paged([90, 1], [600, 30], 2, 128, 32, seed=9), 8, window, sinks)
