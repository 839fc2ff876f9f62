"""Several sequences over a paged cache: attention (fk_sdpa_paged), rotary positions and append (fk_rope_paged_store,
fk_rope_frequencies), pages copied (fk_pages_copy), against plain statements in 64 bits.

Tolerances.  Attention: the probabilities enter the second product as bf16, each off by at most 2^-8 of itself, which moves an
output by at most 2^-8 * A with A = sum p |v| / sum p; the output is rounded once, 2^-8 of it; an fp32 score of 128 products
of values below 4 and 6 sigma, times 128^-1/2, is off by less than 128 * 2^-24 * 245 * 0.09 = 1.7e-4, in numerator and
denominator together 2^-11 * A.  Rotation: one rounding, 2^-8 of the value, and a few fp32 operations, 2^-20 of the pair.  What is
moved is moved exactly."""
import math

import numpy as np
import pytest

from helpers import normal_bf16, rng
from paged_reference import Paged, attention, frequencies, rotated, wide

pytestmark = pytest.mark.gpu


def attend(fk, p, n_heads, seed=3, scale=None, softcap=0.0, window=0, q=None, rows=None, pad=0, workspace=None, **sizes):
    """Runs the operator; returns (q, out bits [rows, heads, dim], whole out buffer)."""
    scale = p.dim ** -0.5 if scale is None else scale
    n = sum(p.rows)
    q = normal_bf16(seed, (n, n_heads, p.dim), std=2.0) if q is None else q
    rows = rows or max(1, n)
    stride = n_heads * p.dim + pad
    qb = np.full((rows, stride), 0x7FC0, np.uint16)
    qb[:n, :n_heads * p.dim] = q.reshape(n, -1)
    batch, pool = p.device(fk, rows=rows, **sizes)
    out = fk.DeviceBuffer.from_numpy(np.full((rows, stride), 0x4242, np.uint16))
    need = fk.sdpa_paged_workspace_bytes(n_heads, p.n_kv, p.dim, len(p.rows), rows, batch.max_len)
    ws = workspace or fk.zeros(need)
    fk.sdpa_paged(fk.DeviceBuffer.from_numpy(qb), stride, out, stride, n_heads, scale, softcap, window, batch, pool, ws, ws.nbytes)
    fk.sync()
    whole = out.to_numpy(np.uint16, (rows, stride))
    assert bool((whole[n:] == 0x4242).all() and (whole[:, n_heads * p.dim:] == 0x4242).all())   # nothing else is written
    return q, whole[:n, :n_heads * p.dim].reshape(n, n_heads, p.dim), whole


def check_attention(fk, p, n_heads, softcap=0.0, window=0, **more):
    q, got, _ = attend(fk, p, n_heads, softcap=softcap, window=window, **more)
    ref, size = attention(p, q, n_heads, p.dim ** -0.5, softcap, window)
    got = wide(got)
    assert np.isfinite(got).all()
    off = np.abs(got - ref) - (2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -11) * size)
    assert off.max() <= 0, (off.max(), np.unravel_index(off.argmax(), off.shape))


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500])
@pytest.mark.parametrize("n_heads,n_kv,dim", [(32, 8, 128), (14, 2, 64)])
def test_one_token(fk, length, n_heads, n_kv, dim):
    check_attention(fk, Paged([1], [length], n_kv, dim, 16, seed=length), n_heads)


@pytest.mark.parametrize("rows,lens", [([5], [5]), ([33], [70]), ([64, 1, 7], [64, 300, 20]), ([0, 3, 0, 1], [40, 3, 0, 129]),
                                       ([130], [131]), ([2, 2, 2, 2, 2], [2, 17, 33, 64, 200]), ([200, 1, 1], [333, 1, 1000])])
@pytest.mark.parametrize("n_heads,n_kv,dim,page_rows", [(8, 2, 128, 16), (7, 1, 64, 32), (6, 6, 64, 128), (4, 2, 128, 256)])
def test_chunks_and_tokens(fk, rows, lens, n_heads, n_kv, dim, page_rows):
    check_attention(fk, Paged(rows, lens, n_kv, dim, page_rows, seed=len(rows)), n_heads)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 1000])
@pytest.mark.parametrize("rows,lens", [([1, 1, 1], [300, 64, 5]), ([90, 1], [250, 129])])
def test_window(fk, window, rows, lens):
    check_attention(fk, Paged(rows, lens, 2, 64, 16, seed=window), 4, window=window)
    check_attention(fk, Paged(rows, lens, 2, 128, 64, seed=window), 8, window=window)


@pytest.mark.parametrize("softcap", [0.5, 5.0, 50.0, 1024.0])
@pytest.mark.parametrize("window", [0, 70])
def test_softcap(fk, softcap, window):
    check_attention(fk, Paged([40, 1, 1], [200, 90, 700], 2, 128, 32, seed=1), 8, softcap=softcap, window=window)
    check_attention(fk, Paged([40, 1], [41, 300], 2, 64, 16, seed=2), 2, softcap=softcap, window=window)


@pytest.mark.parametrize("n_heads,n_kv", [(1, 1), (3, 3), (16, 1), (40, 1), (64, 2), (33, 3), (130, 1)])
def test_head_layouts(fk, n_heads, n_kv):
    check_attention(fk, Paged([3, 1], [100, 260], n_kv, 64, 16, seed=4), n_heads)
    check_attention(fk, Paged([1], [260], n_kv, 128, 16, seed=5), n_heads)


def test_many_sequences(fk):
    lens = [int(n) for n in rng(1).integers(1, 150, 150)]
    check_attention(fk, Paged([1] * 150, lens, 2, 64, 16, seed=6), 4)


def test_long_context_few_heads(fk):
    """Far more positions than one workgroup takes, also beside short ones, and a last page of one row."""
    check_attention(fk, Paged([1], [9985], 1, 128, 64, seed=7), 4)
    check_attention(fk, Paged([1, 1, 2], [6145, 3, 2000], 2, 64, 16, seed=8), 14)


def test_rows_behind_the_last_sequence_and_strides(fk):
    p = Paged([4, 0, 1], [50, 7, 30], 2, 64, 16, seed=9)
    check_attention(fk, p, 4, rows=11, pad=24, max_rows=9, max_len=64)


def test_sizes_of_the_launch_do_not_change_a_row_s_positions(fk):
    """A plan for far longer contexts than the batch holds."""
    p = Paged([1, 6], [75, 20], 2, 128, 16, seed=10, spare_table=300)
    check_attention(fk, p, 8, max_len=4000, max_rows=7)


@pytest.mark.parametrize("dim,page_rows", [(64, 16), (128, 64)])
def test_infinities_and_nan_in_masked_places(fk, dim, page_rows):
    """What a row does not see may hold anything: later rows of its own chunk, positions before its window."""
    for bad_bits in (0x7F80, 0xFF80, 0x7FC0):
        p = Paged([20, 1], [90, 200], 2, dim, page_rows, seed=11)
        page, slot = p.where(0, np.arange(85, 90))          # the last five rows of the chunk
        p.k[page, :, slot] = bad_bits
        p.v[page, :, slot] = bad_bits
        page, slot = p.where(1, np.arange(0, 100))          # before the window of the second sequence
        p.k[page, :, slot] = bad_bits
        p.v[page, :, slot] = bad_bits
        q, got, _ = attend(fk, p, 4, window=100)
        with np.errstate(all="ignore"):
            ref, size = attention(p, q, 4, dim ** -0.5, 0.0, 100)
        fine = np.r_[0:15, 20]                              # rows that see none of them
        off = np.abs(wide(got[fine]) - ref[fine]) - (2.0 ** -8 * np.abs(ref[fine]) + (2.0 ** -8 + 2.0 ** -11) * size[fine])
        assert np.isfinite(wide(got[fine])).all() and off.max() <= 0, hex(bad_bits)
        if bad_bits == 0x7FC0:
            assert np.isnan(wide(got[15:20])).all()


def test_values_of_the_type_s_range(fk):
    """Probabilities sum values near bf16's largest without leaving fp32."""
    p = Paged([1, 3], [130, 40], 1, 64, 16, seed=12)
    for i, n in enumerate(p.lens):
        page, slot = p.where(i, np.arange(n))
        p.v[page, :, slot] = 0x7F70
    q, got, _ = attend(fk, p, 2)
    assert bool((np.abs(wide(got) / wide([0x7F70]) - 1) <= 2.0 ** -7 + 2.0 ** -11).all())   # the probabilities' rounding and the output's


def test_scores_far_apart(fk):
    """One key takes everything; scores of thousands."""
    p = Paged([1, 2], [200, 90], 1, 64, 16, seed=13)
    q = normal_bf16(14, (3, 2, 64), std=100.0)
    _, got, _ = attend(fk, p, 2, q=q)
    ref, size = attention(p, q, 2, 0.125)
    # an fp32 score is off by up to 64 * 2^-24 * sum |q k| / 8, sum |q k| below 64 * 130: 4e-3, in numerator and denominator 8e-3, and 2^-8
    assert bool((np.abs(wide(got) - ref) <= 2.0 ** -6 * size + 2.0 ** -8 * np.abs(ref)).all())


def test_a_row_that_sees_nothing_is_zero_and_reported(fk):
    fault = fk.zeros(4)
    p = Paged([3, 1], [3, 20], 1, 64, 16, seed=15)
    p.kv_len[0] = 2                                          # one row more than positions
    p.lens[0] = 2
    q, got, _ = attend(fk, p, 2, fault=fault)
    assert bool((got[0] == 0).all())
    ref, size = attention(p, q, 2, 0.125)
    assert bool((np.abs(wide(got) - ref) <= 2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -11) * size).all())
    with pytest.raises(fk.InvalidArgument, match="length"):
        fk.paged_check(fault)
    fk.paged_check(fault)                                    # cleared


def test_device_values_beyond_the_launch_are_cut_and_reported(fk):
    for change, word in ((lambda p: p.kv_len.__setitem__(0, 4000000000), "length"), (lambda p: p.row_start.__setitem__(1, 900), "row_start"),
                         (lambda p: p.table.__setitem__((0, 0), p.n_pages), "page id"), (lambda p: p.row_start.__setitem__(0, 0xFFFFFFFF), "row_start")):
        fault = fk.zeros(4)
        p = Paged([3, 1], [40, 20], 1, 64, 16, seed=16, poison=0)
        change(p)
        attend_only = dict(fault=fault, max_len=48)
        n = sum(p.rows)
        batch, pool = p.device(fk, rows=n, **attend_only)
        ws = fk.zeros(fk.sdpa_paged_workspace_bytes(2, 1, 64, 2, n, 48))
        out = fk.DeviceBuffer.from_numpy(np.zeros(n * 128, np.uint16))
        qb = fk.DeviceBuffer.from_numpy(normal_bf16(3, (n, 2, 64)))
        fk.sdpa_paged(qb, 128, out, 128, 2, 0.125, 0.0, 0, batch, pool, ws, ws.nbytes)
        with pytest.raises(fk.InvalidArgument, match=word):
            fk.paged_check(fault)


def test_same_call_again_and_between_other_streams_workspaces(fk):
    """The workspace is ready for the next launch, and a row's result does not depend on what ran before."""
    p = Paged([1, 40, 1], [3000, 100, 700], 2, 64, 16, seed=17)
    ws = fk.zeros(fk.sdpa_paged_workspace_bytes(4, 2, 64, 3, 42, 3000))
    first = attend(fk, p, 4, workspace=ws)[1]
    other = Paged([1], [2500], 2, 64, 32, seed=18)
    attend(fk, other, 4, workspace=ws)
    assert bool((attend(fk, p, 4, workspace=ws)[1] == first).all())
    assert bool((attend(fk, p, 4, workspace=fk.zeros(2 * ws.nbytes))[1] == first).all())


# ---------------------------------------------------------------- rotary positions and append

SCALINGS = [dict(scaling="plain"), dict(scaling="linear", factor=4.0), dict(scaling="parts", factor=8.0, low=1.0, high=4.0, trained=8192),
            dict(scaling="ramp", factor=16.0, low=1.0, high=32.0, trained=4096)]


@pytest.mark.parametrize("kind", SCALINGS, ids=lambda s: s["scaling"])
@pytest.mark.parametrize("dims,theta", [(64, 1e4), (128, 1e6), (16, 5e5), (2, 1e4)])
def test_frequencies(fk, kind, dims, theta):
    out = fk.DeviceBuffer(8 * (dims // 2 + 1))
    fk.rope_frequencies(dims, theta, out, **kind)
    fk.sync()
    ref = frequencies(dims, theta, **kind)
    assert np.abs(out.to_numpy(np.float64) / ref - 1).max() <= 64 * 2.0 ** -53   # a pow, a log, a few operations


def store(fk, p, n_heads, rope_dims, interleaved, freq, norms=(None, None), packed=True, in_place=False, rows=None, eps=1e-6, **sizes):
    n, D, nk = sum(p.rows), p.dim, p.n_kv
    rows = rows or n
    width = (n_heads + 2 * nk) * D
    qkv = normal_bf16(21, (rows, width))
    batch, pool = p.device(fk, rows=rows, **sizes)
    dn = [None if w is None else fk.DeviceBuffer.from_numpy(w) for w in norms]
    f = None if freq is None else fk.DeviceBuffer.from_numpy(freq)
    if packed:
        src = fk.DeviceBuffer.from_numpy(qkv)
        args = (src.ptr, width, src.ptr + 2 * n_heads * D, width, src.ptr + 2 * (n_heads + nk) * D, width)
        qs = width
    else:
        parts = [fk.DeviceBuffer.from_numpy(np.ascontiguousarray(a)) for a in (qkv[:, :n_heads * D], qkv[:, n_heads * D:(n_heads + nk) * D], qkv[:, (n_heads + nk) * D:])]
        args = (parts[0], n_heads * D, parts[1], nk * D, parts[2], nk * D)
        src, qs = parts[0], n_heads * D
    out = src if in_place else fk.DeviceBuffer.from_numpy(np.full((rows, n_heads * D), 0x4242, np.uint16))
    fk.rope_paged_store(*args, out, qs if in_place else n_heads * D, n_heads, *dn, eps, rope_dims, interleaved, f, batch, pool)
    fk.sync()
    got_q = out.to_numpy(np.uint16, (rows, qs if in_place else n_heads * D))[:, :n_heads * D].reshape(rows, n_heads, D)
    got_k, got_v = (p.d[i].to_numpy(np.uint16, p.k.shape) for i in (3, 4))
    return qkv.reshape(rows, n_heads + 2 * nk, D), got_q, got_k, got_v


def check_store(fk, p, n_heads, rope_dims, interleaved, freq, norms=(None, None), **more):
    qkv, got_q, got_k, got_v = store(fk, p, n_heads, rope_dims, interleaved, freq, norms, **more)
    n, nk = sum(p.rows), p.n_kv
    if not more.get("in_place"):
        assert bool((got_q[n:] == 0x4242).all())
    pos = np.concatenate([np.arange(l - r, l) for r, l in zip(p.rows, p.lens)]).astype(np.int64)
    x = wide(qkv[:n])
    wk, wv = p.k.copy(), p.v.copy()
    touched = np.zeros(p.k.shape[:3], bool)
    for part, norm, got in ((x[:, :n_heads], norms[0], got_q[:n]), (x[:, n_heads:n_heads + nk], norms[1], None)):
        ref, size = rotated(part, pos, freq, rope_dims, interleaved, None if norm is None else wide(norm))
        if got is None:
            seq = np.repeat(np.arange(len(p.rows)), p.rows)
            page, slot = p.table[seq, pos // p.page_rows], pos % p.page_rows
            got = got_k[page, :, slot]
            touched[page, :, slot] = True
            assert bool((got_v[page, :, slot] == qkv[:n, n_heads + nk:]).all())
        assert bool((np.abs(wide(got) - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -20 * size).all())
    assert bool((got_k[~touched] == wk[~touched]).all() and (got_v[~touched] == wv[~touched]).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rope_dims", [(64, 64), (64, 32), (64, 16), (128, 128), (128, 64), (128, 48), (64, 0)])
def test_rope_store_layouts(fk, interleaved, dim, rope_dims):
    freq = frequencies(rope_dims, 1e4) if rope_dims else None
    for n_heads, n_kv in ((4, 2), (7, 1), (3, 3)):
        check_store(fk, Paged([1, 5, 0, 17], [100, 20, 4, 17], n_kv, dim, 16, seed=1), n_heads, rope_dims, interleaved, freq)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("packed,in_place", [(True, True), (False, True), (False, False)])
def test_rope_store_norms_and_places(fk, interleaved, packed, in_place):
    for dim in (64, 128):
        norms = (normal_bf16(5, dim, std=0.1, mean=1.0), normal_bf16(6, dim, std=0.1, mean=1.0))
        check_store(fk, Paged([3, 1], [3, 300], 2, dim, 64, seed=2), 8, dim, interleaved, frequencies(dim, 1e6), norms, packed=packed, in_place=in_place)
        check_store(fk, Paged([3, 1], [3, 300], 2, dim, 64, seed=2), 8, dim // 2, interleaved, frequencies(dim // 2, 1e6), (None, norms[1]), packed=packed,
                    in_place=in_place)


@pytest.mark.parametrize("kind", SCALINGS, ids=lambda s: s["scaling"])
def test_rope_store_far_positions(fk, kind):
    """A million positions on, the fastest pair has turned 160000 times: the angle still holds."""
    p = Paged([2], [64], 1, 128, 1024, seed=3)
    n = 1000001
    p.table = np.zeros((1, 1024), np.uint32)
    p.stride = 1024
    p.lens, p.kv_len = [n], np.array([n], np.uint32)
    check_store(fk, p, 4, 128, False, frequencies(128, 1e4, **kind), max_len=n)


def test_rope_store_rows_behind_the_batch_and_bad_values(fk):
    freq = frequencies(64, 1e4)
    check_store(fk, Paged([2, 1], [30, 9], 2, 64, 16, seed=4), 4, 64, False, freq, rows=9, max_rows=5)
    fault = fk.zeros(4)
    p = Paged([2, 1], [30, 9], 2, 64, 16, seed=4)
    p.table[0, 1] = p.n_pages + 7
    _, _, got_k, got_v = store(fk, p, 4, 64, False, freq, fault=fault)
    own = np.zeros(p.k.shape[:3], bool)
    own[p.table[1, 0], :, 8] = True
    assert bool((got_k[~own] == p.k[~own]).all() and (got_v[~own] == p.v[~own]).all())   # the bad page's rows are stored nowhere
    with pytest.raises(fk.InvalidArgument, match="page id"):
        fk.paged_check(fault)


# ---------------------------------------------------------------- pages copied

@pytest.mark.parametrize("planes,n_pages,page_bytes,pairs", [(1, 2, 16, 1), (3, 9, 4096, 4), (2, 40, 16 * 257, 20), (5, 1200, 64, 600), (70, 12, 32768, 5)])
@pytest.mark.parametrize("gap", [0, 48])
def test_pages_copy(fk, planes, n_pages, page_bytes, pairs, gap):
    stride = n_pages * page_bytes + gap
    pool = rng(planes).integers(0, 256, planes * stride, dtype=np.uint8)
    order = rng(pairs).permutation(n_pages)
    src, dst = order[:pairs].copy(), order[pairs:2 * pairs]
    src[1::3] = src[0]                                       # one page forked several times
    d = fk.DeviceBuffer.from_numpy(pool)
    fk.pages_copy(d, planes, stride, n_pages, page_bytes, np.stack([src, dst], 1))
    fk.sync()
    ref = pool.copy()
    for l in range(planes):
        v = ref[l * stride:l * stride + n_pages * page_bytes].reshape(n_pages, page_bytes)
        v[dst] = v[src]
    assert bool((d.to_numpy(np.uint8) == ref).all())
    fk.pages_copy(d, planes, stride, n_pages, page_bytes, [])


def test_pages_beyond_32_bits(fk):
    """Pages around 4 GB, 2^32 values and at the pool's end: attention of a chunk and of single tokens, the append, copies."""
    p = Paged([40, 1, 3], [200, 130, 70], 2, 128, 64, seed=30)
    page_bytes, far = p.k[0].nbytes, 2 ** 33 // p.k[0].nbytes + 40
    ids = np.concatenate([2 ** 32 // page_bytes + np.arange(-2, 2), 2 ** 33 // page_bytes + np.arange(-2, 2), far - 1 - np.arange(p.n_pages)]).astype(np.uint32)
    pools = [fk.DeviceBuffer(far * page_bytes) for _ in range(2)]
    for buf, pages in zip(pools, (p.k, p.v)):
        for i in range(p.n_pages):
            buf.upload(pages[i], int(ids[i]) * page_bytes)
    table = np.where(p.table < p.n_pages, ids[np.minimum(p.table, p.n_pages - 1)], 0xFFFFFFFF).astype(np.uint32)
    d = [fk.DeviceBuffer.from_numpy(a) for a in (p.row_start, p.kv_len, table)]
    n, n_heads = sum(p.rows), 8
    q = normal_bf16(31, (n, n_heads, 128))
    ref, size = attention(p, q, n_heads, 128 ** -0.5)
    pool = fk.PagePool(pools[0], pools[1], far, 64, 2, 128)
    for keep in (slice(0, 3), slice(1, 3)):                   # with the chunk; single tokens and three rows, tiles of 16
        rows = np.array(p.rows[keep])
        start = fk.DeviceBuffer.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32))
        first, m = sum(p.rows[:keep.start]), int(rows.sum())
        batch = fk.PagedBatch(start, d[1].ptr + 4 * keep.start, d[2].ptr + 4 * keep.start * p.stride, p.stride, len(rows), m, int(rows.max()), 200, None)
        out, ws = fk.zeros(m * n_heads * 256), fk.zeros(fk.sdpa_paged_workspace_bytes(n_heads, 2, 128, len(rows), m, 200))
        fk.sdpa_paged(fk.DeviceBuffer.from_numpy(q[first:first + m]), n_heads * 128, out, n_heads * 128, n_heads, 128 ** -0.5, 0.0, 0, batch, pool, ws, ws.nbytes)
        fk.sync()
        got, r, s = wide(out.to_numpy(np.uint16, (m, n_heads, 128))), ref[first:first + m], size[first:first + m]
        assert bool((np.abs(got - r) <= 2.0 ** -8 * np.abs(r) + (2.0 ** -8 + 2.0 ** -11) * s).all())
    kv = normal_bf16(32, (n, 2, 128))
    dk, dq = fk.DeviceBuffer.from_numpy(kv), fk.DeviceBuffer.from_numpy(q)
    batch = fk.PagedBatch(d[0], d[1], d[2], p.stride, 3, n, 40, 200, None)
    fk.rope_paged_store(dq, n_heads * 128, dk, 256, dk, 256, dq, n_heads * 128, n_heads, None, None, 1e-6, 0, False, None, batch, pool)
    at = 0
    for i, (r, length) in enumerate(zip(p.rows, p.lens)):
        page, slot = p.where(i, np.arange(length - r, length))
        p.k[page, :, slot] = p.v[page, :, slot] = kv[at:at + r]
        at += r
    near = np.array([[ids[0], 1], [ids[p.n_pages - 1], 2 ** 32 // page_bytes + 5]], np.uint32)
    for buf, pages in zip(pools, (p.k, p.v)):
        fk.pages_copy(buf, 1, far * page_bytes, far, page_bytes, near)
        fk.sync()
        for i in range(p.n_pages):
            assert bool((buf.to_numpy(np.uint16, p.k[0].shape, int(ids[i]) * page_bytes) == pages[i]).all())
        for src, dst in ((0, near[0, 1]), (p.n_pages - 1, near[1, 1])):
            assert bool((buf.to_numpy(np.uint16, p.k[0].shape, int(dst) * page_bytes) == pages[src]).all())


# ---------------------------------------------------------------- a few hundred positions and few tiles: 64 columns, 128 positions a step

@pytest.mark.parametrize("rows,lens", [([130], [300]), ([40], [700]), ([200, 1], [500, 700]), ([70, 33, 0, 2], [330, 400, 9, 77]), ([65], [321]), ([8], [300]), ([8, 8], [300, 290])])
@pytest.mark.parametrize("n_heads,n_kv,dim,page_rows", [(8, 2, 128, 16), (14, 2, 64, 32), (6, 6, 64, 128), (8, 2, 128, 256)])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (300, 0.0), (0, 20.0), (310, 30.0)])
def test_few_tiles(fk, rows, lens, n_heads, n_kv, dim, page_rows, window, softcap):
    p = Paged(rows, lens, n_kv, dim, page_rows, seed=40 + len(rows))
    check_attention(fk, p, n_heads, softcap=softcap, window=window, rows=max(sum(rows), 40), max_rows=max(rows + [36]))


@pytest.mark.parametrize("edge", [256, 257, 383, 384, 385, 448, 511, 512, 513])
def test_few_tiles_at_the_edges_of_a_step(fk, edge):
    for rows in (1, 33, edge if edge < 400 else 100):
        check_attention(fk, Paged([max(rows, 17)], [edge], 1, 128, 32, seed=edge, spare_table=20), 4, max_len=700)


@pytest.mark.parametrize("dim,page_rows", [(64, 16), (128, 64)])
def test_infinities_and_nan_in_masked_places_of_few_tiles(fk, dim, page_rows):
    for bad_bits in (0x7F80, 0xFF80, 0x7FC0):
        p = Paged([50, 1], [400, 600], 2, dim, page_rows, seed=41)
        for i, at in ((0, np.arange(395, 400)), (1, np.arange(0, 270))):      # the chunk's last five rows; before the window of the other
            page, slot = p.where(i, at)
            p.k[page, :, slot] = bad_bits
            p.v[page, :, slot] = bad_bits
        q, got, _ = attend(fk, p, 8, window=320)
        with np.errstate(all="ignore"):
            ref, size = attention(p, q, 8, dim ** -0.5, 0.0, 320)
        fine = np.r_[0:45, 50]
        off = np.abs(wide(got[fine]) - ref[fine]) - (2.0 ** -8 * np.abs(ref[fine]) + (2.0 ** -8 + 2.0 ** -11) * size[fine])
        assert np.isfinite(wide(got[fine])).all() and off.max() <= 0, hex(bad_bits)
        if bad_bits == 0x7FC0:
            assert np.isnan(wide(got[45:50])).all()


def test_few_tiles_bad_page(fk):
    fault = fk.zeros(4)
    p = Paged([60, 50], [300, 310], 2, 128, 16, seed=42)
    p.table[0, 9] = p.n_pages + 3
    q, got, _ = attend(fk, p, 8, fault=fault)
    p.table[0, 9] = 0
    ref, size = attention(p, q, 8, 128 ** -0.5)
    other = slice(60, 110)
    assert bool((np.abs(wide(got[other]) - ref[other]) <= 2.0 ** -8 * np.abs(ref[other]) + (2.0 ** -8 + 2.0 ** -11) * size[other]).all())
    with pytest.raises(fk.InvalidArgument, match="page id"):
        fk.paged_check(fault)


@pytest.mark.parametrize("rows,lens", [([300, 1, 2], [300, 2500, 1500]), ([1, 140, 1, 0], [4000, 200, 70, 90]), ([1, 1, 150], [2049, 5000, 151])])
@pytest.mark.parametrize("n_heads,dim,window,softcap", [(64, 64, 0, 0.0), (64, 128, 2100, 0.0), (128, 64, 0, 20.0)])
def test_long_tokens_among_more_tiles_than_are_cut(fk, rows, lens, n_heads, dim, window, softcap):
    p = Paged(rows, lens, 64, dim, 32, seed=50 + len(rows))
    ws = fk.zeros(fk.sdpa_paged_workspace_bytes(n_heads, 64, dim, len(rows), sum(rows), max(lens)))
    for _ in range(2):                                       # a workspace is left ready
        check_attention(fk, p, n_heads, softcap=softcap, window=window, workspace=ws)


@pytest.mark.parametrize("n_seqs,long_at,chunk_at", [(300, (7, 290), None), (130, (0,), None), (70, (3, 69), 65), (150, (149,), 0), (200, (), None)])
@pytest.mark.parametrize("dim,window,softcap", [(64, 0, 0.0), (128, 3000, 20.0)])
def test_more_sequences_than_have_slots(fk, n_seqs, long_at, chunk_at, dim, window, softcap):
    lens = [int(n) for n in rng(n_seqs).integers(1, 40, n_seqs)]
    rows = [1] * n_seqs
    for i in long_at:
        lens[i] = 3500 + i
    if chunk_at is not None:
        rows[chunk_at], lens[chunk_at] = 90, 130
    p = Paged(rows, lens, 8, dim, 32, seed=60, spare_table=0)
    ws = fk.zeros(fk.sdpa_paged_workspace_bytes(16, 8, dim, n_seqs, sum(rows), max(lens)))
    for _ in range(2):
        check_attention(fk, p, 16, softcap=softcap, window=window, workspace=ws)


@pytest.mark.parametrize("n_seqs,longest", [(130, 260), (256, 500), (140, 1024), (140, 1025), (300, 129)])
def test_more_sequences_than_have_slots_of_some_rounds(fk, n_seqs, longest):
    lens = [int(n) for n in rng(longest).integers(100, longest + 1, n_seqs)]
    lens[5] = longest
    check_attention(fk, Paged([1] * n_seqs, lens, 8, 64, 64, seed=61, spare_table=0), 8)
