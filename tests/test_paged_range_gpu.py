"""Attention over a paged cache (fk_sdpa_paged) with scores and values of any size, against the statement in 64 bits.

In the tests of scores a query and a key differ from 0 in their first dim only, so that a score is the product of two bf16 values, exact in fp32: what is left of the tolerance is the
probabilities' rounding to bf16, 2^-8 of A = sum p |v| / sum p, that of the output, 2^-8 of it, and 2^-11 A for exponentials and sums in fp32."""
import numpy as np
import pytest

import oracle
from helpers import rng
from paged_reference import Paged, attention, wide
from test_paged_gpu import attend

pytestmark = pytest.mark.gpu


def first_dim(values, dim):
    out = np.zeros((*values.shape, dim), np.uint16)
    out[..., 0] = oracle.f32_to_bf16(values.astype(np.float32))
    return out


# single tokens on 8 and on 16 columns, whole and cut; whole tiles of 128 columns, of 64, cut ones; chunks among tokens
SHAPES = [([1, 1], [200, 33], 4, 2, 128), ([1], [9000], 4, 1, 64), ([3], [150], 8, 1, 64), ([2, 1], [7000, 300], 16, 1, 128),
          ([130], [131], 8, 2, 128), ([130, 17], [300, 310], 8, 2, 64), ([64], [3000], 8, 2, 128), ([150, 1, 1], [2500, 2000, 64], 8, 2, 64)]


@pytest.mark.parametrize("rows,lens,n_heads,n_kv,dim", SHAPES)
@pytest.mark.parametrize("size", [1e3, 1e9, 4e9, 1e11, 1e20, 2.4e38, 3.3e38])
def test_large_scores(fk, rows, lens, n_heads, n_kv, dim, size):
    g = rng(len(rows) + dim)
    for sign in (1, -1):
        p = Paged(rows, lens, n_kv, dim, 32, seed=7)
        for i, n in enumerate(lens):                        # (keys of a few magnitudes: many positions tie)
            page, slot = p.where(i, np.arange(n))
            k = np.sqrt(size) * g.choice([0.25, 0.5, 0.75, 1.0], (n, n_kv)) if size < 1e38 else 1e19 * g.choice([0.5, 1.0], (n, n_kv))
            p.k[page, :, slot] = first_dim(k, dim)
        q = sign * (np.sqrt(size) if size < 1e38 else size / 1e19) * (1 - 0.3 * g.random((sum(rows), n_heads)))
        q[:, 0] = 0.0                                       # (a head without a preference, beside the others in its tile)
        q = first_dim(q, dim)
        _, got, _ = attend(fk, p, n_heads, scale=1.0, q=q)
        ref, a = attention(p, q, n_heads, 1.0)
        assert bool((np.abs(wide(got) - ref) <= 2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -11) * a).all()), sign


def test_a_row_that_sees_nothing_beside_large_scores(fk):
    for rows, lens in (([3], [3]), ([40], [300]), ([140], [140])):
        fault = fk.zeros(4)
        p = Paged(rows, lens, 1, 64, 16, seed=8)
        page, slot = p.where(0, np.arange(lens[0]))
        p.k[page, :, slot] = first_dim(np.full((lens[0], 1), 1e18), 64)
        p.kv_len[0] = p.lens[0] = rows[0] - 1               # one row more than positions
        q = first_dim(rng(9).random((rows[0], 2)) * 1e18, 64)
        _, got, _ = attend(fk, p, 2, scale=1.0, q=q, fault=fault, max_len=lens[0])
        assert bool((got[0] == 0).all())
        ref, a = attention(p, q, 2, 1.0)
        assert bool((np.abs(wide(got) - ref) <= 2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -11) * a).all())
        with pytest.raises(fk.InvalidArgument, match="length"):
            fk.paged_check(fault)


@pytest.mark.parametrize("rows,lens,n_heads,n_kv,dim", SHAPES)
@pytest.mark.parametrize("size", [1e-34, 1e-28, 1e30, 2e37])
def test_values_of_any_size(fk, rows, lens, n_heads, n_kv, dim, size):
    """Values near both ends of bf16's range, weighted by ordinary scores.  An fp32 score of `dim` products of values below 5 and 10, times dim^-1/2, is off
    by less than 128 * 2^-24 * 128 * 50 * 0.09 / 30 = 1.5e-4 with the sums that normal values have: 2^-11 A with the sums' own rounding."""
    p = Paged(rows, lens, n_kv, dim, 32, seed=10)
    for i, n in enumerate(lens):
        page, slot = p.where(i, np.arange(n))
        p.v[page, :, slot] = oracle.f32_to_bf16((size * rng(11 + i).standard_normal((n, n_kv, dim))).astype(np.float32))
    q, got, _ = attend(fk, p, n_heads)
    ref, a = attention(p, q, n_heads, dim ** -0.5)
    off = np.abs(wide(got) - ref) - (2.0 ** -8 * np.abs(ref) + (2.0 ** -8 + 2.0 ** -11) * a + 2.0 ** -126)   # (below the smallest normal number: to 0)
    assert off.max() <= 0, off.max()


@pytest.mark.parametrize("rows,lens,n_heads,n_kv,dim", SHAPES)
def test_the_largest_values(fk, rows, lens, n_heads, n_kv, dim):
    """Sums of probabilities times the type's largest values leave fp32, their average does not."""
    p = Paged(rows, lens, n_kv, dim, 32, seed=12)
    for i, n in enumerate(lens):
        page, slot = p.where(i, np.arange(n))
        p.v[page, :, slot] = np.where(np.arange(dim) % 3 == 0, 0xFF7F, 0x7F60)
    q, got, _ = attend(fk, p, n_heads)
    ref = np.broadcast_to(wide(np.where(np.arange(dim) % 3 == 0, 0xFF7F, 0x7F60).astype(np.uint16)), got.shape)
    assert bool((np.abs(wide(got) / ref - 1) <= 2.0 ** -7 + 2.0 ** -11).all())   # the probabilities' rounding and the output's
