"""Tokens drawn from logits (fk_sample) against a plain statement in 64 bits.

Tolerances.  A token is a whole number and has to be the plain statement's: both form weights and sums in 64 bits, so that a random number has to lie within
some 1e-13 of a border for the two to differ.  A log probability is rounded once, 2^-24 of it; in 64 bits it is off by far less than 2^-26."""
import numpy as np
import pytest

import oracle
from decode_loop_reference import sample
from helpers import rng
from test_paged_graph_gpu import Graph, stream  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
NAMES = ("temperature", "top_k", "top_p", "min_p", "u")


class Draw:
    def __init__(self, fk, bits, pad=0, seed=0, logprobs=True, **settings):
        self.fk, self.rows, self.vocab = fk, *bits.shape
        self.stride = self.vocab + pad
        r = rng(seed + 99)
        whole = np.full((self.rows, self.stride), 0x7F7F, np.uint16)          # (behind a row: larger than what is in it)
        whole[:, :self.vocab] = bits
        with np.errstate(invalid="ignore"):
            self.x = oracle.bf16_to_f32(bits).astype(np.float64)
        usual = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=r.random(self.rows, dtype=np.float32))
        self.v = {n: np.broadcast_to(np.asarray(settings.get(n, usual[n]), np.uint32 if n == "top_k" else np.float32), self.rows).copy() for n in NAMES}
        self.d = {n: fk.DeviceBuffer.from_numpy(a) for n, a in self.v.items() if n == "u" or n in settings}
        self.logits = fk.DeviceBuffer.from_numpy(whole)
        self.out = fk.DeviceBuffer.from_numpy(np.full((4, self.rows + 2), 0x55555555, np.uint32))   # tokens and logprobs, with a border
        at = self.out.ptr + 4
        self.tokens, self.logprobs = at, at + 8 * (self.rows + 2) if logprobs else None
        self.ws = fk.zeros(fk.sample_workspace_bytes(self.rows, self.vocab))

    def run(self, st=None):
        g = self.d.get
        self.fk.sample(self.logits, self.stride, self.rows, self.vocab, g("temperature"), g("top_k"), g("top_p"), g("min_p"), self.d["u"], self.tokens,
                       self.logprobs, self.ws, self.ws.nbytes, st)
        return self

    def got(self):
        whole = self.out.to_numpy(np.uint32, (4, self.rows + 2))
        assert bool((whole[[1, 3]] == 0x55555555).all() and (whole[:, [0, -1]] == 0x55555555).all())      # nothing else is written
        return whole[0, 1:-1], whole[2, 1:-1].view(np.float32)

    def check(self):
        self.fk.sync()
        tokens, logprobs = self.got()
        for i in range(self.rows):
            t, lp = sample(self.x[i], *(self.v[n][i] for n in NAMES))
            assert tokens[i] == t, (i, tokens[i], t, {n: self.v[n][i] for n in NAMES})
            if self.logprobs:
                assert logprobs[i] == lp if not np.isfinite(lp) else abs(logprobs[i] - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -26, (i, logprobs[i], lp)
        return self


def normal(seed, rows, vocab, std=2.5, mean=0.0):
    return oracle.f32_to_bf16((rng(seed).standard_normal((rows, vocab), dtype=np.float32) * np.float32(std) + np.float32(mean)).astype(np.float32))


def mixed(seed, rows):
    """Settings as a server's users have them."""
    r = rng(seed)
    return dict(temperature=np.where(r.random(rows) < 0.1, 0, r.uniform(0.2, 2.0, rows)), top_k=np.where(r.random(rows) < 0.4, 0, r.integers(1, 300, rows)),
                top_p=np.where(r.random(rows) < 0.3, 1, r.uniform(0.1, 1.0, rows)), min_p=np.where(r.random(rows) < 0.5, 0, r.uniform(0, 0.3, rows)))


@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 9, 15, 63, 64, 65, 127, 511, 1000, 1023, 1025, 4096, 8191, 8192, 8193, 16385, 32000, 50257, 151851])
@pytest.mark.parametrize("rows,pad", [(1, 0), (5, 3)])
def test_sizes(fk, vocab, rows, pad):
    Draw(fk, normal(vocab, rows, vocab), pad=pad, seed=vocab, **mixed(vocab, rows)).run().check()


@pytest.mark.parametrize("rows", [1, 2, 3, 16, 33, 64, 100, 257, 700])
def test_rows(fk, rows):
    Draw(fk, normal(rows, rows, 3001), pad=7, seed=rows, **mixed(rows, rows)).run().check()


@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("std", [0.1, 1.0, 4.0, 12.0, 60.0])
def test_spreads(fk, rows, std):
    Draw(fk, normal(7, rows, 40009, std), seed=rows, **mixed(8, rows)).run().check()
    Draw(fk, normal(9, rows, 40009, std), seed=rows).run().check()                                # nothing cut, no array but u
    Draw(fk, normal(9, rows, 20000, std, mean=30 * std), seed=rows, **mixed(9, rows)).run().check()
    Draw(fk, normal(9, rows, 20000, std, mean=-30 * std), seed=rows, **mixed(9, rows)).run().check()


@pytest.mark.parametrize("name,values", [("temperature", [0.0, -1.0, np.nan, 1e-45, 1e-30, 1e-3, 0.05, 5.0, 1e4, 1e30, np.inf, -0.0]),
                                         ("top_k", [0, 1, 2, 3, 10, 997, 998, 999, 1000, 1001, 0xFFFFFFFF]),
                                         ("top_p", [-1.0, 0.0, 1e-30, 1e-6, 0.01, 0.5, 0.999999, 1.0, 2.0, np.inf, np.nan, -np.inf]),
                                         ("min_p", [-1.0, 0.0, 1e-30, 1e-6, 0.01, 0.5, 0.999, 1.0, 2.0, np.inf, np.nan]),
                                         ("u", [0.0, -0.0, -1.0, 1e-30, 1e-7, 0.5, 1 - 2.0 ** -24, 1.0, 2.0, np.inf, np.nan])])
def test_edges_of_a_setting(fk, name, values):
    n = len(values)
    for other in ({}, mixed(4, n)):
        more = dict(other)
        more.pop(name, None)
        with np.errstate(over="ignore"):
            Draw(fk, normal(3, n, 1000), seed=n, **more, **{name: values}).run().check()


@pytest.mark.parametrize("lowest", [0xFF80, 0xFF7F, 0x7FC0, 0xFFFF])       # -inf, the type's lowest, NaN
@pytest.mark.parametrize("share", [0.5, 0.99, 0.9999])
def test_masks(fk, lowest, share):
    for seed, std in ((1, 2.0), (2, 30.0)):
        bits = normal(seed, 6, 30011, std)
        bits[rng(seed).random(bits.shape) < share] = lowest
        Draw(fk, bits, seed=seed, **mixed(seed, 6)).run().check()
        Draw(fk, bits, seed=seed, temperature=[1.0, 8.0, 50.0, 1e3, 1e30, 1e38]).run().check()


def test_rows_that_hold_nothing(fk):
    bits = normal(5, 7, 5000)
    bits[1], bits[3], bits[5] = 0xFF80, 0x7FC0, np.where(np.arange(5000) % 2, 0xFF80, 0xFFC1)
    bits[6] = 0xFF80
    bits[6, 4999] = 0xFF7F
    d = Draw(fk, bits, **mixed(5, 7)).run().check()
    assert d.got()[0][[1, 3, 5, 6]].tolist() == [0, 0, 0, 4999]


@pytest.mark.parametrize("vocab", [9, 5000, 70001])
def test_infinities(fk, vocab):
    bits = normal(6, 4, vocab)
    bits[0, vocab // 2] = 0x7F80
    bits[1, [1, 5, vocab - 1]] = 0x7F80
    bits[2] = 0x7F80
    Draw(fk, bits, temperature=[1.0, 0.5, 1e30, 1.0], u=[0.5, 0.7, 0.99, 0.3]).run().check()
    Draw(fk, bits, temperature=[0.0, np.inf, 1.0, 1.0], top_k=[0, 2, 7, 1], top_p=[0.5, 0.5, 0.5, 1.0]).run().check()


@pytest.mark.parametrize("value", [0x0000, 0x8000, 0x3F80, 0xC2C8, 0x7F7F, 0xFF7F, 0x0001, 0x8001, 0x4680])
@pytest.mark.parametrize("vocab", [1, 64, 1000, 70000])
def test_rows_of_one_value(fk, value, vocab):
    """Every token weighs the same: which one follows from u alone."""
    rows = 8
    u = (np.arange(rows) + 0.5) / rows
    d = Draw(fk, np.full((rows, vocab), value, np.uint16), u=u).run().check()
    assert d.got()[0].tolist() == [int(np.float32(v) * np.float64(vocab)) for v in u]
    Draw(fk, np.full((rows, vocab), value, np.uint16), u=u, top_p=[0.5, 0.25, 0.125, 1.0, 0.0, 0.75, 0.5, 0.5], top_k=[0, 0, 0, 5, 5, 8, 1, 2]).run().check()


def test_zeros_of_both_signs_are_one_value(fk):
    bits = np.where(rng(1).random((4, 3000)) < 0.5, 0x8000, 0x0000).astype(np.uint16)
    Draw(fk, bits, u=[0.1, 0.5, 0.9, 0.9999], top_k=[0, 0, 17, 1000]).run().check()


def test_ties_at_every_border(fk):
    """Few distinct logits: each cut falls inside a run of equal ones, the lower tokens stay."""
    bits = oracle.f32_to_bf16(rng(2).integers(0, 4, (64, 4001)).astype(np.float32))
    Draw(fk, bits, seed=2, top_k=rng(3).integers(0, 4001, 64), top_p=rng(4).uniform(0.05, 1.0, 64), min_p=rng(5).uniform(0, 0.5, 64)).run().check()


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-12, 1e-7, 1e3, 1e12, 1e37])
def test_logits_of_any_size(fk, scale):
    """Values far outside of what models give, in order all the same, with the temperature that makes something of them."""
    for t in (scale, 0.3 * scale, 1.0):
        Draw(fk, normal(11, 5, 9000, scale), seed=3, temperature=t, top_k=[0, 50, 0, 1, 700], top_p=[1.0, 0.9, 0.3, 1.0, 1.0]).run().check()
    Draw(fk, normal(12, 5, 9000, scale), seed=4, temperature=0.0).run().check()


def test_values_of_all_sizes_in_one_row(fk):
    """Every bf16 pattern once: all of the type's range, both zeros, infinities and NaN among them."""
    bits = np.tile(np.arange(65536, dtype=np.uint16), (6, 1))
    for i in range(6):
        bits[i] = rng(i).permutation(bits[i])
    bits[2:][(bits[2:] & 0x7FFF) == 0x7F80] = 0                             # no infinity in these
    Draw(fk, bits, temperature=[1.0, 0.5, 1.0, 1e38, 1e36, 1e30], u=[0.3, 0.7, 0.5, 0.9, 0.2, 0.999]).run().check()
    Draw(fk, bits, temperature=1e38, top_k=[5, 0, 30000, 40000, 65000, 66000], top_p=[1.0, 1.0, 0.5, 0.9, 0.99, 0.999]).run().check()


def test_a_row_does_not_depend_on_the_others(fk):
    bits, more = normal(21, 90, 20011), mixed(21, 90)
    u = rng(22).random(90, dtype=np.float32)
    every = Draw(fk, bits, u=u, **more).run()
    fk.sync()
    tokens, logprobs = every.got()
    for rows in ([3], [3, 77], list(range(40, 57))):
        d = Draw(fk, bits[rows], u=u[rows], **{n: a[rows] for n, a in more.items()}).run()
        fk.sync()
        t, lp = d.got()
        assert np.array_equal(t, tokens[rows]) and np.array_equal(lp, logprobs[rows])


def test_without_log_probabilities(fk):
    Draw(fk, normal(23, 9, 12345), logprobs=False, **mixed(23, 9)).run().check()
    Draw(fk, normal(23, 1, 151851), logprobs=False, **mixed(24, 1)).run().check()


@pytest.mark.parametrize("first", [1, 3])
def test_logits_that_start_anywhere(fk, first):
    d = Draw(fk, normal(24, 4, 9001), pad=2, **mixed(24, 4))
    moved = fk.DeviceBuffer(d.logits.nbytes + 64)
    moved.upload(np.full(moved.nbytes // 2, 0x7F7F, np.uint16))
    moved.upload(d.logits.to_numpy(np.uint16), 2 * first)
    keep, d.logits = d.logits, moved.ptr + 2 * first
    d.run().check()


def test_the_workspace_is_left_ready(fk):
    """One workspace for calls of different shapes, one after another."""
    shapes = [(1, 151851), (40, 3000), (3, 32000), (200, 1000), (1, 151851), (7, 60000)]
    ws = fk.zeros(max(fk.sample_workspace_bytes(*s) for s in shapes))
    every = [Draw(fk, normal(30 + i, *s), seed=i, **mixed(i, s[0])) for i, s in enumerate(shapes)]
    for d in every:
        d.ws = ws
    for _ in range(2):
        for d in every:
            d.run()
    for d in every:
        d.check()


def test_captured_and_on_two_streams(fk, stream):  # noqa: F811
    a, b = stream(), stream()
    one, two = Draw(fk, normal(41, 3, 70001), seed=1, **mixed(41, 3)), Draw(fk, normal(42, 70, 9001), seed=2, **mixed(42, 70))
    one.run(a)
    two.run(b)
    fk.sync(a)
    fk.sync(b)
    g, h = Graph(fk, a, lambda: one.run(a)), Graph(fk, b, lambda: two.run(b))
    for i in range(4):
        for d in (one, two):
            d.v["u"] = rng(50 + i).random(d.rows, dtype=np.float32)
            d.d["u"].upload(d.v["u"])
            d.out.upload(np.full((4, d.rows + 2), 0x55555555, np.uint32))
        g.replay()
        h.replay()
        fk.sync(a)
        fk.sync(b)
        one.check()
        two.check()
    g.free()
    h.free()


@pytest.mark.parametrize("rows,vocab", [(2, 262145), (3, 300001), (1, 1 << 21)])
def test_vocabularies_of_more_groups_than_a_row_has(fk, rows, vocab):
    Draw(fk, normal(61, rows, vocab), pad=1, seed=vocab, **mixed(61, rows)).run().check()
    flat = normal(62, rows, vocab, std=0.01)
    Draw(fk, flat, seed=vocab, u=[0.1, 0.5, 0.97][:rows]).run().check()


def test_many_rows_of_a_large_vocabulary(fk):
    """More rows than the device has CUs, of more than 2^20 tokens."""
    rows, vocab = 257, (1 << 20) + 5
    one = normal(63, 1, vocab)
    d = Draw(fk, np.repeat(one[:, :64], rows, 0), **mixed(63, rows))
    d.vocab, d.stride = vocab, 0                  # (the whole rows: made on the device, one after the other)
    d.logits = fk.DeviceBuffer(2 * rows * (vocab + 3))
    row = fk.DeviceBuffer.from_numpy(np.concatenate([one[0], [0x7F7F] * 3]).astype(np.uint16))
    same = fk.zeros(4 * rows)
    for at in range(0, rows, 64):
        n = min(64, rows - at)
        fk.beam_reorder(row, d.logits.ptr + 2 * at * (vocab + 3), 2 * (vocab + 3), same, 1, 1, n)
    d.stride, d.ws = vocab + 3, fk.zeros(fk.sample_workspace_bytes(rows, vocab))
    d.run()
    fk.sync()
    tokens, logprobs = d.got()
    x = oracle.bf16_to_f32(one[0]).astype(np.float64)
    for i in list(range(0, rows, 37)) + [rows - 1]:
        t, lp = sample(x, *(d.v[n][i] for n in NAMES))
        assert tokens[i] == t and abs(logprobs[i] - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -26, i


def test_few_tokens_that_min_p_cuts(fk):
    """A handful of logits far apart: the cut falls where no logit is, and the next one lies many bins on."""
    bits = np.full((300, 500), 0xFF7F, np.uint16)
    r = rng(64)
    for i in range(300):
        at = r.choice(500, r.integers(1, 9), replace=False)
        bits[i, at] = oracle.f32_to_bf16((r.uniform(-1, 1, len(at)) * 10.0 ** r.uniform(-8, 2, len(at))).astype(np.float32))
    for rows in (300, 20):
        Draw(fk, bits[:rows], min_p=r.uniform(0, 1, rows), temperature=10.0 ** r.uniform(-3, 2, rows), top_k=r.integers(0, 6, rows)).run().check()
        Draw(fk, bits[:rows], top_p=r.uniform(0, 1, rows), temperature=10.0 ** r.uniform(-3, 2, rows)).run().check()


@pytest.mark.parametrize("rows,vocab,share", [(13, 40000, 0.3), (300, 9001, 0.5), (16, 70001, 0.001), (6, 262145, 0.6), (40, 1000, 1.0), (270, 70001, 0.4)])
def test_places_among_equal_logits(fk, rows, vocab, share):
    """From the first of those that hold a logit to the last: they are counted from the nearer end."""
    bits = np.where(rng(71).random((rows, vocab)) < share, 0x4040, 0x4000).astype(np.uint16)      # 3 and 2
    bits[:, ::97] = 0xFF80
    u = np.linspace(0, 1, rows, endpoint=False, dtype=np.float32)
    u[-1] = 1 - 2.0 ** -24
    d = Draw(fk, bits, pad=1, seed=72, u=u, logprobs=False)
    d.run().check()
    Draw(fk, bits, seed=72, u=u[::-1].copy(), temperature=3.0, top_p=0.9).run().check()
