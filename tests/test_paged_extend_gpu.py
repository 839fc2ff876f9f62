"""A batch built on the device from the requests' lengths (fk_paged_extend): whole numbers, equal to a plain statement's."""
import numpy as np
import pytest

from decode_loop_reference import extend
from helpers import rng
from test_paged_graph_gpu import Graph, stream  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
FILL = 0xAAAAAAAA


class Requests:
    """Slots with lengths and pages, a shuffled free stack, and a batch's arrays filled with a pattern."""

    def __init__(self, fk, held, n_slots=None, page_rows=16, room=64, seed=0, spare=5, stride=None, in_place=True):
        self.fk, self.page_rows, self.in_place = fk, page_rows, in_place
        self.lengths = np.array(list(held) + [0] * ((n_slots or len(held)) - len(held)), np.uint32)
        need = -(-self.lengths.astype(np.int64) // page_rows)
        self.stride = stride or int(max(need)) + room
        self.n_pages = int(need.sum()) + room * len(self.lengths) + spare
        order = rng(seed).permutation(self.n_pages).astype(np.uint32)
        self.tables = np.full((len(self.lengths), self.stride), FILL, np.uint32)
        at = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = order[at:at + n]
            at += n
        self.n_free = self.n_pages - at
        self.free = np.full(self.n_pages, 0xFFFFFFFF, np.uint32)
        self.free[:self.n_free] = order[at:]
        up = fk.DeviceBuffer.from_numpy
        self.d_lengths, self.d_tables, self.d_free, self.d_n = up(self.lengths), up(self.tables), up(self.free), up(np.array([self.n_free], np.uint32))
        self.d_lengths_out, self.d_n_out = (self.d_lengths, self.d_n) if in_place else (up(np.full_like(self.lengths, FILL)), up(np.array([FILL], np.uint32)))
        self.counter, self.fault = fk.zeros(4), fk.zeros(4)

    def batch(self, slots, rows, capacity=None, max_rows=None, max_len=None, row_slots=True, stride=None):
        n, up = len(slots) if slots is not None else len(rows), self.fk.DeviceBuffer.from_numpy
        self.slots, self.rows = slots, rows
        self.capacity = capacity or max(1, int(np.sum(rows)))
        stride = stride or self.stride
        self.start = [np.full(n + 1, FILL, np.uint32), np.full(n, FILL, np.uint32), np.full((n, stride), FILL, np.uint32), np.full(self.capacity + 1, FILL, np.uint32)]
        self.d_out = [up(a) for a in self.start]
        self.d_slots = None if slots is None else up(np.array(slots, np.uint32))
        self.d_rows = None if rows is None else up(np.array(rows, np.uint32))
        self.b = self.fk.PagedBatch(*self.d_out[:3], stride, n, self.capacity, max_rows or max([1] + list(rows)), max_len or self.stride * self.page_rows, self.fault)
        self.row_slots = self.d_out[3] if row_slots else None
        return self

    def run(self, st=None, ones=False):
        q = self.fk.PagedRequests(self.d_slots, None if ones else self.d_rows, len(self.lengths), self.d_lengths, self.d_lengths_out, self.d_tables, self.stride,
                                  self.d_free, self.d_n, self.d_n_out, self.counter)
        self.fk.paged_extend(q, self.b, self.n_pages, self.page_rows, self.row_slots, st)
        return self

    def got(self):
        out = [d.to_numpy(np.uint32, a.shape) for d, a in zip(self.d_out, self.start)]
        return out + [self.d_lengths_out.to_numpy(np.uint32), self.d_tables.to_numpy(np.uint32, self.tables.shape), int(self.d_n_out.to_numpy(np.uint32)[0])]

    def check(self):
        self.fk.paged_check(self.fault)
        slots = range(len(self.rows)) if self.slots is None else self.slots
        ref = list(extend(slots, self.rows, self.lengths, self.tables, self.free, self.n_free, self.page_rows, self.start[2], self.start[3]))
        if self.row_slots is None:
            ref[3] = self.start[3]
        for name, a, b in zip(("row_start", "kv_len", "page_table", "row_slots", "lengths", "tables", "n_free"), self.got(), ref):
            assert np.array_equal(a, b), name
        assert self.counter.to_numpy(np.uint32)[0] == 0
        self.lengths, self.tables, self.n_free = ref[4:]
        return self

    def unchanged(self, fk, match):
        with pytest.raises(fk.InvalidArgument, match=match):
            fk.paged_check(self.fault)
        out = self.got()
        assert not out[0].any() and not out[1].any() and bool((out[2] == FILL).all() and (out[3] == FILL).all())
        assert np.array_equal(out[4], self.lengths) and np.array_equal(out[5], self.tables) and out[6] == self.n_free
        assert self.counter.to_numpy(np.uint32)[0] == 0


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("held", [0, 1, 15, 16, 17, 31, 32, 613])
@pytest.mark.parametrize("rows", [0, 1, 2, 15, 16, 17, 33, 200])
def test_one_sequence(fk, held, rows, in_place):
    r = Requests(fk, [held], page_rows=16, in_place=in_place).batch([0], [rows])
    r.run().check()


@pytest.mark.parametrize("page_rows", [16, 64, 1024])
@pytest.mark.parametrize("n", [2, 3, 5, 64, 255, 256, 257, 1003])
def test_many(fk, n, page_rows):
    g = rng(n)
    r = Requests(fk, g.integers(0, 3000, n + 7), page_rows=page_rows, room=48, seed=n)
    for step in range(2):                        # the second goes on from what the first left
        slots = g.permutation(n + 7)[:n]
        rows = np.where(g.random(n) < 0.1, g.integers(0, 300, n), 1)
        r.batch(slots, rows, capacity=int(rows.sum()) + 9).run().check()


def test_far_more_sequences_than_blocks(fk):
    g = rng(5)
    n = 20000
    r = Requests(fk, g.integers(0, 40, n), room=3, seed=5)
    r.batch(g.permutation(n), g.integers(0, 4, n)).run().check()


def test_by_none(fk):
    """Without slots and counts: sequence i in slot i, a row each; and without a slot map."""
    r = Requests(fk, [5, 16, 0, 99], n_slots=9).batch(None, [1, 1, 1, 1])
    r.run(ones=True).check()
    r.batch([3, 0], [1, 7], row_slots=False).run().check()


@pytest.mark.parametrize("rows", [700, 5000])
def test_chunks_among_tokens(fk, rows):
    r = Requests(fk, [33, 1000, 0, 17, 5], page_rows=32, room=400).batch([4, 2, 0, 1, 3], [1, rows, 1, rows - 33, 1])
    r.run().check()


def test_tables_wider_than_the_batch_s(fk):
    r = Requests(fk, [100, 200, 40], room=20).batch([2, 0], [3, 9], stride=15, max_len=230)
    r.run().check()


def test_the_last_free_page(fk):
    r = Requests(fk, [16, 32], room=2, spare=0)
    r.batch([0, 1], [32, 32]).run().check()
    assert r.n_free == 0
    r.batch([0, 1], [0, 0]).run().check()
    r.batch([1, 0], [0, 1], max_len=r.stride * 16).run()
    r.unchanged(fk, "fewer free pages|above max_len")


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("slots,rows,more,match", [([0, 3], [1, 1], {}, "slot beyond"), ([1, 0xFFFFFFFF], [1, 1], {}, "slot beyond"), ([1, 1], [1, 1], {}, "named twice"),
                                                   ([0, 1], [1, 5], dict(max_rows=4), "exceeds the launch"), ([0, 1], [3, 3], dict(capacity=5), "exceeds the launch"),
                                                   ([0, 1], [1, 0xFFFFFFFF], dict(capacity=8, max_rows=8), "exceeds the launch"),
                                                   ([0, 1], [1, 20], dict(max_len=100), "above max_len"), ([2, 1], [1, 1], dict(max_len=100), "above max_len")])
def test_what_does_not_fit_changes_nothing(fk, slots, rows, more, match, in_place):
    r = Requests(fk, [40, 90, 101], in_place=in_place).batch(slots, rows, **{**dict(capacity=64), **more})
    if not in_place:
        r.d_n_out.upload(np.array([7], np.uint32))
    r.run()
    r.unchanged(fk, match)
    r.batch([2, 0], [5, 6]).run().check()


def test_too_few_pages_and_a_broken_stack(fk):
    r = Requests(fk, [40, 90])
    for n, match in ((2, "fewer free pages"), (r.n_pages + 1, "does not have"), (0xFFFFFFFF, "does not have")):
        keep, r.n_free = r.n_free, n
        r.d_n.upload(np.array([n], np.uint32))
        r.batch([0, 1], [30, 40]).run()
        r.unchanged(fk, match)
        r.n_free = keep
    r.d_n.upload(np.array([r.n_free], np.uint32))
    r.d_free.upload(np.full(r.n_pages, r.n_pages, np.uint32))
    r.batch([0, 1], [30, 40]).run()
    with pytest.raises(fk.InvalidArgument, match="does not have"):
        fk.paged_check(r.fault)


@pytest.mark.parametrize("two_sets", [False, True])
def test_replays_of_a_captured_step(fk, stream, two_sets):  # noqa: F811
    """A graph of one step, replayed while the lengths grow in place on the device."""
    st, g = stream(), rng(8)
    r = Requests(fk, g.integers(0, 200, 70), room=40, seed=8).batch(g.permutation(70)[:50], g.integers(0, 9, 50), max_rows=9, capacity=500)
    r.run(st).check()
    work = fk.DeviceBuffer(1 << 20)
    if two_sets:                                # and two batches of it, one after the other in one graph
        s = Requests(fk, g.integers(0, 200, 20), room=40, seed=9).batch(g.permutation(20)[:20], g.integers(0, 9, 20), max_rows=9)
    graph = Graph(fk, st, lambda: (r.run(st), two_sets and s.run(st)))
    for i in range(5):
        graph.replay()
        fk.fill_u32(work, i, 1 << 18, st)
        fk.sync(st)
        r.check()
        if two_sets:
            s.check()
            s.start = s.got()[:4]
        r.start = r.got()[:4]                   # (what is not written stays)
    graph.free()
