"""The operators over a paged cache and of beam search inside captured graphs and on streams of the caller: a graph is replayed while lengths, scores, state
and inputs move on the device, with other work between the replays, and every replay is compared with the same calls made directly."""
import ctypes as C

import numpy as np
import pytest

from helpers import normal_bf16, rng
from paged_reference import frequencies

pytestmark = pytest.mark.gpu


class Graph:
    """Stream capture by the HIP runtime that the library is linked with."""

    def __init__(self, fk, stream, body):
        ok = lambda e: None if e == 0 else pytest.fail(f"HIP error {e}")
        self.hip, self.stream, self.exec, graph = fk.lib, C.c_void_p(stream), C.c_void_p(), C.c_void_p()
        ok(self.hip.hipStreamBeginCapture(self.stream, C.c_int(0)))
        body()
        ok(self.hip.hipStreamEndCapture(self.stream, C.byref(graph)))
        ok(self.hip.hipGraphInstantiate(C.byref(self.exec), graph, None, None, C.c_size_t(0)))
        self.graph, self.ok = graph, ok

    def replay(self):
        self.ok(self.hip.hipGraphLaunch(self.exec, self.stream))

    def free(self):
        self.ok(self.hip.hipGraphExecDestroy(self.exec))
        self.ok(self.hip.hipGraphDestroy(self.graph))


@pytest.fixture
def stream(fk):
    made = []

    def new():
        s = C.c_void_p()
        fk.check(fk.lib.fk_stream_create(C.byref(s)))
        made.append(s)
        return s.value
    yield new
    for s in made:
        fk.check(fk.lib.fk_stream_destroy(s))


class Step:
    """One decode step of a batch: lengths, rotation and append, attention, selection, state that follows; the next step starts from what it left."""

    def __init__(self, fk, stream, n=6, n_heads=8, n_kv=2, dim=64, page_rows=16, start=40, chunk=0, seed=1, beams=3, vocab=5003):
        self.fk, self.st, self.shape = fk, stream, (n, n_heads, n_kv, dim, beams, vocab)
        up = lambda a: fk.DeviceBuffer.from_numpy(np.ascontiguousarray(a))
        rows, most = [chunk] * (chunk > 0) + [1] * (n - (chunk > 0)), 640
        self.rows, pages = sum(rows), n * most // page_rows
        self.table = up(rng(seed).permutation(pages).astype(np.uint32))
        self.k, self.v = (up(normal_bf16(seed + i, pages * n_kv * page_rows * dim)) for i in (1, 2))
        self.start = up(np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32))
        self.steps = up(np.array([start + 17 * i + q - 1 for i, q in enumerate(rows)], np.uint32))
        self.len, self.offset = fk.zeros(4 * n), fk.zeros(4)
        self.width = (n_heads + 2 * n_kv) * dim
        self.qkv = up(normal_bf16(seed + 3, self.rows * self.width))
        self.q, self.out = fk.zeros(2 * self.rows * n_heads * dim), fk.zeros(2 * self.rows * n_heads * dim)
        self.freq = up(frequencies(dim, 1e4))
        self.batch = fk.PagedBatch(self.start, self.len, self.table, most // page_rows, n, self.rows, max(rows), most)
        self.pool = fk.PagePool(self.k, self.v, pages, page_rows, n_kv, dim)
        self.ws = fk.zeros(fk.sdpa_paged_workspace_bytes(n_heads, n_kv, dim, n, self.rows, most))
        g = n // beams
        self.logits, self.scores = up(normal_bf16(seed + 4, n * vocab)), up(-rng(seed).random(n).astype(np.float32))
        self.state = up(rng(seed).integers(0, 1 << 20, (n, 33)).astype(np.uint32))
        self.o_s, self.o_b, self.o_t = (fk.zeros(4 * n) for _ in range(3))
        self.bws = fk.zeros(fk.beam_select_workspace_bytes(g, beams, vocab, beams))
        self.same = up(np.tile(np.arange(beams, dtype=np.uint32), g))
        self.one = fk.zeros(4 * self.rows)
        fk.sync()

    def run(self):
        n, H, K, D, beams, vocab = self.shape
        fk, st, w, g = self.fk, self.st, self.width, self.shape[0] // self.shape[4]
        for i in range(n):
            fk.step_init(self.steps.ptr + 4 * i, self.offset, self.len.ptr + 4 * i, st)
        q = self.qkv.ptr
        fk.rope_paged_store(q, w, q + 2 * H * D, w, q + 2 * (H + K) * D, w, self.q, H * D, H, None, None, 0.0, D, False, self.freq, self.batch, self.pool, st)
        fk.sdpa_paged(self.q, H * D, self.out, H * D, H, D ** -0.5, 0.0, 0, self.batch, self.pool, self.ws, self.ws.nbytes, st)
        fk.beam_select(self.logits, vocab, self.scores, None, 0, g, beams, vocab, beams, self.o_s, self.o_b, self.o_t, self.bws, self.bws.nbytes, st)
        for state, row in ((self.state, 4 * 33), (self.logits, 2 * vocab)):
            fk.beam_reorder(state, state, row, self.o_b, g, beams, beams, st)
        # the next step's inputs: the scores, and what the attention gave as queries
        fk.beam_reorder(self.o_s, self.scores, 4, self.same, g, beams, beams, st)
        fk.beam_reorder(self.out, self.qkv, 2 * H * D, self.one, self.rows, 1, 1, st, dst_stride=2 * w)

    def now(self):
        return [b.to_numpy(np.uint16) for b in (self.out, self.q, self.k, self.v, self.o_s, self.o_b, self.o_t, self.state, self.logits, self.len)]


def same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a.now(), b.now()))


@pytest.mark.parametrize("chunk,start,dim", [(0, 40, 64), (0, 500, 128), (33, 40, 128), (70, 430, 64)])
def test_replays(fk, stream, chunk, start, dim):
    """Replays equal direct calls: lengths that grow within the plan, with single tokens, chunks, and contexts long enough to be cut."""
    st = stream()
    a, b = (Step(fk, st, chunk=chunk, start=start, dim=dim) for _ in range(2))
    a.run()                                            # (what a first call sets up is not captured)
    b.run()
    fk.sync(st)
    g = Graph(fk, st, a.run)
    work = fk.DeviceBuffer(1 << 20)
    for i in range(5):
        g.replay()
        b.run()
        fk.fill_u32(work, i, 1 << 18, st)
        fk.sync(st)
        assert same(a, b), i
        assert bool((work.to_numpy(np.uint32) == i).all())
    g.free()


def test_graphs_that_share_a_workspace_one_after_another(fk, stream):
    """Two captured graphs of other shapes over one workspace, replayed in turn on one stream."""
    st = stream()
    shapes = (dict(start=300, seed=2), dict(n=3, n_heads=16, n_kv=1, dim=128, start=500, seed=3))
    own, plain = [Step(fk, st, **s) for s in shapes], [Step(fk, st, **s) for s in shapes]
    for name in ("ws", "bws"):
        shared = fk.zeros(max(getattr(s, name).nbytes for s in own))
        for s in own:
            setattr(s, name, shared)
    for s in (*own, *plain):
        s.run()
    fk.sync(st)
    graphs = [Graph(fk, st, s.run) for s in own]
    for i in range(4):
        for g, p in zip(graphs, plain):
            g.replay()
            p.run()
        fk.sync(st)
        assert same(own[0], plain[0]) and same(own[1], plain[1]), i
    for g in graphs:
        g.free()


def test_streams_at_the_same_time(fk, stream):
    """Two batches with workspaces of their own on two streams at once."""
    one, two, third = stream(), stream(), stream()
    a, b = Step(fk, one, start=400, seed=4), Step(fk, two, start=400, seed=5)
    c, d = Step(fk, third, start=400, seed=4), Step(fk, third, start=400, seed=5)
    for _ in range(6):
        a.run()
        b.run()
    for st in (one, two):
        fk.sync(st)
    for _ in range(6):
        c.run()
        d.run()
    fk.sync(third)
    assert same(a, c) and same(b, d)


def test_pages_copied_in_a_graph(fk, stream):
    """A captured copy keeps the pairs that it was captured with."""
    st = stream()
    start = np.arange(3 * 40 * 64, dtype=np.uint32).reshape(3, 40, 64)
    pool, pairs = fk.DeviceBuffer.from_numpy(start), np.array([[1, 30], [1, 31], [5, 32]], np.uint32)
    g = Graph(fk, st, lambda: fk.pages_copy(pool, 3, 40 * 256, 40, 256, pairs, st))
    pairs[:] = 7
    for i in range(3):
        ref = start + np.uint32(i)
        pool.upload(ref)
        g.replay()
        fk.sync(st)
        ref = ref.copy()
        ref[:, 30], ref[:, 31], ref[:, 32] = ref[:, 1], ref[:, 1], ref[:, 5]
        assert np.array_equal(pool.to_numpy(np.uint32, ref.shape), ref)
    g.free()
