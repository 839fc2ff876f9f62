"""Continuations drawn on the device (PagedDecoder.sample): batches built there, attention with a window and first positions, tokens drawn there, together as a
decode loop runs them, against the same loop over the host's batches with the plain statement of sampling in 64 bits; and the decoder with first positions
against a plain one in 64 bits.

The two loops launch the same kernels over the same rows, so that their logits are the same bits and their tokens equal.  Tolerance of the plain decoder's
logits: as derived for the decoder's other options (test_paged_decoder_options_gpu.py)."""
import json
import subprocess
import sys

import numpy as np
import pytest

import decode_loop_reference as ref
from helpers import rel_l2, rng
from paged_reference import frequencies, rotated, wide
from test_paged_decoder_gpu import models, paged  # noqa: F401 (a fixture)
from test_paged_decoder_options_gpu import bf16, model  # noqa: F401 (a fixture)
from test_paged_graph_gpu import Graph, stream  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
SETTINGS = dict(temperature=[0.7, 1.3, 0.0, 1.0], top_k=[0, 40, 0, 7], top_p=[0.9, 1.0, 1.0, 0.5], min_p=[0.0, 0.02, 0.0, 0.1])


def by_the_host(d, fk, prompts, max_tokens, temperature, top_k, top_p, min_p, seed, eos=None):
    """PagedDecoder.sample over batches of the host, every token drawn from the logits by the plain statement."""
    n, vocab = len(prompts), d.cfg.vocab
    each = [np.broadcast_to(np.asarray(v, t), (n,)) for v, t in ((temperature, np.float32), (top_k, np.uint32), (top_p, np.float32), (min_p, np.float32))]
    u = [np.random.Generator(np.random.PCG64([seed, i])).random(max_tokens, np.float32) for i in range(n)]
    seqs, out = [d.pages.new() for _ in prompts], [[] for _ in prompts]

    def drawn(rows, who):
        fk.paged_check(d.fault)
        logits = d.logits.to_numpy(np.uint16)[:rows * vocab].reshape(rows, vocab)
        return [ref.sample(wide(row), *(v[i] for v in each), u[i][len(out[i])])[0] for row, i in zip(logits, who)]
    for i, (s, p) in enumerate(zip(seqs, prompts)):
        d.prefill(s, p)
        out[i] += drawn(1, [i])
    ended = lambda t: eos in t if eos is not None else False
    while True:
        live = [i for i in range(n) if not ended(out[i]) and len(out[i]) < max_tokens]
        if not live:
            break
        for _ in range(min(max_tokens - len(out[live[0]]), max_tokens if eos is None else d.LOOK)):     # (those that end meanwhile go on to the round's end)
            d.forward([(seqs[i], out[i][-1:]) for i in live])
            for i, t in zip(live, drawn(len(live), live)):
                out[i].append(t)
    for s in seqs:
        d.pages.release(s)
    return [t[:t.index(eos) + 1] if ended(t) else t for t in out]


def prompts_of(cfg, lengths=(17, 1, 40, 64)):
    return [rng(30 + i).integers(0, cfg.vocab, n).tolist() for i, n in enumerate(lengths)]


@pytest.mark.parametrize("name,more", [("norms", dict(window=20, sinks=3)), ("biases", {}), ("bf16", dict(window=33, sinks=17, softcap=20.0)), ("norms", dict(sinks=4))], ids=str)
def test_the_loop_on_the_device(fk, models, name, more):  # noqa: F811
    cfg, d = paged(models, name, **more)
    e = paged(models, name, **more)[1]
    prompts = prompts_of(cfg)
    # (pages in no order, some held by others)
    for x in (d, e):
        other = [x.pages.new() for _ in range(9)]
        for s in other:
            x.prefill(s, [1] * 20)
        for s in other[1::2]:
            x.pages.release(s)
    free = sorted(d.pages._free)
    got = d.sample(prompts, 50, **SETTINGS, seed=7)
    assert got == by_the_host(e, fk, prompts, 50, **SETTINGS, seed=7)
    assert [len(t) for t in got] == [50] * 4 and sorted(d.pages._free) == free
    assert d.sample(prompts, 50, **SETTINGS, seed=7) == got          # the pages lie elsewhere now
    again = d.sample(prompts, 50, **SETTINGS, seed=8)
    assert again[2] == got[2] and all(a != b for i, (a, b) in enumerate(zip(again, got)) if i != 2)      # temperature 0 draws nothing


@pytest.mark.parametrize("tokens", [1, 2, 17, 18, 40])
def test_continuations_that_end(fk, models, tokens):  # noqa: F811
    cfg, d = paged(models, "norms", window=30, sinks=2)
    e = paged(models, "norms", window=30, sinks=2)[1]
    prompts, free = prompts_of(cfg), d.pages.free_pages
    settings = dict(temperature=0.5, top_k=3, top_p=1.0, min_p=0.0, seed=2)
    open_ended = by_the_host(e, fk, prompts, 40, **settings)
    # (a token that some continuation meets at its third place, so that this one ends)
    eos = open_ended[1][2]
    got = d.sample(prompts, tokens, **settings, eos=eos)
    assert got == by_the_host(e, fk, prompts, tokens, **settings, eos=eos)
    assert all(eos not in t[:-1] for t in got) and got[1] == open_ended[1][:open_ended[1].index(eos) + 1][:tokens] and d.pages.free_pages == free
    assert all(len(t) == tokens or t[-1] == eos for t in got)


def test_temperature_zero_is_greedy(fk, models):  # noqa: F811
    cfg, d = paged(models, "norms")
    prompts = prompts_of(cfg)
    assert d.sample(prompts, 20, temperature=0.0) == d.generate(prompts, 20) == d.sample(prompts, 20, top_k=1, seed=5)


def test_one_prompt_of_one_token(fk, models):  # noqa: F811
    cfg, d = paged(models, "bf16", max_seqs=1, max_rows=1, n_pages=2)
    got = d.sample([[5]], 32, seed=3)
    assert got == by_the_host(d, fk, [[5]], 32, 1.0, 0, 1.0, 0.0, 3) and d.pages.free_pages == 2
    assert d.sample([[5]], 1, seed=3) == [got[0][:1]]


def test_another_stream(fk, models, stream):  # noqa: F811
    cfg, d = paged(models, "norms", window=20, sinks=3)
    other = paged(models, "norms", window=20, sinks=3, stream=stream())[1]
    prompts = prompts_of(cfg)
    assert other.sample(prompts, 24, **SETTINGS, seed=1) == d.sample(prompts, 24, **SETTINGS, seed=1)


@pytest.mark.parametrize("name,nth", [("sample", 0), ("sample", 3), ("sample", 9), ("paged_extend", 0), ("paged_extend", 5), ("sdpa_paged_sinks", 11), ("qgemm", 30)])
def test_a_launch_that_is_refused(fk, models, monkeypatch, name, nth):  # noqa: F811
    cfg, d = paged(models, "norms", window=20, sinks=3)
    prompts, calls, real = prompts_of(cfg), [0], getattr(fk, name)
    kept = d.pages.new()
    d.prefill(kept, [3] * 20)
    before = d.pages.users.tolist(), sorted(d.pages._free)

    def fails(*args, **more):
        calls[0] += 1
        if calls[0] > nth:
            raise fk.InvalidArgument(fk.FK_ERR_INVALID, "refused")
        return real(*args, **more)
    with monkeypatch.context() as m:
        m.setattr(fk, name, fails)
        with pytest.raises(fk.InvalidArgument, match="refused"):
            d.sample(prompts, 20, **SETTINGS)
    assert (d.pages.users.tolist(), sorted(d.pages._free)) == before and kept.length == 20
    e = paged(models, "norms", window=20, sinks=3)[1]
    assert d.sample(prompts, 20, **SETTINGS) == e.sample(prompts, 20, **SETTINGS)


def test_what_a_launch_reports_is_raised(fk, models):  # noqa: F811
    cfg, d = paged(models, "norms")
    want = d.sample([[1], [2, 3]], 5, seed=1)
    d.fault.upload(np.array([2], np.uint32))                  # as a launch that meets a bad length sets it
    with pytest.raises(fk.InvalidArgument, match="length"):
        d.sample([[1], [2, 3]], 5, seed=1)
    assert d.pages.free_pages == 64 and d.sample([[1], [2, 3]], 5, seed=1) == want


def test_a_captured_round(fk, models, stream):  # noqa: F811
    """Six steps in one graph, replayed from the same state and from others, with eager work between the replays."""
    from fusekit_amd.paged import _Steps
    st = stream()
    cfg, d = paged(models, "norms", window=20, sinks=3, stream=st)
    prompts, count = prompts_of(cfg), 6
    word = (np.float32, np.uint32, np.float32, np.float32)
    settings = [np.asarray(v, t) for v, t in zip(SETTINGS.values(), word)]
    seqs = [d.pages.new() for _ in prompts]
    for s, p in zip(seqs, prompts):
        d.prefill(s, p)
    ws, free = fk.zeros(fk.sample_workspace_bytes(4, cfg.vocab)), fk.DeviceBuffer(4 * d.pages.n_pages)
    draws = [rng(i).random((count, 4), np.float32) for i in range(3)]
    make = lambda u: _Steps(d, ws, free, settings, u, [5, 6, 7, 8], seqs)

    def run(steps):
        for j in range(count):
            steps.run(j)

    def left(steps):
        fk.paged_check(d.fault, st)
        return steps.mem.to_numpy(np.uint32), d.logits.to_numpy(np.uint16)[:4 * cfg.vocab]
    eager = []
    for u in draws:
        steps = make(u)
        run(steps)
        eager.append(left(steps))
    steps = make(draws[0])
    graph = Graph(fk, st, lambda: run(steps))
    try:
        for i in (0, 2, 1, 1, 0):
            steps.mem.upload(make(draws[i]).mem.to_numpy(np.uint32))
            graph.replay()
            got = left(steps)
            assert all(np.array_equal(a, b) for a, b in zip(got, eager[i])), i
            other = make(draws[i])                             # eager work between two replays
            run(other)
            assert all(np.array_equal(a, b) for a, b in zip(left(other), eager[i]))
        steps.finish()
        assert [s.length for s in seqs] == [len(p) + count for p in prompts]
    finally:
        graph.free()


def plain(model, tokens, window, sinks, softcap=0.0, stored=lambda x: x):  # noqa: F811
    """Logits behind every token with `sinks` first positions besides the window; `stored`: what becomes of a value that the decoder stores."""
    cfg, _, mats, vecs = model
    n, freq = len(tokens), frequencies(cfg.head_dim, cfg.theta)
    norm = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + cfg.eps) * w
    at = np.arange(n)
    seen = (at <= at[:, None]) & ((at > at[:, None] - window) | (at < sinks))
    x = mats["embed_tokens"][tokens]
    for l in range(cfg.n_layers):
        p = f"layers.{l}."
        h = stored(norm(x, vecs[p + "input_layernorm"]))
        q, k, v = (stored(h @ mats[p + f"self_attn.{i}_proj"].T).reshape(n, -1, cfg.head_dim) for i in "qkv")
        qw, kw = (vecs[p + f"self_attn.{i}_norm"] if cfg.qk_norm else None for i in "qk")
        q, k = (stored(rotated(a, at, freq, cfg.head_dim, False, b, cfg.eps)[0]) for a, b in ((q, qw), (k, kw)))
        k, v = (np.repeat(a, cfg.n_heads // cfg.n_kv, 1) for a in (k, v))
        s = np.einsum("ahd,bhd->hab", q, k) * cfg.head_dim ** -0.5
        s = softcap * np.tanh(s / softcap) if softcap else s
        s = np.exp(np.where(seen, s, -np.inf) - np.where(seen, s, -np.inf).max(-1, keepdims=True))
        x = stored(x + stored(np.einsum("hab,bhd->ahd", stored(s) / s.sum(-1, keepdims=True), v).reshape(n, -1)) @ mats[p + "self_attn.o_proj"].T)
        h = stored(norm(x, vecs[p + "post_attention_layernorm"]))
        g = h @ mats[p + "mlp.gate_proj"].T
        x = stored(x + stored(g / (1 + np.exp(-g)) * (h @ mats[p + "mlp.up_proj"].T)) @ mats[p + "mlp.down_proj"].T)
    return stored(stored(norm(x, vecs["final_norm"])) @ mats.get("lm_head", mats["embed_tokens"]).T)


@pytest.mark.parametrize("options", [dict(window=5, sinks=4), dict(window=20, sinks=1), dict(window=11, sinks=33, softcap=1.5)], ids=str)
def test_first_positions_beside_the_window(fk, model, options):  # noqa: F811
    from fusekit_amd.paged import PagedDecoder
    cfg = model[0]
    d = PagedDecoder(cfg, model[1], n_pages=40, page_rows=16, max_rows=96, max_seqs=4, **options)
    a, b = (rng(20 + i).integers(0, cfg.vocab, 90).tolist() for i in range(2))
    refs = [plain(model, t, **options) for t in (a, b)]
    off = lambda x, r: np.linalg.norm(x - r, axis=-1) / np.linalg.norm(r, axis=-1)
    bar = 2 * max(off(plain(model, t, stored=bf16, **options), r).max() for t, r in zip((a, b), refs))
    assert bar < 0.1 and np.linalg.norm(refs[0] - plain(model, a, **{**options, "sinks": 0})) > 3 * bar * np.linalg.norm(refs[0])     # the option counts
    x, y = d.pages.new(), d.pages.new()
    done = [0, 0]
    for cuts in ((50, 1), (51, 2), (52, 40), (90, 41), (90, 90)):     # chunks, single tokens, both at once
        batch = [(s, t[at:to]) for s, t, at, to in zip((x, y), (a, b), done, cuts) if to > at]
        ends = [(r, to) for r, at, to in zip(refs, done, cuts) if to > at]
        got = d.forward(batch)
        fk.paged_check(d.fault)
        got = got.to_numpy(np.uint16)[:len(batch) * cfg.vocab].reshape(len(batch), cfg.vocab)
        for row, (r, to) in zip(got, ends):
            assert rel_l2(row, r[to - 1]) <= bar, (cuts, to, bar)
        done = list(cuts)


def test_command(fk, tmp_path):
    run = lambda *a: subprocess.run([sys.executable, "-m", "fusekit_amd", *a], capture_output=True, text=True, timeout=100)
    assert run("export-random", "--out", str(tmp_path / "m"), "--vocab", "500").returncode == 0
    from fusekit_amd.checkpoint import load_mlx_checkpoint
    from fusekit_amd.paged import PagedDecoder
    cfg, w = load_mlx_checkpoint(str(tmp_path / "m"), capacity=1024)
    d = PagedDecoder(cfg, w, 8, 16)
    want = [d.sample([[1, 2, 3]], 12, 0.8, 50, 0.95, 0.01, 3)[0], d.sample([[1, 2, 3]], 12, 1.5)[0]]
    for options, tokens in ((["--temperature", "0.8", "--top-k", "50", "--top-p", "0.95", "--min-p", "0.01", "--seed", "3"], want[0]), (["--temperature", "1.5"], want[1]),
                            (["--temperature", "1.5", "--eos", str(want[1][4])], want[1][:want[1].index(want[1][4]) + 1])):
        r = run("generate", "--model", str(tmp_path / "m"), "--ids", "1,2,3", "--max-tokens", "12", *options)
        assert r.returncode == 0, r.stderr[-500:]
        assert json.loads(r.stdout.strip().splitlines()[-1])["tokens"] == tokens
