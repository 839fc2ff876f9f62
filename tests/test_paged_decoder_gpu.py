"""Several sequences of a dense decoder over pages (fusekit_amd/paged.py): the operators together, as a serving loop and a beam search use them,
against the decoder that keeps one sequence in a contiguous cache and against plain beam search.

Tolerance of logits: the two paths round some eight bf16 values a layer in different places, 2 layers: sqrt(2 * 2 * 8) * 2^-8 / sqrt(3) < 1.3e-2 of
their norm; 2e-2 is allowed.  A log probability is then off by at most twice the largest difference of a row's logits."""
import json
import subprocess
import sys

import numpy as np
import pytest

import oracle
from helpers import rel_l2, rng

pytestmark = pytest.mark.gpu
BAR = 2e-2

CONFIGS = {
    "norms": dict(n_layers=2, hidden=512, n_heads=8, n_kv=2, head_dim=64, inter=768, vocab=1003, capacity=256, qk_norm=True),
    "biases": dict(n_layers=2, hidden=512, n_heads=4, n_kv=4, head_dim=128, inter=512, vocab=800, capacity=256, qkv_bias=True),
    "bf16": dict(n_layers=2, hidden=256, n_heads=4, n_kv=1, head_dim=64, inter=512, vocab=640, capacity=256, bits=16),
}


@pytest.fixture(scope="module")
def models(fk):
    from fusekit_amd.decoder import DecoderConfig, DecoderWeights
    made = {}

    def get(name):
        if name not in made:
            cfg = DecoderConfig(**CONFIGS[name])
            made[name] = cfg, DecoderWeights.random_init(cfg, seed=3, std=0.05)
        return made[name]
    return get


def paged(models, name, **more):
    from fusekit_amd.paged import PagedDecoder
    cfg, w = models(name)
    return cfg, PagedDecoder(cfg, w, **{**dict(n_pages=64, page_rows=16, max_rows=96, max_seqs=12), **more})


def logits_of(models, name, tokens):
    """Logits behind the last token, by the decoder with a contiguous cache."""
    from fusekit_amd.decoder import DecoderRuntime
    cfg, w = models(name)
    rt = DecoderRuntime(cfg, w)
    rt.prefill_rows(tokens)
    return rt.logits.to_numpy(np.uint16)


def wide(bits):
    return oracle.bf16_to_f32(bits).astype(np.float64)


@pytest.mark.parametrize("name", CONFIGS)
def test_batches_of_chunks_and_tokens(fk, models, name):
    cfg, d = paged(models, name, max_rows=192)
    text = rng(5).integers(0, cfg.vocab, (4, 80)).tolist()
    cuts = [[30, 31, 60], [1, 2, 40], [33, 64, 70], [5, 5, 80]]     # what each sequence has seen after each batch
    seqs, done = [d.pages.new() for _ in text], [0] * 4
    for step in range(3):
        batch = [(s, t[a:c[step]]) for s, t, a, c in zip(seqs, text, done, cuts) if c[step] > a]
        who = [i for i in range(4) if cuts[i][step] > done[i]]
        got = d.forward(batch)
        fk.sync()
        got = got.to_numpy(np.uint16)[:len(who) * cfg.vocab].reshape(len(who), cfg.vocab)
        done = [max(a, c[step]) for a, c in zip(done, cuts)]
        for row, i in zip(got, who):
            ref = logits_of(models, name, text[i][:done[i]])
            assert rel_l2(row, wide(ref)) <= BAR, (step, i)
    fk.paged_check(d.fault)


def test_forks_share_pages_and_compacting_keeps_them(fk, models):
    cfg, d = paged(models, "norms")
    text = rng(6).integers(0, cfg.vocab, 60).tolist()
    a, other = d.pages.new(), d.pages.new()
    d.forward([(other, text[:50]), (a, text[:37])])
    b, c = d.pages.fork(a), d.pages.fork(a)
    assert d.pages.free_pages == 64 - 4 - 3
    tails = {id(a): text[37:39], id(b): [7, 8, 9], id(c): [11]}
    got = d.forward([(s, tails[id(s)]) for s in (a, b, c)])
    fk.sync()
    first = got.to_numpy(np.uint16)[:3 * cfg.vocab].reshape(3, -1)
    assert d.pages.free_pages == 64 - 4 - 2 - 3                    # two pages shared, a tail each
    d.pages.release(other)
    assert d.compact() > 0 and sorted({p for s in (a, b, c) for p in s.pages}) == list(range(5))
    got = d.forward([(c, [3]), (a, [4]), (b, [5])])
    fk.sync()
    second = got.to_numpy(np.uint16)[:3 * cfg.vocab].reshape(3, -1)
    for row, tokens in [(first[0], text[:39]), (first[1], text[:37] + [7, 8, 9]), (first[2], text[:37] + [11]), (second[0], text[:37] + [11, 3]),
                        (second[1], text[:39] + [4]), (second[2], text[:37] + [7, 8, 9, 5])]:
        assert rel_l2(row, wide(logits_of(models, "norms", tokens))) <= BAR


@pytest.mark.parametrize("name", ["norms", "bf16"])
def test_generate_takes_the_likeliest_tokens(fk, models, name):
    cfg, d = paged(models, name, max_rows=24)
    prompts = [rng(7 + i).integers(0, cfg.vocab, n).tolist() for i, n in enumerate((3, 50, 17))]
    out = d.generate(prompts, 6)
    assert d.pages.free_pages == 64
    for p, tokens in zip(prompts, out):
        assert len(tokens) == 6
        for i, t in enumerate(tokens):
            x = wide(logits_of(models, name, p + tokens[:i]))
            assert x[t] >= x.max() - 2 * BAR * np.linalg.norm(x) / 8    # (a row's largest difference is far below its norm's share of it)


def log_probabilities(models, name, tokens):
    x = wide(logits_of(models, name, tokens))
    return x - x.max() - np.log(np.exp(x - x.max()).sum())


@pytest.mark.parametrize("beams,eos", [(1, None), (4, None), (5, 1)])
def test_beam_search(fk, models, beams, eos):
    name, steps = "norms", 5
    cfg, d = paged(models, name, max_rows=192)
    prompt = rng(9).integers(0, cfg.vocab, 21).tolist()
    if eos is not None:     # a token that the search does meet
        eos = int(np.argsort(-log_probabilities(models, name, prompt))[1])
    found = d.beam_search(prompt, beams, steps, eos)
    assert d.pages.free_pages == 64 and len(found) == beams and len({tuple(t) for t, _ in found}) == beams
    # plain: every continuation of every beam, from logits of its own
    plain = [([], 0.0)]
    for _ in range(steps):
        nxt = []
        for tokens, p in plain:
            if eos is not None and tokens and tokens[-1] == eos:
                nxt.append((tokens, p))
                continue
            lp = log_probabilities(models, name, prompt + tokens)
            nxt += [(tokens + [int(t)], p + float(lp[t])) for t in np.argsort(-lp)[:beams]]
        plain = sorted(nxt, key=lambda x: -x[1])[:beams]
    off = 2 * BAR * np.linalg.norm(wide(logits_of(models, name, prompt))) / 8 * steps
    for (tokens, p), (_, q) in zip(found, plain):
        assert abs(p - q) <= off
        assert eos is None or eos not in tokens[:-1]
        assert len(tokens) == steps or tokens[-1] == eos
        total = 0.0
        for i, t in enumerate(tokens):                              # the sum is that of its own tokens
            total += float(log_probabilities(models, name, prompt + tokens[:i])[t])
        assert abs(total - p) <= off
    if eos is not None:
        assert any(t[-1] == eos for t, _ in found)


def test_refusals(fk, models):
    from fusekit_amd.paged import OutOfPages
    cfg, d = paged(models, "norms", n_pages=4)
    s = d.pages.new()
    for bad in ([], [(s, [])], [(s, [1] * 97)], [(s, [1]), (s, [2])]):
        with pytest.raises(ValueError):
            d.forward(bad)
    with pytest.raises(OutOfPages):
        d.forward([(s, [1] * 65)])
    assert s.length == 0 and d.pages.free_pages == 4
    for bad in (dict(beams=0, max_tokens=1), dict(beams=13, max_tokens=1), dict(beams=2, max_tokens=0)):
        with pytest.raises(ValueError):
            d.beam_search([1], **bad)
    with pytest.raises(OutOfPages):
        d.beam_search([1] * 40, 4, 40)
    assert d.pages.free_pages == 4                                  # what a search held is given back


def test_command(fk, tmp_path):
    run = lambda *a: subprocess.run([sys.executable, "-m", "fusekit_amd", *a], capture_output=True, text=True, timeout=100)
    assert run("export-random", "--out", str(tmp_path / "m"), "--vocab", "500").returncode == 0
    r = run("generate", "--model", str(tmp_path / "m"), "--ids", "1,2,3,4,5", "--beams", "3", "--max-tokens", "4")
    assert r.returncode == 0, r.stderr[-500:]
    beams = json.loads(r.stdout.strip().splitlines()[-1])["beams"]
    assert len(beams) == 3 and all(len(b["tokens"]) == 4 for b in beams)
    assert beams[0]["log_probability"] >= beams[1]["log_probability"] >= beams[2]["log_probability"]


@pytest.mark.parametrize("tokens", [[1, 1003], [-1], [2 ** 32]])
def test_tokens_outside_of_the_vocabulary_change_nothing(fk, models, tokens):
    cfg, d = paged(models, "norms")
    s = d.pages.new()
    with pytest.raises(ValueError):
        d.forward([(s, tokens)])
    assert s.length == 0 and d.pages.free_pages == 64


def test_a_large_pool_sends_only_the_pages_of_the_batch(fk, models):
    cfg, d = paged(models, "norms", n_pages=5000)
    a, b = d.pages.new(), d.pages.new()
    tokens = rng(8).integers(0, cfg.vocab, 40).tolist()
    got = d.forward([(a, tokens), (b, tokens[:3])]).to_numpy(np.uint16)[:2 * cfg.vocab].reshape(2, -1)
    for row, t in zip(got, (tokens, tokens[:3])):
        assert rel_l2(row, wide(logits_of(models, "norms", t))) <= BAR
