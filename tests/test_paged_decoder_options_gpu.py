"""PagedDecoder's window, cap of scores and rotary options, through prompts in chunks and single tokens, against a plain decoder in 64 bits over the same bf16
weights.

Tolerance of logits: the decoder rounds to bf16 what it stores between its kernels, and a layer's scores, 2.6 in the mean here, carry their operands' roundings
into the probabilities.  What that amounts to is computed: the plain decoder with the same values rounded, off by D of a row's norm at most (1 to 4 %), is
one draw of these errors and the decoder another, which shares most of them; two that share none are sqrt(2) D apart, and a draw's norm, over the 256 dims that the
logits come from, is within a few times 256^-1/2 of its mean: 2 D from the unrounded one is allowed.  Every option moves the logits by more than three times
that, which is asserted."""
import numpy as np
import pytest

import oracle
from helpers import rel_l2, rng
from paged_reference import frequencies, rotated, wide

pytestmark = pytest.mark.gpu
SCALED = dict(scaling="parts", factor=8.0, low=1.0, high=4.0, trained=64)
OPTIONS = [dict(window=5), dict(window=37), dict(softcap=0.7), dict(window=20, softcap=1.5), dict(interleaved=True), dict(rope_dims=32), dict(rope_dims=0),
           dict(rope_dims=16, interleaved=True), dict(rope=SCALED), dict(rope=dict(scaling="linear", factor=4.0), window=33),
           dict(rope=dict(scaling="ramp", factor=16.0, low=1.0, high=8.0, trained=128), rope_dims=48, softcap=2.0)]


@pytest.fixture(scope="module", params=[(64, True), (128, False)], ids=["64-dims-norms", "128-dims"])
def model(fk, request):
    from fusekit_amd.decoder import DecoderConfig, DecoderWeights
    dim, norms = request.param
    cfg = DecoderConfig(n_layers=2, hidden=256, n_heads=4, n_kv=2, head_dim=dim, inter=384, vocab=512, theta=1e4, bits=16, qk_norm=norms)
    w = DecoderWeights.random_init(cfg, seed=5, std=0.1)
    return cfg, w, {n: wide(m.w.to_numpy(np.uint16, (m.n, m.k))) for n, m in w.mats.items()}, {n: wide(v.to_numpy(np.uint16)) for n, v in w.vecs.items()}


def bf16(x):
    return wide(oracle.f32_to_bf16(x.astype(np.float32)))


def plain(model, tokens, window=0, softcap=0.0, rope_dims=None, interleaved=False, rope=None, stored=lambda x: x):
    """Logits behind every token; `stored`: what becomes of a value that the decoder stores."""
    cfg, _, mats, vecs = model
    n, dims = len(tokens), cfg.head_dim if rope_dims is None else rope_dims
    norm = lambda x, w: x / np.sqrt((x * x).mean(-1, keepdims=True) + cfg.eps) * w
    freq = frequencies(dims, cfg.theta, **(rope or {})) if dims else np.ones(1)
    back = np.arange(n)[:, None] - np.arange(n)
    seen = (back >= 0) & (back < (window or n))
    x = mats["embed_tokens"][tokens]
    for l in range(cfg.n_layers):
        p = f"layers.{l}."
        h = stored(norm(x, vecs[p + "input_layernorm"]))
        q, k, v = (stored(h @ mats[p + f"self_attn.{i}_proj"].T).reshape(n, -1, cfg.head_dim) for i in "qkv")
        qw, kw = (vecs[p + f"self_attn.{i}_norm"] if cfg.qk_norm else None for i in "qk")
        q, k = (stored(rotated(a, np.arange(n), freq, dims, interleaved, b, cfg.eps)[0]) for a, b in ((q, qw), (k, kw)))
        k, v = (np.repeat(a, cfg.n_heads // cfg.n_kv, 1) for a in (k, v))
        s = np.einsum("ahd,bhd->hab", q, k) * cfg.head_dim ** -0.5
        s = softcap * np.tanh(s / softcap) if softcap else s
        s = np.exp(np.where(seen, s, -np.inf) - np.where(seen, s, -np.inf).max(-1, keepdims=True))
        att = np.einsum("hab,bhd->ahd", stored(s) / s.sum(-1, keepdims=True), v).reshape(n, -1)
        x = stored(x + stored(att) @ mats[p + "self_attn.o_proj"].T)
        h = stored(norm(x, vecs[p + "post_attention_layernorm"]))
        g = h @ mats[p + "mlp.gate_proj"].T
        x = stored(x + stored(g / (1 + np.exp(-g)) * (h @ mats[p + "mlp.up_proj"].T)) @ mats[p + "mlp.down_proj"].T)
    return stored(stored(norm(x, vecs["final_norm"])) @ mats.get("lm_head", mats["embed_tokens"]).T)


@pytest.mark.parametrize("options", [{}, *OPTIONS], ids=str)
def test_options(fk, model, options):
    from fusekit_amd.paged import PagedDecoder
    cfg = model[0]
    d = PagedDecoder(cfg, model[1], n_pages=40, page_rows=16, max_rows=96, max_seqs=4, **options)
    a, b = (rng(20 + i).integers(0, cfg.vocab, 90).tolist() for i in range(2))
    refs = [plain(model, t, **options) for t in (a, b)]
    off = lambda x, ref: np.linalg.norm(x - ref, axis=-1) / np.linalg.norm(ref, axis=-1)
    bar = 2 * max(off(plain(model, t, stored=bf16, **options), ref).max() for t, ref in zip((a, b), refs))
    assert bar < 0.1
    if options:                                               # the option counts
        assert np.linalg.norm(refs[0] - plain(model, a)) > 3 * bar * np.linalg.norm(refs[0])
    x, y = d.pages.new(), d.pages.new()
    done = [0, 0]
    for cuts in ((50, 1), (51, 2), (52, 40), (90, 41), (90, 90)):     # chunks, single tokens, both at once
        batch = [(s, t[at:to]) for s, t, at, to in zip((x, y), (a, b), done, cuts) if to > at]
        ends = [(r, to) for r, at, to in zip(refs, done, cuts) if to > at]
        got = d.forward(batch)
        fk.paged_check(d.fault)
        got = got.to_numpy(np.uint16)[:len(batch) * cfg.vocab].reshape(len(batch), cfg.vocab)
        for row, (ref, to) in zip(got, ends):
            assert rel_l2(row, ref[to - 1]) <= bar, (cuts, to, bar)
        done = list(cuts)
