"""What several sequences over a paged cache need, as cases that can be timed and compared.

    attend   attention of new rows (a chunk of a prompt, single tokens, both in one batch) over a paged cache
             (fk_sdpa_paged)
    rope     rotary positions of q and k, half-split or interleaved, part of a head, scaled for long contexts, and the
             append of k and v to the pages (fk_rope_paged_store)
    pages    pages copied inside a pool: what a fork leaves to copy, what compacting moves (fk_pages_copy)
    select   beam search's selection over the beams and the vocabulary (fk_beam_select)
    reorder  rows of per-beam state taken from the beams that were chosen (fk_beam_reorder)

A case is a dict of plain values; listed() gives the fixed ones, draw() more of the same ranges.  With `own` the passes are
calls of the framework; without, elementary torch operations in 32 bits or more, rounded once at the end.
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # a small assistant's single token behind a chat turn: launch latency and the host's call are nearly all of it
        {"name": "attend-1-token-613", "kind": "attend", "chunks": 0, "chunk_rows": 1, "decodes": 1, "shortest": 613, "longest": 613,
         "n_heads": 14, "n_kv": 2, "dim": 64, "page_rows": 16, "window": 0, "softcap": 0.0},
        # a server's decode step: 64 users, contexts from a short question to a long document
        {"name": "attend-64-tokens-ragged", "kind": "attend", "chunks": 0, "chunk_rows": 1, "decodes": 64, "shortest": 190, "longest": 9000,
         "n_heads": 32, "n_kv": 8, "dim": 128, "page_rows": 64, "window": 0, "softcap": 0.0},
        # a prompt's chunk and other users' single tokens in one pass, of a model whose layers look back 2000 positions and cap their scores
        {"name": "attend-chunk-among-tokens", "kind": "attend", "chunks": 1, "chunk_rows": 509, "decodes": 24, "shortest": 300, "longest": 4100,
         "n_heads": 32, "n_kv": 8, "dim": 128, "page_rows": 16, "window": 2000, "softcap": 30.0},
        # two long documents, a large chunk of each a pass
        {"name": "attend-2-chunks-2048", "kind": "attend", "chunks": 2, "chunk_rows": 2048, "decodes": 0, "shortest": 4000, "longest": 6000,
         "n_heads": 32, "n_kv": 8, "dim": 128, "page_rows": 32, "window": 0, "softcap": 0.0},
        # the small assistant's token: half-split pairs over the whole head
        {"name": "rope-1-token", "kind": "rope", "chunks": 0, "chunk_rows": 1, "decodes": 1, "shortest": 613, "longest": 613, "n_heads": 14,
         "n_kv": 2, "dim": 64, "rope_dims": 64, "interleaved": False, "norm": False, "scaling": "none", "page_rows": 16},
        # chunks of three prompts far into a stretched context among single tokens: interleaved pairs of half the head, head norms
        {"name": "rope-chunks-4000", "kind": "rope", "chunks": 3, "chunk_rows": 1371, "decodes": 13, "shortest": 2000, "longest": 60000,
         "n_heads": 32, "n_kv": 8, "dim": 128, "rope_dims": 64, "interleaved": True, "norm": True, "scaling": "ramp", "page_rows": 64},
        # a beam search of the small model forks its tail pages
        {"name": "pages-fork-4", "kind": "pages", "planes": 48, "n_pages": 640, "page_bytes": 4096, "pairs": 4},
        # a pool of the 4B class is compacted: its 36 layers' K and V
        {"name": "pages-compact-307", "kind": "pages", "planes": 72, "n_pages": 900, "page_bytes": 32768, "pairs": 307},
        # one request, four beams, a small vocabulary
        {"name": "select-4-beams-32000", "kind": "select", "groups": 1, "beams": 4, "vocab": 32000, "k": 8, "finished": False, "first": False},
        # sixteen requests of eight beams over a large vocabulary, twice as many candidates as beams; an odd row length
        {"name": "select-16x8-beams-151851", "kind": "select", "groups": 16, "beams": 8, "vocab": 151851, "k": 16, "finished": True, "first": False},
        # one request's page tables and token histories follow its four beams
        {"name": "reorder-4-beams-8KB", "kind": "reorder", "groups": 1, "beams": 4, "words": 2051},
        # recurrent or short-window states of eight requests of eight beams
        {"name": "reorder-8x8-beams-2MB", "kind": "reorder", "groups": 8, "beams": 8, "words": 600000},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Sizes spread over their ranges; none costs more than the largest listed case of its kind."""
    kind = rng.choice(("attend", "attend", "attend", "rope", "pages", "select", "reorder"))
    most = {}
    for c in listed():
        w = work(c)
        at = most.setdefault(c["kind"], {"bytes": 0.0, "flops": 0.0})
        most[c["kind"]] = {k: max(at[k], w[k]) for k in at}
    while True:
        if kind in ("attend", "rope"):
            n_kv, dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 128))
            shortest = _log(rng, 1, 4000)
            c = {"kind": kind, "chunks": rng.choice((0, 0, 1, 2, 3)), "chunk_rows": _log(rng, 2, 2500), "decodes": _log(rng, 1, 97) - rng.randint(0, 1),
                 "shortest": shortest, "longest": _log(rng, shortest, 12000), "n_heads": n_kv * rng.choice((1, 2, 4, 7, 8)), "n_kv": n_kv,
                 "dim": dim, "page_rows": rng.choice((16, 32, 64, 128, 256))}
            c["decodes"] = max(c["decodes"], 0 if c["chunks"] else 1)
            if kind == "attend":
                c.update(window=rng.choice((0, 0, _log(rng, 1, 4000))), softcap=rng.choice((0.0, 0.0, 20.0, 50.0)))
                rows, lens = _batch(c)
                if c["n_heads"] * max(c["chunks"] * max(rows), len(rows)) * max(lens) > 2.2e9:     # the plain form's scores have to fit
                    continue
            else:
                c.update(rope_dims=rng.choice((dim, dim, dim // 2, dim // 4)), interleaved=rng.choice((False, True)), norm=rng.choice((False, True)),
                         scaling=rng.choice(("none", "linear", "parts", "ramp")))
        elif kind == "pages":
            n = _log(rng, 8, 1500)
            c = {"kind": kind, "planes": _log(rng, 1, 96), "n_pages": n, "page_bytes": 16 * _log(rng, 16, 8192), "pairs": rng.randint(1, n // 2)}
            if c["planes"] * c["n_pages"] * c["page_bytes"] > 2.5e9:
                continue
        elif kind == "select":
            beams = rng.randint(1, 16)
            c = {"kind": kind, "groups": _log(rng, 1, 64), "beams": beams, "vocab": _log(rng, 500, 260000), "k": beams * rng.choice((1, 2)),
                 "finished": rng.choice((False, True)), "first": rng.choice((False, False, True))}
        else:
            c = {"kind": kind, "groups": _log(rng, 1, 32), "beams": rng.randint(2, 16), "words": _log(rng, 1, 600000)}
        w = work(c)
        if all(w[k] <= most[kind][k] for k in w):
            return c


# ---------------------------------------------------------------- inputs

def _batch(case):
    """(new rows, positions) of each sequence: contexts spread over their logarithm, long and short ones mixed."""
    n = case["chunks"] + case["decodes"]
    step = next(p for p in (7, 11, 13, 17, 19, 23) if math.gcd(p, n) == 1)
    lo, hi = math.log(case["shortest"]), math.log(case["longest"])
    before = [int(round(math.exp(lo + (hi - lo) * (i * step % n + 1) / n))) for i in range(n)]
    rows = [max(1, case["chunk_rows"] - 37 * i) for i in range(case["chunks"])] + [1] * case["decodes"]
    return rows, [b - 1 + r for b, r in zip(before, rows)]


def _frequencies(case):
    """Revolutions a position of every rotary pair, and last the factor of cos and sin (64 bits)."""
    dims, theta, factor, trained = case["rope_dims"], 1e6, 8.0, 8192
    inv = theta ** (-np.arange(0, dims, 2, dtype=np.float64) / dims)
    gain = 1.0
    if case["scaling"] == "linear":
        inv = inv / factor
    elif case["scaling"] == "parts":    # wavelengths longer than the trained context are stretched, short ones kept
        turns = trained * inv / (2 * math.pi)
        keep = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        inv = inv * (keep + (1 - keep) / factor)
    elif case["scaling"] == "ramp":     # a ramp over the pairs, from those that turn 32 times in the trained context to those that turn once
        at = [dims * math.log(trained / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dims - 1)
        ramp = np.clip((np.arange(dims // 2) - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
        inv = inv * (1 - ramp + ramp / factor)
        gain = 0.1 * math.log(factor) + 1.0
    return np.concatenate([inv / (2 * math.pi), [gain]])


def _normal(g, *shape, mean=0.0, std=1.0):
    return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(mean, std, generator=g)


def _dev(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _paged(s, case, g):
    """The batch's arrays, and pages for every position, anywhere in the pool."""
    rows, lens = _batch(case)
    need = [-(-n // case["page_rows"]) for n in lens]
    total, widest = sum(need), max(need)
    order = torch.randperm(total + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(rows), widest), 0, dtype=torch.int32)
    flat = order.cpu()
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = flat[at:at + n]
        at += n
    starts = np.concatenate([[0], np.cumsum(rows)]).tolist()
    s.update(rows=starts[-1], max_rows=max(rows), max_len=max(lens), n_pages=total + 3, row_start=_dev(starts), kv_len=_dev(lens), table=table.cuda())
    s.update(k_pages=_normal(g, total + 3, case["n_kv"], case["page_rows"], case["dim"]), v_pages=_normal(g, total + 3, case["n_kv"], case["page_rows"], case["dim"]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = case["kind"]
    s = {"case": case}
    if kind in ("attend", "rope"):
        _paged(s, case, g)
        nh, nk, d = case["n_heads"], case["n_kv"], case["dim"]
        if kind == "attend":
            s.update(q=_normal(g, s["rows"], nh, d, std=3.0), out=torch.empty(s["rows"], nh, d, dtype=torch.bfloat16, device="cuda"),
                     scratch=torch.zeros(64 << 20, dtype=torch.uint8, device="cuda"))
        else:
            # the projections' packed output rows
            s.update(qkv=_normal(g, s["rows"], nh + 2 * nk, d), q_out=torch.empty(s["rows"], nh, d, dtype=torch.bfloat16, device="cuda"),
                     freq=_dev(_frequencies(case).tolist(), torch.float64))
            s.update(q_norm=_normal(g, d, mean=1.0, std=0.1) if case["norm"] else None, k_norm=_normal(g, d, mean=1.0, std=0.1) if case["norm"] else None)
        if own:
            import fusekit_amd.native as fk
            s.update(pool=fk.PagePool(s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), s["n_pages"], case["page_rows"], nk, d),
                     batch=fk.PagedBatch(s["row_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1],
                                         s["table"].shape[0], s["rows"], s["max_rows"], s["max_len"]))
    elif kind == "pages":
        s["pool"] = torch.empty(case["planes"], case["n_pages"], case["page_bytes"] // 4, dtype=torch.int32, device="cuda").random_(generator=g)
        order = torch.randperm(case["n_pages"], generator=g, device="cuda").to(torch.int64)
        s["src"], s["dst"] = order[:case["pairs"]].clone(), order[case["pairs"]:2 * case["pairs"]].clone()
        s["pairs"] = np.ascontiguousarray(torch.stack([s["src"], s["dst"]], 1).cpu().numpy().astype(np.uint32))   # as the page allocator has them
    elif kind == "select":
        n = case["groups"] * case["beams"]
        s["logits"] = _normal(g, n, case["vocab"], std=3.0)
        s["scores"] = -5.0 * torch.rand(n, generator=g, device="cuda") - 10.0
        if case["first"]:       # the first step: all beams are the prompt, only the first counts
            s["scores"] = s["scores"].view(case["groups"], -1).masked_fill_(torch.arange(case["beams"], device="cuda") > 0, -math.inf).view(-1)
        s["finished"] = (torch.rand(n, generator=g, device="cuda") < 0.15).to(torch.int32) if case["finished"] else None
        shape = (case["groups"], case["k"])
        s.update(out_scores=torch.empty(shape, dtype=torch.float32, device="cuda"), out_beams=torch.empty(shape, dtype=torch.int32, device="cuda"),
                 out_tokens=torch.empty(shape, dtype=torch.int32, device="cuda"), scratch=torch.zeros(64 << 20, dtype=torch.uint8, device="cuda"))
    else:
        n = case["groups"] * case["beams"]
        s["state"] = torch.empty(n, case["words"], dtype=torch.int32, device="cuda").random_(generator=g)
        s["moved"] = torch.empty_like(s["state"])
        s["parents"] = torch.randint(0, case["beams"], (case["groups"], case["beams"]), generator=g, device="cuda").to(torch.int32)
    return s


# ---------------------------------------------------------------- one pass

def _rows_of(s):
    """For each new row: its sequence, its place in the sequence's chunk, its position."""
    starts, lens = s["row_start"].long(), s["kv_len"].long()
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(starts[1:], row, right=True)
    place = row - starts[seq]
    return seq, place, lens[seq] - (starts[seq + 1] - starts[seq]) + place


def _attend_some(s, seqs, rows, most):
    """The rows `rows` of the sequences `seqs` (slices), at most `most` rows a sequence, as one padded batch."""
    case = s["case"]
    nh, nk, d = case["n_heads"], case["n_kv"], case["dim"]
    table = s["table"][seqs].long()
    n_seqs = table.shape[0]
    seq, place, pos = (x[rows] for x in _rows_of(s))
    seq = seq - seqs.start
    k, v = (s[n][table].permute(0, 2, 1, 3, 4).reshape(n_seqs, nk, -1, d).float() for n in ("k_pages", "v_pages"))
    q = torch.zeros(n_seqs, most, nh, d, device="cuda")
    q[seq, place] = s["q"][rows].float()
    at = torch.full((n_seqs, most), -1, dtype=torch.int64, device="cuda")
    at[seq, place] = pos
    scores = torch.matmul(q.view(n_seqs, most, nk, nh // nk, d).permute(0, 2, 3, 1, 4).reshape(n_seqs, nk, -1, d), k.transpose(2, 3)) / math.sqrt(d)
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= at[..., None]
    if case["window"]:
        seen &= key > at[..., None] - case["window"]
    scores = scores.view(n_seqs, nk, nh // nk, most, -1).masked_fill(~seen[:, None, None], -math.inf)
    scores = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-3e38)).view(n_seqs, nk, -1, k.shape[2])
    out = torch.matmul(scores, v) / scores.sum(-1, keepdim=True)
    return out.view(n_seqs, nk, nh // nk, most, d).permute(0, 3, 1, 2, 4).reshape(n_seqs, most, nh, d)[seq, place].to(torch.bfloat16)


def _attend(s):
    """Chunks and single tokens apart, so that a token is not padded to a chunk."""
    chunks, decodes = s["case"]["chunks"], s["case"]["decodes"]
    cut = s["rows"] - decodes
    parts = []
    if chunks:
        parts.append(_attend_some(s, slice(0, chunks), slice(0, cut), s["max_rows"]))
    if decodes:
        parts.append(_attend_some(s, slice(chunks, chunks + decodes), slice(cut, s["rows"]), 1))
    return torch.cat(parts)


def _normed(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()


def _turned(x, cos, sin, interleaved):
    dims = 2 * cos.shape[-1]
    lo, hi = (x[..., 0:dims:2], x[..., 1:dims:2]) if interleaved else (x[..., :dims // 2], x[..., dims // 2:dims])
    turned = (lo * cos - hi * sin, hi * cos + lo * sin)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat([turned, x[..., dims:]], -1).to(torch.bfloat16)


def _rope(s):
    case = s["case"]
    nh, nk = case["n_heads"], case["n_kv"]
    seq, _, pos = _rows_of(s)
    angle = 2 * math.pi * torch.frac(pos[:, None].double() * s["freq"][:-1])
    cos, sin = ((f(angle) * s["freq"][-1]).float()[:, None] for f in (torch.cos, torch.sin))
    q, k, v = s["qkv"].split((nh, nk, nk), 1)
    page, slot = s["table"].long()[seq, pos // case["page_rows"]], pos % case["page_rows"]
    s["k_pages"][page, :, slot] = _turned(_normed(k, s["k_norm"]), cos, sin, case["interleaved"])
    s["v_pages"][page, :, slot] = v
    return {"q": _turned(_normed(q, s["q_norm"]), cos, sin, case["interleaved"]), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _select(s):
    case = s["case"]
    groups, beams, vocab, k = case["groups"], case["beams"], case["vocab"], case["k"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    total = s["scores"].double()[:, None] + (x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))))
    if s["finished"] is not None:   # a finished beam goes on as it is, with token 0
        over = s["finished"].bool()[:, None]
        token = torch.arange(vocab, device="cuda")
        total = torch.where(over, torch.where(token == 0, s["scores"].double()[:, None], -math.inf), total)
    scores, at = torch.sort(total.view(groups, beams * vocab), dim=-1, descending=True, stable=True)
    at = at[:, :k]
    return {"scores": scores[:, :k].float(), "beams": (at // vocab).to(torch.int32), "tokens": (at % vocab).to(torch.int32)}


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        import fusekit_amd.native as fk
        stream = torch.cuda.current_stream().cuda_stream
        if kind == "attend":
            nh, d = case["n_heads"], case["dim"]
            fk.sdpa_paged(s["q"].data_ptr(), nh * d, s["out"].data_ptr(), nh * d, nh, 1.0 / math.sqrt(d), case["softcap"], case["window"],
                          s["batch"], s["pool"], s["scratch"].data_ptr(), s["scratch"].numel(), stream)
            return s["out"]
        if kind == "rope":
            nh, nk, d = case["n_heads"], case["n_kv"], case["dim"]
            q, row = s["qkv"].data_ptr(), (nh + 2 * nk) * d
            norms = [None if s[n] is None else s[n].data_ptr() for n in ("q_norm", "k_norm")]
            fk.rope_paged_store(q, row, q + 2 * nh * d, row, q + 2 * (nh + nk) * d, row, s["q_out"].data_ptr(), nh * d, nh, norms[0], norms[1], 1e-6,
                                case["rope_dims"], case["interleaved"], s["freq"].data_ptr(), s["batch"], s["pool"], stream)
            return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if kind == "pages":
            fk.pages_copy(s["pool"].data_ptr(), case["planes"], case["n_pages"] * case["page_bytes"], case["n_pages"], case["page_bytes"], s["pairs"], stream)
            return s["pool"]
        if kind == "select":
            over = None if s["finished"] is None else s["finished"].data_ptr()
            fk.beam_select(s["logits"].data_ptr(), case["vocab"], s["scores"].data_ptr(), over, 0, case["groups"], case["beams"], case["vocab"], case["k"],
                           s["out_scores"].data_ptr(), s["out_beams"].data_ptr(), s["out_tokens"].data_ptr(), s["scratch"].data_ptr(),
                           s["scratch"].numel(), stream)
            return {"scores": s["out_scores"], "beams": s["out_beams"], "tokens": s["out_tokens"]}
        fk.beam_reorder(s["state"].data_ptr(), s["moved"].data_ptr(), 4 * case["words"], s["parents"].data_ptr(), case["groups"], case["beams"],
                        case["beams"], stream)
        return s["moved"]
    if kind == "attend":
        return _attend(s)
    if kind == "rope":
        return _rope(s)
    if kind == "pages":
        s["pool"][:, s["dst"]] = s["pool"][:, s["src"]]
        return s["pool"]
    if kind == "select":
        return _select(s)
    first = torch.arange(case["groups"], device="cuda")[:, None] * case["beams"]
    return s["state"][(s["parents"].long() + first).view(-1)]


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("pages", "reorder"):
        return None                 # whole numbers that are moved
    if kind == "select":
        lp = torch.log_softmax(s["logits"].double(), -1) + s["scores"].double()[:, None]
        if s["finished"] is not None:
            for r in torch.nonzero(s["finished"]).view(-1).tolist():
                lp[r] = -math.inf
                lp[r, 0] = s["scores"][r].double()
        lp = lp.view(case["groups"], -1)
        return {"scores": torch.topk(lp, case["k"]).values, "beams": None, "tokens": None}
    rows, lens = _batch(case)
    nh, nk, d, per = case["n_heads"], case["n_kv"], case["dim"], case["page_rows"]
    table = s["table"].cpu().long()
    if kind == "attend":
        out = torch.empty(s["rows"], nh, d, dtype=torch.float64, device="cuda")
        at = 0
        for i, (r, n) in enumerate(zip(rows, lens)):
            pages = table[i, :-(-n // per)].cuda()
            where = n - r + torch.arange(r, device="cuda")[:, None] - torch.arange(n, device="cuda")      # how far back a key lies
            hidden = (where < 0) | (where >= case["window"]) if case["window"] else where < 0
            for h in range(nk):
                kk, vv = (s[p][pages, h].reshape(-1, d)[:n].double() for p in ("k_pages", "v_pages"))
                for j in range(h * (nh // nk), (h + 1) * (nh // nk)):
                    x = s["q"][at:at + r, j].double() @ kk.T * d ** -0.5
                    if case["softcap"]:
                        x = torch.tanh(x / case["softcap"]) * case["softcap"]
                    out[at:at + r, j] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ vv
            at += r
        return out
    f = torch.from_numpy(_frequencies(case)).cuda()
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    x = s["qkv"].double()
    if case["norm"]:
        for part, w in ((x[:, :nh], s["q_norm"]), (x[:, nh:nh + nk], s["k_norm"])):
            part /= torch.sqrt((part * part).sum(-1, keepdim=True) / d + 1e-6)
            part *= w.double()
    pos = torch.cat([torch.arange(n - r, n) for r, n in zip(rows, lens)]).cuda()
    phase = pos.double()[:, None] * f[:-1]
    spin = torch.polar(f[-1].expand_as(phase).contiguous(), 2 * math.pi * (phase - torch.floor(phase)))[:, None]
    m = case["rope_dims"]
    part = x[:, :nh + nk, :m]
    z = torch.complex(part[..., 0::2].contiguous(), part[..., 1::2].contiguous()) if case["interleaved"] else torch.complex(part[..., :m // 2].contiguous(), part[..., m // 2:].contiguous())
    z = z * spin
    x[:, :nh + nk, :m] = torch.view_as_real(z).reshape(part.shape) if case["interleaved"] else torch.cat([z.real, z.imag], -1)
    seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows))
    page, slot = table[seq, pos.cpu() // per].cuda(), pos % per
    for h in range(nk):
        k_pages[page, h, slot] = x[:, nh + h]
        v_pages[page, h, slot] = x[:, nh + nk + h]
    return {"q": x[:, :nh].contiguous(), "k_pages": k_pages, "v_pages": v_pages}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind in ("attend", "rope"):
        rows, lens = _batch(case)
        nh, nk, d = case["n_heads"], case["n_kv"], case["dim"]
        if kind == "rope":
            return {"bytes": 4.0 * sum(rows) * (nh + 2 * nk) * d, "flops": 3.0 * sum(rows) * (nh + nk) * case["rope_dims"]}
        window = case["window"] or max(lens)
        pairs = sum(min(p + 1, window) for r, n in zip(rows, lens) for p in range(n - r, n))
        read = sum(n - max(0, n - r - window + 1) for r, n in zip(rows, lens))
        return {"bytes": 4.0 * nk * d * read + 4.0 * sum(rows) * nh * d, "flops": 4.0 * nh * d * pairs}
    if kind == "pages":
        return {"bytes": 2.0 * case["planes"] * case["pairs"] * case["page_bytes"], "flops": 0.0}
    n = case["groups"] * case["beams"]
    if kind == "select":
        return {"bytes": 2.0 * n * case["vocab"] + 4.0 * n + 12.0 * case["groups"] * case["k"], "flops": 4.0 * n * case["vocab"]}
    return {"bytes": 8.0 * n * case["words"] + 4.0 * n, "flops": 0.0}
