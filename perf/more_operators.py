"""What a decode loop over a paged cache needs so that it stays on the device, as cases that can be timed and compared.

    sample   tokens drawn from logits with a temperature, top-k, top-p and min-p of each row's own, from given random numbers (fk_sample)
    attend   attention over a paged cache through a sliding window, with the first positions visible besides (fk_sdpa_paged_sinks)
    extend   row starts, lengths, page tables and slot map of a batch built from the requests' lengths, pages taken from the free ones (fk_paged_extend)

A case is a dict of plain values; listed() gives the fixed ones, draw() more of the same ranges.  With `own` the passes are calls of the framework;
without, elementary torch operations in 32 bits or more, rounded once at the end.
"""
import math

import numpy as np
import torch

own = False


def listed():
    return [
        # one user of a small model, the usual settings: launch latency is nearly all of it
        {"name": "sample-1-row-32000", "kind": "sample", "rows": 1, "vocab": 32000, "spread": 2.5, "peaks": 40, "masked": 0.0, "lowest": False},
        # one user of a large vocabulary, an odd row, a grammar that forbids nine tokens in ten
        {"name": "sample-1-row-151851-masked", "kind": "sample", "rows": 1, "vocab": 151851, "spread": 2.0, "peaks": 30, "masked": 0.9, "lowest": False},
        # a server's decode step: 64 users, each with settings of its own
        {"name": "sample-64-rows-151936", "kind": "sample", "rows": 64, "vocab": 151936, "spread": 2.2, "peaks": 50, "masked": 0.0, "lowest": False},
        # many continuations of few prompts, as a trainer rolls them out: flat rows, where large parts of the vocabulary stay
        {"name": "sample-389-rows-151851-flat", "kind": "sample", "rows": 389, "vocab": 151851, "spread": 2.8, "peaks": 0, "masked": 0.0, "lowest": False},
        # a small assistant that chats without an end: one token, a window of 1000 positions and four first ones
        {"name": "attend-1-token-2611", "kind": "attend", "chunks": 0, "chunk_rows": 1, "decodes": 1, "shortest": 2611, "longest": 2611, "n_heads": 14,
         "n_kv": 2, "dim": 64, "page_rows": 16, "window": 1000, "sinks": 4, "softcap": 0.0},
        # a server's decode step: 64 conversations of up to 20000 positions, of which a token sees the last 4096 and the system prompt's start
        {"name": "attend-64-tokens-ragged", "kind": "attend", "chunks": 0, "chunk_rows": 1, "decodes": 64, "shortest": 190, "longest": 20000, "n_heads": 32,
         "n_kv": 8, "dim": 128, "page_rows": 64, "window": 4096, "sinks": 100, "softcap": 0.0},
        # a prompt's chunk and other users' single tokens in one pass, capped scores, a first position that lies alone
        {"name": "attend-chunk-among-tokens", "kind": "attend", "chunks": 1, "chunk_rows": 509, "decodes": 24, "shortest": 700, "longest": 9100,
         "n_heads": 32, "n_kv": 8, "dim": 128, "page_rows": 16, "window": 1500, "sinks": 1, "softcap": 30.0},
        # two long documents, a large chunk of each a pass
        {"name": "attend-2-chunks-2048", "kind": "attend", "chunks": 2, "chunk_rows": 2048, "decodes": 0, "shortest": 8000, "longest": 11000,
         "n_heads": 32, "n_kv": 8, "dim": 128, "page_rows": 32, "window": 4096, "sinks": 128, "softcap": 0.0},
        # one conversation's next token
        {"name": "extend-1-token", "kind": "extend", "seqs": 1, "slots": 4, "chunks": 0, "chunk_rows": 1, "shortest": 613, "longest": 613, "page_rows": 16},
        # a decode step of 256 of 320 conversations
        {"name": "extend-256-tokens", "kind": "extend", "seqs": 256, "slots": 320, "chunks": 0, "chunk_rows": 1, "shortest": 100, "longest": 30000,
         "page_rows": 16},
        # a thousand conversations, nine of them with a chunk of a new prompt
        {"name": "extend-1003-mixed", "kind": "extend", "seqs": 1003, "slots": 1100, "chunks": 9, "chunk_rows": 811, "shortest": 300, "longest": 60000,
         "page_rows": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Sizes spread over their ranges; none costs more than the largest listed case of its kind."""
    kind = rng.choice(("sample", "sample", "attend", "attend", "extend"))
    most = {}
    for c in listed():
        w = work(c)
        at = most.setdefault(c["kind"], {"bytes": 0.0, "flops": 0.0})
        most[c["kind"]] = {k: max(at[k], w[k]) for k in at}
    while True:
        if kind == "sample":
            c = {"kind": kind, "rows": _log(rng, 1, 600), "vocab": _log(rng, 150, 260000), "spread": rng.uniform(0.5, 4.0),
                 "peaks": rng.choice((0, 10, 60)), "masked": rng.choice((0.0, 0.0, 0.5, 0.98)), "lowest": rng.choice((False, True))}
        elif kind == "attend":
            n_kv, shortest = rng.choice((1, 2, 4, 8)), _log(rng, 1, 9000)
            c = {"kind": kind, "chunks": rng.choice((0, 0, 1, 2, 3)), "chunk_rows": _log(rng, 2, 2500), "decodes": _log(rng, 1, 97) - rng.randint(0, 1),
                 "shortest": shortest, "longest": _log(rng, shortest, 20000), "n_heads": n_kv * rng.choice((1, 2, 4, 7, 8)), "n_kv": n_kv,
                 "dim": rng.choice((64, 128)), "page_rows": rng.choice((16, 32, 64, 128, 256)), "window": _log(rng, 1, 6000),
                 "sinks": rng.choice((1, 4, _log(rng, 2, 600))), "softcap": rng.choice((0.0, 0.0, 20.0, 50.0))}
            c["decodes"] = max(c["decodes"], 0 if c["chunks"] else 1)
            rows, lens = _batch(c)
            if c["n_heads"] * c["chunks"] * max(rows) * max(lens) > 2.2e9 or len(rows) * c["n_kv"] * c["dim"] * max(lens) > 1.5e9:   # the plain form has to fit
                continue
        else:
            seqs, shortest = _log(rng, 1, 1400), _log(rng, 1, 4000)
            c = {"kind": kind, "seqs": seqs, "slots": seqs + _log(rng, 1, 200) - 1, "chunks": rng.randint(0, min(seqs, 9)), "chunk_rows": _log(rng, 2, 2500),
                 "shortest": shortest, "longest": _log(rng, shortest, 60000), "page_rows": rng.choice((16, 32, 64, 128, 256))}
        w = work(c)
        if all(w[k] <= most[kind][k] for k in w):
            return c


# ---------------------------------------------------------------- inputs

def _spread(n, shortest, longest):
    """n contexts spread over their logarithm, long and short ones mixed."""
    step = next(p for p in (7, 11, 13, 17, 19, 23, 29) if math.gcd(p, n) == 1)
    lo, hi = math.log(shortest), math.log(longest)
    return [int(round(math.exp(lo + (hi - lo) * (i * step % n + 1) / n))) for i in range(n)]


def _batch(case):
    """(new rows, positions) of each sequence, chunks first."""
    n = case["chunks"] + case["decodes"] if "decodes" in case else case["seqs"]
    rows = [max(1, case["chunk_rows"] - 37 * i) for i in range(case["chunks"])] + [1] * (n - case["chunks"])
    return rows, [b - 1 + r for b, r in zip(_spread(n, case["shortest"], case["longest"]), rows)]


def _pages(length, page_rows):
    return -(-length // page_rows)


def _normal(g, *shape, std=1.0):
    return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(0.0, std, generator=g)


def _dev(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _table(case, lens, rows_of_table, order):
    """Page ids of each length in turn, in a table of as many rows; order: the pool's pages shuffled."""
    need = [_pages(n, case["page_rows"]) for n in lens]
    table = torch.zeros(rows_of_table, max(max(need), 1), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, at


def _prepare_sample(s, case, g):
    rows, vocab = case["rows"], case["vocab"]
    s["logits"] = _normal(g, rows, vocab, std=case["spread"])
    if case["peaks"]:           # what a trained model's rows look like: a few tokens far above the others
        at = torch.randint(0, vocab, (rows, case["peaks"]), generator=g, device="cuda")
        s["logits"].scatter_(1, at, 9.0 + 3.0 * _normal(g, rows, case["peaks"]))
    if case["masked"]:
        hidden = torch.rand(rows, vocab, generator=g, device="cuda") < case["masked"]
        s["logits"].masked_fill_(hidden, torch.finfo(torch.bfloat16).min if case["lowest"] else -math.inf)
    some = lambda share: torch.rand(rows, generator=g, device="cuda") < share
    uniform = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g, device="cuda")
    s["temperature"] = torch.where(some(0.1), 0.0, uniform(0.3, 1.5))
    s["top_k"] = torch.where(some(0.5), 0, torch.randint(1, 200, (rows,), generator=g, device="cuda")).to(torch.int32)
    s["top_p"] = torch.where(some(0.3), 1.0, uniform(0.5, 1.0))
    s["min_p"] = torch.where(some(0.6), 0.0, uniform(0.0, 0.2))
    s["u"] = torch.rand(rows, generator=g, device="cuda")
    s.update(tokens=torch.zeros(rows, dtype=torch.int32, device="cuda"), logprobs=torch.zeros(rows, dtype=torch.float32, device="cuda"))


def _prepare_attend(s, case, g):
    rows, lens = _batch(case)
    nh, nk, d, per = case["n_heads"], case["n_kv"], case["dim"], case["page_rows"]
    n_pages = sum(_pages(n, per) for n in lens) + 3
    table, _ = _table(case, lens, len(lens), torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu())
    starts = np.concatenate([[0], np.cumsum(rows)]).tolist()
    s.update(rows=starts[-1], max_rows=max(rows), max_len=max(lens), n_pages=n_pages, row_start=_dev(starts), kv_len=_dev(lens), table=table.cuda(),
             k_pages=_normal(g, n_pages, nk, per, d), v_pages=_normal(g, n_pages, nk, per, d), q=_normal(g, starts[-1], nh, d, std=3.0),
             out=torch.empty(starts[-1], nh, d, dtype=torch.bfloat16, device="cuda"))


def _prepare_extend(s, case, g):
    """Requests in slots of a server's tables; the batch names its slots in an order of its own."""
    rows, lens = _batch(case)
    per, seqs, slots = case["page_rows"], case["seqs"], case["slots"]
    chosen = torch.randperm(slots, generator=g, device="cuda")[:seqs].to(torch.int32)
    held = torch.arange(slots) * 3 + 5          # (of the slots that are not in the batch)
    held[chosen.cpu().long()] = torch.tensor([n - r for n, r in zip(lens, rows)])
    held = held.tolist()
    need = sum(_pages(n, per) - _pages(n - r, per) for n, r in zip(lens, rows))
    n_pages = sum(_pages(n, per) for n in held) + need + 50
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu()
    table, used = _table(case, held, slots, order)
    stride = max(_pages(n, per) for n in lens + held)
    tables = torch.zeros(slots, stride, dtype=torch.int32)
    tables[:, :table.shape[1]] = table
    free = torch.zeros(n_pages, dtype=torch.int32)
    free[:n_pages - used] = order[used:]
    s.update(rows=sum(rows), max_rows=max(rows), max_len=stride * per, n_pages=n_pages, stride=stride, slot=chosen, new_rows=_dev(rows), lengths=_dev(held),
             tables=tables.cuda(), free=free.cuda(), n_free=_dev([n_pages - used]), n_free_out=_dev([0]), counter=_dev([0]),
             lengths_out=_dev([0] * slots), row_start=_dev([0] * (seqs + 1)), kv_len=_dev([0] * seqs),
             page_table=torch.zeros(seqs, stride, dtype=torch.int32, device="cuda"), row_slots=_dev([0] * sum(rows)), fault=_dev([0]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = case["kind"]
    s = {"case": case}
    {"sample": _prepare_sample, "attend": _prepare_attend, "extend": _prepare_extend}[kind](s, case, g)
    if own:
        import fusekit_amd.native as fk
        at = lambda name: s[name].data_ptr()
        if kind == "sample":
            s["scratch"] = torch.zeros(fk.sample_workspace_bytes(case["rows"], case["vocab"]), dtype=torch.uint8, device="cuda")
        elif kind == "attend":
            s["scratch"] = torch.zeros(fk.SDPA_PAGED_WORKSPACE_MOST, dtype=torch.uint8, device="cuda")
            s["pool"] = fk.PagePool(at("k_pages"), at("v_pages"), s["n_pages"], case["page_rows"], case["n_kv"], case["dim"])
            s["batch"] = fk.PagedBatch(at("row_start"), at("kv_len"), at("table"), s["table"].shape[1], s["table"].shape[0], s["rows"], s["max_rows"], s["max_len"])
        else:
            s["requests"] = fk.PagedRequests(at("slot"), at("new_rows"), case["slots"], at("lengths"), at("lengths_out"), at("tables"), s["stride"], at("free"),
                                             at("n_free"), at("n_free_out"), at("counter"))
            s["batch"] = fk.PagedBatch(at("row_start"), at("kv_len"), at("page_table"), s["stride"], case["seqs"], s["rows"], s["max_rows"], s["max_len"], at("fault"))
    return s


# ---------------------------------------------------------------- one pass

def _sample(s):
    """The whole vocabulary in order, running sums in 64 bits (a token next to the border of a sum must not depend on the sum's rounding)."""
    x, at = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True)
    x = x.double()
    vocab, n = x.shape[1], torch.arange(x.shape[1], device="cuda")
    top = x[:, :1]
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    k = s["top_k"].long()[:, None]
    k = torch.where(greedy, 1, torch.where(k == 0, vocab, k))
    w = torch.exp((x - top) / torch.where(greedy, 1.0, t))
    w = torch.where((n < k) & (x > -math.inf), w, 0.0)
    upto = torch.cumsum(w, -1)
    p = s["top_p"].double()[:, None]
    keep = (upto - w < p * upto[:, -1:]) & (w >= s["min_p"].double()[:, None]) | (n == 0)
    w = torch.where(keep, w, 0.0)
    upto = torch.cumsum(w, -1)
    first = (upto > s["u"].double()[:, None] * upto[:, -1:]).to(torch.int8).argmax(-1, keepdim=True)
    whole = torch.log(torch.where(x > -math.inf, torch.exp(x - top), 0.0).sum(-1, keepdim=True))
    empty = top == -math.inf
    lp = torch.where(empty, -math.inf, x.gather(1, first) - top - whole)
    return {"tokens": torch.where(empty, 0, at.gather(1, first)).view(-1).to(torch.int32), "logprobs": lp.view(-1).float()}


def _rows_of(s):
    """For each new row: its sequence, its place in the sequence's chunk, its position."""
    starts, lens = s["row_start"].long(), s["kv_len"].long()
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(starts[1:], row, right=True)
    place = row - starts[seq]
    return seq, place, lens[seq] - (starts[seq + 1] - starts[seq]) + place


def _weights(case, scores, seen):
    """exp(score - largest) of what is seen, [..., positions], and its sum."""
    if case["softcap"]:
        scores = case["softcap"] * torch.tanh(scores / case["softcap"])
    scores = scores.masked_fill(~seen, -math.inf)
    scores = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-3e38))
    return scores, scores.sum(-1, keepdim=True)


def _attend_tokens(s, seqs, rows):
    """Single tokens: the positions that each sees, gathered."""
    case = s["case"]
    nh, nk, d, per = case["n_heads"], case["n_kv"], case["dim"], case["page_rows"]
    pos = s["kv_len"][seqs].long()[:, None] - 1
    low = (pos - case["window"] + 1).clamp_min(0)
    near = pos - torch.arange(min(case["window"], s["max_len"]), device="cuda")
    far = torch.arange(min(case["sinks"], s["max_len"]), device="cuda").expand(pos.shape[0], -1)
    where, seen = torch.cat([far, near.clamp_min(0)], 1), torch.cat([far < low, near >= 0], 1)
    page = s["table"][seqs].long().gather(1, (where // per).clamp_max(s["table"].shape[1] - 1))
    k, v = (s[n][page, :, where % per].permute(0, 2, 1, 3).float() for n in ("k_pages", "v_pages"))       # [sequences, n_kv, positions, d]
    scores = torch.matmul(s["q"][rows].float().view(-1, nk, nh // nk, d), k.transpose(2, 3)) / math.sqrt(d)
    w, total = _weights(case, scores, seen[:, None, None])
    return (torch.matmul(w, v) / total).view(-1, nh, d).to(torch.bfloat16)


def _attend_chunks(s, seqs, rows):
    """Chunks as one padded batch, every position's score masked or not."""
    case = s["case"]
    nh, nk, d, most = case["n_heads"], case["n_kv"], case["dim"], s["max_rows"]
    table = s["table"][seqs].long()
    n = table.shape[0]
    seq, place, pos = (x[rows] for x in _rows_of(s))
    k, v = (s[m][table].permute(0, 2, 1, 3, 4).reshape(n, nk, -1, d).float() for m in ("k_pages", "v_pages"))
    q = torch.zeros(n, most, nh, d, device="cuda")
    q[seq, place] = s["q"][rows].float()
    at = torch.full((n, most, 1), -1, dtype=torch.int64, device="cuda")
    at[seq, place, 0] = pos
    scores = torch.matmul(q.view(n, most, nk, nh // nk, d).permute(0, 2, 3, 1, 4).reshape(n, nk, -1, d), k.transpose(2, 3)) / math.sqrt(d)
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key <= at) & ((key > at - case["window"]) | (key < case["sinks"]))
    w, total = _weights(case, scores.view(n, nk, nh // nk, most, -1), seen[:, None, None])
    out = torch.matmul(w.view(n, nk, -1, k.shape[2]), v) / total.view(n, nk, -1, 1)
    return out.view(n, nk, nh // nk, most, d).permute(0, 3, 1, 2, 4).reshape(n, most, nh, d)[seq, place].to(torch.bfloat16)


def _attend(s):
    """Chunks and single tokens apart, so that a token is not padded to a chunk."""
    chunks, decodes = s["case"]["chunks"], s["case"]["decodes"]
    cut = s["rows"] - decodes
    parts = [_attend_chunks(s, slice(0, chunks), slice(0, cut))] if chunks else []
    return torch.cat(parts + ([_attend_tokens(s, slice(chunks, chunks + decodes), slice(cut, s["rows"]))] if decodes else []))


def _extend(s):
    per = s["case"]["page_rows"]
    slot, rows = s["slot"].long(), s["new_rows"].long()
    held = s["lengths"].long()[slot]
    length = held + rows
    before, after = (held + per - 1) // per, (length + per - 1) // per
    taken = torch.cumsum(after - before, 0)
    column = torch.arange(s["stride"], device="cuda")
    fresh = (column >= before[:, None]) & (column < after[:, None])
    place = s["n_free"].long() - 1 - ((taken - (after - before) - before)[:, None] + column)      # in the free pages, the last is taken first
    pages = torch.where(fresh, s["free"][place.clamp(0, s["n_pages"] - 1)], s["tables"][slot])
    s["tables"][slot] = pages
    page_table = torch.where(column < after[:, None], pages, s["page_table"])
    ends = torch.cumsum(rows, 0)
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(ends, row, right=True)
    pos = held[seq] + row - (ends - rows)[seq]
    lengths = s["lengths"].clone()
    lengths[slot] = length.to(torch.int32)
    return {"row_start": torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32), "kv_len": length.to(torch.int32), "page_table": page_table,
            "row_slots": (page_table.long()[seq, pos // per] * per + pos % per).to(torch.int32), "tables": s["tables"], "lengths": lengths,
            "n_free": (s["n_free"] - taken[-1:]).to(torch.int32)}


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        import fusekit_amd.native as fk
        stream = torch.cuda.current_stream().cuda_stream
        at = lambda name: s[name].data_ptr()
        if kind == "sample":
            fk.sample(at("logits"), case["vocab"], case["rows"], case["vocab"], at("temperature"), at("top_k"), at("top_p"), at("min_p"), at("u"), at("tokens"),
                      at("logprobs"), at("scratch"), s["scratch"].numel(), stream)
            return {"tokens": s["tokens"], "logprobs": s["logprobs"]}
        if kind == "attend":
            nh, d = case["n_heads"], case["dim"]
            fk.sdpa_paged_sinks(at("q"), nh * d, at("out"), nh * d, nh, 1.0 / math.sqrt(d), case["softcap"], case["window"], case["sinks"], s["batch"], s["pool"],
                                at("scratch"), s["scratch"].numel(), stream)
            return s["out"]
        fk.paged_extend(s["requests"], s["batch"], s["n_pages"], case["page_rows"], at("row_slots"), stream)
        return {"row_start": s["row_start"], "kv_len": s["kv_len"], "page_table": s["page_table"], "row_slots": s["row_slots"], "tables": s["tables"],
                "lengths": s["lengths_out"], "n_free": s["n_free_out"]}
    return {"sample": _sample, "attend": _attend, "extend": _extend}[kind](s)


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_sample(s, case):
    """Row by row over the distinct logits, the largest first: how many tokens hold each, and what they weigh."""
    out = torch.empty(case["rows"], dtype=torch.float64)
    settings = [s[n].double().tolist() for n in ("temperature", "top_k", "top_p", "min_p", "u")]
    for r, (t, k, p, m, u) in enumerate(zip(*settings)):
        row = s["logits"][r].float()
        value, count = (x.double().cpu().numpy()[::-1] for x in torch.unique(row[row > -math.inf], return_counts=True))
        if not len(value):
            out[r] = -math.inf
            continue
        share = np.exp(value - value[0])
        if t == 0:
            out[r] = -math.log((share * count).sum())
            continue
        weight = np.exp((value - value[0]) / t)
        left = np.minimum(count, np.maximum((k if k else count.sum()) - (np.cumsum(count) - count), 0))     # tokens of each value that top-k leaves
        mass = np.cumsum(weight * left)
        need = np.ceil((p * mass[-1] - (mass - weight * left)) / np.maximum(weight, 1e-300))                # and that top-p needs of it
        left = np.where(weight >= m, np.minimum(left, np.maximum(need, 0)), 0)
        left[0] = max(left[0], 1)
        mass = np.cumsum(weight * left)
        out[r] = value[np.searchsorted(mass, u * mass[-1], side="right")] - value[0] - math.log((share * count).sum())
    return {"tokens": None, "logprobs": out.cuda()}


def _exact_attend(s, case):
    rows, lens = _batch(case)
    nh, nk, d, per = case["n_heads"], case["n_kv"], case["dim"], case["page_rows"]
    table = s["table"].cpu().long()
    out = torch.empty(s["rows"], nh, d, dtype=torch.float64, device="cuda")
    at = 0
    for i, (r, n) in enumerate(zip(rows, lens)):
        pages = table[i, :_pages(n, per)].cuda()
        back = n - r + torch.arange(r, device="cuda")[:, None] - torch.arange(n, device="cuda")     # how far back a key lies
        hidden = (back < 0) | (back >= case["window"])
        hidden[:, :case["sinks"]] &= back[:, :case["sinks"]] < 0
        for h in range(nk):
            kk, vv = (s[m][pages, h].reshape(-1, d)[:n].double() for m in ("k_pages", "v_pages"))
            for j in range(h * (nh // nk), (h + 1) * (nh // nk)):
                x = s["q"][at:at + r, j].double() @ kk.T * d ** -0.5
                if case["softcap"]:
                    x = torch.tanh(x / case["softcap"]) * case["softcap"]
                out[at:at + r, j] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ vv
        at += r
    return out


def exact(case, seed):
    if case["kind"] == "extend":
        return None                 # whole numbers
    s = prepare(case, seed)
    return _exact_sample(s, case) if case["kind"] == "sample" else _exact_attend(s, case)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["kind"] == "sample":
        return {"bytes": 2.0 * case["rows"] * case["vocab"] + 28.0 * case["rows"], "flops": 3.0 * case["rows"] * case["vocab"]}
    rows, lens = _batch(case)
    if case["kind"] == "extend":
        used = sum(_pages(n, case["page_rows"]) for n in lens)
        fresh = used - sum(_pages(n - r, case["page_rows"]) for r, n in zip(rows, lens))
        return {"bytes": 8.0 * used + 4.0 * fresh + 4.0 * sum(rows) + 16.0 * case["seqs"] + 8.0 * case["slots"], "flops": 0.0}
    nh, nk, d, window, sinks = case["n_heads"], case["n_kv"], case["dim"], case["window"], case["sinks"]
    pairs = read = 0
    for r, n in zip(rows, lens):
        pos = np.arange(n - r, n)
        low = np.maximum(pos - window + 1, 0)
        pairs += int((pos + 1 - low + np.minimum(low, sinks)).sum())
        read += n - int(low[0]) + min(int(low[0]), sinks)
    return {"bytes": 4.0 * nk * d * read + 4.0 * sum(rows) * nh * d, "flops": 4.0 * nh * d * pairs}
