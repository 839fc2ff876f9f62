"""Several sequences of a dense decoder over one pool of pages: prompts in chunks among single tokens, forks that share pages, beam search.

PageAllocator keeps, on the host, which sequence has which pages: reference counts, a copy of the tail page where a shared one is about to be
written, compaction.  It moves no memory: what has to be copied it returns as pairs for fk_pages_copy.  PagedDecoder holds the pools of a
model's layers and runs batches over them; the kernels are rope_paged_store, sdpa_paged (sdpa_paged_sinks), beam_select, beam_reorder, paged_extend,
sample and those that prompt passes use.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np

from . import native
from .decoder import DecoderConfig, DecoderWeights
from .native import DeviceBuffer


class OutOfPages(RuntimeError):
    """The pool has fewer free pages than a call needs; nothing was changed."""


class PagedSequence:
    """Pages in order and positions held.  Made by PageAllocator.new / fork, given back with release."""

    __slots__ = ("pages", "length", "live")

    def __init__(self, pages: List[int], length: int):
        self.pages, self.length, self.live = pages, length, True


class PageAllocator:
    def __init__(self, n_pages: int, page_rows: int):
        if n_pages < 1 or page_rows < 1:
            raise ValueError("a pool has pages, and pages have rows")
        self.n_pages, self.page_rows = n_pages, page_rows
        self.users = np.zeros(n_pages, np.int64)              # sequences that hold a page
        self._free = list(range(n_pages - 1, -1, -1))         # the lowest is taken first
        self._sequences: Dict[int, PagedSequence] = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _mine(self, seq: PagedSequence) -> None:
        if not seq.live or self._sequences.get(id(seq)) is not seq:
            raise ValueError("not a sequence of this pool, or released")

    def new(self) -> PagedSequence:
        seq = PagedSequence([], 0)
        self._sequences[id(seq)] = seq
        return seq

    def fork(self, seq: PagedSequence) -> PagedSequence:
        """A sequence of its own with the same past; the pages are shared until one of the two writes into the last."""
        self._mine(seq)
        child = PagedSequence(list(seq.pages), seq.length)
        for p in child.pages:
            self.users[p] += 1
        self._sequences[id(child)] = child
        return child

    def release(self, seq: PagedSequence) -> None:
        self._mine(seq)
        for p in seq.pages:
            self.users[p] -= 1
            if self.users[p] == 0:
                self._free.append(p)
        seq.pages, seq.length, seq.live = [], 0, False
        del self._sequences[id(seq)]

    def extend(self, seqs: Sequence[PagedSequence], rows: Sequence[int]) -> List[Tuple[int, int]]:
        """Makes room for rows[i] further positions of seqs[i] (each sequence once) and counts them in.  Returns the page copies, (from, to), that
        have to run before anything is written and before a sequence is released."""
        seqs, rows = list(seqs), [int(r) for r in rows]
        if len(rows) != len(seqs) or len({id(s) for s in seqs}) != len(seqs) or any(r < 0 for r in rows):
            raise ValueError("one count of rows, not negative, for each of several sequences")
        need, users = 0, self.users.copy()
        shared = []
        for seq, r in zip(seqs, rows):
            self._mine(seq)
            own = bool(r and seq.length % self.page_rows and users[seq.pages[-1]] > 1)   # a tail page that others see too
            if own:
                users[seq.pages[-1]] -= 1
            shared.append(own)
            need += -(-(seq.length + r) // self.page_rows) - len(seq.pages) + own
        if need > len(self._free):
            raise OutOfPages(f"{need} pages wanted, {len(self._free)} free")
        copies = []
        for seq, r, own in zip(seqs, rows, shared):
            if own:
                page = self._take()
                copies.append((seq.pages[-1], page))
                self.users[seq.pages[-1]] -= 1
                seq.pages[-1] = page
            while len(seq.pages) * self.page_rows < seq.length + r:
                seq.pages.append(self._take())
            seq.length += r
        return copies

    def restore(self, seqs: Sequence[PagedSequence], held: Sequence[Tuple[List[int], int]]) -> None:
        """Takes an extend() of `seqs` back: held[i] is (list(seqs[i].pages), seqs[i].length) from before it, and nothing else has happened since."""
        for seq, (pages, length) in reversed(list(zip(seqs, held))):
            for i in reversed(range(len(seq.pages))):
                if i < len(pages) and pages[i] == seq.pages[i]:
                    continue
                self.users[seq.pages[i]] = 0
                self._free.append(seq.pages[i])
                if i < len(pages):                             # the tail that others see too
                    self.users[pages[i]] += 1
            seq.pages, seq.length = list(pages), length

    def _take(self) -> int:
        page = self._free.pop()
        self.users[page] = 1
        return page

    def adopt(self, seqs: Sequence[PagedSequence], lengths: Sequence[int], tables: np.ndarray, n_free: int) -> None:
        """What launches of paged_extend did to `seqs` since their lengths, pages and the stack of free pages were handed to the device: the lengths they
        have now, their rows of the tables and the free pages that are left.  Nothing else has happened to the pool meanwhile."""
        taken = [[int(p) for p in row[len(s.pages):-(-int(length) // self.page_rows)]] for s, length, row in zip(seqs, lengths, tables)]
        for seq in seqs:
            self._mine(seq)
        if sorted(p for pages in taken for p in pages) != sorted(self._free[n_free:]) or any(n < s.length for s, n in zip(seqs, lengths)):
            raise RuntimeError("the device's pages are not the host's")
        for seq, length, pages in zip(seqs, lengths, taken):
            seq.pages.extend(pages)
            seq.length = int(length)
            self.users[pages] = 1
        del self._free[n_free:]

    def truncate(self, seq: PagedSequence, length: int) -> None:
        """Drops the positions from `length` on."""
        self._mine(seq)
        if not 0 <= length <= seq.length:
            raise ValueError("a sequence is cut to a length that it has")
        keep = -(-length // self.page_rows)
        for p in seq.pages[keep:]:
            self.users[p] -= 1
            if self.users[p] == 0:
                self._free.append(p)
        del seq.pages[keep:]
        seq.length = length

    def compact(self) -> List[Tuple[int, int]]:
        """Moves the pages in use to the lowest ids.  Returns the copies; the sequences already name the new places."""
        used = int((self.users > 0).sum())
        holes = [p for p in range(used) if self.users[p] == 0]
        moved = dict(zip((int(p) for p in np.nonzero(self.users[used:])[0] + used), holes))
        for src, dst in moved.items():
            self.users[dst], self.users[src] = self.users[src], 0
        for seq in self._sequences.values():
            seq.pages = [moved.get(p, p) for p in seq.pages]
        self._free = list(range(self.n_pages - 1, used - 1, -1))
        return list(moved.items())

    def table(self, seqs: Sequence[PagedSequence], stride: int) -> np.ndarray:
        """The page table of a batch, [n, stride]; places without a page hold 0."""
        t = np.zeros((len(seqs), stride), np.uint32)
        for i, s in enumerate(seqs):
            self._mine(s)
            t[i, :len(s.pages)] = s.pages
        return t


def largest_rows(most: int) -> List[int]:
    """Row counts whose qgemm workspaces serve all counts up to `most`: the split of k differs between the forms of up to 32, up to 64 and more rows and
    with the number of 128-row tiles, so that more rows can need less."""
    return sorted({most, *(m for m in (32, 64) if m < most), *range(128, most, 128)})


class PagedDecoder:
    """A dense decoder over pages.  forward() takes any mix of sequences, each with its new tokens, and leaves the logits behind the last token
    of each."""

    def __init__(self, cfg: DecoderConfig, weights: DecoderWeights, n_pages: int, page_rows: int = 64, max_rows: int = 512, max_seqs: int = 64,
                 rope_dims: Optional[int] = None, interleaved: bool = False, rope: Optional[dict] = None, window: int = 0, softcap: float = 0.0,
                 stream=None, sinks: int = 0):
        """rope: scaling and its numbers as native.rope_frequencies takes them; window, softcap: of every layer; sinks: first positions that stay visible
        besides the window."""
        if cfg.kv_bits:
            raise ValueError("pages hold a bf16 cache")
        if cfg.head_dim not in (64, 128) or cfg.n_kv < 1 or cfg.n_heads % cfg.n_kv:
            raise ValueError("paged attention takes heads of 64 or 128 dims, and as many query heads for each KV head")
        if not 16 <= page_rows <= 1024 or page_rows & (page_rows - 1):
            raise ValueError("page_rows: a power of two from 16 to 1024")
        if min(n_pages, max_rows, max_seqs) < 1:
            raise ValueError("a decoder has pages, rows and sequences")
        if rope_dims is not None and (rope_dims % 16 or not 0 <= rope_dims <= cfg.head_dim):
            raise ValueError("rope_dims: a multiple of 16 up to head_dim, or 0")
        if not 0 <= window < 1 << 31 or not 0.0 <= softcap <= 1024.0:
            raise ValueError("window and softcap are not negative, softcap up to 1024 (0: none)")
        if not 0 <= sinks < 1 << 31:
            raise ValueError("sinks are not negative")
        self.cfg, self.w, self.stream = cfg, weights, stream
        self.pages = PageAllocator(n_pages, page_rows)
        self.max_rows, self.max_seqs, self.window, self.sinks, self.softcap = max_rows, max_seqs, window, sinks, softcap
        self.interleaved, self.rope_dims = interleaved, cfg.head_dim if rope_dims is None else rope_dims
        c, R, S = cfg, max_rows, max_seqs
        self.page_bytes = c.n_kv * page_rows * c.head_dim * 2
        self.plane_bytes = n_pages * self.page_bytes
        self.pool = DeviceBuffer(2 * c.n_layers * self.plane_bytes)               # layer l: plane 2 l keys, 2 l + 1 values
        self.layers = [native.PagePool(self.pool.ptr + 2 * l * self.plane_bytes, self.pool.ptr + (2 * l + 1) * self.plane_bytes, n_pages, page_rows,
                                       c.n_kv, c.head_dim) for l in range(c.n_layers)]
        self.freq = None
        if self.rope_dims:
            self.freq = DeviceBuffer(8 * (self.rope_dims // 2 + 1))
            native.rope_frequencies(self.rope_dims, c.theta, self.freq, **(rope or {}), stream=stream)
        # row starts, lengths, tokens and page tables of a batch, sent in one piece (a sequence may hold every page)
        self.batch_words = DeviceBuffer(4 * (S + 1 + S + R + S * n_pages))
        self.fault = native.zeros(4)
        self.x, self.x2, self.xn = (DeviceBuffer(R * c.hidden * 2) for _ in range(3))
        self.q, self.att = DeviceBuffer(R * c.n_q * 2), DeviceBuffer(R * c.n_q * 2)
        self.k, self.v = DeviceBuffer(R * c.n_kvd * 2), DeviceBuffer(R * c.n_kvd * 2)
        self.mid = DeviceBuffer(R * c.inter * 2)
        self.last = DeviceBuffer(S * c.hidden * 2)
        self.head = weights.mats.get("lm_head", weights.mats["embed_tokens"])
        self.logits = DeviceBuffer(S * c.vocab * 2)
        g = 0 if c.bits == 16 else c.group
        shapes = ((c.n_q + 2 * c.n_kvd, c.hidden), (c.hidden, c.n_q), (c.inter, c.hidden), (c.hidden, c.inter))
        ws = max(native.qgemm_workspace_bytes(m, n, k, g) for m in largest_rows(R) for n, k in shapes)
        ws = max(2 * ws, max(native.qgemm_workspace_bytes(m, c.vocab, c.hidden, 0 if self.head.bits == 16 else self.head.group) for m in largest_rows(S)))
        self.ws = DeviceBuffer(ws)
        self.sdpa_ws = native.zeros(native.SDPA_PAGED_WORKSPACE_MOST)

    def forward(self, batch: Sequence[Tuple[PagedSequence, Sequence[int]]]) -> DeviceBuffer:
        """Each sequence takes its new tokens (one at least); returns the logits [len(batch), vocab], overwritten by the next call.  A call that raises
        leaves the sequences as they were.  Does not wait for the device: what a launch finds wrong in a batch is in `fault`, for native.paged_check
        (beam_search and generate look at every step, sample at every round of steps)."""
        c = self.cfg
        seqs, tokens = [s for s, _ in batch], [list(t) for _, t in batch]
        n, rows = len(seqs), [len(t) for t in tokens]
        R = sum(rows)
        if not 0 < n <= self.max_seqs or R > self.max_rows or min(rows) < 1:
            raise ValueError("a batch has sequences with tokens, no more than max_seqs and max_rows")
        flat = [t for ts in tokens for t in ts]
        if min(flat) < 0 or max(flat) >= c.vocab:
            raise ValueError("a token outside of the vocabulary")
        held = [(list(s.pages), s.length) for s in seqs]
        copies = self.pages.extend(seqs, rows)
        try:
            self.copy_pages(copies)
            return self._launch(seqs, rows, flat)
        except BaseException:
            self.pages.restore(seqs, held)
            raise

    def _launch(self, seqs: List[PagedSequence], rows: List[int], flat: List[int]) -> DeviceBuffer:
        """The launches of forward(), for sequences that have room for their rows."""
        c, st = self.cfg, self.stream
        n, R = len(seqs), len(flat)
        starts = np.concatenate([[0], np.cumsum(rows)])
        stride = max(len(s.pages) for s in seqs)
        words = np.concatenate([starts, [s.length for s in seqs], flat, self.pages.table(seqs, stride).ravel()]).astype(np.uint32)
        if st is not None:
            native.sync(st)                                    # (the upload below does not wait for another stream's batch)
        self.batch_words.upload(words)
        at = [self.batch_words.ptr + 4 * i for i in (0, n + 1, 2 * n + 1, 2 * n + 1 + R)]
        b = native.PagedBatch(at[0], at[1], at[3], stride, n, R, max(rows), max(s.length for s in seqs), self.fault)
        self._layers(b, at[2])
        last = self.x
        if R > n:                                              # the last row of each sequence
            last = self.last
            for i in range(n):
                native.copy(self.last.ptr + i * c.hidden * 2, self.x.ptr + (int(starts[i + 1]) - 1) * c.hidden * 2, c.hidden * 2, st)
        return self._head(last, n)

    def _layers(self, b: native.PagedBatch, tokens) -> None:
        """A batch of rows from their tokens, on the device, to what the last layer leaves in self.x."""
        c, w, st, R = self.cfg, self.w, self.stream, b.rows
        native.embed_lookup_rows(w.mats["embed_tokens"], tokens, R, c.embed_scale, self.x, st)
        scale = float(c.head_dim) ** -0.5
        for l in range(c.n_layers):
            p = f"layers.{l}."
            m, vec = (lambda name: w.mats[p + name]), (lambda name: w.vecs[p + name])
            native.rmsnorm_rows(self.x, vec("input_layernorm"), c.eps, R, c.hidden, self.xn, st)
            biases = [vec(f"self_attn.{i}_proj.bias") for i in "qkv"] if c.qkv_bias else None
            native.qgemm_fanout([m(f"self_attn.{i}_proj") for i in "qkv"], self.xn, R, biases, [self.q, self.k, self.v], self.ws, st)
            norms = [vec("self_attn.q_norm"), vec("self_attn.k_norm")] if c.qk_norm else [None, None]
            native.rope_paged_store(self.q, c.n_q, self.k, c.n_kvd, self.v, c.n_kvd, self.q, c.n_q, c.n_heads, *norms, c.eps, self.rope_dims,
                                    self.interleaved, self.freq, b, self.layers[l], st)
            if self.sinks:
                native.sdpa_paged_sinks(self.q, c.n_q, self.att, c.n_q, c.n_heads, scale, self.softcap, self.window, self.sinks, b, self.layers[l],
                                        self.sdpa_ws, self.sdpa_ws.nbytes, st)
            else:
                native.sdpa_paged(self.q, c.n_q, self.att, c.n_q, c.n_heads, scale, self.softcap, self.window, b, self.layers[l], self.sdpa_ws,
                                  self.sdpa_ws.nbytes, st)
            native.qgemm(m("self_attn.o_proj"), self.att, R, None, self.x, self.x2, self.ws, st)
            native.rmsnorm_rows(self.x2, vec("post_attention_layernorm"), c.eps, R, c.hidden, self.xn, st)
            native.qgemm_swiglu(m("mlp.gate_proj"), m("mlp.up_proj"), self.xn, R, c.swiglu_variant, self.mid, self.ws, st)
            native.qgemm(m("mlp.down_proj"), self.mid, R, None, self.x2, self.x, self.ws, st)

    def _head(self, last, n: int) -> DeviceBuffer:
        """The logits of n rows of what the last layer left."""
        c, st = self.cfg, self.stream
        native.rmsnorm_rows(last, self.w.vecs["final_norm"], c.eps, n, c.hidden, self.xn, st)
        native.qgemm(self.head, self.xn, n, None, None, self.logits, self.ws, st)
        return self.logits

    def copy_pages(self, copies: Sequence[Tuple[int, int]]) -> None:
        """Page copies in every layer's pool."""
        if copies:
            native.pages_copy(self.pool, 2 * self.cfg.n_layers, self.plane_bytes, self.pages.n_pages, self.page_bytes, copies, self.stream)

    def compact(self) -> int:
        """Moves the pages in use to the front of the pool; returns how many were moved.  A call that raises leaves the sequences as they were."""
        a = self.pages
        held = a.users.copy(), list(a._free), [(s, s.pages) for s in a._sequences.values()]
        copies = a.compact()
        try:
            self.copy_pages(copies)
        except BaseException:
            a.users, a._free = held[0], held[1]
            for seq, pages in held[2]:
                seq.pages = pages
            raise
        return len(copies)

    def prefill(self, seq: PagedSequence, prompt: Sequence[int]) -> DeviceBuffer:
        """A prompt in chunks of max_rows tokens; the logits behind its last token are the first row.  A call that raises leaves the sequence at the
        positions that it had."""
        prompt, before = list(prompt), seq.length
        if not prompt:
            raise ValueError("empty prompt")
        try:
            for i in range(0, len(prompt), self.max_rows):
                logits = self.forward([(seq, prompt[i:i + self.max_rows])])
        except BaseException:
            if seq.live and seq.length > before:
                self.pages.truncate(seq, before)
            raise
        return logits

    def beam_search(self, prompt: Sequence[int], beams: int, max_tokens: int, eos: Optional[int] = None) -> List[Tuple[List[int], float]]:
        """The `beams` continuations that beam search ends with, the likeliest first: (tokens, sum of log probabilities).  A beam that
        takes `eos` (its last token then) goes on unchanged.  Pages are shared as far as the beams' pasts are the same."""
        if not 1 <= beams <= min(64, self.max_seqs) or max_tokens < 1 or beams > self.cfg.vocab:
            raise ValueError("beams: 1 to 64, max_seqs and the vocabulary at most, and a token at least")
        if beams > self.max_rows and max_tokens > 1:
            raise ValueError("a step takes a row for every beam: max_rows at most")
        c, st = self.cfg, self.stream
        u32 = lambda a: np.asarray(a, dtype=np.uint32)
        ws = native.zeros(max(native.beam_select_workspace_bytes(1, b, c.vocab, beams) for b in (1, beams)))
        chosen = DeviceBuffer(12 * beams)                       # scores, beams, tokens
        scores, finished = native.zeros(4 * beams), native.zeros(4 * beams)
        history = native.zeros(4 * beams * max_tokens)          # [beams, max_tokens]: follows the beams
        same = DeviceBuffer.from_numpy(np.arange(beams, dtype=np.uint32))
        live = [self.pages.new()]
        try:
            logits = self.prefill(live[0], prompt)
            over, lengths = [False], [0]
            for step in range(max_tokens):
                n = len(live)
                out = [chosen.ptr + 4 * beams * i for i in range(3)]
                native.beam_select(logits, c.vocab, scores, finished, 0, 1, n, c.vocab, beams, *out, ws, ws.nbytes, st)
                if step:
                    native.beam_reorder(history, history, 4 * max_tokens, out[1], 1, beams, beams, st)
                native.beam_reorder(out[2], history.ptr + 4 * step, 4, same, 1, beams, beams, st, dst_stride=4 * max_tokens)
                native.paged_check(self.fault, st)                 # (waits for the stream)
                total, parent, token = chosen.to_numpy(np.uint32, (3, beams))
                grown = [not over[p] for p in parent]
                over = [over[p] or (eos is not None and int(t) == eos) for p, t in zip(parent, token)]
                lengths = [lengths[p] + int(g) for p, g in zip(parent, grown)]
                scores.upload(total)
                finished.upload(u32(over))
                children = [self.pages.fork(live[p]) for p in parent]
                for s in live:
                    self.pages.release(s)
                live = children
                if step + 1 == max_tokens or all(over):
                    break
                # finished beams stand still: the others' rows are computed, and every beam's logits lie in its row
                order = sorted(range(beams), key=lambda i: over[i])
                if order != list(range(beams)):
                    live, over, lengths, token = ([a[i] for i in order] for a in (live, over, lengths, token))
                    perm = DeviceBuffer.from_numpy(u32(order))
                    for state, row in ((scores, 4), (finished, 4), (history, 4 * max_tokens)):
                        native.beam_reorder(state, state, row, perm, 1, beams, beams, st)
                    native.sync(st)
                logits = self.forward([(s, [int(t)]) for s, t, o in zip(live, token, over) if not o])
            native.sync(st)
            rows, total = history.to_numpy(np.uint32, (beams, max_tokens)), scores.to_numpy(np.float32)
            return [(rows[i, :lengths[i]].tolist(), float(total[i])) for i in sorted(range(beams), key=lambda i: -total[i])]
        finally:
            for s in live:
                if s.live:
                    self.pages.release(s)

    def generate(self, prompts: Sequence[Sequence[int]], max_tokens: int) -> List[List[int]]:
        """Greedy continuations of several prompts, decoded together."""
        c, st = self.cfg, self.stream
        prompts = [list(p) for p in prompts]
        n = len(prompts)
        if not 0 < n <= self.max_seqs or max_tokens < 1 or not all(prompts):
            raise ValueError("one prompt at least, max_seqs at most, none empty, and a token at least")
        if n > self.max_rows and max_tokens > 1:
            raise ValueError("a step takes a row for every prompt: max_rows at most")
        ws = native.zeros(max(native.beam_select_workspace_bytes(g, 1, c.vocab, 1) for g in range(1, n + 1)))
        zero, chosen = native.zeros(4 * n), DeviceBuffer(12 * n)
        out = [chosen.ptr + 4 * n * i for i in range(3)]

        def best(logits: DeviceBuffer, rows: int) -> List[int]:
            native.beam_select(logits, c.vocab, zero, None, 0, rows, 1, c.vocab, 1, *out, ws, ws.nbytes, st)
            native.paged_check(self.fault, st)                     # (waits for the stream)
            return [int(t) for t in chosen.to_numpy(np.uint32, (3, n))[2, :rows]]

        seqs = [self.pages.new() for _ in prompts]
        try:
            tokens = [best(self.prefill(s, p), 1) for s, p in zip(seqs, prompts)]
            for _ in range(max_tokens - 1):
                for t, nxt in zip(tokens, best(self.forward([(s, t[-1:]) for s, t in zip(seqs, tokens)]), n)):
                    t.append(nxt)
            return tokens
        finally:
            for s in seqs:
                self.pages.release(s)

    def sample(self, prompts: Sequence[Sequence[int]], max_tokens: int, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, seed: int = 0,
               eos: Optional[int] = None) -> List[List[int]]:
        """Continuations of several prompts, decoded together, each token drawn as fk_sample draws it.  The settings are one value for all or one a
        prompt; prompt i draws with random numbers of its own, from (seed, i).  A continuation ends behind `eos` or with max_tokens.

        The steps run on the device, which makes the batches (paged_extend), takes free pages and hands a step's tokens to the next: without `eos` the
        host does not wait between them.  With `eos` it looks after every 16 steps which have ended; those go no further then,
        and what they drew behind `eos` is dropped.  A call that raises leaves pages and sequences as they were."""
        c, pages = self.cfg, self.pages
        prompts = [list(p) for p in prompts]
        n = len(prompts)
        if not 0 < n <= self.max_seqs or max_tokens < 1 or not all(prompts):
            raise ValueError("one prompt at least, max_seqs at most, none empty, and a token at least")
        if n > self.max_rows and max_tokens > 1:
            raise ValueError("a step takes a row for every prompt: max_rows at most")
        if not 0 <= seed < 1 << 64:
            raise ValueError("a seed is a number of 64 bits, not negative")
        settings = []
        for name, value, word, sound in (("temperature", temperature, np.float32, lambda v: (v >= 0) & (v < np.inf)),
                                         ("top_k", top_k, np.uint32, lambda v: (v >= 0) & (v < 1 << 32) & (v == np.floor(v))),
                                         ("top_p", top_p, np.float32, lambda v: (v > 0) & (v <= 1)), ("min_p", min_p, np.float32, lambda v: (v >= 0) & (v <= 1))):
            v = np.asarray(value, np.float64)
            if v.shape not in ((), (n,)) or not sound(v).all():
                raise ValueError(f"{name}: one for all or one a prompt; a temperature is finite and not negative, top_k a count (0: all), top_p in (0, 1], min_p in [0, 1]")
            settings.append(np.broadcast_to(v, (n,)).astype(word))
        held = lambda length: -(-length // pages.page_rows)
        need = sum(held(len(p) + max_tokens - 1) for p in prompts)
        if need > pages.free_pages:
            raise OutOfPages(f"{need} pages wanted, {pages.free_pages} free")
        draws = np.stack([np.random.Generator(np.random.PCG64([seed, i])).random(max_tokens, np.float32) for i in range(n)], 1)
        ws = native.zeros(max(native.sample_workspace_bytes(r, c.vocab) for r in range(1, n + 1)))
        free = DeviceBuffer(4 * pages.n_pages)
        seqs = [pages.new() for _ in prompts]
        try:
            start = _Steps(self, ws, free, settings, draws[:1], [0] * n)
            for i, (s, p) in enumerate(zip(seqs, prompts)):
                start.draw(self.prefill(s, p), 0, i, 1)
            out = [[int(t)] for t in start.finish()[0]]
            while True:
                live = [i for i in range(n) if out[i][-1] != eos and len(out[i]) < max_tokens]
                if not live:
                    return out
                done = len(out[live[0]])                       # (all that live have as many)
                count = min(max_tokens - done, max_tokens if eos is None else self.LOOK)
                steps = _Steps(self, ws, free, [v[live] for v in settings], draws[done:done + count, live], [out[i][-1] for i in live], [seqs[i] for i in live])
                for j in range(count):
                    steps.run(j)
                for row in steps.finish():
                    for i, t in zip(live, row):
                        if out[i][-1] != eos:
                            out[i].append(int(t))
        finally:
            for s in seqs:
                pages.release(s)

    LOOK = 16   # steps of sample() between two looks for `eos`


class _Steps:
    """Steps of PagedDecoder.sample for a number of sequences, one row each: what they read and write lies on the device, in one piece."""

    def __init__(self, dec: PagedDecoder, ws: DeviceBuffer, free: DeviceBuffer, settings, draws: np.ndarray, tokens: Sequence[int],
                 seqs: Sequence[PagedSequence] = ()):
        """free: room for the stack of free pages; settings: temperature, top_k, top_p and min_p of each sequence; draws: random numbers
        [steps, sequences]; tokens: what the first step reads."""
        pages = dec.pages
        self.dec, self.ws, self.seqs, self.shape = dec, ws, list(seqs), draws.shape
        self.longest = max([s.length for s in seqs], default=0)
        self.stride = -(-(self.longest + len(draws)) // pages.page_rows)
        parts = [*settings, draws, tokens, np.zeros(draws.shape, np.uint32),                       # (the tokens drawn lie behind those read first)
                 [s.length for s in seqs], pages.table(seqs, self.stride), [pages.free_pages], [0],
                 np.zeros(len(seqs) + 1, np.uint32), np.zeros(len(seqs), np.uint32), np.zeros((len(seqs), self.stride), np.uint32)]
        words = [(a if isinstance(a, np.ndarray) and a.dtype == np.float32 else np.asarray(a, np.uint32)).ravel().view(np.uint32) for a in parts]
        self.mem = DeviceBuffer.from_numpy(np.concatenate(words))
        self.at = np.concatenate([[0], np.cumsum([4 * len(w) for w in words])]).tolist()
        place = [self.mem.ptr + a for a in self.at]
        self.settings, self.draws, self.tokens = place[:4], place[4], place[5]
        if seqs:
            lengths, tables, n_free, counter, *self.batch = place[7:14]
            need = sum(-(-(s.length + len(draws)) // pages.page_rows) - len(s.pages) for s in seqs)
            if need:                                           # (of the stack the steps read no more)
                free.upload(np.asarray(pages._free[-need:], np.uint32), 4 * (pages.free_pages - need))
            self.requests = native.PagedRequests(None, None, len(seqs), lengths, lengths, tables, self.stride, free, n_free, n_free, counter)

    def draw(self, logits, step: int, row: int, rows: int) -> None:
        """Tokens of the sequences row .. row + rows - 1 from their logits."""
        c, n, st = self.dec.cfg, self.shape[1], self.dec.stream
        native.sample(logits, c.vocab, rows, c.vocab, *(p + 4 * row for p in self.settings), self.draws + 4 * (n * step + row),
                      self.tokens + 4 * (n * (step + 1) + row), None, self.ws, self.ws.nbytes, st)

    def run(self, step: int) -> None:
        dec, n = self.dec, self.shape[1]
        b = native.PagedBatch(*self.batch, self.stride, n, n, 1, self.longest + step + 1, dec.fault)
        native.paged_extend(self.requests, b, dec.pages.n_pages, dec.pages.page_rows, None, dec.stream)
        dec._layers(b, self.tokens + 4 * n * step)
        self.draw(dec._head(dec.x, n), step, 0, n)

    def finish(self) -> np.ndarray:
        """Waits for the steps, hands what they took to the host's pages and returns the tokens drawn, [steps, sequences]."""
        dec, at = self.dec, self.at
        native.paged_check(dec.fault, dec.stream)
        words = self.mem.to_numpy(np.uint32)
        part = lambda i: words[at[i] // 4:at[i + 1] // 4]
        if self.seqs:
            dec.pages.adopt(self.seqs, part(7), part(8).reshape(-1, self.stride), int(part(9)[0]))
        return part(6).reshape(self.shape)
