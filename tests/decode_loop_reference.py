"""Plain statements in 64 bits of what a decode loop on the device is made of, for the tests: sampling, attention with a window and first positions, a batch
built from request lengths."""
from __future__ import annotations

import numpy as np

from paged_reference import Paged, wide


def sample(logits, t, k, p, m, u):
    """(token, log probability) of one row: logits float64, settings plain numbers."""
    x = np.where(np.isnan(logits), -np.inf, logits)
    top = x.max()
    if top == -np.inf:
        return 0, -np.inf
    with np.errstate(all="ignore"):
        away = np.where(x == top, 0.0, x - top)                         # (of an infinity: nothing beside it)
        lp = away - np.log(np.exp(away).sum())
        greedy = not t > 0
        order = np.argsort(-x, kind="stable")
        order = order[x[order] > -np.inf]
        order = order[:1] if greedy else order[:k] if k else order
        w = np.exp(away[order] / np.float64(1 if greedy else t))
    if p < 1:
        upto = np.cumsum(w)
        order = order[(upto - w < np.float64(p) * upto[-1]) | (np.arange(len(w)) == 0)]
        w = w[:len(order)]
    least = min(np.float64(m), 1.0) if m > 0 else 0.0
    order, w = order[w >= least], w[w >= least]
    upto = np.cumsum(w)
    u = min(np.float64(u), 1 - 2.0 ** -24) if u > 0 else 0.0             # (the nearest fp32 value in [0, 1); NaN as 0)
    at = int(np.searchsorted(upto, u * upto[-1], side="right"))
    return int(order[at]), float(lp[order[at]])


def attention(p: Paged, q, n_heads, scale, window, sinks, softcap=0.0):
    """(outputs [rows, n_heads, dim], sum p |v| / sum p of each): q bf16 bits [rows, n_heads, dim]."""
    out = np.zeros((sum(p.rows), n_heads, p.dim))
    size = np.zeros_like(out)
    at = 0
    for i, (r, n) in enumerate(zip(p.rows, p.lens)):
        k, v = p.gathered(i, p.k), p.gathered(i, p.v)
        for j in range(r):
            pos = n - r + j
            if pos < 0:
                continue
            key = np.arange(pos + 1)
            seen = (key < sinks) | (key > pos - window) if window else key >= 0
            for h in range(n_heads):
                g = h // (n_heads // p.n_kv)
                x = k[:pos + 1][seen, g] @ wide(q[at + j, h]) * scale
                if softcap:
                    x = softcap * np.tanh(x / softcap)
                w = np.exp(x - x.max())
                w /= w.sum()
                out[at + j, h] = w @ v[:pos + 1][seen, g]
                size[at + j, h] = w @ np.abs(v[:pos + 1][seen, g])
        at += r
    return out, size


def extend(slots, new_rows, lengths, tables, free, n_free, page_rows, page_table, row_slots):
    """(row_start, kv_len, page_table, row_slots, lengths, tables, n_free) behind a call that fits; the arrays given stay as they are."""
    lengths, tables, page_table, row_slots = (np.array(a) for a in (lengths, tables, page_table, row_slots))
    row_start, kv_len = [0], []
    for i, (s, r) in enumerate(zip(slots, new_rows)):
        held, length = int(lengths[s]), int(lengths[s]) + int(r)
        before, after = -(-held // page_rows), -(-length // page_rows)
        for c in range(before, after):
            n_free -= 1
            tables[s, c] = free[n_free]
        page_table[i, :after] = tables[s, :after]
        pos = np.arange(held, length)
        row_slots[row_start[-1]:row_start[-1] + int(r)] = tables[s, pos // page_rows].astype(np.int64) * page_rows + pos % page_rows
        row_start.append(row_start[-1] + int(r))
        kv_len.append(length)
        lengths[s] = length
    return np.array(row_start, np.uint32), np.array(kv_len, np.uint32), page_table, row_slots, lengths, tables, n_free
