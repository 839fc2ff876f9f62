"""Plain statements in 64 bits of the operators over a paged cache and of beam search's selection, for the tests."""
from __future__ import annotations

import numpy as np

import oracle
from helpers import normal_bf16, rng


def wide(bits):
    """bf16 bit patterns as float64."""
    return oracle.bf16_to_f32(np.asarray(bits)).astype(np.float64)


class Paged:
    """A batch and one layer's pages: rows[i] new rows of sequence i, lens[i] positions with them.  The pages lie in a random
    order; slots that hold no position, and whole pages that belong to nobody, are NaN unless `poison` is another pattern."""

    def __init__(self, rows, lens, n_kv, dim, page_rows, seed=0, spare_pages=3, spare_table=2, poison=0x7FC0, shared=None):
        self.rows, self.lens, self.n_kv, self.dim, self.page_rows = list(rows), list(lens), n_kv, dim, page_rows
        need = [-(-n // page_rows) for n in lens]
        self.n_pages, self.stride = sum(need) + spare_pages, max(need + [1]) + spare_table
        order = rng(seed).permutation(self.n_pages).astype(np.uint32)
        self.table = np.full((len(lens), self.stride), 0xFFFFFFFF, np.uint32)   # what is behind a sequence's pages is not read
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        shape = (self.n_pages, n_kv, page_rows, dim)
        self.k = np.full(shape, poison, np.uint16)
        self.v = np.full(shape, poison, np.uint16)
        for i, n in enumerate(lens):
            self.fill(i, normal_bf16(seed * 1000 + 2 * i + 1, (n, n_kv, dim)), normal_bf16(seed * 1000 + 2 * i + 2, (n, n_kv, dim)))
        self.row_start = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.uint32)
        self.kv_len = np.array(self.lens, np.uint32)

    def where(self, i, pos):
        pos = np.asarray(pos)
        return self.table[i, pos // self.page_rows], pos % self.page_rows

    def fill(self, i, k, v):
        page, slot = self.where(i, np.arange(len(k)))
        self.k[page, :, slot] = k
        self.v[page, :, slot] = v

    def gathered(self, i, pages):
        page, slot = self.where(i, np.arange(self.lens[i]))
        return wide(pages[page, :, slot])          # [n, n_kv, dim]

    def device(self, fk, rows=None, max_rows=None, max_len=None, fault=None):
        self.d = [fk.DeviceBuffer.from_numpy(a) for a in (self.row_start, self.kv_len, self.table, self.k, self.v)]
        batch = fk.PagedBatch(self.d[0], self.d[1], self.d[2], self.stride, len(self.rows), rows or max(1, sum(self.rows)),
                              max_rows or max(self.rows + [1]), max_len or max(self.lens + [1]), fault)
        return batch, fk.PagePool(self.d[3], self.d[4], self.n_pages, self.page_rows, self.n_kv, self.dim)


def attention(p: Paged, q, n_heads, scale, softcap=0.0, window=0):
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
            lo = max(0, pos - window + 1) if window else 0
            for h in range(n_heads):
                g = h // (n_heads // p.n_kv)
                x = k[lo:pos + 1, g] @ wide(q[at + j, h]) * scale
                if softcap:
                    x = softcap * np.tanh(x / softcap)
                w = np.exp(x - x.max())
                w /= w.sum()
                out[at + j, h] = w @ v[lo:pos + 1, g]
                size[at + j, h] = w @ np.abs(v[lo:pos + 1, g])
        at += r
    return out, size


def frequencies(dims, theta, scaling="plain", factor=1.0, low=0.0, high=0.0, trained=0):
    """Revolutions a position of each pair, then the factor of cos and sin."""
    i = np.arange(dims // 2, dtype=np.float64)
    rev = theta ** (-2 * i / dims) / (2 * np.pi)
    gain = 1.0
    if scaling == "linear":
        rev = rev / factor
    elif scaling == "parts":
        keep = np.clip((trained * rev - low) / (high - low), 0, 1)
        rev = rev * keep + rev / factor * (1 - keep)
    elif scaling == "ramp":
        pair = lambda turns: dims * np.log(trained / (turns * 2 * np.pi)) / (2 * np.log(theta))
        a, b = max(np.floor(pair(high)), 0), min(np.ceil(pair(low)), dims - 1)
        stretched = np.clip((i - a) / max(b - a, 1e-3), 0, 1)
        rev = rev * (1 - stretched) + rev / factor * stretched
        gain = 0.1 * np.log(factor) + 1
    return np.concatenate([rev, [gain]])


def rotated(x, pos, freq, dims, interleaved, norm=None, eps=1e-6):
    """(rotated heads, |lo| + |hi| of each value's pair): x float64 [..., heads, dim], pos [...]."""
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm
    out, size = x.copy(), np.abs(x)
    if dims:
        angle = 2 * np.pi * np.mod(np.asarray(pos, np.float64)[..., None] * freq[:-1], 1.0)
        c, s = np.cos(angle)[..., None, :] * freq[-1], np.sin(angle)[..., None, :] * freq[-1]
        lo, hi = (slice(0, dims, 2), slice(1, dims, 2)) if interleaved else (slice(0, dims // 2), slice(dims // 2, dims))
        out[..., lo] = x[..., lo] * c - x[..., hi] * s
        out[..., hi] = x[..., hi] * c + x[..., lo] * s
        size[..., lo] = size[..., hi] = (np.abs(x[..., lo]) + np.abs(x[..., hi])) * freq[-1]
    return out, size


def beams(logits, scores, finished, pad, groups, n_beams, k):
    """(scores, beams, tokens) of the k best of each group; logits float64 [groups * beams, vocab]."""
    x = np.where(np.isnan(logits), -np.inf, logits)
    with np.errstate(all="ignore"):
        m = x.max(-1, keepdims=True)
        total = scores.astype(np.float64)[:, None] - (m + np.log(np.exp(x - m).sum(-1, keepdims=True))) + x
    if finished is not None:
        over = finished != 0
        total[over] = -np.inf
        total[over, pad] = scores[over]
    total = np.where(np.isnan(total), -np.inf, total).reshape(groups, -1)
    order = np.argsort(-total, axis=-1, kind="stable")[:, :k]
    vocab = logits.shape[1]
    return np.take_along_axis(total, order, -1), order // vocab, order % vocab
