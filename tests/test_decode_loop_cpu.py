"""Refusals of sampling, of attention with first positions and of batches built on the device: they come before a device is looked for.  Plain numbers stand
for addresses; nothing is launched."""
import numpy as np
import pytest

import decode_loop_reference as ref
import fusekit_amd.native as fk
from test_paged_cpu import BATCHES, POOLS, batch, pool, refused

A, B, C = 0x10000, 0x100000, 0x200000   # aligned addresses that nothing reads


def draw(**change):
    v = dict(logits=C, stride=100, rows=4, vocab=100, temperature=A, top_k=A + 64, top_p=A + 128, min_p=A + 192, u=A + 256, tokens=B, logprobs=B + 64,
             workspace=B + 4096, size=1 << 30)
    v.update(change)
    fk.sample(v["logits"], v["stride"], v["rows"], v["vocab"], v["temperature"], v["top_k"], v["top_p"], v["min_p"], v["u"], v["tokens"], v["logprobs"],
              v["workspace"], v["size"])


@pytest.mark.parametrize("change", [dict(logits=None), dict(u=None), dict(tokens=None), dict(workspace=None), dict(rows=0), dict(vocab=0), dict(stride=99), dict(size=0),
                                    dict(logits=C + 1), dict(temperature=A + 2), dict(top_k=A + 1), dict(top_p=A + 3), dict(min_p=A + 2), dict(u=A + 258),
                                    dict(tokens=B + 1), dict(logprobs=B + 66), dict(workspace=B + 4100), dict(rows=65536), dict(vocab=(1 << 24) + 1, stride=1 << 25),
                                    dict(stride=1 << 62), dict(tokens=A), dict(tokens=A + 52), dict(tokens=C + 780), dict(tokens=A + 256), dict(logprobs=A + 128),
                                    dict(logprobs=B + 12), dict(logprobs=B + 4096), dict(tokens=B + 4096)], ids=str)
def test_sample(change):
    refused(lambda: draw(**change))


def test_sample_workspaces():
    assert fk.sample_workspace_bytes(1, 1) > 0 and fk.sample_workspace_bytes(65535, 1 << 24) > 0
    for bad in ((0, 10), (10, 0), (65536, 10), (1, (1 << 24) + 1)):
        refused(lambda: fk.sample_workspace_bytes(*bad))


def attend(b=None, p=None, **change):
    v = dict(q=B, q_stride=256, out=C, out_stride=256, n_heads=4, scale=0.125, softcap=0.0, window=100, sinks=4, workspace=A, workspace_bytes=64 << 20)
    v.update(change)
    fk.sdpa_paged_sinks(v["q"], v["q_stride"], v["out"], v["out_stride"], v["n_heads"], v["scale"], v["softcap"], v["window"], v["sinks"], b or batch(),
                        p or pool(), v["workspace"], v["workspace_bytes"])


@pytest.mark.parametrize("change", [dict(b=batch(**c)) for c in BATCHES] + [dict(p=pool(**c)) for c in POOLS] +
                         [dict(q=None), dict(out=None), dict(workspace=None), dict(n_heads=3), dict(q_stride=248), dict(q_stride=260), dict(out=B), dict(scale=0.0),
                          dict(softcap=-1.0), dict(workspace_bytes=0), dict(q=A + 2)], ids=lambda c: "-".join(c))
def test_attention(change):
    refused(lambda: attend(**change))


def extend(b=None, n_pages=64, page_rows=16, row_slots=C, **change):
    v = dict(slot=A, new_rows=A + 0x100, n_slots=4, lengths=A + 0x200, lengths_out=A + 0x200, tables=A + 0x1000, table_stride=8, free_pages=A + 0x300,
             n_free=A + 0x500, n_free_out=A + 0x500, counter=A + 0x510)
    v.update(change)
    fk.paged_extend(fk.PagedRequests(**v), b or target(), n_pages, page_rows, row_slots)


def target(**change):
    return batch(**{**dict(row_start=B, kv_len=B + 0x100, page_table=B + 0x200, fault=B + 0x800), **change})


@pytest.mark.parametrize("change", [dict(lengths=None), dict(lengths_out=None), dict(tables=None), dict(free_pages=None), dict(n_free=None), dict(n_free_out=None),
                                    dict(counter=None), dict(n_slots=0), dict(n_slots=1), dict(n_slots=(1 << 18) + 1), dict(table_stride=7), dict(slot=A + 1),
                                    dict(new_rows=A + 2), dict(lengths=A + 3), dict(lengths_out=A + 0x204), dict(lengths_out=A + 0x1f8), dict(tables=A + 2),
                                    dict(n_free=A + 0x510), dict(n_free_out=A + 0x510), dict(counter=A), dict(n_free_out=A + 0x304), dict(tables=A + 0x200),
                                    dict(lengths=A + 0x1000, lengths_out=A + 0x1000), dict(n_pages=0), dict(page_rows=8), dict(page_rows=24), dict(page_rows=2048),
                                    dict(row_slots=C + 1), dict(row_slots=B), dict(row_slots=A + 0x300), dict(n_pages=1 << 28), dict(tables=B + 0x200),
                                    dict(b=target(row_start=None)), dict(b=target(kv_len=None)), dict(b=target(page_table=None)), dict(b=target(n_seqs=0)),
                                    dict(b=target(rows=0)), dict(b=target(max_rows=0)), dict(b=target(max_rows=5)), dict(b=target(max_len=0)),
                                    dict(b=target(max_len=129)), dict(b=target(n_seqs=5)), dict(b=target(kv_len=B + 2)), dict(b=target(fault=B + 0x801)),
                                    dict(b=target(kv_len=B)), dict(b=target(page_table=B + 0x100)), dict(b=target(fault=B)), dict(b=target(row_start=A))],
                         ids=lambda c: "-".join(f"{k}" for k in c))
def test_extend(change):
    refused(lambda: extend(**change))


def test_extend_by_none():
    for args in ((None, target()), (fk.PagedRequests(A, A, 4, A, A, A, 8, A, A, A, A), None)):
        refused(lambda: fk.paged_extend(args[0], args[1], 64, 16))


def test_the_plain_statement_of_sampling():
    """The statement that the kernels are held to, on rows whose answer can be said by hand."""
    x = np.array([1.0, 3.0, 3.0, -np.inf, 2.0])
    one = lambda **v: ref.sample(x, **{**dict(t=1.0, k=0, p=1.0, m=0.0, u=0.0), **v})[0]
    assert one() == 1 and one(t=0.0, u=0.9) == 1 and one(k=1, u=0.99) == 1 and one(k=2, u=0.99) == 2 and one(k=2, u=0.49) == 1
    assert one(u=0.9999999) == 0 and one(p=0.0, u=0.99) == 1 and one(m=1.0, u=0.99) == 2 and one(m=0.3, u=0.9999) == 4
    w = np.exp([0.0, 0.0, -1.0, -2.0])
    assert one(p=float(w[:3].sum() / w.sum()) - 1e-6, u=0.9999) == 4 and one(p=float(w[:3].sum() / w.sum()) + 1e-6, u=0.9999) == 0
    assert ref.sample(np.full(4, -np.inf), 1.0, 0, 1.0, 0.0, 0.5) == (0, -np.inf)
    assert abs(ref.sample(x, 0.3, 0, 1.0, 0.0, 0.0)[1] + np.log(w.sum())) < 1e-12
