"""Refusals of the operators over a paged cache and of beam search: they come before a device is looked for.  Plain numbers stand for
addresses; nothing is launched."""
import numpy as np
import pytest

import fusekit_amd.native as fk

A, B, C = 0x10000, 0x100000, 0x200000   # aligned addresses that nothing reads


def batch(**change):
    v = dict(row_start=A, kv_len=A, page_table=A, table_stride=8, n_seqs=2, rows=4, max_rows=3, max_len=128, fault=None)
    v.update(change)
    return fk.PagedBatch(**v)


def pool(**change):
    v = dict(k=A, v=A, n_pages=10, page_rows=16, n_kv=2, head_dim=64)
    v.update(change)
    return fk.PagePool(**v)


BATCHES = [dict(row_start=None), dict(kv_len=None), dict(page_table=None), dict(n_seqs=0), dict(rows=0), dict(max_rows=0), dict(max_len=0),
           dict(max_rows=5), dict(max_len=129), dict(max_len=0x80000000, table_stride=0x10000000), dict(kv_len=A + 2), dict(fault=A + 1)]
POOLS = [dict(k=None), dict(v=None), dict(n_pages=0), dict(n_kv=0), dict(page_rows=8), dict(page_rows=24), dict(page_rows=2048), dict(head_dim=96),
         dict(head_dim=0), dict(k=A + 8), dict(v=A + 2)]


def refused(call):
    with pytest.raises(fk.FusekitError) as e:
        call()
    assert e.value.status in (fk.FK_ERR_INVALID, fk.FK_ERR_UNSUPPORTED), e.value
    return e.value


def attend(b=None, p=None, **change):
    v = dict(q=B, q_stride=256, out=C, out_stride=256, n_heads=4, scale=0.125, softcap=0.0, window=0, workspace=A, workspace_bytes=64 << 20)
    v.update(change)
    fk.sdpa_paged(v["q"], v["q_stride"], v["out"], v["out_stride"], v["n_heads"], v["scale"], v["softcap"], v["window"], b or batch(), p or pool(),
                  v["workspace"], v["workspace_bytes"])


def store(b=None, p=None, **change):
    v = dict(q=B, q_stride=512, k=B + 512, k_stride=512, v=B + 768, v_stride=512, q_out=C, q_out_stride=256, n_heads=4, q_norm=None, k_norm=None, eps=1e-6,
             rope_dims=64, interleaved=0, freq=A)
    v.update(change)
    fk.rope_paged_store(*v.values(), b or batch(), p or pool())


@pytest.mark.parametrize("change", BATCHES, ids=str)
def test_batches(change):
    refused(lambda: attend(b=batch(**change)))
    refused(lambda: store(b=batch(**change)))


@pytest.mark.parametrize("change", POOLS, ids=str)
def test_pools(change):
    refused(lambda: attend(p=pool(**change)))
    refused(lambda: store(p=pool(**change)))


@pytest.mark.parametrize("change", [dict(q=None), dict(out=None), dict(workspace=None), dict(n_heads=0), dict(n_heads=3), dict(n_heads=65536 * 2),
                                    dict(q_stride=255), dict(q_stride=260), dict(out_stride=248), dict(q=A + 2), dict(out=A + 8), dict(workspace=A + 4),
                                    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(softcap=-1.0),
                                    dict(softcap=float("nan")), dict(softcap=float("inf")), dict(softcap=1025.0), dict(softcap=1e-40), dict(scale=3e38), dict(workspace_bytes=0),
                                    dict(out=B), dict(out=B + 512 * 3), dict(out=B + 2 * 128), dict(out=B - 512), dict(out=B + 2 * 256, q_stride=512, out_stride=264)], ids=str)
def test_attention(change):
    refused(lambda: attend(**change))


@pytest.mark.parametrize("change", [dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(n_heads=0), dict(rope_dims=8), dict(rope_dims=80),
                                    dict(rope_dims=128), dict(freq=None), dict(freq=A + 4), dict(q_stride=248), dict(q_stride=260), dict(k_stride=120),
                                    dict(v_stride=130), dict(q_out_stride=255), dict(q=A + 2), dict(k=A + 8), dict(v=A + 4), dict(q_out=A + 2),
                                    dict(q_norm=A + 1), dict(k_norm=A + 1), dict(eps=-1.0), dict(eps=float("nan")),
                                    dict(q_out=B), dict(q_out=B + 16, q_out_stride=512), dict(q_out=B + 512, q_out_stride=512), dict(q_out=B + 1024 * 3)], ids=str)
def test_rope_store(change):
    refused(lambda: store(**change))


def test_workspaces():
    assert fk.sdpa_paged_workspace_bytes(32, 8, 128, 64, 64, 9000) > 0
    for bad in ((0, 1, 64, 1, 1, 1), (3, 2, 64, 1, 1, 1), (4, 2, 80, 1, 1, 1), (4, 2, 64, 0, 1, 1), (4, 2, 64, 1, 0, 1), (4, 2, 64, 1, 1, 0)):
        refused(lambda: fk.sdpa_paged_workspace_bytes(*bad))
    assert fk.beam_select_workspace_bytes(2, 4, 100, 8) > 0
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0), (1, 65, 10, 1), (1, 1, 100, 65), (1, 2, 3, 7), (2000, 64, 10, 1)):
        refused(lambda: fk.beam_select_workspace_bytes(*bad))


@pytest.mark.parametrize("bad", [(0, 1e4), (7, 1e4), (64, 1.0), (64, 0.0), (64, float("nan")), (64, float("inf"))])
def test_frequencies(bad):
    refused(lambda: fk.rope_frequencies(*bad, A))


@pytest.mark.parametrize("bad", [dict(scaling="linear", factor=0.5), dict(scaling="linear", factor=float("nan")), dict(scaling="parts", factor=8.0, low=1.0, high=4.0),
                                 dict(scaling="parts", factor=8.0, low=4.0, high=1.0, trained=100), dict(scaling="ramp", factor=8.0, low=0.0, high=4.0, trained=100),
                                 dict(scaling="ramp", factor=8.0, low=1.0, high=float("inf"), trained=100)], ids=str)
def test_frequency_scalings(bad):
    refused(lambda: fk.rope_frequencies(64, 1e4, A, **bad))
    with pytest.raises(KeyError):
        fk.rope_frequencies(64, 1e4, A, scaling="other")


@pytest.mark.parametrize("pairs,word", [([[0, 10]], "does not have"), ([[10, 0]], "does not have"), ([[0, 1], [2, 1]], "written twice"),
                                        ([[0, 1], [1, 2]], "read and written"), ([[3, 3]], "read and written"), ([[0, 1], [2, 0]], "read and written"),
                                        ([[0xFFFFFFFF, 1]], "does not have"), ([[-1, 1]], "page ids"), ([[0, 1 << 32]], "page ids"), ([0, 1], r"\[n, 2\]"),
                                        ([[0.0, 1.0]], "page ids")])
def test_page_pairs(pairs, word):
    with pytest.raises(fk.InvalidArgument, match=word):
        fk.pages_copy(A, 2, 640, 10, 64, pairs)


@pytest.mark.parametrize("change", [dict(base=None), dict(base=A + 8), dict(planes=0), dict(planes=70000), dict(stride=624), dict(stride=648), dict(pages=0),
                                    dict(bytes=0), dict(bytes=40), dict(bytes=(1 << 64) - 16)], ids=str)
def test_pools_to_copy_in(change):
    v = dict(base=A, planes=2, stride=640, pages=10, bytes=64)
    v.update(change)
    refused(lambda: fk.pages_copy(v["base"], v["planes"], v["stride"], v["pages"], v["bytes"], [[0, 1]]))


def test_no_pairs_is_nothing_to_do():
    fk.pages_copy(None, 0, 0, 0, 0, [])
    fk.pages_copy(A, 2, 640, 10, 64, np.zeros((0, 2), np.uint32))


@pytest.mark.parametrize("change", [dict(logits=None), dict(scores=None), dict(os=None), dict(ob=None), dict(ot=None), dict(ws=None), dict(stride=99),
                                    dict(logits=A + 1), dict(scores=A + 2), dict(ws=A + 8), dict(size=0), dict(finished=A, pad=100), dict(finished=A + 1),
                                    dict(groups=0), dict(beams=65), dict(k=65), dict(vocab=0), dict(beams=1, vocab=4, k=5)], ids=str)
def test_select(change):
    v = dict(logits=A, stride=100, scores=A, finished=None, pad=0, groups=2, beams=4, vocab=100, k=8, os=A, ob=A, ot=A, ws=A, size=1 << 20)
    v.update(change)
    refused(lambda: fk.beam_select(*v.values()))


@pytest.mark.parametrize("change", [dict(src=None), dict(dst=None), dict(parents=None), dict(row=0), dict(groups=0), dict(beams=0), dict(out=0),
                                    dict(beams=65), dict(out=65), dict(groups=70000), dict(parents=A + 2), dict(dst=A, out=3), dict(dst=A + 100),
                                    dict(dst=A - 100), dict(row=1 << 60), dict(src_stride=63), dict(dst_stride=60), dict(dst=A, dst_stride=128),
                                    dict(dst=A + 64, src_stride=256, dst_stride=256), dict(src_stride=2048)], ids=str)
def test_reorder(change):
    v = dict(src=A, dst=A + 8192, row=64, parents=A, groups=2, beams=4, out=4, stream=None, src_stride=None, dst_stride=None)
    v.update(change)
    refused(lambda: fk.beam_reorder(*v.values()))


def make(n_pages=8, page_rows=4):
    from fusekit_amd.paged import PageAllocator
    return PageAllocator(n_pages, page_rows)


def test_allocator_takes_shares_and_gives_back():
    from fusekit_amd.paged import OutOfPages
    a = make()
    s, t = a.new(), a.new()
    assert a.extend([s, t], [6, 0]) == [] and s.pages == [0, 1] and s.length == 6 and t.pages == []
    f = a.fork(s)
    assert f.pages == s.pages and a.users[0] == 2
    # both write into the shared tail page: the first copies it, the second then has it to itself
    assert a.extend([f, s], [1, 1]) == [(1, 2)] and f.pages == [0, 2] and s.pages == [0, 1]
    assert a.extend([s], [2]) == [] and s.pages == [0, 1, 3]                       # 7 + 2 positions: a page more, nothing shared is written
    g = a.fork(f)
    a.extend([f], [1])                                                             # (its tail page was shared)
    assert f.pages == [0, 4] and g.pages == [0, 2]
    h = a.fork(f)
    assert a.extend([h], [1]) == [] and h.pages == [0, 4, 5] and a.users[4] == 2   # a full tail page stays shared
    before = (a.users.copy(), a.free_pages, list(s.pages), s.length)
    with pytest.raises(OutOfPages):
        a.extend([s, t], [4, 8])
    assert (a.users == before[0]).all() and (a.free_pages, s.pages, s.length) == before[1:]
    for x in (s, f, g, h, t):
        a.release(x)
    assert a.free_pages == 8 and not a.users.any()


def test_allocator_copies_are_what_pages_copy_takes():
    """Sources are never destinations, and no destination comes twice, whatever is forked."""
    a, rng = make(200, 4), np.random.Generator(np.random.PCG64(1))
    live = [a.new()]
    a.extend(live, [7])
    for _ in range(200):
        parents = rng.integers(0, len(live), 5)
        children = [a.fork(live[p]) for p in parents]
        for s in live:
            a.release(s)
        live = children
        pairs = a.extend(live, rng.integers(0, 6, 5))
        src, dst = {p for p, _ in pairs}, [q for _, q in pairs]
        assert len(set(dst)) == len(dst) and not src & set(dst)
        held = [p for s in live for p in s.pages]
        assert all(a.users[p] == held.count(p) for p in set(held)) and a.free_pages == 200 - len(set(held))
        if max(s.length for s in live) > 60:
            for s in live:
                a.truncate(s, min(s.length, 5))
            assert all(-(-s.length // 4) == len(s.pages) for s in live)


def test_allocator_compacts():
    a = make(10, 4)
    s = [a.new() for _ in range(5)]
    a.extend(s, [8] * 5)
    f = a.fork(s[4])
    a.release(s[0])
    a.release(s[2])
    pairs = a.compact()
    assert sorted(p for x in (s[1], s[3], s[4]) for p in x.pages) == list(range(6)) and f.pages == s[4].pages
    assert {q for _, q in pairs} == {0, 1, 4, 5} and {p for p, _ in pairs} == {6, 7, 8, 9} and a.compact() == [] and a.free_pages == 4
    a.extend([s[1]], [4])
    assert s[1].pages[-1] == 6


def test_allocator_refusals():
    a = make()
    s, other = a.new(), make().new()
    a.extend([s], [5])
    for bad in (lambda: make(0, 4), lambda: make(4, 0), lambda: a.extend([s, s], [1, 1]), lambda: a.extend([s], [1, 2]), lambda: a.extend([s], [-1]),
                lambda: a.extend([other], [1]), lambda: a.fork(other), lambda: a.release(other), lambda: a.truncate(s, 6), lambda: a.truncate(s, -1)):
        with pytest.raises(ValueError):
            bad()
    a.release(s)
    for bad in (lambda: a.release(s), lambda: a.fork(s), lambda: a.extend([s], [1]), lambda: a.table([s], 4)):
        with pytest.raises(ValueError):
            bad()


def test_sound_calls_ask_for_the_device():
    if fk.has_device():
        pytest.skip("a HIP device is present: the addresses are not real")
    for call in (attend, store, lambda: store(q_out=B, q_out_stride=512), lambda: attend(q_stride=1024, out=B + 512, out_stride=1024), lambda: fk.rope_frequencies(64, 1e4, A), lambda: fk.pages_copy(A, 2, 640, 10, 64, [[0, 1], [0, 2]]),
                 lambda: fk.beam_select(A, 100, A, A, 3, 2, 4, 100, 8, A, A, A, A, 1 << 20), lambda: fk.beam_reorder(A, A, 64, A, 2, 4, 4)):
        with pytest.raises(fk.FusekitError) as e:
            call()
        assert e.value.status == fk.FK_ERR_HIP


def test_one_workspace_serves_every_shape():
    draw = np.random.default_rng(0)
    for _ in range(3000):
        n_kv, group = int(draw.integers(1, 129)), int(draw.integers(1, 33))
        n_seqs, rows = (int(np.exp(draw.uniform(0, np.log(20000)))) for _ in range(2))
        need = fk.sdpa_paged_workspace_bytes(n_kv * group, n_kv, int(draw.choice([64, 128])), n_seqs, rows, int(draw.integers(1, 10 ** 6)))
        assert need <= fk.SDPA_PAGED_WORKSPACE_MOST
