"""Refusals of the operators over a paged cache and of beam search: they come before a device is looked for.  Plain numbers stand for
addresses; nothing is launched."""
import numpy as np
import pytest

import fusekit_amd.native as fk

A = 0x10000   # an aligned address that nothing reads


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
    v = dict(q=A, q_stride=256, out=A, out_stride=256, n_heads=4, scale=0.125, softcap=0.0, window=0, workspace=A, workspace_bytes=64 << 20)
    v.update(change)
    fk.sdpa_paged(v["q"], v["q_stride"], v["out"], v["out_stride"], v["n_heads"], v["scale"], v["softcap"], v["window"], b or batch(), p or pool(),
                  v["workspace"], v["workspace_bytes"])


def store(b=None, p=None, **change):
    v = dict(q=A, q_stride=512, k=A, k_stride=512, v=A, v_stride=512, q_out=A, q_out_stride=256, n_heads=4, q_norm=None, k_norm=None, eps=1e-6,
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
                                    dict(softcap=float("nan")), dict(softcap=float("inf")), dict(workspace_bytes=0)], ids=str)
def test_attention(change):
    refused(lambda: attend(**change))


@pytest.mark.parametrize("change", [dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(n_heads=0), dict(rope_dims=8), dict(rope_dims=80),
                                    dict(rope_dims=128), dict(freq=None), dict(freq=A + 4), dict(q_stride=248), dict(q_stride=260), dict(k_stride=120),
                                    dict(v_stride=130), dict(q_out_stride=255), dict(q=A + 2), dict(k=A + 8), dict(v=A + 4), dict(q_out=A + 2),
                                    dict(q_norm=A + 1), dict(k_norm=A + 1), dict(eps=-1.0), dict(eps=float("nan"))], ids=str)
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
                                    dict(dst=A - 100), dict(row=1 << 60)], ids=str)
def test_reorder(change):
    v = dict(src=A, dst=A + 8192, row=64, parents=A, groups=2, beams=4, out=4)
    v.update(change)
    refused(lambda: fk.beam_reorder(*v.values()))


def test_sound_calls_ask_for_the_device():
    if fk.has_device():
        pytest.skip("a HIP device is present: the addresses are not real")
    for call in (attend, store, lambda: fk.rope_frequencies(64, 1e4, A), lambda: fk.pages_copy(A, 2, 640, 10, 64, [[0, 1], [0, 2]]),
                 lambda: fk.beam_select(A, 100, A, A, 3, 2, 4, 100, 8, A, A, A, A, 1 << 20), lambda: fk.beam_reorder(A, A, 64, A, 2, 4, 4)):
        with pytest.raises(fk.FusekitError) as e:
            call()
        assert e.value.status == fk.FK_ERR_HIP
