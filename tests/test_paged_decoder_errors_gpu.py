"""PagedDecoder when a call fails: sequences and pages are as they were, and the next call is sound."""
import numpy as np
import pytest

from helpers import rng
from test_paged_decoder_gpu import models, paged  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def state(d, *seqs):
    return d.pages.users.tolist(), d.pages.free_pages, [(list(s.pages), s.length) for s in seqs]


def rows(d, cfg, n):
    return d.logits.to_numpy(np.uint16)[:n * cfg.vocab].reshape(n, cfg.vocab)


@pytest.mark.parametrize("name,nth", [("rope_paged_store", 0), ("sdpa_paged", 1), ("qgemm", 3), ("pages_copy", 0), ("rmsnorm_rows", 4)])
def test_a_launch_that_is_refused(fk, models, monkeypatch, name, nth):  # noqa: F811
    cfg, d = paged(models, "norms")
    text = rng(3).integers(0, cfg.vocab, 60).tolist()
    a = d.pages.new()
    d.forward([(a, text[:21])])
    b = d.pages.fork(a)                                       # both are about to write into the page that they share
    batch = [(a, text[21:40]), (b, text[40:43])]
    before, calls, real = state(d, a, b), [0], getattr(fk, name)

    def fails(*args, **more):
        calls[0] += 1
        if calls[0] > nth:
            raise fk.InvalidArgument(fk.FK_ERR_INVALID, "refused")
        return real(*args, **more)

    with monkeypatch.context() as m:
        m.setattr(fk, name, fails)
        with pytest.raises(fk.InvalidArgument, match="refused"):
            d.forward(batch)
    assert state(d, a, b) == before
    d.forward(batch)
    fk.paged_check(d.fault)
    got = rows(d, cfg, 2)
    e = paged(models, "norms")[1]
    x, y = e.pages.new(), e.pages.new()
    e.forward([(x, text[:21])])
    e.forward([(y, text[:21])])
    e.forward([(x, text[21:40]), (y, text[40:43])])
    fk.sync()
    assert np.array_equal(got, rows(e, cfg, 2))


def test_a_prompt_that_does_not_fit(fk, models):  # noqa: F811
    from fusekit_amd.paged import OutOfPages
    cfg, d = paged(models, "norms", n_pages=6, max_rows=40)
    s = d.pages.new()
    d.forward([(s, [1, 2, 3])])
    before = state(d, s)
    with pytest.raises(OutOfPages):
        d.prefill(s, [5] * 100)                               # two chunks of 40 fit, the third does not
    assert state(d, s) == before
    d.prefill(s, [5] * 60)
    assert s.length == 63


def test_more_beams_or_prompts_than_rows_of_a_pass_are_refused_before_any_work(fk, models, monkeypatch):  # noqa: F811
    cfg, d = paged(models, "norms", max_rows=4, max_seqs=8)
    monkeypatch.setattr(d, "forward", lambda batch: pytest.fail("a pass was run"))
    for bad in (lambda: d.beam_search([1, 2], 5, 3), lambda: d.generate([[1]] * 5, 2), lambda: d.generate([[1], []], 2)):
        with pytest.raises(ValueError):
            bad()
    monkeypatch.undo()
    assert len(d.beam_search([1, 2], 5, 1)) == 5 and len(d.generate([[1]] * 5, 1)) == 5      # (a first token takes no step)
    assert len(d.beam_search([1, 2], 4, 2)) == 4 and len(d.generate([[1]] * 4, 2)) == 4 and d.pages.free_pages == 64


@pytest.mark.parametrize("call", [lambda d: d.beam_search([1, 2], 2, 3), lambda d: d.generate([[1], [2, 3]], 3)])
def test_what_a_launch_reports_is_raised(fk, models, call):  # noqa: F811
    cfg, d = paged(models, "norms")
    want = call(d)
    d.fault.upload(np.array([2], np.uint32))                  # as a launch that meets a bad length sets it
    with pytest.raises(fk.InvalidArgument, match="length"):
        call(d)
    assert d.pages.free_pages == 64 and call(d) == want


def test_a_compaction_that_is_refused(fk, models, monkeypatch):  # noqa: F811
    cfg, d = paged(models, "norms")
    text = rng(4).integers(0, cfg.vocab, 50).tolist()
    a, b = d.pages.new(), d.pages.new()
    d.forward([(a, text[:40]), (b, text)])
    c = d.pages.fork(b)
    d.pages.release(a)
    before, free = state(d, b, c), list(d.pages._free)

    def fails(*args, **more):
        raise fk.InvalidArgument(fk.FK_ERR_INVALID, "refused")
    with monkeypatch.context() as m:
        m.setattr(fk, "pages_copy", fails)
        with pytest.raises(fk.InvalidArgument, match="refused"):
            d.compact()
    assert state(d, b, c) == before and d.pages._free == free
    first = d.forward([(c, [7])]).to_numpy(np.uint16)[:cfg.vocab]
    assert d.compact() > 0
    fk.sync()
    assert np.array_equal(d.forward([(b, [7])]).to_numpy(np.uint16)[:cfg.vocab], first)
