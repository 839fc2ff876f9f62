"""Drawing continuations over pages, on the host: what PagedDecoder.sample and the command refuse, and how the pages that the device took come back."""
import subprocess
import sys

import numpy as np
import pytest


def decoder(n_pages=8, max_rows=4, max_seqs=6):
    """What sample() reads before it asks a device for anything."""
    from fusekit_amd.decoder import DecoderConfig
    from fusekit_amd.paged import PageAllocator, PagedDecoder
    d = PagedDecoder.__new__(PagedDecoder)
    d.cfg = DecoderConfig(n_layers=1, hidden=256, n_heads=4, n_kv=4, head_dim=64, inter=256, vocab=100)
    d.pages, d.max_rows, d.max_seqs, d.stream = PageAllocator(n_pages, 16), max_rows, max_seqs, None
    return d


@pytest.mark.parametrize("change", [dict(prompts=[]), dict(prompts=[[1], []]), dict(prompts=[[1]] * 7), dict(prompts=[[1]] * 5), dict(max_tokens=0), dict(seed=-1),
                                    dict(seed=1 << 64), dict(temperature=-0.5), dict(temperature=np.nan), dict(temperature=np.inf), dict(temperature=[1.0]),
                                    dict(temperature=[1.0, 1.0, 1.0]), dict(temperature=[[1.0, 1.0]]), dict(top_k=-1), dict(top_k=2.5), dict(top_k=1 << 32), dict(top_p=0.0),
                                    dict(top_p=1.5), dict(top_p=np.nan), dict(top_p=[0.5, -1]), dict(min_p=-0.1), dict(min_p=1.1), dict(min_p=[0.1, np.nan])], ids=str)
def test_settings(change):
    d = decoder()
    with pytest.raises(ValueError):
        d.sample(**{**dict(prompts=[[1], [2, 3]], max_tokens=2), **change})
    assert d.pages.free_pages == 8


def test_pages_are_counted_before_any_work():
    from fusekit_amd.paged import OutOfPages
    d = decoder(n_pages=4)
    for prompts, tokens in (([[1] * 65], 1), ([[1] * 16] * 2, 18), ([[1]], 65), ([[1] * 48, [1], [1]], 1)):
        with pytest.raises(OutOfPages):
            d.sample(prompts, tokens)
    assert d.pages.free_pages == 4


def test_sinks_are_not_negative():
    from fusekit_amd.decoder import DecoderConfig
    from fusekit_amd.paged import PagedDecoder
    c = DecoderConfig(n_layers=1, hidden=256, n_heads=4, n_kv=4, head_dim=64, inter=256, vocab=100)
    for bad in (-1, 1 << 31):
        with pytest.raises(ValueError, match="sinks"):
            PagedDecoder(c, None, n_pages=4, page_rows=16, window=5, sinks=bad)


def device(a, seqs, rows, stride):
    """(lengths, tables, n_free) as paged_extend leaves them."""
    import decode_loop_reference as ref
    n = len(seqs)
    free = np.array(a._free + [0] * (a.n_pages - len(a._free)))
    got = ref.extend(range(n), rows, [s.length for s in seqs], a.table(seqs, stride), free, len(a._free), a.page_rows, np.zeros((n, stride), np.uint32),
                     np.zeros(sum(rows) + 1, np.uint32))
    return got[4], got[5], got[6]


def test_what_the_device_took_is_what_the_host_would_have():
    from fusekit_amd.paged import PageAllocator
    rng = np.random.Generator(np.random.PCG64(1))
    for _ in range(50):
        a, b = PageAllocator(60, 4), PageAllocator(60, 4)
        sa, sb = ([x.new() for _ in range(5)] for x in (a, b))
        held = rng.integers(0, 12, 5)
        for x, s in ((a, sa), (b, sb)):
            x.extend(s, held)
            x.release(s.pop(2))
        rows = rng.integers(0, 9, 4)
        a.adopt(sa, *device(a, sa, rows, 8))
        b.extend(sb, rows)
        assert [(s.pages, s.length) for s in sa] == [(s.pages, s.length) for s in sb] and (a.users == b.users).all() and a._free == b._free
        for s in sa:
            a.release(s)
        assert a.free_pages == 60 and not a.users.any()


@pytest.mark.parametrize("plant", [lambda l, t, f: (l, t, f - 1), lambda l, t, f: (l, t, f + 1), lambda l, t, f: (l, np.where(t == t[1, 1], t[0, 1], t), f),
                                   lambda l, t, f: (l - 5, t, f)])
def test_pages_that_are_not_the_hosts_are_refused_and_change_nothing(plant):
    from fusekit_amd.paged import PageAllocator
    a = PageAllocator(20, 4)
    seqs = [a.new(), a.new()]
    a.extend(seqs, [3, 4])
    before = a.users.tolist(), list(a._free), [(list(s.pages), s.length) for s in seqs]
    with pytest.raises(RuntimeError):
        a.adopt(seqs, *plant(*device(a, seqs, [4, 4], 4)))
    assert (a.users.tolist(), a._free, [(s.pages, s.length) for s in seqs]) == before


@pytest.mark.parametrize("options,word", [(["--top-k", "3"], "--temperature"), (["--top-p", "0.5"], "--temperature"), (["--min-p", "0"], "--temperature"),
                                          (["--seed", "1"], "--temperature"), (["--temperature", "-1"], "not negative"), (["--temperature", "nan"], "not negative"),
                                          (["--temperature", "1", "--beams", "2"], "without --beams"), (["--temperature", "1", "--artifact", "x"], "artifact"),
                                          (["--temperature", "1", "--top-p", "0"], "above 0"), (["--temperature", "1", "--min-p", "2"], "0 to 1"),
                                          (["--temperature", "1", "--top-k", "-1"], "count"), (["--temperature", "1", "--seed", "-1"], "2^64"),
                                          (["--temperature", "1", "--max-tokens", "0"], "one at least")], ids=str)
def test_commands_that_are_refused(options, word):
    r = subprocess.run([sys.executable, "-m", "fusekit_amd", "generate", "--model", "nowhere", "--ids", "1", *options], capture_output=True, text=True, timeout=100)
    assert r.returncode == 2 and word in r.stderr
