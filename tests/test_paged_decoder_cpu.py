"""PagedDecoder on the host: what it sizes and what it refuses before a device is asked for anything."""
import subprocess
import sys

import numpy as np
import pytest

from fusekit_amd.paged import largest_rows


@pytest.mark.parametrize("most", [1, 31, 32, 33, 64, 65, 128, 129, 500, 512, 600, 4096, 4097, 10000])
def test_workspaces_are_sized_for_every_count_of_rows(most):
    """A workspace grows with the rows between two of 32, 64 and the multiples of 128: the last count before each, and the largest of all."""
    counts = largest_rows(most)
    assert max(counts) == most and min(counts) >= 1
    for m in range(1, most + 1):
        edge = 32 if m <= 32 else 64 if m <= 64 else -(-m // 128) * 128
        assert min(edge, most) in counts


@pytest.mark.parametrize("cfg,change", [(dict(kv_bits=8), {}), (dict(head_dim=96), {}), (dict(head_dim=256), {}), (dict(n_heads=6), {}), ({}, dict(page_rows=8)),
                                        ({}, dict(page_rows=48)), ({}, dict(page_rows=2048)), ({}, dict(page_rows=0)), ({}, dict(n_pages=0)), ({}, dict(max_rows=0)),
                                        ({}, dict(max_seqs=-1)), ({}, dict(rope_dims=8)), ({}, dict(rope_dims=80)), ({}, dict(rope_dims=-16)), ({}, dict(window=-1)),
                                        ({}, dict(softcap=-1.0)), ({}, dict(softcap=2000.0)), ({}, dict(softcap=float("nan")))], ids=str)
def test_what_the_operators_do_not_take_is_refused_at_once(cfg, change):
    from fusekit_amd.decoder import DecoderConfig
    from fusekit_amd.paged import PagedDecoder
    c = DecoderConfig(**{**dict(n_layers=1, hidden=256, n_heads=4, n_kv=4, head_dim=64, inter=256, vocab=100), **cfg})
    with pytest.raises(ValueError):
        PagedDecoder(c, None, **{**dict(n_pages=4, page_rows=16), **change})


def test_an_extension_taken_back_leaves_the_pool_as_it_was():
    from fusekit_amd.paged import PageAllocator
    a, rng = PageAllocator(120, 4), np.random.Generator(np.random.PCG64(2))
    live = [a.new() for _ in range(3)]
    for step in range(300):
        live = live[:6] + [a.fork(live[int(rng.integers(0, len(live)))])]
        before = a.users.copy(), list(a._free), [(list(s.pages), s.length) for s in live]
        some = [live[i] for i in rng.permutation(len(live))[:int(rng.integers(1, len(live) + 1))]]
        rows = rng.integers(0, 7, len(some))
        held = [(list(s.pages), s.length) for s in some]
        a.extend(some, rows)
        a.restore(some, held)
        assert (a.users == before[0]).all() and a._free == before[1] and [(s.pages, s.length) for s in live] == before[2]
        a.extend(some, rows)
        for s in live[6:]:
            a.release(s)
        live = live[:6]
        for s in live:
            a.truncate(s, min(s.length, int(rng.integers(0, 50))))


@pytest.mark.parametrize("options,word", [(["--beams", "-1"], "1 to 64"), (["--beams", "65"], "1 to 64"), (["--eos", "3"], "--beams")])
def test_commands_that_beam_search_does_not_take(options, word):
    r = subprocess.run([sys.executable, "-m", "fusekit_amd", "generate", "--model", "nowhere", "--ids", "1", *options], capture_output=True, text=True, timeout=100)
    assert r.returncode == 2 and word in r.stderr
