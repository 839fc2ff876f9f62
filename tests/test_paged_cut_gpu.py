"""Attention over a paged cache (fk_sdpa_paged) where tiles are cut along their positions and joined: what the parts are, what they leave in the workspace, against
the statement in 64 bits.  Tolerances: those of test_paged_gpu.py."""
import numpy as np
import pytest

from helpers import normal_bf16, rng
from paged_reference import Paged, attention, wide
from test_paged_gpu import attend, check_attention

pytestmark = pytest.mark.gpu


def test_a_falling_row_start_leaves_the_workspace_ready(fk):
    """More tiles than rows account for, the last of them long: what such a batch writes is undefined, what the next one does is not."""
    n_heads, n_kv, dim, rows = 64, 8, 64, 30
    starts = [0]
    while len(starts) < 131:                                  # ten sequences of three rows, then back to the first row
        starts.append(starts[-1] + 3 if starts[-1] < 30 else 0)
    lens = np.full(130, 3, np.uint32)
    lens[[i for i in range(120, 130) if starts[i + 1] > starts[i]][-3:]] = 60000
    fault = fk.zeros(4)
    up = fk.DeviceBuffer.from_numpy
    pages = [up(normal_bf16(i, (4, n_kv, 64, dim))) for i in (1, 2)]
    d = [up(np.array(starts, np.uint32)), up(lens), up(np.zeros((130, 938), np.uint32))]
    q, out = up(normal_bf16(3, (rows, n_heads * dim))), fk.zeros(2 * rows * n_heads * dim)
    ws = fk.zeros(fk.SDPA_PAGED_WORKSPACE_MOST)
    fk.sdpa_paged(q, n_heads * dim, out, n_heads * dim, n_heads, 0.125, 0.0, 0, fk.PagedBatch(*d, 938, 130, rows, 4, 60000, fault),
                  fk.PagePool(*pages, 4, 64, n_kv, dim), ws, ws.nbytes)
    with pytest.raises(fk.InvalidArgument, match="row_start"):
        fk.paged_check(fault)
    assert not ws.to_numpy(np.uint8)[:16384].any()
    check_attention(fk, Paged([1], [9000], n_kv, dim, 64, seed=1), n_heads, workspace=ws)


def test_a_falling_row_start_with_chunks_leaves_the_workspace_ready(fk):
    n_heads, n_kv, dim = 64, 64, 64
    starts = [0, 400, 401, 0, 400, 401, 402]                  # two chunks over the same rows, long tokens behind both
    lens = np.array([400, 60000, 500, 400, 60000, 60000], np.uint32)
    fault = fk.zeros(4)
    up = fk.DeviceBuffer.from_numpy
    pages = [up(normal_bf16(i, (4, n_kv, 64, dim))) for i in (1, 2)]
    d = [up(np.array(starts, np.uint32)), up(lens), up(np.zeros((6, 938), np.uint32))]
    q, out = up(normal_bf16(3, (402, n_heads * dim))), fk.zeros(2 * 402 * n_heads * dim)
    ws = fk.zeros(fk.SDPA_PAGED_WORKSPACE_MOST)
    fk.sdpa_paged(q, n_heads * dim, out, n_heads * dim, n_heads, 0.125, 0.0, 0, fk.PagedBatch(*d, 938, 6, 402, 400, 60000, fault),
                  fk.PagePool(*pages, 4, 64, n_kv, dim), ws, ws.nbytes)
    with pytest.raises(fk.InvalidArgument, match="row_start"):
        fk.paged_check(fault)
    assert not ws.to_numpy(np.uint8)[:16384].any()
    check_attention(fk, Paged([1], [9000], 8, dim, 64, seed=1), n_heads, workspace=ws)
