"""PagedDecoder on the host: what it sizes and what it refuses before a device is asked for anything."""
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
