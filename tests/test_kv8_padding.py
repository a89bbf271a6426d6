"""Page items of batches with rows that go to no page. No GPU."""

import numpy as np
import pytest

from quail_amd.chunk import page_writes


def test_rows_of_no_page_come_as_items_of_page_minus_one():
    dst = np.r_[32:50, [-1] * 3, 64:66]
    phases = page_writes(np.arange(23), dst, rows=25)
    assert [p.tolist() for p in phases] == [[[2, 2, 0, 0, 16], [3, 3, 0, 16, 2], [4, 4, 0, 21, 2],
                                             [-1, -1, 0, 18, 3], [-1, -1, 0, 23, 2]]]
    assert all(p.dtype == np.int32 and p.flags.c_contiguous for p in phases)
    assert [p.tolist() for p in page_writes([0, 1], [-1, -1], rows=2)] == [[[-1, -1, 0, 0, 2]]]
    assert [p.tolist() for p in page_writes([], [], rows=20)] == [[[-1, -1, 0, 0, 16],
                                                                  [-1, -1, 0, 16, 4]]]
    assert page_writes([], [], rows=0) == ()
    assert page_writes([0], [16], rows=1)[0].tolist() == [[1, 1, 0, 0, 1]]


@pytest.mark.parametrize("seed", range(4))
def test_every_row_is_in_one_item(seed):
    rng = np.random.default_rng(seed)
    n = int(rng.integers(1, 300))
    dst = np.arange(n) + 16
    dst[rng.random(n) < 0.2] = -1
    phases = page_writes(np.arange(n), dst, rows=n + 5)
    rows = [r for p in phases for _, _, _, r0, c in p.tolist() for r in range(r0, r0 + c)]
    assert sorted(rows) == list(range(n + 5))
    assert all(0 < c and k + c <= 16 for p in phases for _, _, k, _, c in p.tolist())


def test_rows_past_the_batch_are_refused():
    for src in ([3], [-1]):
        with pytest.raises(ValueError, match="of 3"):
            page_writes(src, [16], rows=3)
