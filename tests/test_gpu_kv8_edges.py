"""The 8-bit KV arena on the GPU where masks, infinities, NaN and long keys
meet: what test_gpu_kv8.py's sizes leave out. Bounds as there."""

import pytest
import torch

from tests.test_gpu_kv8 import DEV, PAGE, engine_arena, engine_of, fill, plan_of, same_codes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (24, 8, 64), (8, 8, 128), (6, 2, 128)])
@pytest.mark.parametrize("q_len,used", [(2, 40), (3, 64), (5, 40), (5, 96), (4, 3000), (3, 9000)])
@pytest.mark.parametrize("back", [0, 1, 3, 9])
def test_nan_values_below_the_cut_reach_every_row_that_sees_them(hq, hk, d, q_len, used, back):
    """A NaN code of V `back` keys before the first key that some row does
    not see, in few rows (split over the keys past 768 of them): every row that
    sees it is NaN in its column, the others are as without it, bit for bit."""
    g = torch.Generator().manual_seed(51)
    arena = engine_arena(-(-used // PAGE) + 1, hk, d)
    fill(arena, g)
    plan, cu_q, u, table = plan_of(arena, hq, (q_len,), (used,), g)
    assert plan["work_rows"] > 0
    q = torch.randn(q_len, hq, d, generator=g).to(torch.bfloat16).to(DEV)
    eng = engine_of(arena, hq)
    clean, clean_lse = eng.read_pages(q, plan, 0)
    at = used - q_len + 1 - back
    row = int(table[0, at // PAGE]) * PAGE + at % PAGE
    v = arena.layer_kv(0)[1]
    v.view(torch.uint8)[row, 0, 5] = 0x7f
    v.view(torch.uint8)[row, hk - 1, d - 1] = 0xff
    out, lse = eng.read_pages(q, plan, 0)
    seen = [i for i in range(q_len) if at <= used - q_len + i]
    want = clean.view(q_len, hq, d).clone()
    want[seen, :hq // hk, 5] = float("nan")
    want[seen, -(hq // hk):, d - 1] = float("nan")
    assert same_codes(out.view(q_len, hq, d), want)
    assert torch.equal(lse, clean_lse)
