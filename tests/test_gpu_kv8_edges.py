"""The 8-bit KV arena on the GPU where masks, infinities, NaN and long keys
meet: what test_gpu_kv8.py's sizes leave out. Bounds as there."""

import numpy as np
import pytest
import torch

from oracle import kv8_ref as ref
from tests.test_gpu_kv8 import (DEV, PAGE, check_rows, engine_arena, engine_of, fill, plan_of,
                                same_codes)

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


def write_rows(arena, hq, k3, v3, table):
    """Rows 0.. of one sequence into its pages, as they are."""
    items = torch.tensor([(int(table[0, p]), int(table[0, p]), 0, PAGE * p,
                           min(PAGE, len(k3) - PAGE * p)) for p in range(-(-len(k3) // PAGE))],
                         dtype=torch.int32, device=DEV)
    engine_of(arena, hq)._write_page_rows(k3, v3, (items,), 0)
    return items.tolist()


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (24, 8, 64), (8, 8, 128), (4, 2, 64)])
@pytest.mark.parametrize("value", [float("inf"), 3.3895313892515355e38])
@pytest.mark.parametrize("side", ["k", "v"])
def test_infinite_keys_and_values_stay_out_of_rows_that_do_not_see_them(hq, hk, d, value, side):
    """An infinity, or bf16's largest number, is stored as a finite value (at
    most 240 * 2^120), so that a weight of 0 times it is 0: rows that do not
    see its page are as without it, bit for bit, and those that see a V one
    match float64 over the stored codes."""
    g = torch.Generator().manual_seed(52)
    used, at = 48, 36
    arena = engine_arena(4, hk, d)
    fill(arena, g)
    k3, v3 = (torch.randn(used, hk, d, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    bad = [k3.clone(), v3.clone()]
    bad["kv".index(side)][at, 0, 5] = value
    bad["kv".index(side)][at + 1, hk - 1, 3] = -value
    for q_len in (40, 33, 8, 1):
        plan, cu_q, u, table = plan_of(arena, hq, (q_len,), (used,), torch.Generator().manual_seed(1))
        q = torch.randn(q_len, hq, d, generator=g).to(torch.bfloat16).to(DEV)
        eng = engine_of(arena, hq)
        write_rows(arena, hq, k3, v3, table)
        clean, clean_lse = eng.read_pages(q, plan, 0)
        pools = [p.cpu() for p in arena.layer_kv(0)] + [arena.layer_scales(0).cpu()]
        items = write_rows(arena, hq, *bad, table)
        ref.write_items(*pools, *(t.double().cpu() for t in bad), items)
        for got, want in zip(arena.layer_kv(0), pools):
            assert same_codes(got, want)
        assert torch.equal(arena.layer_scales(0).cpu(), pools[2])
        for i in (0, 1):
            size = ref.values(pools[i], pools[2], i)[np.r_[tuple(
                slice(PAGE * p, PAGE * p + PAGE) for p in table[0, :3].tolist())]]
            assert float(size.abs().max()) <= 240 * 2.0 ** 120
        out, lse = eng.read_pages(q, plan, 0)
        before = max(0, 2 * PAGE - (used - q_len))      # rows that see none of the last page
        assert torch.equal(out[:before], clean[:before])
        assert torch.equal(lse[:, :before], clean_lse[:, :before])
        if side == "v":
            check_rows(out, lse, q, arena, cu_q, u, table, True)


@pytest.mark.parametrize("q_len", [1, 2, 40])
@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (24, 8, 64)])
def test_nan_values_of_a_split_without_weight_reach_the_rows(q_len, hq, hk, d):
    """A NaN of V among keys that a row sees with a weight that underflows,
    in a split of its own: the row is NaN there, as it is unsplit."""
    from quail_amd.chunk import attention_plan
    g = torch.Generator().manual_seed(53)
    used = 9000
    arena = engine_arena(-(-used // PAGE), hk, d)
    fill(arena, g)
    k, v = arena.layer_kv(0)
    arena.layer_scales(0).fill_(127)
    k.fill_(400.0)
    k[:4096] = -400.0       # whole splits, of 2048 keys at most
    v.view(torch.uint8)[5, 0, 7] = 0x7f
    table = torch.arange(arena.num_pages, dtype=torch.int32, device=DEV).view(1, -1)
    ints = lambda *a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    q = torch.full((q_len, hq, d), 8.0, dtype=torch.bfloat16, device=DEV)
    plan = attention_plan(ints(0, q_len), ints(used), table, heads=(hq, hk, d))
    assert 0 < abs(plan["work_rows"]) < used
    out, lse = engine_of(arena, hq).read_pages(q, plan, 0)
    nan = torch.zeros(hq, d, dtype=torch.bool, device=DEV)
    nan[:hq // hk, 7] = True
    assert torch.equal(torch.isnan(out.view(q_len, hq, d)), nan.expand(q_len, -1, -1))
    assert bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (24, 8, 64), (8, 8, 128), (64, 8, 128)])
@pytest.mark.parametrize("q_lens,used", [([100] * 12 + [21, 3], [100] * 12 + [20000, 9000]),
                                         ([1, 2, 1, 2, 0], [30, 9000, 64, 2100, 5]),
                                         ([40, 150], [9000, 150])])
def test_joins_give_the_rows_of_the_call_that_looks_at_every_sequence(hq, hk, d, q_lens, used):
    """A few rows over long keys among many rows: bit for bit the rows that
    the list without joins gives, in scratch memory of the split rows alone."""
    from quail_amd import _lib
    g = torch.Generator().manual_seed(54)
    arena = engine_arena(sum(-(-u // PAGE) for u in used) + 3, hk, d)
    fill(arena, g)
    plan, cu_q, u, table = plan_of(arena, hq, q_lens, used, g)
    n_joins, part_rows = plan["work_joins"]
    assert 0 < n_joins and part_rows < 4096
    n = int(cu_q[-1])
    q = torch.randn(n, hq, d, generator=g).to(torch.bfloat16).to(DEV)
    eng = engine_of(arena, hq)
    out, lse = eng.read_pages(q, plan, 0)
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    torch.cuda.reset_peak_memory_stats()
    out, lse = eng.read_pages(q, plan, 0)
    torch.cuda.synchronize()
    scratch = part_rows * hq * (d + 2) * 4
    rows = out.numel() * 2 + lse.numel() * 4
    # as asked for (a cached block may be up to 1 MiB larger)
    peak = torch.cuda.memory_stats()["requested_bytes.all.peak"] - before
    assert peak <= 2 * rows + scratch + (1 << 16)
    # the same list, every row in as many splits as the longest sequence has
    sizes = len(q_lens), n, plan["max_q"], plan["max_used"], hq, hk, d
    size = _lib.count("qx_paged_attention8_workspace", *sizes, 1, plan["work_rows"])
    space = torch.empty(size, dtype=torch.uint8, device=DEV)
    out2, lse2 = torch.empty_like(out), torch.empty_like(lse)
    _lib.call("qx_paged_attention8", q.data_ptr(), q.stride(0), None, *arena.layer_pointers(0),
              plan["cu_q"].data_ptr(), plan["used"].data_ptr(), plan["table"].data_ptr(),
              plan["table"].stride(0), *sizes, PAGE, d ** -0.5, 1, out2.data_ptr(), None,
              out2.stride(0), None, 0, lse2.data_ptr(), lse2.stride(0), plan["work"].data_ptr(),
              plan["n_work"], plan["work_rows"], space.data_ptr(), size, None, None, 0, None, 0.0,
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    for s in (i for i, m in enumerate(q_lens) if m and used[i] != 100):
        at = slice(int(cu_q[s]), int(cu_q[s + 1]))
        if q_lens[s] > 100:
            at = slice(at.start, at.start + 2)          # its first rows: the fewest keys
            part = np.asarray([0, 2], dtype=np.int32), u[s:s + 1] - q_lens[s] + 2
        else:
            part = np.asarray([0, q_lens[s]], dtype=np.int32), u[s:s + 1]
        check_rows(out[at], lse[:, at], q[at], arena, *part, table[s:s + 1], True)


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (24, 8, 64), (16, 8, 128)])
@pytest.mark.parametrize("q_len,used", [(40, 9000), (70, 700), (130, 130), (200, 20000)])
@pytest.mark.parametrize("back", [-30, 0, 1, 40, 64, 65, 129])
def test_nan_values_near_the_cut_of_query_tiles(hq, hk, d, q_len, used, back):
    """The same over query tiles, whole and split over their keys: the NaN
    `back` keys before the first that the first row does not see."""
    g = torch.Generator().manual_seed(55)
    arena = engine_arena(-(-used // PAGE) + 1, hk, d)
    fill(arena, g)
    plan, cu_q, u, table = plan_of(arena, hq, (q_len,), (used,), g)
    assert plan["work_rows"] <= 0
    q = torch.randn(q_len, hq, d, generator=g).to(torch.bfloat16).to(DEV)
    eng = engine_of(arena, hq)
    clean, clean_lse = eng.read_pages(q, plan, 0)
    at = max(0, used - q_len + 1 - back)
    row = int(table[0, at // PAGE]) * PAGE + at % PAGE
    v = arena.layer_kv(0)[1]
    v.view(torch.uint8)[row, 0, 5] = 0x7f
    v.view(torch.uint8)[row, hk - 1, d - 1] = 0xff
    out, lse = eng.read_pages(q, plan, 0)
    first = max(0, at - (used - q_len))
    want = clean.view(q_len, hq, d).clone()
    want[first:, :hq // hk, 5] = float("nan")
    want[first:, -(hq // hk):, d - 1] = float("nan")
    assert same_codes(out.view(q_len, hq, d), want)
    assert torch.equal(lse, clean_lse)


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (24, 8, 64), (16, 8, 128), (64, 8, 128)])
@pytest.mark.parametrize("q_lens,used", [((1,), (300,)), ((2, 1), (40, 3000)), ((3, 1, 1), (9000, 17, 200)),
                                         ((1,) * 20, tuple(range(5, 105, 5)))])
def test_few_rows_are_off_by_the_rounding_of_the_output(hq, hk, d, q_lens, used):
    """P goes into the products to 2^-16 of a weight (its rounding to bf16 and
    what that left, rounded again): beside the output's own rounding there are
    only that, the exponent's 2^-20, the scores' and fp32 sums' errors."""
    g = torch.Generator().manual_seed(56)
    arena = engine_arena(sum(-(-u // PAGE) for u in used) + 3, hk, d)
    fill(arena, g)
    plan, cu_q, u, table = plan_of(arena, hq, q_lens, used, g)
    assert plan["work_rows"] > 0
    n = int(cu_q[-1])
    q = torch.randn(n, hq, d, generator=g).to(torch.bfloat16).to(DEV)
    out, _ = engine_of(arena, hq).read_pages(q, plan, 0)
    k, v = arena.layer_kv(0)
    want, _, size, reach = ref.attend(q, k, v, arena.layer_scales(0), cu_q.tolist(), u.tolist(),
                                      table, True)
    score = (d + 8) * 2.0 ** -24 * reach[..., None]
    weight = 2.0 ** -16 + 2 * score + 2.0 ** -20 + max(used) * 2.0 ** -24
    bound = 2.0 ** -8 * want.abs() + 1.01 * weight * size
    over = (out.view(n, hq, d).double() - want).abs() - bound
    assert float(over.max()) <= 1e-30
