"""Plans and tables of Engine.read_pages that change between calls.
Bounds as in test_gpu_kv8.py."""

import numpy as np
import pytest
import torch

from tests.test_gpu_kv8 import DEV, PAGE, check_rows, engine_arena, engine_of, fill, sequences

pytestmark = pytest.mark.gpu


def on_gpu(*arrays):
    return [torch.from_numpy(a).to(DEV) for a in arrays]


@pytest.mark.parametrize("q_lens,start", [((1, 1, 1), (700, 3, 1990)), ((40, 21), (9000, 100))])
def test_a_plan_reads_what_it_was_made_for(q_lens, start):
    """The caller's lengths grow past a multiple of the split afterwards: the
    plan's rows stay as they were."""
    from quail_amd.chunk import attention_plan
    g = torch.Generator().manual_seed(71)
    hq, hk, d = 32, 8, 128
    arena = engine_arena(sum(-(-(u + 600) // PAGE) for u in start) + 3)
    fill(arena, g)
    cu_q, used, table = sequences(g, q_lens, [u + 600 for u in start], arena.num_pages)
    used -= 600
    tables = on_gpu(cu_q, used, table)
    plan = attention_plan(*tables, heads=(hq, hk, d))
    q = torch.randn(int(cu_q[-1]), hq, d, generator=g).to(torch.bfloat16).to(DEV)
    eng = engine_of(arena, hq)
    want = eng.read_pages(q, plan, 0)
    tables[1].add_(600)
    tables[2].fill_(0)
    got = eng.read_pages(q, plan, 0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    check_rows(*got, q, arena, cu_q, used, table, True)


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (24, 8, 64)])
def test_captured_reads_of_growing_sequences_take_tables_without_a_plan(hq, hk, d):
    """One capture, lengths grown in place between replays (from one key,
    past a page, past a split): each replay as the eager call and float64."""
    g = torch.Generator().manual_seed(72)
    bound = 2600
    arena = engine_arena(3 * -(-bound // PAGE), hk, d)
    fill(arena, g)
    cu_q, full, table = sequences(g, (1, 1, 1), [bound] * 3, arena.num_pages, width_extra=0)
    used = np.asarray([1, 15, 2040], dtype=np.int32)
    tables = on_gpu(cu_q, used, table)
    tables = dict(zip(("cu_q", "used", "table"), tables), causal=True, max_q=1, max_used=bound)
    q = torch.randn(3, hq, d, generator=g).to(torch.bfloat16).to(DEV)
    eng = engine_of(arena, hq)
    eng.read_pages(q, tables, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = eng.read_pages(q, tables, 0)
    for step in (0, 1, 2, 300, 255):
        used = used + np.int32(step)
        tables["used"].add_(step)
        eager = [t.clone() for t in eng.read_pages(q, tables, 0)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))
        check_rows(*held, q, arena, cu_q, used, table, True)


def test_tables_without_a_plan_that_do_not_hold_their_bound_are_refused():
    arena = engine_arena(8)
    fill(arena, torch.Generator().manual_seed(73))
    eng = engine_of(arena, 32)
    ints = lambda *a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    q = torch.zeros(1, 32, 128, dtype=torch.bfloat16, device=DEV)
    tables = dict(cu_q=ints(0, 1), used=ints(5), table=ints(1, 2).view(1, 2), causal=True, max_q=1,
                  max_used=32)
    assert bool(torch.isfinite(eng.read_pages(q, tables, 0)[0]).all())
    for bad in (dict(max_used=33), dict(table=ints(1, 2).view(1, 2)[:0])):
        with pytest.raises(ValueError, match="in a table of"):
            eng.read_pages(q, dict(tables, **bad), 0)
