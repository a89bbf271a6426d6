"""Plans of attention over an arena's pages, on the CPU: what they hold."""

import torch

from quail_amd.chunk import attention_plan


def ints(*a):
    return torch.tensor(a, dtype=torch.int32)


def test_a_plan_keeps_the_tables_it_was_made_of():
    cu_q, used, table = ints(0, 1, 3), ints(20, 900), torch.arange(120, dtype=torch.int32).view(2, 60)
    plan = attention_plan(cu_q, used, table[:, :58], heads=(32, 8, 128))
    want = {k: plan[k].clone() for k in ("cu_q", "used", "table", "work")}
    assert torch.equal(want["used"], ints(20, 900)) and torch.equal(want["table"], table[:, :58])
    for t in (cu_q, used, table):
        t.fill_(99)
    for k, w in want.items():
        assert torch.equal(plan[k], w) and plan[k].stride(-1) == 1
