"""What the engine's calls over an 8-bit arena refuse, on the CPU: nothing is
launched before the checks."""

from types import SimpleNamespace

import pytest
import torch

from quail_amd.arena import FP8, KVArena
from quail_amd.chunk import attention_plan
from quail_amd.engine import Engine


def ints(*a):
    return torch.tensor(a, dtype=torch.int32)


@pytest.fixture
def engine(monkeypatch):
    from quail_amd import _lib
    monkeypatch.setattr(_lib.load(), "qx_device_is_gfx950", lambda: 1)
    return make_engine


def make_engine(heads=(4, 2, 128), pages=8):
    hq, hk, d = heads
    arena = KVArena(1, pages, 16, hk, d, dtype=FP8, device="cpu")
    return Engine(arena, num_q_heads=hq, num_kv_heads=hk, head_dim=d,
                  rotary=SimpleNamespace(cos_sin_cache=torch.zeros(64, d, dtype=torch.bfloat16)))


@pytest.mark.parametrize("positions", [torch.zeros(6, dtype=torch.int64)[::2],
                                       torch.zeros(3, dtype=torch.int32),
                                       torch.zeros(2, dtype=torch.int64)])
def test_q_norm_on_load_takes_contiguous_int64_positions(engine, positions):
    eng = engine()
    plan = attention_plan(ints(0, 1, 3), ints(20, 5), ints(1, 2, 3, 0).view(2, 2), heads=(4, 2, 128))
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    out = torch.empty(3, 512, dtype=torch.bfloat16)
    norm = SimpleNamespace(weight=torch.ones(128, dtype=torch.bfloat16), variance_epsilon=1e-6)
    with pytest.raises(ValueError, match="positions"):
        eng._attend8(q, plan, 0, 0.1, out=out, qnorm=(positions, SimpleNamespace(q_norm=norm)))


@pytest.mark.parametrize("causal", [True, False])
def test_sequences_without_a_key_need_no_page(engine, causal):
    """A table of no columns: rows of 0, log-sum-exps of -inf."""
    eng = engine()
    plan = attention_plan(ints(0, 1, 3), ints(0, 0), torch.zeros(2, 0, dtype=torch.int32),
                          heads=(4, 2, 128), causal=causal)
    out, lse = eng.read_pages(torch.ones(3, 4, 128, dtype=torch.bfloat16), plan, 0)
    assert out.shape == (3, 512) and not out.any() and lse.shape == (4, 3)
    assert bool((lse == -float("inf")).all())


@pytest.mark.parametrize("name,bad", [("used", torch.tensor([20, 5])), ("cu_q", torch.tensor([0, 1, 3])),
                                      ("table", torch.zeros(2, 2, dtype=torch.int64)),
                                      ("table", torch.zeros(2, 2, dtype=torch.int32).t()),
                                      ("table", torch.zeros(4, dtype=torch.int32)),
                                      ("used", torch.zeros(4, dtype=torch.int32)[::2]),
                                      ("used", ints(20, 5, 3)), ("max_used", 33)])
def test_tables_without_a_plan_are_checked(engine, name, bad):
    tables = dict(cu_q=ints(0, 1, 3), used=ints(20, 5), table=ints(1, 2, 3, 0).view(2, 2), causal=True,
                  max_q=2, max_used=32)
    with pytest.raises(ValueError, match=f"^{name}: int32|bounds of query|in a table of"):
        engine().read_pages(torch.zeros(3, 4, 128, dtype=torch.bfloat16), {**tables, name: bad}, 0)
