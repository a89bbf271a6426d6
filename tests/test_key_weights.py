"""Accumulated key weights on the CPU: the oracle against a softmax, and what
the engine and the C entry refuse."""

from types import SimpleNamespace

import pytest
import torch

from oracle.thin_ref import key_weights
from quail_amd.arena import FP8, KVArena
from quail_amd.chunk import attention_plan
from quail_amd.engine import Engine


@pytest.mark.parametrize("causal", [True, False])
def test_the_oracles_weights_are_the_softmaxs_column_sums(causal):
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(9, 6, 8, generator=g), torch.randn(12, 2, 8, generator=g)
    score = torch.einsum("ihd,jhd->hij", q[2:7].double(), k.double().repeat_interleave(3, 1)) * 0.3
    if causal:
        score.masked_fill_(torch.arange(12) > 7 + torch.arange(5)[:, None], -torch.inf)
    lse = torch.zeros(6, 9, dtype=torch.float64)
    lse[:, 2:7] = score.logsumexp(-1)
    want = score.softmax(-1).sum(1).view(2, 3, 12).sum(1)
    got, _ = key_weights(q, lse, k, 2, 5, causal, 0.3, 2)
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-14)
    assert float(got.sum()) == pytest.approx(30)


def ints(*a):
    return torch.tensor(a, dtype=torch.int32)


@pytest.fixture(params=[torch.bfloat16, FP8])
def engine(request, monkeypatch):
    from quail_amd import _lib
    monkeypatch.setattr(_lib.load(), "qx_device_is_gfx950", lambda: 1)
    arena = KVArena(1, 8, 16, 2, 128, dtype=request.param, device="cpu")
    return Engine(arena, num_q_heads=4, num_kv_heads=2, head_dim=128,
                  rotary=SimpleNamespace(cos_sin_cache=None))


def tables(**kw):
    return dict(dict(cu_q=ints(0, 1, 3), used=ints(20, 5), table=ints(1, 2, 3, 0).view(2, 2),
                     causal=True, max_q=2, max_used=20), **kw)


Q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
LSE = torch.zeros(4, 3)


@pytest.mark.parametrize("kw,match", [
    (dict(q3=Q[:, :2]), "heads"), (dict(q3=Q.float()), "heads"),
    (dict(q3=torch.zeros(3, 8, 128, dtype=torch.bfloat16)[:, ::2]), "contiguous"),
    (dict(lse=LSE.t()), "log-sum"), (dict(lse=LSE.double()), "log-sum"), (dict(lse=LSE[:, :2]), "log-sum"),
    (dict(lse=torch.zeros(4, 6)[:, ::2]), "log-sum"),
    (dict(weights=torch.zeros(2, 2, 19)), "columns"), (dict(weights=torch.zeros(2, 4, 32)), "weights"),
    (dict(weights=torch.zeros(1, 2, 32)), "weights"), (dict(weights=torch.zeros(2, 2, 32).double()), "weights"),
    (dict(weights=torch.zeros(2, 2, 64)[..., ::2]), "weights"),
    (dict(weights=torch.zeros(2, 2, 32), out=torch.zeros(2, 2, 48)), "weights"),
    (dict(out=torch.zeros(2, 2, 48)[:, :1]), "out"), (dict(out=torch.zeros(2, 1, 48).expand(2, 2, 48)), "overlap"),
    (dict(tables=tables(used=torch.tensor([20, 5]))), "used"),
    (dict(tables=tables(cu_q=ints(0, 3))), "bounds"),
    (dict(tables=tables(max_used=33)), "table"),
    (dict(), "on cpu")])
def test_calls_that_are_refused(engine, kw, match):
    args = dict(dict(q3=Q, lse=LSE, tables=tables(), layer=0), **kw)
    with pytest.raises(ValueError, match=match):
        engine.key_weights(**args)


def test_plans_made_for_others_are_refused(engine):
    eight = engine.arena.eight_bit
    plan = attention_plan(ints(0, 1, 3), ints(20, 5), ints(1, 2, 3, 0).view(2, 2), heads=(4, 2, 128),
                          eight_bit=not eight)
    with pytest.raises(ValueError, match="plan"):
        engine.key_weights(Q, LSE, plan, 0)
    plan = attention_plan(ints(0, 1, 3), ints(20, 5), ints(1, 99, 3, 0).view(2, 2), heads=(4, 2, 128),
                          eight_bit=eight)
    with pytest.raises(ValueError, match="arena"):
        engine.key_weights(Q, LSE, plan, 0)


def test_c_entry_refuses_what_the_kernels_do_not_take():
    from quail_amd import _lib
    ok = dict(q=16, q_ld=512, lse=16, lse_ld=60, k=16, scales=None, cu_q=16, used=16, table=16, table_ld=4,
              seqs=1, rows=60, max_q=60, max_used=64, HQ=4, HK=2, D=128, page=16, scale=0.1, causal=1,
              base=None, base_seq=0, base_head=0, out=16, out_seq=128, out_head=64, cols=64, workspace=None,
              bytes=0, stream=None)
    assert _lib.count("qx_key_weights_workspace", 1, 60, 64, 4, 2) == 0
    for name, value, match in [
            ("D", 96, "head_dim"), ("HQ", 5, "heads"), ("HK", 0, "heads"), ("page", 32, "page"),
            ("max_used", 65, "columns"), ("max_used", -1, "rows"), ("rows", -1, "rows"), ("lse_ld", 59, "strides"),
            ("q_ld", 513, "strides"), ("q_ld", 1 << 19, "apart"), ("q", 8, "alignment"), ("k", 24, "alignment"), ("scale", float("nan"), "scale"),
            ("scale", float("inf"), "scale"), ("scale", 3e38, "scale"), ("q", None, "null"), ("lse", None, "null"), ("table", None, "null"),
            ("out", None, "null"), ("cu_q", None, "null"), ("max_q", 1 << 30, "sequence of")]:
        with pytest.raises(_lib.QxError, match=match):
            _lib.call("qx_key_weights", *dict(ok, **{name: value}).values())
    with pytest.raises(_lib.QxError, match="at most 40960"):
        _lib.call("qx_key_weights", *dict(ok, max_used=40961, cols=50000).values())
    long = dict(ok, rows=5000, max_q=5000, lse_ld=5000)
    need = _lib.count("qx_key_weights_workspace", 1, 5000, 64, 4, 2)
    assert need > 0
    for bad in (dict(), dict(workspace=16, bytes=need - 1), dict(workspace=8, bytes=need)):
        with pytest.raises(_lib.QxError, match="workspace"):
            _lib.call("qx_key_weights", *dict(long, **bad).values())
    with pytest.raises(_lib.QxError):
        _lib.count("qx_key_weights_workspace", -1, 1, 1, 4, 2)


def test_scratch_memory_is_bounded():
    from quail_amd import _lib
    one = _lib.count("qx_key_weights_workspace", 1, 40000, 40960, 32, 8)
    assert _lib.count("qx_key_weights_workspace", 900, 40000, 40960, 32, 8) <= max(one, 128 << 20)
    assert _lib.count("qx_key_weights_workspace", 900, 40000, 40960, 32, 8) > 64 << 20
    few = [_lib.count("qx_key_weights_workspace", n, 40000, 2000, 32, 8) for n in (1, 2, 5)]
    assert few[2] - few[0] == 4 * (few[1] - few[0])
