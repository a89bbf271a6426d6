"""Thinning on the CPU: the oracle against a brute-force definition, what the
arena refuses, and the page accounting of thinned keys."""

import random

import numpy as np
import pytest
import torch

from oracle.thin_ref import kept_slots
from quail_amd.arena import FP8, KVArena
from quail_amd.chunk import pack_chunk


def test_the_oracles_slots_hold_the_heaviest_rows():
    rng = random.Random(1)
    for _ in range(300):
        used = rng.randrange(0, 30)
        keep = rng.randrange(0, 30)
        sinks = rng.randrange(0, keep + 1)
        recent = rng.randrange(0, keep - sinks + 1)
        w = [rng.choice([0.0, 1.0, 2.5, rng.random()]) for _ in range(used)]
        got = kept_slots(w, used, keep, sinks, recent)
        k = min(used, keep)
        assert len(got) == k and len(set(got)) == k and all(0 <= i < used for i in got)
        # rows below k stay; the others go up in order
        assert all(i == slot or i >= k for slot, i in enumerate(got))
        moved = [i for slot, i in enumerate(got) if i != slot]
        assert moved == sorted(moved)
        if used > keep:
            safe = set(range(sinks)) | set(range(used - recent, used))
            assert safe <= set(got)
            dropped = set(range(used)) - set(got)
            for i in set(got) - safe:
                assert all((w[j], -j) < (w[i], -i) for j in dropped)


def cpu_arena(dtype=torch.bfloat16, layers=2, pages=16, heads=2, d=64):
    return KVArena(layers, pages, 16, heads, d, dtype=dtype, device="cpu")


def call(arena=None, used=(5, 20), width=2, max_used=20, cols=32, keep=16, weights=None, **kw):
    arena = arena or cpu_arena()
    tables = dict(used=torch.tensor(used, dtype=torch.int32),
                  table=torch.zeros(len(used), width, dtype=torch.int32), max_used=max_used)
    tables.update({k: kw.pop(k) for k in ("table", "used_tensor", "pages") if k in kw})
    if "used_tensor" in tables:
        tables["used"] = tables.pop("used_tensor")
    weights = torch.zeros(2, len(used), 2, cols) if weights is None else weights
    return arena.thin_rows(tables, weights, keep, **kw)


@pytest.mark.parametrize("kw,match", [
    (dict(weights=torch.zeros(2, 2, 2, 32, dtype=torch.float64)), "weights"),
    (dict(weights=torch.zeros(1, 2, 2, 32)), "weights"),
    (dict(weights=torch.zeros(2, 3, 2, 32)), "weights"),
    (dict(weights=torch.zeros(2, 2, 4, 32)), "weights"),
    (dict(weights=torch.zeros(2, 2, 64)), "weights"),
    (dict(weights=torch.zeros(2, 2, 2, 64)[..., ::2]), "weights"),
    (dict(cols=19), "columns"), (dict(max_used=33), "table"),
    (dict(table=torch.zeros(1, 2, dtype=torch.int32)), "table"),
    (dict(table=torch.zeros(2, 2, dtype=torch.int64)), "table"),
    (dict(table=torch.zeros(2, 4, dtype=torch.int32)[:, ::2]), "table"),
    (dict(used_tensor=torch.zeros(2)), "used"), (dict(pages=17), "arena"),
    (dict(keep=-1), "stay"), (dict(sinks=-1), "stay"), (dict(recent=-1), "stay"),
    (dict(keep=8, sinks=5, recent=4), "stay"),
    (dict(), "on the CPU")])
def test_calls_that_are_refused(kw, match):
    with pytest.raises(ValueError, match=match):
        call(**kw)


def test_8_bit_pages_are_kept_whole():
    with pytest.raises(ValueError, match="whole"):
        call(cpu_arena(FP8), keep=17)


def test_c_entry_refuses_what_the_kernels_do_not_take():
    from quail_amd import _lib
    ok = dict(pools=16, pool_stride=1 << 20, element_bytes=2, scales=None, scale_stride=0, weights=16,
              w_layer=0, w_seq=0, w_head=0, used=16, table=16, table_ld=4, layers=1, seqs=1, HK=2, D=64,
              page=16, max_used=64, cols=64, keep=32, sinks=0, recent=0, kept=16, out=16, stream=None)
    bad = [("D", 96, "head_dim"), ("page", 32, "page"), ("element_bytes", 1, "scales"),
           ("element_bytes", 4, "values"), ("max_used", 65, "columns"), ("max_used", -1, "rows"),
           ("keep", -1, "stay"), ("recent", 33, "stay"), ("pools", 8, "alignment"),
           ("pool_stride", 8, "alignment"), ("weights", None, "null"), ("table", None, "null"),
           ("kept", None, "null"), ("HK", 0, "heads"), ("layers", 1 << 21, "launch")]
    for name, value, match in bad:
        with pytest.raises(_lib.QxError, match=match):
            _lib.call("qx_thin_rows", *dict(ok, **{name: value}).values())
    with pytest.raises(_lib.QxError, match="at most 40960"):
        _lib.call("qx_thin_rows", *dict(ok, max_used=40961, cols=50000).values())
    with pytest.raises(_lib.QxError, match="whole"):
        _lib.call("qx_thin_rows", *dict(ok, element_bytes=1, scales=16, keep=30).values())


@pytest.fixture
def thinned(monkeypatch):
    """An arena whose keys are thinned on paper (no kernel)."""
    arena = cpu_arena(pages=24)
    monkeypatch.setattr(KVArena, "thin_rows", lambda self, tables, weights, keep, **kw: tables)
    return arena


def test_thinning_frees_the_pages_past_what_stays(thinned):
    arena = thinned
    for key, n in (("a", 100), ("b", 20), ("c", 33)):
        assert arena.activate(key, n, capacity_tokens=n + 30) is not None
    pages = arena.owned_pages("a")
    free = arena.free_pages
    tables = arena.thin(["a", "b"], torch.zeros(2, 2, 2, 112), 40)
    assert tables["used"].tolist() == [100, 20] and tables["max_used"] == 100
    assert tables["table"][0, :7].tolist() == pages[:7]
    assert arena.tokens("a") == 40 and arena.owned_pages("a") == pages[:3]
    assert arena.tokens("b") == 20 and arena.free_pages == free + len(pages) - 3
    assert arena.is_thinned("a") and not arena.is_thinned("b") and not arena.is_thinned("c")
    rows = arena.append_rows("a", 9)
    assert rows.tolist() == [pages[2] * 16 + 8 + i for i in range(8)] + [arena.owned_pages("a")[3] * 16]
    assert arena.tokens("a") == 49 and arena.append_rows("a", 10000) is None and arena.tokens("a") == 49
    with pytest.raises(ValueError, match="more rows"):
        arena.append_rows("a", -1)


def test_a_thinned_key_is_not_taken_for_its_first_tokens(thinned):
    arena = thinned
    arena.activate("a", 100)
    arena.thin(["a"], torch.zeros(2, 1, 2, 112), 48)
    for use in (lambda: arena.activate("a", 100), lambda: arena.alloc("x", 60, borrow=("a", 32)),
                lambda: arena.activate("x", 60, borrow=("a", 32)),
                lambda: arena.reserve("a", 100, capacity_tokens=100),
                lambda: arena.reserve("x", 60, capacity_tokens=60, borrow=("a", 32)),
                lambda: arena.fork("a", ["x"], 32), lambda: arena.retain("a", 32),
                lambda: pack_chunk(arena, [dict(key="a", f=48, suffixes=[[1, 2]])]),
                lambda: pack_chunk(arena, [dict(key="a", f=48, suffixes=[[1, 2]])], attention_mode="tree")):
        with pytest.raises(ValueError, match="thinned"):
            use()
    assert not arena.can_borrow("a", 16) and not arena.is_resident("x")
    # forks of all it holds are thinned too, and go on with it
    arena.fork("a", ["x"])
    assert arena.is_thinned("x") and arena.tokens("x") == 48
    with pytest.raises(ValueError, match="borrows"):
        arena.thin(["x"], torch.zeros(2, 1, 2, 112), 16)
    with pytest.raises(ValueError, match="borrows pages of"):
        arena.thin(["a"], torch.zeros(2, 1, 2, 112), 16)
    arena.free_key("x")
    arena.retain("a")
    # a key of the same name that comes later is whole
    arena.free_key("a")
    assert arena.activate("a", 50) is not None and not arena.is_thinned("a") and arena.can_borrow("a", 48)
    arena.thin(["a"], torch.zeros(2, 1, 2, 64), 48)
    arena.accounting.free_key("a")
    arena.accounting.alloc("a", 30)
    assert not arena.is_thinned("a") and arena.can_borrow("a", 16)


def test_keys_in_use_are_not_thinned(thinned):
    arena = thinned
    arena.activate("a", 64)
    arena.activate("b", 80, borrow=("a", 32))
    w = torch.zeros(2, 1, 2, 96)
    with pytest.raises(ValueError, match="borrows pages of"):
        arena.thin(["a"], w, 16)
    with pytest.raises(ValueError, match="'b' borrows pages"):
        arena.thin(["b"], w, 16)
    arena.free_key("b")
    with pytest.raises(ValueError, match="once"):
        arena.thin(["a", "a"], w, 16)
    with pytest.raises(KeyError):
        arena.thin(["nobody"], w, 16)
    arena.hold("a", 1)
    with pytest.raises(ValueError, match="held"):
        arena.thin(["a"], w, 16)
    arena.release("a")
    arena.thin(["a"], w, 64)        # nothing to drop: still whole
    assert not arena.is_thinned("a") and arena.tokens("a") == 64
    assert arena.thin([], torch.zeros(2, 0, 2, 96), 16)["used"].numel() == 0


def test_rows_are_not_appended_behind_dropped_pages():
    arena = cpu_arena()
    arena.activate("a", 64)
    arena.accounting.drop_leading("a", 1)
    with pytest.raises(ValueError, match="dropped"):
        arena.append_rows("a", 1)
    with pytest.raises(ValueError, match="dropped"):
        arena.thin(["a"], torch.zeros(2, 1, 2, 64), 16)


def test_refused_thinning_changes_no_key():
    arena = cpu_arena()
    arena.activate("a", 64)
    with pytest.raises(ValueError, match="on the CPU"):
        arena.thin(["a"], torch.zeros(2, 1, 2, 64), 16)
    assert arena.tokens("a") == 64 and not arena.is_thinned("a")
    assert np.array_equal(arena.capacity_rows("a"), np.arange(64))
