"""Rows appended to resident keys: the page accounting, on the CPU."""

import pytest
import torch

from quail_amd.arena import KVArena


def cpu_arena(pages=16):
    return KVArena(2, pages, 16, 2, 64, device="cpu")


def state(arena):
    acct = arena.accounting
    return {key: acct._table(key) for key in acct.resident_keys()}, acct.free_list(), arena.retained_pages


def test_rows_of_a_page_that_another_key_reads_are_not_handed_out():
    arena = cpu_arena()
    arena.activate("a", 64)
    arena.fork("a", ["x"])
    arena.retain("a", 40)           # x reads tokens 40..47 in the page of a's next rows
    arena.pin("a")
    before = state(arena)
    for count in (1, 8, 9, 100):
        with pytest.raises(ValueError, match="another key reads the page of row 40"):
            arena.append_rows("a", count)
        assert state(arena) == before
    assert len(arena.append_rows("a", 0)) == 0 and state(arena) == before
    rows = arena.append_rows("x", 20)           # its own pages from there on
    assert not set(rows.tolist()) & set(arena.capacity_rows("a").tolist())
    # nobody else's any more
    arena.free_key("x")
    assert arena.append_rows("a", 8).tolist() == arena.capacity_rows("a")[40:48].tolist()


def test_rows_past_a_lent_page_are_the_keys_own():
    arena = cpu_arena()
    arena.activate("a", 64, capacity_tokens=80)
    arena.fork("a", ["x", "y"], 32)
    assert arena.append_rows("a", 5).tolist() == arena.capacity_rows("a")[64:69].tolist()
    arena.retain("a", 48)           # a whole page: the next row begins one of its own
    arena.pin("a")
    assert len(arena.append_rows("a", 30)) == 30
    # a later page of the rows asked for is lent
    arena.fork("a", ["z"], 64)
    arena.retain("a", 33)
    arena.pin("a")
    with pytest.raises(ValueError, match="another key reads"):
        arena.append_rows("a", 1)
    arena.accounting.set_tokens("a", 16)
    with pytest.raises(ValueError, match="another key reads"):
        arena.append_rows("a", 40)


def test_a_key_that_holds_fewer_tokens_than_it_borrows_is_refused():
    arena = cpu_arena()
    arena.activate("a", 64)
    arena.activate("b", 40, borrow=("a", 32))
    arena.accounting.set_tokens("b", 20)
    with pytest.raises(ValueError, match="another key reads the page of row 20"):
        arena.append_rows("b", 1)
    arena.accounting.set_tokens("b", 32)
    assert arena.append_rows("b", 20).tolist() == arena.capacity_rows("b")[32:52].tolist()


def test_holders_of_pages():
    arena = cpu_arena()
    acct = arena.accounting
    arena.activate("a", 64)
    arena.activate("b", 64, borrow=("a", 32))
    arena.activate("c", 64, borrow=("a", 16))
    assert [acct.holders("a", i, i + 1) for i in range(5)] == [3, 2, 1, 1, 0]
    assert acct.holders("a", 1, 99) == 2 and acct.holders("a", -5, 2) == 3 and acct.holders("a", 3, 2) == 0
    assert acct.holders("b", 0, 2) == 3 and acct.holders("b", 2, 4) == 1
    with pytest.raises(KeyError):
        acct.holders("nobody", 0, 1)


def test_retained_keys_are_pinned_before_they_are_continued():
    """Their pages counted as retained, and the victims' sizes, stay true."""
    arena = cpu_arena(8)
    arena.activate("a", 64)
    arena.retain("a", priority=7.0)
    before = state(arena)
    with pytest.raises(ValueError, match="pin it first"):
        arena.append_rows("a", 10)
    with pytest.raises(ValueError, match="pin it first"):
        arena.thin(["a"], torch.zeros(2, 1, 2, 64), 16)
    assert state(arena) == before and arena.retained_pages == 4 and not arena.is_thinned("a")
    arena.pin("a")
    assert len(arena.append_rows("a", 50)) == 50 and arena.retained_pages == 0
    assert arena.activate("b", 64) is None and arena.is_resident("a")     # nothing to evict
    arena.retain("a")
    assert arena.retained_pages == 8
    assert arena.activate("b", 64) is not None and not arena.is_resident("a")
    assert (arena.evicted_pages, arena.evicted_prefix_tokens) == (8, 114)


def test_the_priority_of_a_key_that_was_thinned_is_the_one_it_is_retained_with(monkeypatch):
    monkeypatch.setattr(KVArena, "thin_rows", lambda self, tables, weights, keep, **kw: tables)
    arena = cpu_arena(8)
    for key in "ab":
        arena.activate(key, 64)
    arena.retain("a", priority=9.0)
    arena.retain("b", priority=5.0)
    arena.pin("a")
    arena.thin(["a"], torch.zeros(2, 1, 2, 64), 32)
    arena.append_rows("a", 16)
    arena.retain("a", priority=9.0)
    assert arena.retained_pages == 7
    assert arena.activate("c", 48) is not None
    assert arena.is_resident("a") and not arena.is_resident("b")
