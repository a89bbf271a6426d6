"""Packs over an 8-bit arena at the edges of what a pack holds. No GPU."""

import numpy as np
import pytest
import torch

from quail_amd import chunk as chunks
from quail_amd.arena import FP8, KVArena
from quail_amd.chunk import pack_chunk


def arena_of(dtype=FP8):
    arena = KVArena(1, 40, 16, 2, 64, dtype=dtype, device="cpu")
    arena.activate("d", 21, capacity_tokens=21)
    return arena


def group(*suffixes):
    return [dict(key="d", prefix=np.arange(21), f=21, start=0,
                 suffixes=[np.asarray(s, dtype=np.int64) for s in suffixes])]


@pytest.mark.parametrize("suffixes", [((1, 2), ()), ((), (1,)), ((), ()), ((3,), (), (4, 5))])
def test_a_suffix_of_no_row_packs_as_on_a_16_bit_arena(suffixes):
    plain, eight = arena_of(torch.bfloat16), arena_of()
    want, got = (pack_chunk(a, group(*suffixes), attention_heads=(4, 2, 64)) for a in (plain, eight))
    assert eight.free_pages == plain.free_pages
    for name in ("src", "dst", "cu_q", "used", "table"):
        assert np.array_equal(want.meta["unified"][name], got.meta["unified"][name])
    rows = [r for p in got.meta["unified"]["page_writes"] for _, _, _, r0, c in p.tolist()
            for r in range(r0, r0 + c)]
    assert sorted(rows) == list(range(got.tokens))


@pytest.mark.parametrize("name", ["page_writes", "_add_work"])
def test_a_pack_that_fails_late_leaves_nothing_allocated(name, monkeypatch):
    arena = arena_of()
    free = arena.free_pages

    def fail(*args, **kw):
        raise ValueError("late")

    monkeypatch.setattr(chunks, name, fail)
    with pytest.raises(ValueError, match="late"):
        pack_chunk(arena, group((1, 2), (3,)), attention_heads=(4, 2, 64))
    assert arena.free_pages == free and arena.resident_keys() == ["d"]
