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
