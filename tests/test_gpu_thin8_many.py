"""What rows of 8-bit pages lose over many thinnings, on the GPU.

A row that moves (or stays where one moves in, or where a larger row is written
beside it) takes its page's new scale: its code shifts down by the power of two
between, exact unless the code becomes subnormal, then off by half of that step,
2^-10 of the new scale. Each such shift at least doubles the scale, so all of them
together are off by less than 2^-10 (1 + 1/2 + 1/4 + ...) = 2^-9 of the scale that the
row has now. And a scale is one that some row of its head was written with: it never
passes the largest of those.
"""

import numpy as np
import pytest
import torch

from quail_amd.arena import FP8, KVArena
from tests.test_gpu_kv8 import engine_of
from tests.test_gpu_long_documents import held, write

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("growth", [3, 16, 40])
def test_rows_against_what_was_first_written_over_many_thinnings(growth):
    g = torch.Generator().manual_seed(growth)
    heads, d, keep, steps = 3, 64, 96, 40
    arena = KVArena(1, 20, 16, heads, d, dtype=FP8)
    eng = engine_of(arena, heads)
    count, total = 150, 0
    arena.activate("a", count)
    rows = arena.capacity_rows("a")[:count]
    numbers = np.zeros((0, heads), dtype=np.int64)          # the token in each slot of each head
    first = torch.zeros(2, 0, heads, d, dtype=torch.float64)
    largest = torch.zeros(2, heads, dtype=torch.float64)
    w = torch.zeros(1, 1, heads, 176, device=DEV)
    moved = 0
    for step in range(steps):
        n = len(rows)
        # most rows small, a few 2^9 times as large, which soon leave
        size = torch.where(torch.rand(n, heads, 1, generator=g) < 0.03, 512.0, 1.0) * \
            torch.exp2(torch.randn(n, heads, 1, generator=g))
        kv = [(torch.randn(n, heads, d, generator=g) * size).to(torch.bfloat16).to(DEV) for _ in range(2)]
        write(eng, *kv, rows, 0)
        value, scale = held(arena, rows, 0)
        first = torch.cat([first, value], 1)
        largest = torch.maximum(largest, scale.amax((1, 3)))
        numbers = np.concatenate([numbers, np.arange(total, total + n)[:, None].repeat(heads, 1)])
        total += n
        used = arena.tokens("a")
        assert used == len(numbers) <= w.shape[-1]
        # the large rows weigh least
        w[0, 0, :, used - n:used] = (1 / size[..., 0].t()).to(DEV)
        w += 0.01 * torch.rand(w.shape, generator=g).to(DEV)
        kept, w = arena.thin(["a"], w, keep, sinks=2, newest=8)
        slots = kept[0, 0, :, :min(used, keep)].cpu().numpy()
        moved += int((slots != np.arange(slots.shape[1])).sum())
        numbers = np.stack([numbers[slots[h], h] for h in range(heads)], 1)
        value, scale = held(arena, arena.capacity_rows("a")[:arena.tokens("a")], 0)
        for h in range(heads):
            off = (value[:, :, h] - first[:, numbers[:, h], h]).abs()
            assert bool((off <= 2.0 ** -9 * scale[:, :, h]).all())
        assert bool((scale.amax((1, 3)) <= largest).all())
        rows = arena.append_rows("a", growth)
    assert moved > steps * heads
