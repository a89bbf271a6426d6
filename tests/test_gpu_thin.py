"""Thinning on the GPU against oracle/thin_ref.py: which rows stay and where is
exact, moved 16-bit rows and weights are equal bit for bit, and 8-bit rows are
the definition's codes."""

import math

import numpy as np
import pytest
import torch

from oracle.thin_ref import kept_slots
from quail_amd.arena import FP8, KVArena

pytestmark = pytest.mark.gpu

DEV = "cuda"
PAGE = 16


def make(layers, pages, heads, d, bits, g):
    dtype = FP8 if bits == 8 else torch.bfloat16
    arena = KVArena(layers, pages, PAGE, heads, d, dtype=dtype, v_dtype=dtype if bits == 8 else torch.float16)
    raw = torch.randint(0, 256, (arena.storage.numel() * arena.storage.element_size(),), generator=g,
                        dtype=torch.uint8)
    arena.storage.view(torch.uint8).copy_(raw)
    if bits == 8:
        arena.scales.copy_(torch.randint(118, 124, arena.scales.shape, generator=g, dtype=torch.uint8))
    return arena


def tables_of(used, pages, g, extra=2):
    perm = torch.randperm(pages, generator=g).tolist()
    need = [-(-u // PAGE) for u in used]
    table = np.full((len(used), max([*need, 0]) + extra), -7, dtype=np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[at:at + n]
        at += n
    return table


def raw_pools(arena):
    """(layers, K and V, rows, heads, d) as bytes or 16-bit words, on the CPU."""
    heads, d = arena.kv_shape
    kind = torch.uint8 if arena.eight_bit else torch.int16
    return arena.storage.view(kind).view(arena.num_layers, 2, -1, heads, d).cpu().clone()


def expect(arena, weights, used, table, keep, sinks, recent):
    """(kept, weights, pools, scales) after the definition."""
    L, S, H, cols = weights.shape
    w = weights.cpu()
    slots = min(keep, cols)
    kept = torch.full((L, S, H, slots), -1, dtype=torch.int32)
    out = torch.zeros(L, S, H, cols)
    pools = raw_pools(arena)
    old = pools.clone()
    scales = None if arena.scales is None else arena.scales.cpu().clone()
    old_scales = None if scales is None else scales.clone()
    row = lambda s, i: int(table[s, i // PAGE]) * PAGE + i % PAGE  # noqa: E731
    for layer in range(L):
        for s in range(S):
            for h in range(H):
                src = kept_slots(w[layer, s, h].tolist(), used[s], keep, sinks, recent)
                n = len(src)
                kept[layer, s, h, :n] = torch.tensor(src, dtype=torch.int32)
                out[layer, s, h, :n] = w[layer, s, h][torch.tensor(src, dtype=torch.long)]
                if scales is None:
                    to = [row(s, i) for i in range(n) if src[i] != i]
                    of = [row(s, src[i]) for i in range(n) if src[i] != i]
                    pools[layer, :, to, h] = old[layer, :, of, h]
                    continue
                for p in range(n // PAGE):
                    here = src[p * PAGE:(p + 1) * PAGE]
                    if all(i == p * PAGE + j for j, i in enumerate(here)):
                        continue
                    of = [row(s, i) for i in here]
                    b = old_scales[layer, [r // PAGE for r in of], h].int()       # (16, K and V)
                    top = b.amax(0)
                    for side in range(2):
                        value = old[layer, side, of, h].view(FP8).float()
                        value = value * torch.exp2((b[:, side] - top[side]).float())[:, None]
                        page = int(table[s, p])
                        pools[layer, side, page * PAGE:(page + 1) * PAGE, h] = value.to(FP8).view(torch.uint8)
                        scales[layer, page, h, side] = int(top[side])
    return kept, out, pools, scales


def check(arena, weights, used, table, keep, sinks=0, recent=0, max_used=None, repeat=True):
    want = expect(arena, weights, used, table, keep, sinks, recent)
    tables = dict(used=torch.tensor(used, dtype=torch.int32, device=DEV),
                  table=torch.from_numpy(table).to(DEV),
                  max_used=max([*used, 0]) if max_used is None else max_used)
    before = weights.clone()
    for _ in range(2 if repeat else 1):        # a second call changes nothing
        kept, out = arena.thin_rows(tables, weights, keep, sinks=sinks, recent=recent)
        assert torch.equal(weights.view(torch.int32), before.view(torch.int32))
        assert torch.equal(kept.cpu(), want[0])
        same = out.cpu().view(torch.int32) == want[1].view(torch.int32)
        assert bool((same | (torch.isnan(out.cpu()) & torch.isnan(want[1]))).all())
        pools = raw_pools(arena)
        if arena.eight_bit:
            a, b = pools.view(FP8).float(), want[2].view(FP8).float()
            assert bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())
            assert torch.equal(arena.scales.cpu(), want[3])
        else:
            assert torch.equal(pools, want[2])
    return kept, out


def heavy_tailed(shape, g):
    w = torch.exp(2.5 * torch.randn(shape, generator=g))
    return torch.where(w < 0.05, torch.zeros_like(w), w).to(DEV)


CASES = [
    # used, keep (16 bits), sinks, recent
    ([0, 1, 5], 3, 0, 0),
    ([16, 17, 15], 16, 1, 2),
    ([40, 0, 33, 64], 32, 4, 16),
    ([100, 300, 77], 77, 4, 16),
    ([1024, 1000], 512, 0, 100),
    ([1025, 2048], 1000, 5, 0),
    ([2049], 2048, 0, 0),
    ([3000, 17], 64, 64, 0),
    ([500], 48, 16, 32),
    ([4096, 4097], 4000, 1, 63),
    ([8193], 300, 4, 64),
    ([20000], 5008, 4, 64),
    ([39999, 25], 10000, 4, 128),
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("layers,heads,d", [(2, 2, 64), (1, 3, 128)])
@pytest.mark.parametrize("used,keep,sinks,recent", CASES)
def test_against_the_definition(bits, layers, heads, d, used, keep, sinks, recent):
    if bits == 8:
        keep = -(-keep // PAGE) * PAGE
    g = torch.Generator().manual_seed(sum(used) + keep)
    pages = sum(-(-u // PAGE) for u in used) + 3
    arena = make(layers, pages, heads, d, bits, g)
    table = tables_of(used, pages, g)
    weights = heavy_tailed((layers, len(used), heads, max(used) + 5), g)
    check(arena, weights, used, table, keep, sinks, recent)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("kind", ["zeros", "one value", "two values", "negative", "special", "rising",
                                  "falling", "low bits"])
@pytest.mark.parametrize("n", [90, 3000, 9000])
def test_ties_and_values_that_are_not_numbers(bits, kind, n):
    g = torch.Generator().manual_seed(n)
    shape = (1, 1, 2, n)
    w = {"zeros": torch.zeros(shape), "one value": torch.full(shape, 0.3),
         "two values": torch.randint(0, 2, shape, generator=g).float(),
         "negative": -torch.exp(torch.randn(shape, generator=g)),
         "special": torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, -math.nan, 1e-45, -1e-45, 3e38,
                                  1.0])[torch.randint(0, 10, shape, generator=g)],
         "rising": torch.arange(n).float().expand(shape).contiguous(),
         "falling": -torch.arange(n).float().expand(shape).contiguous(),
         "low bits": (torch.randint(0, 40, shape, generator=g) + 0x3f800000).int().view(torch.float32)}[kind]
    pages = -(-n // PAGE) + 2
    arena = make(1, pages, 2, 64, bits, g)
    for keep, sinks, recent in ((64, 0, 0), (n // 2 // PAGE * PAGE, 3, 5), (32, 16, 16), (0, 0, 0)):
        check(arena, w.to(DEV), [n], tables_of([n], pages, g), keep, sinks, recent, repeat=False)


def test_strided_weights_and_bounds_past_the_sequences():
    g = torch.Generator().manual_seed(8)
    arena = make(2, 20, 2, 64, 16, g)
    used = [100, 40]
    table = tables_of(used, 20, g, extra=40)
    wide = heavy_tailed((4, 3, 5, 700), g)
    check(arena, wide[1:3, 1:, ::3, 13:700], used, table, 33, 2, 7, max_used=600)
    # layers and heads that share their weights
    shared = heavy_tailed((1, 2, 1, 128), g).expand(2, 2, 2, 128)
    check(arena, shared, used, table, 20)


def test_rows_a_bound_cuts_off_and_tables_without_rows():
    g = torch.Generator().manual_seed(9)
    arena = make(1, 20, 2, 64, 16, g)
    table = tables_of([100], 20, g)
    w = heavy_tailed((1, 1, 2, 128), g)
    tables = dict(used=torch.tensor([100], dtype=torch.int32, device=DEV),
                  table=torch.from_numpy(table).to(DEV), max_used=60)
    kept, out = arena.thin_rows(tables, w, 20)      # used counts as 60
    for h in range(2):
        assert kept[0, 0, h].tolist() == kept_slots(w[0, 0, h].tolist(), 60, 20, 0, 0)
    tables["used"].fill_(-5)
    kept, out = arena.thin_rows(tables, w, 20)
    assert bool((kept == -1).all()) and not bool(out.any())
    none = dict(used=torch.zeros(0, dtype=torch.int32, device=DEV),
                table=torch.zeros(0, 0, dtype=torch.int32, device=DEV), max_used=0)
    kept, out = arena.thin_rows(none, w[:, :0], 20)
    assert kept.shape == (1, 0, 2, 20) and out.shape == (1, 0, 2, 128)


def test_a_page_takes_the_largest_scale_its_rows_come_with():
    """Codes shift down by whole powers of two; the last scale and NaN codes among them."""
    g = torch.Generator().manual_seed(10)
    arena = make(1, 12, 1, 64, 8, g)
    arena.scales.copy_(torch.tensor([1, 30, 120, 122, 125, 127, 130, 200, 246, 247, 2, 140],
                                    dtype=torch.uint8).view(1, 12, 1, 1).expand(1, 12, 1, 2))
    codes = arena.storage.view(torch.uint8)
    codes[(codes & 0x7f) > 0x77] = 0x77                 # 240, what the last scale allows
    codes[::97] = 0x7f                                  # NaN
    check(arena, heavy_tailed((1, 1, 1, 192), g), [190], tables_of([190], 12, g, extra=0), 96, 0, 10)


@pytest.mark.parametrize("bits", [16, 8])
def test_growing_sequences_thinned_in_a_captured_call(bits):
    """The lengths and weights are read as they are at each replay."""
    g = torch.Generator().manual_seed(11)
    arena = make(2, 40, 2, 128, bits, g)
    used = [150, 90]
    table = tables_of(used, 40, g, extra=4)
    tables = dict(used=torch.tensor(used, dtype=torch.int32, device=DEV),
                  table=torch.from_numpy(table).to(DEV), max_used=192)
    w = heavy_tailed((2, 2, 2, 192), g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    snapshot = arena.storage.clone(), None if bits == 16 else arena.scales.clone()
    with torch.cuda.stream(side):
        arena.thin_rows(tables, w, 80, sinks=2, recent=8)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, out = arena.thin_rows(tables, w, 80, sinks=2, recent=8)
    for step, lengths in enumerate([(150, 90), (120, 90), (60, 80), (81, 40)]):
        arena.storage.copy_(snapshot[0])
        if bits == 8:
            arena.scales.copy_(snapshot[1])
        w.copy_(heavy_tailed(w.shape, g))
        tables["used"].copy_(torch.tensor(lengths, dtype=torch.int32))
        want = expect(arena, w, lengths, table, 80, 2, 8)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept.cpu(), want[0]) and torch.equal(out.cpu(), want[1])
        if bits == 16:
            assert torch.equal(raw_pools(arena), want[2])
        else:
            a, b = raw_pools(arena).view(FP8).float(), want[2].view(FP8).float()
            assert bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())
            assert torch.equal(arena.scales.cpu(), want[3])


def test_a_pool_past_4_gib():
    """Rows past 2^32 bytes of the storage: 2 layers of 40,000 pages of 8 heads."""
    g = torch.Generator().manual_seed(12)
    arena = KVArena(2, 40000, PAGE, 8, 128)
    arena.storage.view(torch.int16).zero_()
    table = torch.tensor([[39999, 39001, 20000, 5]], dtype=torch.int32)
    rows = (table[0].long()[:, None] * PAGE + torch.arange(PAGE)).view(-1)
    for layer in range(2):
        for pool in arena.layer_kv(layer):
            pool[rows] = torch.randn(64, 8, 128, generator=g).to(pool.dtype).to(DEV)
    old = [p[rows].clone() for layer in range(2) for p in arena.layer_kv(layer)]
    w = heavy_tailed((2, 1, 8, 64), g)
    kept, _ = arena.thin_rows(dict(used=torch.tensor([64], dtype=torch.int32, device=DEV),
                                   table=table.to(DEV), max_used=64), w, 24)
    new = [p[rows] for layer in range(2) for p in arena.layer_kv(layer)]
    for i, (a, b) in enumerate(zip(old, new)):
        for h in range(8):
            src = kept[i // 2, 0, h].long()
            assert src.tolist() == kept_slots(w[i // 2, 0, h].tolist(), 64, 24, 0, 0)
            assert torch.equal(b[:24, h], a[src, h]) and torch.equal(b[24:, h], a[24:, h])


def test_keys_are_thinned_with_their_accounting():
    g = torch.Generator().manual_seed(13)
    arena = make(2, 60, 2, 64, 16, g)
    for key, n in (("a", 200), ("b", 31), ("c", 90)):
        assert arena.activate(key, n, capacity_tokens=n + 20) is not None
    table, used = arena.block_table(["c", "a"])
    w = heavy_tailed((2, 2, 2, 224), g)
    want = expect(arena, w, used.tolist(), table, 50, 4, 9)
    kept, out = arena.thin(["c", "a"], w, 50, sinks=4, recent=9)
    assert torch.equal(kept.cpu(), want[0]) and torch.equal(out.cpu(), want[1])
    assert torch.equal(raw_pools(arena), want[2])
    assert [arena.tokens(k) for k in "abc"] == [50, 31, 50] and len(arena.owned_pages("a")) == 4
    before = arena.owned_pages("a")
    arena.free_key("b")
    arena.retain("a")       # compaction moves the pages of keys that no pack has pinned
    arena.retain("c")
    arena.compact()
    pools = raw_pools(arena)
    rows = lambda pages: [p * PAGE + i for p in pages for i in range(PAGE)][:50]  # noqa: E731
    assert torch.equal(pools[:, :, rows(arena.owned_pages("a"))], want[2][:, :, rows(before)])


def test_another_stream_than_the_arenas():
    g = torch.Generator().manual_seed(14)
    arena = make(1, 20, 2, 64, 16, g)
    table = tables_of([250], 20, g)
    w = heavy_tailed((1, 1, 2, 256), g)
    want = expect(arena, w, [250], table, 100, 0, 0)
    tables = dict(used=torch.tensor([250], dtype=torch.int32, device=DEV),
                  table=torch.from_numpy(table).to(DEV), max_used=250)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        kept, out = arena.thin_rows(tables, w, 100)
        torch.cuda.current_stream().synchronize()
    assert torch.equal(kept.cpu(), want[0]) and torch.equal(raw_pools(arena), want[2])
