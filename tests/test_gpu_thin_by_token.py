"""Thinning by token on the GPU against oracle/thin_ref.py: which rows stay, where,
and their numbers are exact, moved 16-bit rows and weights are equal bit for bit,
8-bit rows are the definition's codes; and sequences and keys that are thinned as
they grow hold their first and last tokens, by token number."""

import math
import warnings

import pytest
import torch

from oracle.thin_ref import kept_slots_by_token
from quail_amd.arena import FP8, KVArena
from tests.test_gpu_thin import heavy_tailed, make, raw_pools, tables_of

pytestmark = pytest.mark.gpu

DEV = "cuda"
PAGE = 16


def numbers_of(layers, used, totals, heads, cols, fresh, g):
    """Numbers of the tokens that rows hold after earlier thinnings: the last
    `fresh` rows of each sequence were appended since (negative), the others hold
    tokens before those in an order of each head's own."""
    tokens = torch.full((layers, len(used), heads, cols), -1, dtype=torch.int32)
    for s, (n, total) in enumerate(zip(used, totals)):
        new = min(fresh, n)
        for layer in range(layers):
            for h in range(heads):
                tokens[layer, s, h, :n - new] = torch.randperm(total - new, generator=g)[:n - new]
        tokens[:, s, :, n - new:] = -1 - torch.arange(cols - n + new)
    return tokens


def expect(weights, tokens, totals, used, keep, sinks, newest):
    """(kept, weights, numbers) after the definition."""
    L, S, H, cols = weights.shape
    w, t = weights.cpu(), tokens.cpu()
    kept = torch.full((L, S, H, min(keep, cols)), -1, dtype=torch.int32)
    out, left = torch.zeros(L, S, H, cols), torch.full((L, S, H, cols), -1, dtype=torch.int32)
    for layer in range(L):
        for s in range(S):
            for h in range(H):
                slots, numbers = kept_slots_by_token(w[layer, s, h].tolist(), t[layer, s, h].tolist(), totals[s],
                                                     used[s], keep, sinks, newest)
                n = len(slots)
                kept[layer, s, h, :n] = torch.tensor(slots, dtype=torch.int32)
                out[layer, s, h, :n] = w[layer, s, h][torch.tensor(slots, dtype=torch.long)]
                left[layer, s, h, :n] = torch.tensor(numbers, dtype=torch.int32)
    return kept, out, left


def moved(pools, scales, kept, table):
    """Pools and scales before -> after the moves that `kept` names."""
    new, new_scales = pools.clone(), None if scales is None else scales.clone()
    row = lambda s, i: int(table[s, i // PAGE]) * PAGE + i % PAGE  # noqa: E731
    L, S, H, _ = kept.shape
    for layer in range(L):
        for s in range(S):
            for h in range(H):
                src = [i for i in kept[layer, s, h].tolist() if i >= 0]
                if scales is None:
                    at = [i for i in range(len(src)) if src[i] != i]
                    new[layer, :, [row(s, i) for i in at], h] = pools[layer, :, [row(s, src[i]) for i in at], h]
                    continue
                for p in range(len(src) // PAGE):
                    here = src[p * PAGE:(p + 1) * PAGE]
                    if here == list(range(p * PAGE, (p + 1) * PAGE)):
                        continue
                    of = [row(s, i) for i in here]
                    b = scales[layer, [r // PAGE for r in of], h].int()
                    top = b.amax(0)
                    page = int(table[s, p])
                    for side in range(2):
                        value = pools[layer, side, of, h].view(FP8).float()
                        value = value * torch.exp2((b[:, side] - top[side]).float())[:, None]
                        new[layer, side, page * PAGE:(page + 1) * PAGE, h] = value.to(FP8).view(torch.uint8)
                        new_scales[layer, page, h, side] = int(top[side])
    return new, new_scales


def check_rows(arena, before, kept, table):
    want, want_scales = moved(*before, kept, table)
    if not arena.eight_bit:
        assert torch.equal(raw_pools(arena), want)
        return
    a, b = raw_pools(arena).view(FP8).float(), want.view(FP8).float()
    assert bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())
    assert torch.equal(arena.scales.cpu(), want_scales)


def rows_of(arena):
    return raw_pools(arena), None if arena.scales is None else arena.scales.cpu().clone()


def tables_for(used, totals, table, max_used=None):
    return dict(used=torch.tensor(used, dtype=torch.int32, device=DEV), table=torch.from_numpy(table).to(DEV),
                max_used=max([*used, 0]) if max_used is None else max_used,
                tokens=torch.tensor(totals, dtype=torch.int32, device=DEV))


def check(arena, weights, tokens, totals, used, table, keep, sinks=0, newest=0, max_used=None):
    want = expect(weights, tokens, totals, used, keep, sinks, newest)
    before, given = rows_of(arena), (weights.clone(), tokens.clone())
    kept, out, left = arena.thin_rows(tables_for(used, totals, table, max_used), weights, keep, sinks=sinks,
                                      newest=newest, tokens=tokens)
    assert torch.equal(weights.view(torch.int32), given[0].view(torch.int32)) and torch.equal(tokens, given[1])
    assert torch.equal(kept.cpu(), want[0]) and torch.equal(left.cpu(), want[2])
    same = out.cpu().view(torch.int32) == want[1].view(torch.int32)
    assert bool((same | (torch.isnan(out.cpu()) & torch.isnan(want[1]))).all())
    check_rows(arena, before, want[0], table)
    return kept, out, left


CASES = [
    # used, keep (16 bits), sinks, newest, rows appended since
    ([0, 1, 5], 3, 0, 1, 1),
    ([16, 17, 15], 16, 1, 2, 1),
    ([40, 0, 33, 64], 32, 4, 16, 1),
    ([100, 300, 77], 77, 4, 16, 20),
    ([1024, 1000], 512, 0, 100, 99),
    ([1025, 2048], 1000, 5, 0, 3),
    ([2049], 2048, 0, 0, 1),
    ([3000, 17], 64, 64, 0, 0),
    ([500], 48, 16, 32, 500),
    ([4096, 4097], 4000, 1, 63, 1),
    ([8193], 300, 4, 64, 7),
    ([20000], 5008, 4, 64, 1),
    ([39999, 25], 10000, 4, 128, 1),
    ([40960], 40944, 0, 40944, 16),
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("layers,heads,d", [(2, 2, 64), (1, 3, 128)])
@pytest.mark.parametrize("used,keep,sinks,newest,fresh", CASES)
def test_against_the_definition(bits, layers, heads, d, used, keep, sinks, newest, fresh):
    if bits == 8:
        keep = -(-keep // PAGE) * PAGE
    g = torch.Generator().manual_seed(sum(used) + keep)
    pages = sum(-(-u // PAGE) for u in used) + 3
    arena = make(layers, pages, heads, d, bits, g)
    totals = [n + n // 3 + s for s, n in enumerate(used)]
    cols = max(used) + 5
    tokens = numbers_of(layers, used, totals, heads, cols, fresh, g).to(DEV)
    weights = heavy_tailed((layers, len(used), heads, cols), g)
    check(arena, weights, tokens, totals, used, tables_of(used, pages, g), keep, sinks, newest)


@pytest.mark.parametrize("kind", ["zeros", "two values", "special", "rising", "falling"])
@pytest.mark.parametrize("n", [90, 3000, 9000])
def test_ties_and_values_that_are_not_numbers(kind, n):
    """A NaN is heavier than every number and lighter than a protected row."""
    g = torch.Generator().manual_seed(n)
    shape = (1, 1, 2, n)
    w = {"zeros": torch.zeros(shape), "two values": torch.randint(0, 2, shape, generator=g).float(),
         "special": torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, -math.nan, 1e-45, -1e-45, 3e38,
                                  1.0])[torch.randint(0, 10, shape, generator=g)],
         "rising": torch.arange(n).float().expand(shape).contiguous(),
         "falling": -torch.arange(n).float().expand(shape).contiguous()}[kind]
    pages = -(-n // PAGE) + 2
    arena = make(1, pages, 2, 64, 16, g)
    tokens = numbers_of(1, [n], [2 * n], 2, n, 3, g).to(DEV)
    for keep, sinks, newest in ((64, 0, 0), (n // 2, n // 8, n // 4), (32, 16, 16), (0, 0, 0)):
        check(arena, w.to(DEV), tokens, [2 * n], [n], tables_of([n], pages, g), keep, sinks, newest)


def test_numbers_that_no_sequence_has():
    """All alike, past the tokens there are, or more protected than stay: the first rows
    of those that rank alike stay, `keep` in all."""
    g = torch.Generator().manual_seed(21)
    arena = make(1, 12, 2, 64, 16, g)
    table = tables_of([150], 12, g)
    w = heavy_tailed((1, 1, 2, 160), g)
    for fill, total, newest in ((0, 150, 3), (2 ** 31 - 1, 150, 3), (149, 150, 40), (7, 2 ** 31 - 1, 4),
                                (-2 ** 31, 150, 5)):
        tokens = torch.full((1, 1, 2, 160), fill, dtype=torch.int32, device=DEV)
        check(arena, w, tokens, [total], [150], table, 40, 0, newest)
    # fewer tokens so far than rows: as many as rows
    tokens = torch.full((1, 1, 2, 160), -1, dtype=torch.int32, device=DEV)
    want = expect(w, tokens, [150], [150], 40, 2, 9)
    for total in (149, 0, -5, -2 ** 31):
        got = arena.thin_rows(tables_for([150], [total], table), w, 40, sinks=2, newest=9, tokens=tokens)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_strided_numbers_and_weights_and_bounds_past_the_sequences():
    g = torch.Generator().manual_seed(22)
    arena = make(2, 20, 2, 64, 16, g)
    used, totals = [100, 40], [220, 41]
    table = tables_of(used, 20, g, extra=40)
    wide = heavy_tailed((4, 3, 5, 700), g)
    numbers = torch.zeros(3, 4, 6, 800, dtype=torch.int32, device=DEV)
    part = numbers[1:, 1:3, ::3, 9:696]
    part.copy_(numbers_of(2, used, totals, 2, 687, 5, g))
    check(arena, wide[1:3, 1:, ::3, 13:700], part, totals, used, table, 33, 2, 7, max_used=600)
    # layers and heads that share their numbers
    shared = numbers_of(1, used, totals, 1, 128, 9, g).to(DEV).expand(2, 2, 2, 128)
    check(arena, heavy_tailed((2, 2, 2, 128), g), shared, totals, used, table, 20, 1, 12)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("growth", [1, 15, 16, 17])
def test_sequences_thinned_as_they_grow_hold_their_newest_tokens(bits, growth):
    """A newest of 16 and growths about it, 30 thinnings: by number, and by the numbers
    that this test follows through `kept` itself."""
    g = torch.Generator().manual_seed(growth)
    layers, heads, keep, sinks, newest = 2, 3, 64, 4, 16
    arena = make(layers, 14, heads, 64, bits, g)
    used, totals = [90, 30], [90, 30]
    table = tables_of([96, 96], 14, g)
    cols = 112
    tokens = torch.full((layers, 2, heads, cols), -1, dtype=torch.int32, device=DEV)
    w = torch.zeros(layers, 2, heads, cols, device=DEV)
    held = {(layer, s, h): list(range(n)) for s, n in enumerate(used) for layer in range(layers)
            for h in range(heads)}
    for step in range(30):
        # the newest have gathered least
        w = w + torch.rand(w.shape, generator=g).to(DEV)
        kept, w, tokens = check(arena, w, tokens, totals, used, table, keep, sinks, newest, max_used=96)
        for (layer, s, h), numbers in held.items():
            slots = [i for i in kept[layer, s, h].tolist() if i >= 0]
            numbers[:] = [numbers[i] for i in slots]
            assert tokens[layer, s, h, :len(slots)].tolist() == numbers
            want = set(range(min(sinks, totals[s]))) | set(range(max(0, totals[s] - newest), totals[s]))
            assert want <= set(numbers) and len(set(numbers)) == min(totals[s], keep)
        used = [min(n, keep) + growth for n in used]
        for (layer, s, h), numbers in held.items():
            numbers += range(totals[s], totals[s] + growth)
        totals = [n + growth for n in totals]


@pytest.mark.parametrize("bits", [16, 8])
def test_a_captured_token_at_a_time(bits):
    """One graph that appends a token to each sequence and thins, its numbers, lengths and
    weights as they then are; after every replay the last tokens are held."""
    g = torch.Generator().manual_seed(23)
    layers, heads, keep, newest = 2, 2, 48, 8
    arena = make(layers, 12, heads, 128, bits, g)
    table = tables_of([64, 64], 12, g, extra=0)
    tables = tables_for([48, 20], [48, 20], table, max_used=49)
    w = heavy_tailed((layers, 2, heads, 64), g)
    more = torch.zeros_like(w)
    tokens = torch.full((layers, 2, heads, 64), -1, dtype=torch.int32, device=DEV)

    def step():
        tables["used"].add_(1)
        tables["tokens"].add_(1)
        w.add_(more)
        kept, out, left = arena.thin_rows(tables, w, keep, sinks=2, newest=newest, tokens=tokens)
        w.copy_(out)
        tokens.copy_(left)
        tables["used"].clamp_(max=keep)
        return kept

    state = [tables["used"], tables["tokens"], w, tokens, arena.storage.view(torch.uint8)]
    state += [] if bits == 16 else [arena.scales]
    saved = [t.clone() for t in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for t, x in zip(state, saved):
        t.copy_(x)
    used, totals = [48, 20], [48, 20]
    for _ in range(40):
        more.copy_(torch.rand(w.shape, generator=g))
        used, totals = [n + 1 for n in used], [n + 1 for n in totals]
        want = expect(w + more, tokens, totals, used, keep, 2, newest)
        before = rows_of(arena)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept.cpu(), want[0]) and torch.equal(w.cpu(), want[1]) and torch.equal(tokens.cpu(), want[2])
        check_rows(arena, before, want[0], table)
        used = [min(n, keep) for n in used]
        assert tables["used"].tolist() == used and tables["tokens"].tolist() == totals
        for s, (n, total) in enumerate(zip(used, totals)):
            for numbers in tokens[:, s, :, :n].reshape(-1, n).tolist():
                assert set(numbers) >= {0, 1} | set(range(total - newest, total))


def test_keys_thinned_as_they_grow_hold_their_newest_tokens():
    """KVArena.thin with the numbers that the arena keeps: a row of K per token that says
    which one it is, so that the pages themselves are asked."""
    g = torch.Generator().manual_seed(24)
    layers, heads, d, keep, sinks, newest = 2, 2, 64, 48, 2, 12
    arena = KVArena(layers, 30, PAGE, heads, d)
    totals = {"a": 70, "b": 10}

    def write(rows, first):
        for layer in range(layers):
            for pool in arena.layer_kv(layer):
                # (to 2048 in fp16, to 256 in bf16: two columns)
                n = torch.arange(first, first + len(rows), device=DEV)
                pool[torch.from_numpy(rows).to(DEV), :, 0] = (n // 100).to(pool.dtype)[:, None]
                pool[torch.from_numpy(rows).to(DEV), :, 1] = (n % 100).to(pool.dtype)[:, None]

    for key, n in totals.items():
        assert arena.activate(key, n) is not None
        write(arena.capacity_rows(key)[:n], 0)
    w = torch.zeros(layers, 2, heads, 96, device=DEV)
    for step in range(40):
        if step:
            for key in totals:
                write(arena.append_rows(key, 1 + step % 13), totals[key])
                totals[key] += 1 + step % 13
        w = w + torch.rand(w.shape, generator=g).to(DEV)
        stream = torch.cuda.Stream()        # each thinning on a stream of its own
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream), warnings.catch_warnings():
            warnings.simplefilter("error")
            _, w = arena.thin(["b", "a"], w, keep, sinks=sinks, newest=newest)
        torch.cuda.current_stream().wait_stream(stream)
        w.record_stream(torch.cuda.current_stream())
        for key, total in totals.items():
            rows = torch.from_numpy(arena.capacity_rows(key)[:arena.tokens(key)]).to(DEV)
            assert len(rows) == min(total, keep)
            for layer in range(layers):
                for pool in arena.layer_kv(layer):
                    n = (pool[rows, :, 0].float() * 100 + pool[rows, :, 1].float()).int().cpu()
                    for h in range(heads):
                        got = set(n[:, h].tolist())
                        assert len(got) == len(rows)
                        assert got >= set(range(sinks)) | set(range(max(0, total - newest), total))
