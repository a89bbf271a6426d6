"""Accumulated key weights on the GPU against oracle/thin_ref.py in 64 bits.

Bounds: a score is a sum of D products in fp32 and three more roundings, off by
(D + 16) 2^-24 of the sum of its products' sizes and of the log-sum-exp; the
hardware's exp2 adds 2^-20 of a weight; both times the weights (the oracle's
second result), and sums of n weights at most (n / 32 + 16) 2^-24 of
themselves (32 lanes, then a tree), one rounding for `weights`.
"""

import math

import numpy as np
import pytest
import torch

from oracle import thin_ref as ref
from quail_amd.arena import FP8, KVArena
from quail_amd.chunk import attention_plan
from tests.test_gpu_kv8 import engine_of, sequences

pytestmark = pytest.mark.gpu

DEV = "cuda"
PAGE = 16
HEADS = [(4, 2, 64), (32, 8, 128), (64, 8, 128), (3, 3, 64), (20, 4, 128), (6, 1, 128)]


def make(pages, hk, d, bits, g, layers=1):
    arena = KVArena(layers, pages, PAGE, hk, d, dtype=FP8 if bits == 8 else torch.bfloat16)
    for layer in range(layers):
        k = arena.layer_kv(layer)[0]
        if bits == 8:
            k.copy_((torch.randn(k.shape, generator=g) * 60).clamp(-448, 448).to(FP8))
            s = arena.layer_scales(layer)
            s.copy_(torch.randint(119, 123, s.shape, generator=g, dtype=torch.uint8))
        else:
            k.copy_(torch.randn(k.shape, generator=g).to(k.dtype))
        arena.layer_kv(layer)[1].copy_((torch.randn(k.shape, generator=g) * 3).to(arena.v_dtype))
    return arena


def keys_of(arena, table, n, layer=0):
    rows = (torch.from_numpy(np.asarray(table)).long()[:, None] * PAGE + torch.arange(PAGE)).reshape(-1)[:n]
    k = arena.layer_kv(layer)[0].cpu()[rows].double()
    if arena.eight_bit:
        k = k * torch.exp2(arena.layer_scales(layer)[..., 0].cpu().double() - 127)[rows // PAGE][..., None]
    return k


def check(got, q, lse, arena, cu_q, used, table, causal, weights=None, scale=None, layer=0):
    hk, d = arena.kv_shape
    hq = q.shape[1]
    scale = d ** -0.5 if scale is None else scale
    got = got.cpu().double()
    base = torch.zeros_like(got) if weights is None else weights.cpu().double()
    want = base.clone()
    bound = 2.0 ** -24 * base.abs()
    q, lse = q.cpu(), lse.cpu()
    for s, n in enumerate(used):
        count = int(cu_q[s + 1] - cu_q[s])
        if not n or not count:
            continue
        w, off = ref.key_weights(q, lse, keys_of(arena, table[s], n, layer), int(cu_q[s]), count, causal, scale, hk)
        terms = count * (hq // hk)
        want[s, :, :n] += w
        bound[s, :, :n] += ((d + 16) * 2.0 ** -24 + 2.0 ** -20) * off + (terms / 32 + 16) * 2.0 ** -24 * w \
            + 2.0 ** -24 * want[s, :, :n].abs() + terms * 2.0 ** -126
    assert bool(torch.isfinite(got).all())
    over = (got - want).abs() - bound
    assert float(over.max()) <= 0, float(((got - want).abs() / (bound + 1e-300)).max())


def run_case(bits, heads, q_lens, used, causal, prior=False, plan=True, seed=0, width_extra=2):
    g = torch.Generator().manual_seed(seed + sum(q_lens) + sum(used))
    hq, hk, d = heads
    pages = sum(-(-u // PAGE) for u in used) + 4
    arena = make(pages, hk, d, bits, g)
    eng = engine_of(arena, hq)
    cu_q, used, table = sequences(g, q_lens, used, pages, width_extra)
    q = torch.randn(int(cu_q[-1]), hq, d, generator=g).to(torch.bfloat16).to(DEV)
    on = [torch.from_numpy(a).to(DEV) for a in (cu_q, used, table)]
    if plan:
        tables = attention_plan(*on, heads=heads, causal=causal, eight_bit=bits == 8)
    else:
        tables = dict(zip(("cu_q", "used", "table"), on), causal=causal, max_q=max(q_lens) + 3,
                      max_used=min(max(used.tolist()) + 40, table.shape[1] * PAGE))
    _, lse = eng.read_pages(q, tables, 0)
    weights = None
    if prior:
        weights = torch.rand(len(used), hk, table.shape[1] * PAGE + 7, generator=g).to(DEV) * 5
    got = eng.key_weights(q, lse, tables, 0, weights=weights)
    check(got, q, lse, arena, cu_q, used.tolist(), table, causal, weights)
    return eng, arena, q, lse, tables, got


CASES = [
    ((1,), (1,), True), ((1,), (300,), True),
    ((1, 1, 1, 1, 1, 1), (1, 15, 16, 17, 33, 2049), True),
    ((3, 1, 2), (127, 128, 129), True), ((5, 0, 7), (40, 50, 0), True),
    ((9, 30), (4, 20), True),                                  # rows that see no key
    ((64, 100), (255, 513), True), ((64, 100), (255, 513), False),
    ((257,), (257,), True), ((300, 20, 411), (300, 700, 430), True),
    ((1100,), (1500,), True), ((1100, 7, 600), (1100, 3000, 640), True), ((900, 40), (300, 77), False),
    ((2500,), (2500,), True),
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("q_lens,used,causal", CASES)
def test_against_the_definition(bits, heads, q_lens, used, causal):
    run_case(bits, heads, q_lens, used, causal, prior=len(used) % 2 == 0)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("q_lens,used,causal", [CASES[2], CASES[4], CASES[9], CASES[11]])
def test_tables_without_a_plan(bits, q_lens, used, causal):
    run_case(bits, (32, 8, 128), q_lens, used, causal, plan=False, seed=5, width_extra=40)


def test_a_whole_context():
    run_case(16, (32, 8, 128), (3,), (40960,), True, prior=True, width_extra=0)
    run_case(8, (8, 2, 128), (700,), (39999,), True)


def test_a_row_adds_a_head_groups_size_and_calls_repeat_bit_for_bit():
    eng, arena, q, lse, plan, got = run_case(16, (32, 8, 128), (1200, 90), (1200, 1000), True)
    total = got.sum(-1, dtype=torch.float64)
    assert torch.allclose(total, torch.tensor([[1200.0 * 4], [90.0 * 4]], device=DEV, dtype=torch.float64)
                          .expand(2, 8), rtol=1e-5)
    for _ in range(3):
        assert torch.equal(eng.key_weights(q, lse, plan, 0), got)


def test_results_in_place_and_strided():
    eng, arena, q, lse, plan, got = run_case(16, (4, 2, 64), (50, 3), (60, 400), True)
    cols = got.shape[2]
    wide = torch.full((4, 5, cols + 9), -1.0, device=DEV)
    part = wide[1:3, 1:4:2, 5:5 + cols]
    part.copy_(torch.rand(part.shape, device=DEV))
    before = part.clone()
    again = eng.key_weights(q, lse, plan, 0, weights=part, out=part)
    assert again is part and torch.equal(part, before + got)
    part.fill_(-1.0)
    assert bool((wide == -1).all())
    out = torch.empty_like(got)
    assert eng.key_weights(q, lse, plan, 0, out=out) is out and torch.equal(out, got)


def test_query_rows_apart_and_a_softmax_scale():
    g = torch.Generator().manual_seed(3)
    arena = make(30, 2, 128, 16, g)
    eng = engine_of(arena, 4)
    cu_q, used, table = sequences(g, (20, 5), (200, 100), 30)
    qkv = torch.randn(25, 8 * 128 + 64, generator=g).to(torch.bfloat16).to(DEV)
    q = qkv[:, 64:64 + 512].unflatten(1, (4, 128))
    plan = attention_plan(*(torch.from_numpy(a).to(DEV) for a in (cu_q, used, table)), heads=(4, 2, 128),
                          eight_bit=False)
    _, lse = eng.read_pages(q, plan, 0, softmax_scale=0.2)
    got = eng.key_weights(q, lse, plan, 0, softmax_scale=0.2)
    check(got, q, lse, arena, cu_q, used.tolist(), table, True, scale=0.2)
    wide = torch.full((6, 40), 3.0, device=DEV)     # log-sum-exps apart
    wide[1:5, 8:33] = lse
    assert torch.equal(eng.key_weights(q, wide[1:5, 8:33], plan, 0, softmax_scale=0.2), got)


def test_one_row_of_a_wide_tensor():
    g = torch.Generator().manual_seed(31)
    arena = make(8, 2, 64, 16, g)
    eng = engine_of(arena, 4)
    cu_q, used, table = sequences(g, (1,), (90,), 8, 1)
    tables = attention_plan(*(torch.from_numpy(a).to(DEV) for a in (cu_q, used, table)), heads=(4, 2, 64),
                            causal=True, eight_bit=False)
    wide = torch.randn(2, 2 ** 19 + 3, generator=g).to(torch.bfloat16).to(DEV)
    q = wide[:1, 8:8 + 256].view(1, 4, 64)
    _, lse = eng.read_pages(q.contiguous(), tables, 0)
    check(eng.key_weights(q, lse, tables, 0), q, lse, arena, cu_q, used.tolist(), table, True)


@pytest.mark.parametrize("bits", [16, 8])
def test_what_lies_past_the_keys_and_in_masked_ones_stays_out(bits):
    """NaN rows past each sequence's keys, and NaN in a key that only the last
    rows see: that key's weight alone is NaN, and those rows' (their
    log-sum-exps are)."""
    g = torch.Generator().manual_seed(4)
    hq, hk, d = 4, 2, 64
    arena = make(40, hk, d, bits, g)
    eng = engine_of(arena, hq)
    cu_q, used, table = sequences(g, (100, 3), (120, 300), 40)
    k = arena.layer_kv(0)[0]
    live = torch.zeros(k.shape[0], dtype=torch.bool)
    for s, n in enumerate(used):
        live[(torch.from_numpy(table[s]).long()[:, None] * PAGE + torch.arange(PAGE)).reshape(-1)[:n]] = True
    raw, nan = (k.view(torch.uint8), 0x7f) if bits == 8 else (k.view(torch.int16), 0x7fc0)
    raw[~live.to(DEV)] = nan
    q = torch.randn(103, hq, d, generator=g).to(torch.bfloat16).to(DEV)
    plan = attention_plan(*(torch.from_numpy(a).to(DEV) for a in (cu_q, used, table)), heads=(hq, hk, d),
                          eight_bit=bits == 8)
    _, lse = eng.read_pages(q, plan, 0)
    got = eng.key_weights(q, lse, plan, 0)
    check(got, q, lse, arena, cu_q, used.tolist(), table, True)
    # key 119 of the first sequence, which its last row alone sees
    bad = int(table[0, 119 // PAGE]) * PAGE + 119 % PAGE
    raw[bad] = nan
    lse2 = lse.clone()
    lse2[:, 99] = 0.0           # a log-sum-exp that is a number: the key's own NaN is what is left
    again = eng.key_weights(q, lse2, plan, 0)
    assert bool(torch.isnan(again[0, :, 119]).all())
    again[0, :, 119] = 0
    assert bool(torch.isfinite(again).all())
    assert torch.equal(again[1], got[1])


def test_sequences_that_grow_in_a_captured_call():
    """One capture over bounds, weights gathered in place; lengths grow
    between the replays, a token each, as a generating caller's do."""
    g = torch.Generator().manual_seed(6)
    hq, hk, d = 32, 8, 128
    arena = make(48, hk, d, 16, g)
    eng = engine_of(arena, hq)
    cu_q, used, table = sequences(g, (1, 1, 1), (1, 250, 400), 48)
    tables = dict(cu_q=torch.from_numpy(cu_q).to(DEV), used=torch.from_numpy(used).to(DEV),
                  table=torch.from_numpy(table).to(DEV), causal=True, max_q=1, max_used=432)
    q = torch.randn(3, hq, d, generator=g).to(torch.bfloat16).to(DEV)
    held = torch.zeros(3, hk, 448, device=DEV)

    def step():
        _, lse = eng.read_pages(q, tables, 0)
        eng.key_weights(q, lse, tables, 0, weights=held, out=held)
        return lse

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lse = step()
    held.zero_()
    want = torch.zeros(3, hk, 448, dtype=torch.float64)
    for t in range(12):
        q.copy_(torch.randn(3, hq, d, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        now = tables["used"].cpu().tolist()
        for s, n in enumerate(now):
            w, _ = ref.key_weights(q.cpu(), lse.cpu(), keys_of(arena, table[s], n), s, 1, True, d ** -0.5, hk)
            want[s, :, :n] += w
        tables["used"].add_(1)
    assert torch.allclose(held.cpu().double(), want, rtol=1e-4, atol=1e-6)


def test_two_captured_calls_and_an_eager_one_share_nothing():
    """Calls over chunks (scratch memory) captured twice, replayed on two
    streams at once beside an eager one."""
    g = torch.Generator().manual_seed(7)
    hq, hk, d = 8, 2, 128
    arena = make(300, hk, d, 16, g)
    eng = engine_of(arena, hq)
    parts = []
    for i in range(3):
        cu_q, used, table = sequences(g, (900 + i, 40), (1000, 90 + i), 300)
        q = torch.randn(int(cu_q[-1]), hq, d, generator=g).to(torch.bfloat16).to(DEV)
        plan = attention_plan(*(torch.from_numpy(a).to(DEV) for a in (cu_q, used, table)),
                              heads=(hq, hk, d), eight_bit=False)
        _, lse = eng.read_pages(q, plan, 0)
        parts.append((q, lse, plan, eng.key_weights(q, lse, plan, 0)))
    torch.cuda.synchronize()
    graphs = []
    for q, lse, plan, _ in parts[:2]:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eng.key_weights(q, lse, plan, 0)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = eng.key_weights(q, lse, plan, 0)
        graphs.append((graph, got, torch.cuda.Stream()))
    for _ in range(5):
        for graph, got, stream in graphs:
            got.fill_(-1.0)
        torch.cuda.synchronize()
        for graph, got, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        eager = eng.key_weights(*parts[2][:3], 0)
        torch.cuda.synchronize()
        assert torch.equal(eager, parts[2][3])
        for (graph, got, stream), part in zip(graphs, parts):
            assert torch.equal(got, part[3])


def test_many_sequences_in_one_call():
    """More sequences than one launch takes, few rows and chunked ones."""
    g = torch.Generator().manual_seed(8)
    hq, hk, d = 4, 1, 64
    arena = make(64, hk, d, 16, g)
    eng = engine_of(arena, hq)
    seqs = 2100
    for longest in (3, 600):
        q_lens = [int(n) for n in torch.randint(0, 4, (seqs,), generator=g)]
        q_lens[7], q_lens[2060] = longest, longest
        used = [int(n) for n in torch.randint(0, 60, (seqs,), generator=g)]
        used[7], used[2060] = 64, 64
        table = torch.stack([torch.randperm(64, generator=g)[:4] for _ in range(seqs)]).to(torch.int32).numpy()
        cu_q = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        q = torch.randn(int(cu_q[-1]), hq, d, generator=g).to(torch.bfloat16).to(DEV)
        plan = attention_plan(torch.from_numpy(cu_q).to(DEV), torch.tensor(used, dtype=torch.int32, device=DEV),
                              torch.from_numpy(table).to(DEV), heads=(hq, hk, d), eight_bit=False)
        _, lse = eng.read_pages(q, plan, 0)
        got = eng.key_weights(q, lse, plan, 0)
        check(got, q, lse, arena, cu_q, used, table, True)


def test_no_rows_and_no_keys():
    g = torch.Generator().manual_seed(9)
    arena = make(4, 2, 64, 16, g)
    eng = engine_of(arena, 4)
    none = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=DEV)
    tables = dict(cu_q=torch.zeros(3, dtype=torch.int32, device=DEV),
                  used=torch.tensor([5, 0], dtype=torch.int32, device=DEV),
                  table=torch.zeros(2, 1, dtype=torch.int32, device=DEV), causal=True, max_q=0, max_used=16)
    w = torch.rand(2, 2, 16, device=DEV)
    assert torch.equal(eng.key_weights(none, torch.zeros(4, 0, device=DEV), tables, 0, weights=w), w)
    assert not bool(eng.key_weights(none, torch.zeros(4, 0, device=DEV), tables, 0).any())
    q = torch.randn(2, 4, 64, generator=g).to(torch.bfloat16).to(DEV)
    tables.update(cu_q=torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV),
                  used=torch.zeros(2, dtype=torch.int32, device=DEV), max_q=1, max_used=0,
                  table=torch.zeros(2, 0, dtype=torch.int32, device=DEV))
    _, lse = eng.read_pages(q, tables, 0)
    assert eng.key_weights(q, lse, tables, 0).shape == (2, 2, 0)
    assert torch.equal(eng.key_weights(q, lse, tables, 0, weights=w), w)
    assert math.isinf(float(lse[0, 0]))
