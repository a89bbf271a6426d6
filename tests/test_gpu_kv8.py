"""The 8-bit KV arena on the GPU: page writes, attention over the pages and
page copies against float64 restatements of their definitions
(oracle/kv8_ref.py), and runs of them together.

Error bounds, counted in roundings (half a step: bf16 2^-8, e4m3 2^-4, fp32
2^-24 of the value). Attention: P is rounded to bf16 (2^-8 of each weight),
the row to bf16 (2^-8 of the value); a score is a sum of D fp32 products,
off by at most (D + 8) 2^-24 of scale * sum |q||k|, and so is the logarithm
of a weight, twice (score and maximum); the hardware's exp2 and log2 add
2^-20 of a weight or of 1 + |lse|.
"""

import numpy as np
import pytest
import torch

from oracle import kv8_ref as ref
from quail_amd.arena import FP8, KVArena

pytestmark = pytest.mark.gpu

DEV = "cuda"
PAGE = 16
HEADS = [(4, 2, 64), (24, 8, 64), (32, 8, 128), (64, 8, 128), (8, 8, 128), (6, 2, 128)]


def same_codes(a, b):
    """Equal values (e4m3 has two codes of zero and two of NaN)."""
    a, b = a.float().cpu(), b.float().cpu()
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


class _Rotary:
    def __init__(self, cache):
        self.cos_sin_cache = cache


class _Norm:
    def __init__(self, weight):
        self.weight, self.variance_epsilon = weight, 1e-6


class _Attn:
    def __init__(self, d, g):
        self.q_norm = _Norm((1 + 0.2 * torch.randn(d, generator=g)).to(torch.bfloat16).to(DEV))
        self.k_norm = _Norm((1 + 0.2 * torch.randn(d, generator=g)).to(torch.bfloat16).to(DEV))


def engine_of(arena, hq, cache=None):
    from quail_amd.engine import Engine
    hk, d = arena.kv_shape
    return Engine(arena, num_q_heads=hq, num_kv_heads=hk, head_dim=d, rotary=_Rotary(cache))


def rope_cache(rows, d, dtype):
    inv = 1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).to(dtype).to(DEV)


def fill(arena, g, stale=0x7f):
    """Random codes and scales in every page; returns nothing."""
    k, v = arena.layer_kv(0)
    for pool in (k, v):
        x = torch.randn(pool.shape, generator=g) * 60
        pool.copy_(x.clamp(-448, 448).to(FP8))
    s = arena.layer_scales(0)
    s.copy_(torch.randint(117, 123, s.shape, generator=g, dtype=torch.uint8))


def sequences(g, q_lens, used, num_pages, width_extra=2):
    """cu_q, used and a block table of distinct random pages (rows past each
    sequence's pages name page 0)."""
    perm = torch.randperm(num_pages, generator=g).tolist()
    width = max(-(-u // PAGE) for u in used) + width_extra
    table, at = np.zeros((len(used), width), dtype=np.int32), 0
    for s, u in enumerate(used):
        need = -(-u // PAGE)
        table[s, :need] = perm[at:at + need]
        at += need
    cu_q = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    return cu_q, np.asarray(used, dtype=np.int32), table


def spoil_unused_rows(arena, used, table):
    """NaN codes in every row that no sequence may read."""
    k, v = arena.layer_kv(0)
    live = np.zeros(k.shape[0], dtype=bool)
    for s, u in enumerate(used):
        rows = (table[s][:, None] * PAGE + np.arange(PAGE)).reshape(-1)[:u]
        live[rows] = True
    dead = torch.from_numpy(~live).to(DEV)
    for pool in (k, v):
        pool.view(torch.uint8)[dead] = 0x7f


def check_rows(out, lse, q, arena, cu_q, used, table, causal, scale=None):
    k, v = arena.layer_kv(0)
    d = q.shape[2]
    want, want_lse, size, reach = ref.attend(q, k, v, arena.layer_scales(0), cu_q.tolist(),
                                             used.tolist(), table, causal, scale)
    got = out.view(want.shape).double()
    score = (d + 8) * 2.0 ** -24 * reach
    bound = 2.0 ** -8 * (size + want.abs()) + (2 * score[..., None] + 2.0 ** -20 + 2.0 ** -16) * size
    assert bool(torch.isfinite(got).all())
    over = (got - want).abs() - bound
    assert float(over.max()) <= 1e-30, float(((got - want).abs() / (bound + 1e-30)).max())
    empty = torch.isinf(want_lse)
    got_lse = lse.t().double()
    assert bool((torch.isinf(got_lse) == empty).all())
    err = (got_lse - want_lse).abs()[~empty]
    assert bool((err <= (2 * score + 2.0 ** -20 * (1 + want_lse.abs()))[~empty]).all())


CASES = [
    # (query rows, keys) per sequence; causal
    ((1,), (1,), True),
    ((1,), (300,), True),
    ((1, 1, 1, 1, 1, 1), (1, 15, 16, 17, 33, 2049), True),
    ((3, 1, 2), (127, 128, 129), True),
    ((5, 0, 1, 8), (3, 20, 0, 64), True),          # rows that see no key, no rows, no keys
    ((7, 40, 1), (31, 96, 500), False),
    ((21, 33, 64, 100), (70, 33, 700, 101), True),
    ((2, 1), (5000, 9000), False),                  # split over the keys
    ((130, 3), (130, 1), True),
    ((40, 21, 70), (9000, 100, 1500), True),        # tiles split over the keys
    ((33, 9), (6000, 640), False),
]


@pytest.mark.parametrize("hq,hk,d", HEADS)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_read_pages_matches_float64(hq, hk, d, case):
    from quail_amd.chunk import attention_plan
    q_lens, used, causal = CASES[case]
    g = torch.Generator().manual_seed(100 + case)
    pages = sum(-(-u // PAGE) for u in used) + 3
    arena = KVArena(1, pages, PAGE, hk, d, dtype=FP8)
    fill(arena, g)
    cu_q, used, table = sequences(g, q_lens, used, pages)
    spoil_unused_rows(arena, used, table)
    q = torch.randn(int(cu_q[-1]), hq, d, generator=g).to(torch.bfloat16).to(DEV)
    plan = attention_plan(*(torch.from_numpy(a).to(DEV) for a in (cu_q, used, table)),
                          heads=(hq, hk, d), causal=causal)
    out, lse = engine_of(arena, hq).read_pages(q, plan, 0)
    check_rows(out, lse, q, arena, cu_q, used, table, causal)


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (32, 8, 128), (6, 2, 128)])
@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, torch.float32])
def test_page_writes_match_float64(hq, hk, d, cache_dtype):
    """Fresh pages, appends to part-filled pages (with smaller, larger and
    equal scales), a copied partial page, one token, a page of zeros."""
    g = torch.Generator().manual_seed(7)
    arena = KVArena(2, 12, PAGE, hk, d, dtype=FP8)
    phases = [[(3, 3, 0, 0, 16), (5, 5, 0, 16, 3), (0, 0, 7, 19, 9), (1, 1, 15, 28, 1),
               (7, 7, 4, 29, 2), (9, 9, 0, 31, 4)],
              [(11, 5, 3, 35, 6), (2, 3, 16, 41, 0), (10, 0, 9, 41, 7)]]
    n = 48
    qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g)
    qkv[19:28] *= 1000
    qkv[31:35, (hq + hk) * d:] = 0
    qkv[29, (hq + hk) * d] = float("inf")
    qkv[30, (hq + hk) * d + 1] = float("nan")
    qkv = qkv.to(torch.bfloat16).to(DEV)
    positions = torch.randint(0, 500, (n,), generator=g).to(DEV)
    cache = rope_cache(500, d, cache_dtype)
    attn = _Attn(d, g)
    for layer in range(2):
        k, v = arena.layer_kv(layer)
        for pool in (k, v):
            pool.copy_((torch.randn(pool.shape, generator=g) * 100).clamp(-448, 448).to(FP8))
        arena.layer_scales(layer).copy_(torch.randint(110, 135, (12, hk, 2), generator=g,
                                                      dtype=torch.uint8))
    layer = 1
    before = [t.clone() for t in (*arena.layer_kv(0), arena.layer_scales(0))]
    k0, v0 = (p.cpu() for p in arena.layer_kv(layer))
    s0 = arena.layer_scales(layer).cpu().clone()
    eng = engine_of(arena, hq, cache)
    items = tuple(torch.tensor(p, dtype=torch.int32, device=DEV) for p in phases)
    meta = dict(layer=layer, unified=dict(page_writes=items))
    q = eng.qk_norm_rope_kv(qkv, positions, attn, meta)
    assert meta["kv_fresh_layer"] == layer
    # float64 rows
    x = qkv.double().cpu().view(n, -1, d)
    cs = cache.double().cpu()[positions.cpu()][:, None]
    cos, sin = cs[..., :d // 2], cs[..., d // 2:]

    def turn(x, w):
        y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double().cpu()
        a, b = y[..., :d // 2], y[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    k_rows, v_rows = turn(x[:, hq:hq + hk], attn.k_norm.weight), x[:, hq + hk:]
    for phase in phases:
        ref.write_items(k0, v0, s0, k_rows, v_rows, phase)
    k, v = (p.cpu() for p in arena.layer_kv(layer))
    assert torch.equal(arena.layer_scales(layer).cpu(), s0)
    assert same_codes(v, v0)    # V is only rounded, and once
    # K's fp32 norm and RoPE are off by a few 2^-24 of the row's size: a code
    # may be the neighbour only where the exact value is that near a border
    assert bool((torch.isnan(k.float()) == torch.isnan(k0.float())).all())
    off = (k.float() != k0.float()) & ~torch.isnan(k.float())
    assert float(off.float().mean()) < 1e-4
    exact = ref.values(k0, s0, 0)
    assert bool(((ref.values(k, s0, 0) - exact).abs() <= 0.126 * exact.abs() + 2.0 ** -9 *
                 torch.exp2(s0[:, :, 0].double() - 127).repeat_interleave(PAGE, 0)[..., None]).all())
    # q's rows
    want = turn(x[:, :hq], attn.q_norm.weight)
    written = sorted({r for p in phases for _, _, _, r0, c in p for r in range(r0, r0 + c)})
    assert written == list(range(n))
    err = (q.view(n, hq, d).double().cpu() - want).abs()
    assert bool((err <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * want.abs().amax(-1, keepdim=True)).all())
    # the other layer is untouched
    for a, b in zip(before, (*arena.layer_kv(0), arena.layer_scales(0))):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    # the same from rows, V bit for bit
    again = KVArena(1, 12, PAGE, hk, d, dtype=FP8)
    k1, v1, s1 = k0.clone(), v0.clone(), s0.clone()
    for pool, h in zip(again.layer_kv(0), (k1, v1)):
        pool.copy_(h)
    again.layer_scales(0).copy_(s1)
    k3 = k_rows.to(torch.bfloat16).to(DEV)
    v3 = qkv.view(n, -1, d)[:, hq + hk:]
    engine_of(again, hq).write_kv(k3, v3, dict(layer=0, unified=dict(page_writes=items)))
    for phase in phases:
        ref.write_items(k1, v1, s1, k3.double().cpu(), v3.double().cpu(), phase)
    for pool, h in zip(again.layer_kv(0), (k1, v1)):
        assert same_codes(pool, h)
    assert torch.equal(again.layer_scales(0).cpu(), s1)


@pytest.mark.parametrize("dtype", [FP8, torch.bfloat16])
@pytest.mark.parametrize("layers,hk,d,pages,moved", [(1, 2, 64, 7, 3), (36, 8, 128, 1001, 500),
                                                     (3, 1, 64, 20, 1), (2, 3, 128, 9, 0)])
def test_copy_pages_is_exact_in_every_layer(dtype, layers, hk, d, pages, moved):
    g = torch.Generator().manual_seed(3)
    arena = KVArena(layers, pages, PAGE, hk, d, dtype=dtype)
    raw = arena.storage.view(torch.uint8)
    raw.copy_(torch.randint(0, 256, (1 << 20,), generator=g, dtype=torch.uint8).to(DEV).repeat(
        -(-raw.numel() // (1 << 20)))[:raw.numel()])
    if arena.eight_bit:
        arena.scales.copy_(torch.randint(0, 256, arena.scales.shape, generator=g,
                                         dtype=torch.uint8))
    order = torch.randperm(pages, generator=g).tolist()
    src, dst = order[:moved], order[moved:2 * moved]
    if moved > 1:
        src[1] = src[0]    # one source for two destinations
    want = raw.clone().view(2 * layers, pages, -1)
    want[:, dst] = want[:, src]
    scales = None if arena.scales is None else arena.scales.clone()
    if scales is not None:
        scales[:, dst] = scales[:, src]
    arena.copy_pages(src, dst)
    assert torch.equal(raw, want.view(-1))
    if scales is not None:
        assert torch.equal(arena.scales, scales)


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (24, 8, 64), (8, 8, 128)])
@pytest.mark.parametrize("q_len,used", [(5, 40), (40, 40), (70, 300), (33, 64)])
def test_nan_keys_and_values_reach_only_the_rows_that_see_them(hq, hk, d, q_len, used):
    """NaN codes in K and V of one late token: rows before it are as they are
    without it, bit for bit; rows that see it are NaN (V: in its columns)."""
    from quail_amd.chunk import attention_plan
    g = torch.Generator().manual_seed(5)
    pages = -(-used // PAGE) + 1
    arena = KVArena(1, pages, PAGE, hk, d, dtype=FP8)
    fill(arena, g)
    cu_q, u, table = sequences(g, (q_len,), (used,), pages)
    plan = attention_plan(*(torch.from_numpy(a).to(DEV) for a in (cu_q, u, table)),
                          heads=(hq, hk, d))
    q = torch.randn(q_len, hq, d, generator=g).to(torch.bfloat16).to(DEV)
    eng = engine_of(arena, hq)
    clean, clean_lse = eng.read_pages(q, plan, 0)
    at = used - 3                                   # seen by the last 3 rows
    row = int(table[0, at // PAGE]) * PAGE + at % PAGE
    k, v = arena.layer_kv(0)
    keep = v.view(torch.uint8)[row].clone()
    v.view(torch.uint8)[row, 0, 5] = 0x7f
    v.view(torch.uint8)[row, hk - 1, d - 1] = 0xff
    out, lse = eng.read_pages(q, plan, 0)
    group = hq // hk
    want = clean.view(q_len, hq, d).clone()
    want[-3:, :group, 5] = float("nan")
    want[-3:, -group:, d - 1] = float("nan")
    got = out.view(q_len, hq, d)
    assert bool(((got == want) | (torch.isnan(got) & torch.isnan(want))).all())
    assert torch.equal(lse, clean_lse)
    v.view(torch.uint8)[row] = keep
    k.view(torch.uint8)[row, 0, 7] = 0x7f
    out, lse = eng.read_pages(q, plan, 0)
    got = out.view(q_len, hq, d)
    assert torch.equal(got[:-3], clean.view(q_len, hq, d)[:-3])
    assert torch.equal(got[:, group:], clean.view(q_len, hq, d)[:, group:])
    assert bool(torch.isnan(got[-3:, :group]).all() and torch.isnan(lse[:group, -3:]).all())
    assert torch.equal(lse[:, :-3], clean_lse[:, :-3])


def engine_arena(pages, hk=8, d=128, layers=1, dtype=FP8):
    return KVArena(layers, pages, PAGE, hk, d, dtype=dtype)


@pytest.mark.parametrize("attention_mode", ["unified", "tree"])
@pytest.mark.parametrize("kind", ["one question", "questions"])
def test_stage_runs_on_an_8_bit_arena(attention_mode, kind):
    """A whole stage of the small model (head_dim 64): documents behind a
    shared prefix, packed, borrowed and read through 8-bit pages. Its margins
    differ from a bf16 arena's by the codes' roundings (2^-4 of a value each,
    many of either sign): within 0.5 of margins that spread over several."""
    from quail_amd import readout as ro
    from quail_amd.executor import StageRun
    from quail_amd.model import CONFIGS, build_synthetic, retain_answer_head
    from quail_amd.qwen3 import Qwen3Pipeline
    from quail_amd.workload import make_workload

    wl = make_workload("tiny", seed=0)
    model = build_synthetic(CONFIGS["tiny"], seed=0, device="cuda", gen_device="cpu",
                            norm_init="random")
    cfg = model.config
    rng = np.random.default_rng(1)
    prefixes, suffixes = wl.groups_input()
    if kind == "questions":
        suffixes = [[rng.integers(0, 4096, int(n)) for n in rng.integers(2, 9, 3)]
                    for _ in prefixes]
    got = {}
    for dtype in (torch.bfloat16, FP8):
        arena = KVArena(cfg.layers, 3 * wl.chunk_budget // PAGE + 64, PAGE, cfg.kv_heads,
                        cfg.head_dim, dtype=dtype)
        retain_answer_head(model, wl.label_ids[:2])
        rows = ro.AnswerRows(model, [wl.label_ids[0]], [wl.label_ids[1]])
        run = StageRun(Qwen3Pipeline(model, arena), arena, ro.AsyncMargins(rows), prefixes,
                       suffixes, wl.chunk_budget // 4, attention_mode=attention_mode)
        results = run.run()
        torch.cuda.synchronize()
        assert run.stats["chunks"] > 1
        flat = [m for r in results for m in (r if isinstance(r, list) else [r])]
        got[dtype] = np.array([y - n for y, n in flat])
    off = np.abs(got[FP8] - got[torch.bfloat16])
    print("margins", got[torch.bfloat16].std(), "off", off.max(), np.sqrt((off ** 2).mean()))
    assert np.isfinite(got[FP8]).all()
    assert off.max() < 0.5 and off.max() > 0
