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


def through_pages(x, cu):
    """float64 rows (n, HK, D) as 8-bit pages of each sequence hold them."""
    out = x.double().clone()
    for r0, r1 in zip(cu[:-1], cu[1:]):
        for p in range(int(r0), int(r1), PAGE):
            rows = out[p:min(p + PAGE, int(r1))]
            b = torch.tensor([ref.scale_byte(float(a)) for a in rows.abs().amax((0, 2))])[None, :, None]
            rows.copy_(ref.codes_of(rows, b).double() * torch.exp2(b.double() - 127))
    return out


@pytest.mark.parametrize("attention_mode", ["unified", "tree"])
@pytest.mark.parametrize("kind", ["one question", "questions"])
def test_stage_runs_on_an_8_bit_arena(attention_mode, kind, monkeypatch):
    """A whole stage of the small model (head_dim 64): documents behind a
    shared prefix, packed, borrowed and read through 8-bit pages, against the
    oracle's pass over each prompt with its K and V rounded as pages hold
    them. How far the codes move a margin at all is what the oracle says with
    and without them; the engine's other roundings flip some codes (a K or V
    that a bf16 rounding moves by 2^-8 changes its code once in 16 times), so
    it is held to less than that, not to the 16-bit pages' bound. (The tree
    path reads a pack's own rows unrounded.)"""
    from oracle import qwen3_ref
    from quail_amd import readout as ro
    from quail_amd.executor import StageRun
    from quail_amd.model import CONFIGS, build_synthetic, retain_answer_head
    from quail_amd.qwen3 import Qwen3Pipeline
    from quail_amd.workload import make_workload
    from tests.helpers import ref_model

    wl = make_workload("tiny", seed=0)
    model = build_synthetic(CONFIGS["tiny"], seed=0, device="cuda", gen_device="cpu",
                            norm_init="random")
    cfg = model.config
    rng = np.random.default_rng(1)
    prefixes, suffixes = wl.groups_input()
    if kind == "questions":
        suffixes = [[rng.integers(0, 4096, int(n)) for n in rng.integers(2, 9, 3)]
                    for _ in prefixes]
    arena = KVArena(cfg.layers, 3 * wl.chunk_budget // PAGE + 64, PAGE, cfg.kv_heads,
                    cfg.head_dim, dtype=FP8)
    labels = list(wl.label_ids[:2])
    retain_answer_head(model, labels)
    rows = ro.AnswerRows(model, labels[:1], labels[1:])
    run = StageRun(Qwen3Pipeline(model, arena), arena, ro.AsyncMargins(rows), prefixes, suffixes,
                   wl.chunk_budget // 4, attention_mode=attention_mode)
    results = run.run()
    torch.cuda.synchronize()
    assert run.stats["chunks"] > 1 and run.stats["borrowed_tokens"] > 0
    got = np.array([y - n for r in results for y, n in (r if isinstance(r, list) else [r])])
    prompts = [np.concatenate([p, s]) for p, sufs in zip(prefixes, suffixes) for s in sufs]
    m = ref_model(model)

    def margins():
        normed = qwen3_ref.forward_documents(m, prompts)
        yes, no, _, _ = qwen3_ref.answer(normed, m.head[labels], [1, 0])
        return (yes - no).double().numpy()

    plain = margins()
    exact = qwen3_ref.varlen_attention
    monkeypatch.setattr(qwen3_ref, "varlen_attention", lambda q, k, v, cu: exact(
        q, through_pages(k, cu), through_pages(v, cu), cu))
    paged = margins()
    codes = float(np.sqrt(((paged - plain) ** 2).mean()))
    off = got - (paged if attention_mode == "unified" else plain)
    print("codes move margins by", codes, "engine off", np.sqrt((off ** 2).mean()), abs(off).max())
    assert float(np.sqrt((off ** 2).mean())) <= 2 ** 0.5 * codes
    assert float(np.abs(off).max()) <= 4 * 2 ** 0.5 * codes


def plan_of(arena, hq, q_lens, used, g, causal=True):
    from quail_amd.chunk import attention_plan
    pages = arena.num_pages
    cu_q, u, table = sequences(g, q_lens, used, pages)
    hk, d = arena.kv_shape
    plan = attention_plan(*(torch.from_numpy(a).to(DEV) for a in (cu_q, u, table)),
                          heads=(hq, hk, d), causal=causal)
    return plan, cu_q, u, table


@pytest.mark.parametrize("q_lens,used", [((1, 2), (300, 1500)), ((40, 70), (40, 200))])
def test_o_proj_input_is_the_quantized_rows(q_lens, used):
    """The fused e4m3 output is the group quant of the bf16 rows, bit for bit
    (D = 128), through the engine's unified attention."""
    g = torch.Generator().manual_seed(11)
    arena = engine_arena(200)
    fill(arena, g)
    plan, cu_q, _, _ = plan_of(arena, 32, q_lens, used, g)
    eng = engine_of(arena, 32)
    q = torch.randn(int(cu_q[-1]), 32, 128, generator=g).to(torch.bfloat16).to(DEV)
    out, _ = eng.read_pages(q, plan, 0)
    want_q, want_s = eng.quant(out)
    got_q, got_s = eng._paged(q, plan, 0, None, None)
    assert torch.equal(got_q.view(torch.uint8), want_q.view(torch.uint8))
    assert torch.equal(got_s, want_s)


@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_lens,used", [((1, 3, 1), (300, 1500, 7)), ((40, 70, 1), (40, 200, 90)),
                                         ((12,), (9000,))])
def test_q_norm_on_load_is_the_pass_then_the_attention(q_lens, used, cache_dtype):
    """The projection's q, normed and rotated as the attention loads it, gives
    what the pass's bf16 q gives: bit for bit over query tiles (one sum
    tree); over few rows the sum of squares adds in another order, so a q may
    be the next bf16: 2^-7 of a score's products, and of the weights."""
    g = torch.Generator().manual_seed(21)
    hq, hk, d = 32, 8, 128
    arena = engine_arena(1000)
    fill(arena, g)
    attn, cache = _Attn(d, g), rope_cache(10000, d, cache_dtype)
    eng = engine_of(arena, hq, cache)
    plan, cu_q, u, table = plan_of(arena, hq, q_lens, used, g)
    n = int(cu_q[-1])
    qkv = torch.randn(n, 48 * d, generator=g).to(torch.bfloat16).to(DEV)
    pos = torch.cat([torch.arange(b - a, b) for a, b in zip(q_lens, used)]).clamp(min=0).to(DEV)
    normed, _ = eng.qk_norm_rope(qkv, pos, attn)
    want, want_lse = eng.read_pages(normed.view(n, hq, d), plan, 0)
    got, lse = torch.empty_like(want), torch.empty_like(want_lse)
    eng._attend8(qkv[:, :hq * d].view(n, hq, d), plan, 0, d ** -0.5, out=got, lse=lse,
                 qnorm=(pos, attn))
    if plan["work_rows"] <= 0:
        assert torch.equal(got, want) and torch.equal(lse, want_lse)
    else:
        k, v = arena.layer_kv(0)
        _, _, size, reach = ref.attend(normed.view(n, hq, d), k, v, arena.layer_scales(0),
                                       cu_q.tolist(), u.tolist(), table, True)
        off = 2.0 ** -7 * reach
        assert bool(((lse - want_lse).abs().t() <= off + 1e-5).all())
        bound = 2 * (2.0 ** -7 + torch.expm1(2 * off))[..., None] * size
        assert bool(((got.float() - want.float()).abs().view(n, hq, d) <= bound).all())
    with pytest.raises(ValueError, match="positions"):
        eng._attend8(qkv[:, :hq * d].view(n, hq, d), plan, 0, d ** -0.5, out=got, lse=lse,
                     qnorm=(pos[1:], attn))


def test_rows_do_not_depend_on_the_list_or_on_padding_columns():
    """A plan without its list of items, a table of more columns than the
    sequences have pages, query rows that are columns of wider rows: the same
    rows; and rows behind the last sequence stay as they were."""
    g = torch.Generator().manual_seed(12)
    arena = engine_arena(300)
    fill(arena, g)
    eng = engine_of(arena, 32)
    for q_lens, used in (((40, 3, 65), (700, 64, 65)), ((1, 2, 1), (900, 5, 64))):
        plan, cu_q, u, table = plan_of(arena, 32, q_lens, used, g)
        n = int(cu_q[-1])
        wide = torch.randn(n + 2, 48 * 128, generator=g).to(torch.bfloat16).to(DEV)
        q = wide[:n, 128 * 8:128 * 40].view(n, 32, 128)
        out, lse = eng.read_pages(q, plan, 0)
        again, lse2 = eng.read_pages(q.contiguous(), plan, 0)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
        bare = {k: v for k, v in plan.items() if not k.startswith(("work", "n_work"))}
        bare["table"] = torch.cat([plan["table"], torch.full((len(used), 7), 1 << 30,
                                                             dtype=torch.int32, device=DEV)], 1)
        other, lse3 = eng.read_pages(q, bare, 0)
        # another split of the keys sums in another order: each within the
        # bound of the exact rows
        check_rows(out, lse, q, arena, cu_q, u, table, True)
        check_rows(other, lse3, q, arena, cu_q, u, table, True)
        padded = torch.cat([q, q[:2]])
        tail = torch.full((n + 2, 32 * 128), 7.0, dtype=torch.bfloat16, device=DEV)
        tail_lse = torch.full((32, n + 2), 7.0, device=DEV)
        eng._attend8(padded, plan, 0, 128 ** -0.5, out=tail, lse=tail_lse)
        assert torch.equal(tail[:n], out) and torch.equal(tail_lse[:, :n], lse)
        assert bool((tail[n:] == 7).all() and (tail_lse[:, n:] == 7).all())


def test_pools_past_32_bit_offsets():
    """Pages whose codes lie past 4 GiB of a pool: written, read and copied."""
    pages = 270000                                   # 16 KiB a page and pool: 4.4 GB
    arena = engine_arena(pages)
    g = torch.Generator().manual_seed(13)
    far = [pages - 1, pages - 7, 3, pages - 20, 262143, 262144]
    n = 16 * len(far)
    qkv = torch.randn(n, 48 * 128, generator=g).to(torch.bfloat16).to(DEV)
    attn = _Attn(128, g)
    cache = rope_cache(n, 128, torch.bfloat16)
    eng = engine_of(arena, 32, cache)
    items = torch.tensor([(p, p, 0, 16 * i, 16) for i, p in enumerate(far)], dtype=torch.int32,
                         device=DEV)
    q = eng.qk_norm_rope_kv(qkv, torch.arange(n, device=DEV), attn,
                            dict(layer=0, unified=dict(page_writes=(items,))))
    small = engine_arena(len(far))
    here = torch.tensor([(i, i, 0, 16 * i, 16) for i in range(len(far))], dtype=torch.int32,
                        device=DEV)
    eng2 = engine_of(small, 32, cache)
    q2 = eng2.qk_norm_rope_kv(qkv, torch.arange(n, device=DEV), attn,
                              dict(layer=0, unified=dict(page_writes=(here,))))
    assert torch.equal(q, q2)
    from quail_amd.chunk import attention_plan
    ints = lambda *a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    for rows in (1, n):
        plans = [attention_plan(ints(0, rows), ints(n), ints(*t).view(1, -1), heads=(32, 8, 128))
                 for t in (far, range(len(far)))]
        a = eng.read_pages(q[:rows].view(rows, 32, 128), plans[0], 0)
        b = eng2.read_pages(q[:rows].view(rows, 32, 128), plans[1], 0)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    arena.copy_pages([pages - 1, 3], [pages - 2, 11])
    k, v = arena.paged_kv(0)
    for src, dst in ((pages - 1, pages - 2), (3, 11)):
        assert same_codes(k[src], k[dst]) and same_codes(v[src], v[dst])
        assert torch.equal(arena.layer_scales(0)[src], arena.layer_scales(0)[dst])


def test_tokens_appended_one_by_one_read_as_a_whole_write_does():
    """Single-token decoding: each token's K and V appended to its sequence's
    last page, then its row attends. A page's scale only grows while it
    fills, so its codes end as one write's, but for what was rounded under a
    smaller scale and became subnormal: within 2^-9 of the page's scale."""
    g = torch.Generator().manual_seed(14)
    hq, hk, d, seqs, steps = 32, 8, 128, 5, 37
    arena, whole = engine_arena(40), engine_arena(40)
    for a in (arena, whole):        # what the rows before each start hold
        fill(a, torch.Generator().manual_seed(140))
    attn, cache = _Attn(d, g), rope_cache(200, d, torch.bfloat16)
    eng = engine_of(arena, hq, cache)
    tables = torch.randperm(40, generator=g)[:35].view(seqs, 7).to(torch.int32)
    start = [0, 3, 15, 16, 40]
    size = torch.exp2(torch.randn(seqs, steps, 1, generator=g) * 2)
    qkv = (torch.randn(seqs, steps, 48 * d, generator=g) * size).to(torch.bfloat16).to(DEV)
    from quail_amd.chunk import attention_plan, page_writes
    used = list(start)
    for t in range(steps):
        pos = np.array(used)
        dst = np.array([int(tables[s, p // PAGE]) * PAGE + p % PAGE for s, p in enumerate(used)])
        phases = page_writes(np.arange(seqs), dst)
        meta = dict(layer=0, unified=dict(page_writes=tuple(torch.from_numpy(p).to(DEV)
                                                            for p in phases)))
        q = eng.qk_norm_rope_kv(qkv[:, t], torch.from_numpy(pos).to(DEV), attn, meta)
        used = [u + 1 for u in used]
    rows = np.concatenate([[int(tables[s, (start[s] + t) // PAGE]) * PAGE + (start[s] + t) % PAGE
                            for t in range(steps)] for s in range(seqs)])
    pos = np.concatenate([start[s] + np.arange(steps) for s in range(seqs)])
    phases = page_writes(np.arange(seqs * steps), rows)
    assert len(phases) == 1
    one = engine_of(whole, hq, cache)
    one.qk_norm_rope_kv(qkv.reshape(seqs * steps, -1), torch.from_numpy(pos).to(DEV), attn,
                        dict(layer=0, unified=dict(page_writes=(torch.from_numpy(
                            phases[0]).to(DEV),))))
    at = torch.from_numpy(rows).to(DEV)
    # pages that began empty hold the same rows either way
    full = torch.from_numpy(np.isin(rows // PAGE, [int(tables[s, p]) for s in range(seqs)
                                                   for p in range(-(-start[s] // PAGE), 7)])).to(DEV)
    for side in (0, 1):
        a = ref.values(arena.layer_kv(0)[side], arena.layer_scales(0), side)[at][full]
        b = ref.values(whole.layer_kv(0)[side], whole.layer_scales(0), side)[at][full]
        scale = torch.exp2(whole.layer_scales(0)[:, :, side].double() - 127)
        scale = scale.repeat_interleave(PAGE, 0)[at][full][..., None]
        assert bool(((a - b).abs() <= 2.0 ** -9 * scale).all())
        assert torch.equal(arena.layer_scales(0)[:, :, side][at[full] // PAGE],
                           whole.layer_scales(0)[:, :, side][at[full] // PAGE])
    # the last token's rows against the definition
    plan = attention_plan(torch.arange(seqs + 1, dtype=torch.int32, device=DEV),
                          torch.tensor(used, dtype=torch.int32, device=DEV), tables.to(DEV),
                          heads=(hq, hk, d))
    out, lse = eng.read_pages(q.view(seqs, hq, d), plan, 0)
    check_rows(out, lse, q.view(seqs, hq, d), arena, np.arange(seqs + 1), np.array(used),
               tables.numpy(), True)


def test_forks_continue_apart_and_compaction_keeps_what_they_read():
    """A document of 40 tokens, forked twice (borrowed full pages, its partial
    page copied in every layer), the forks continued with different tokens;
    then freed neighbours, compaction, and the same rows read again."""
    from quail_amd.chunk import attention_plan, page_writes
    g = torch.Generator().manual_seed(15)
    hq, hk, d, layers = 32, 8, 128, 3
    arena = KVArena(layers, 30, PAGE, hk, d, dtype=FP8)
    attn, cache = _Attn(d, g), rope_cache(100, d, torch.bfloat16)
    eng = engine_of(arena, hq, cache)

    def append(key, first, qkv):
        """Write qkv's rows at the key's slots first.. in every layer."""
        rows = arena.capacity_rows(key)[first:first + len(qkv)]
        phases = tuple(torch.from_numpy(p).to(DEV)
                       for p in page_writes(np.arange(len(qkv)), rows))
        pos = torch.arange(first, first + len(qkv), device=DEV)
        return [eng.qk_norm_rope_kv(qkv * (layer + 1), pos, attn, dict(
            layer=layer, unified=dict(page_writes=phases))) for layer in range(layers)]

    def read(key, tokens, q):
        table = torch.tensor([arena.owned_pages(key)], dtype=torch.int32, device=DEV)
        ints = lambda *a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
        plan = attention_plan(ints(0, len(q)), ints(tokens), table, heads=(hq, hk, d))
        return torch.stack([eng.read_pages(q.view(-1, hq, d), plan, layer)[0]
                            for layer in range(layers)])

    rows = lambda n: torch.randn(n, 48 * d, generator=g).to(torch.bfloat16).to(DEV)  # noqa: E731
    for k, n in (("hole1", 50), ("doc", 40), ("hole2", 33), ("straight a", 60), ("straight b", 60)):
        arena.alloc(k, n, capacity_tokens=n)
    doc, a, b = rows(40), rows(20), rows(9)
    append("doc", 0, doc)
    pages = arena.fork("doc", ["a", "b"], capacity_tokens=60)
    assert [len(p) for p in pages] == [2, 2]
    qa, qb = append("a", 40, a), append("b", 40, b)
    got = read("a", 60, qa[0]), read("b", 49, qb[0]), read("doc", 40, qa[0][:4])
    # the same tokens written straight
    for key, more in (("straight a", a), ("straight b", b)):
        append(key, 0, doc)
        append(key, 40, more)
    assert torch.equal(got[0], read("straight a", 60, qa[0]))
    assert torch.equal(got[1], read("straight b", 49, qb[0]))
    for k in ("hole1", "hole2", "straight a"):
        arena.free_key(k)
    before = {k: arena.owned_pages(k) for k in ("doc", "a", "b", "straight b")}
    assert arena.compact() > 0
    after = {k: arena.owned_pages(k) for k in before}
    assert after != before
    live = {p for pages in after.values() for p in pages}
    assert live == set(range(len(live)))
    assert torch.equal(read("a", 60, qa[0]), got[0])
    assert torch.equal(read("b", 49, qb[0]), got[1])
    assert torch.equal(read("doc", 40, qa[0][:4]), got[2])
    arena.free_key("doc")
    assert torch.equal(read("a", 60, qa[0]), got[0])      # its borrowed pages stay


def test_captured_calls_replay_with_eager_work_between_and_streams_run_apart():
    """A write, a split attention and a page copy captured into one graph,
    replayed with other inputs and eager calls between; and two streams at
    once, each with its own workspace."""
    g = torch.Generator().manual_seed(16)
    arena = engine_arena(700)
    fill(arena, g)
    attn, cache = _Attn(128, g), rope_cache(10000, 128, torch.bfloat16)
    eng = engine_of(arena, 32, cache)
    plan, cu_q, u, table = plan_of(arena, 32, (1, 1, 1), (2000, 4000, 9), g)
    assert plan["work_rows"] > 0
    end = [(int(table[s, (n - 1) // PAGE]), (n - 1) % PAGE) for s, n in enumerate(u)]
    items = torch.tensor([(p, p, r, s, 1) for s, (p, r) in enumerate(end)], dtype=torch.int32,
                         device=DEV)
    pos = torch.tensor([int(n) - 1 for n in u], dtype=torch.int64, device=DEV)
    spare = sorted(set(range(700)) - set(table.reshape(-1).tolist()))[:2]
    qkv = torch.randn(3, 48 * 128, generator=g).to(torch.bfloat16).to(DEV)

    def once(x):
        q = eng.qk_norm_rope_kv(x, pos, attn, dict(layer=0, unified=dict(page_writes=(items,))))
        out = eng.read_pages(q.view(3, 32, 128), plan, 0)
        arena.copy_pages([end[0][0], end[1][0]], spare)
        return out

    state = [t.clone() for t in (arena.storage, arena.scales)]

    def reset():
        for t, s in zip((arena.storage, arena.scales), state):
            t.view(torch.uint8).copy_(s.view(torch.uint8))

    once(qkv)
    reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once(qkv)
    for i in range(4):
        x = torch.randn(3, 48 * 128, generator=g).to(torch.bfloat16).to(DEV)
        reset()
        want = [t.clone() for t in once(x)]
        pools = [t.clone() for t in (arena.storage, arena.scales)]
        reset()
        qkv.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*held, arena.storage, arena.scales), (*want, *pools)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    # two streams, many calls in flight
    q = torch.randn(3, 32, 128, generator=g).to(torch.bfloat16).to(DEV)
    want = [eng.read_pages(x, plan, 0) for x in (q, q * 2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(eng.read_pages(q if i == 0 else q * 2, plan, 0))
    torch.cuda.synchronize()
    for i in (0, 1):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


def test_the_engine_refuses_what_8_bit_pages_do_not_take():
    arena = engine_arena(4)
    eng = engine_of(arena, 32)
    rows = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="page items"):
        eng.kv_row_scatter(rows, rows, torch.zeros(1, dtype=torch.int64, device=DEV),
                           torch.zeros(1, dtype=torch.int64, device=DEV), 0)
    items = torch.zeros(1, 5, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="bf16"):
        eng._write_page_rows(rows.half(), rows, (items,), 0)
    with pytest.raises(ValueError, match="int32"):
        eng._write_page_rows(rows, rows, (items.long(),), 0)
    attn = _Attn(128, torch.Generator().manual_seed(1))
    rope = engine_of(arena, 32, rope_cache(8, 128, torch.bfloat16))
    qkv = torch.zeros(1, 48 * 128, dtype=torch.bfloat16, device=DEV)
    where = torch.zeros(1, dtype=torch.int64, device=DEV)
    meta = dict(layer=0, unified=dict(page_writes=(items,)))
    for bad_qkv, bad_pos, match in ((qkv, where.int(), "positions"), (qkv, where[:0], "positions"),
                                    (qkv.half(), where, "bf16"), (qkv[:, :-8], where, "width")):
        with pytest.raises(ValueError, match=match):
            rope.qk_norm_rope_kv(bad_qkv, bad_pos, attn, dict(meta))
    from quail_amd.chunk import attention_plan
    ints = lambda *a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    plan = attention_plan(ints(0, 1), ints(20), ints(1, 2).view(1, 2), heads=(32, 8, 128))
    q = torch.zeros(1, 32, 128, dtype=torch.bfloat16, device=DEV)
    for bad in (q.half(), q[:, :16], torch.zeros(1, 32, 64, dtype=torch.bfloat16, device=DEV)):
        with pytest.raises(ValueError, match="query rows"):
            eng.read_pages(bad, plan, 0)
    with pytest.raises(ValueError, match="contiguous"):
        eng.read_pages(torch.zeros(1, 128, 32, dtype=torch.bfloat16, device=DEV).mT, plan, 0)
    for args, match in (((ints(0, 1), ints(33), ints(1, 2).view(1, 2)), "keys"),
                        ((ints(0, 1), ints(3, 4), ints(1, 2).view(1, 2)), "sequences"),
                        ((ints(1, 2), ints(3), ints(1, 2).view(1, 2)), "rises"),
                        ((ints(0, 1), ints(-1), ints(1, 2).view(1, 2)), "negative"),
                        ((ints(0, 1).long(), ints(3), ints(1, 2).view(1, 2)), "int32")):
        with pytest.raises(ValueError, match=match):
            attention_plan(*args, heads=(32, 8, 128))
    for src, dst in (([0], [4]), ([0, 1], [2, 2]), ([0, 1], [1, 2])):
        with pytest.raises(ValueError):
            arena.copy_pages(src, dst)
    out, lse = eng.read_pages(q[:0], attention_plan(ints(0), ints(), torch.zeros(
        0, 1, dtype=torch.int32, device=DEV), heads=(32, 8, 128)), 0)
    assert out.shape == (0, 4096) and lse.shape == (32, 0)


def test_read_pages_refuses_a_plan_made_for_other_rows_heads_or_pages():
    from quail_amd.chunk import attention_plan
    arena = engine_arena(4)
    eng = engine_of(arena, 32)
    ints = lambda *a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    where = ints(0, 2), ints(20), ints(1, 2).view(1, 2)
    q = torch.zeros(2, 32, 128, dtype=torch.bfloat16, device=DEV)
    for rows, heads, eight_bit in ((1, (32, 8, 128), True), (2, (16, 8, 128), True),
                                   (2, (32, 8, 128), False)):
        plan = attention_plan(*where, heads=heads, eight_bit=eight_bit)
        with pytest.raises(ValueError, match="a plan for"):
            eng.read_pages(q[:rows], plan, 0)
    with pytest.raises(ValueError, match="of 4"):
        arena.copy_pages([0], [(1 << 32) + 1])
    rows = torch.zeros(1, 8, 256, dtype=torch.bfloat16, device=DEV)[:, :, :128]
    with pytest.raises(ValueError, match="contiguous"):
        eng._write_page_rows(rows, rows, (torch.zeros(1, 5, dtype=torch.int32, device=DEV),), 0)


def test_a_long_sequence_of_many_heads_per_kv_head():
    """40,000 rows at 16 heads a KV head: more rows than few-row blocks fit
    in a grid. The last rows against float64; the rest finite."""
    from quail_amd.chunk import attention_plan
    hq, hk, d, n = 128, 8, 64, 40000
    pages = -(-n // PAGE)
    arena = KVArena(1, pages, PAGE, hk, d, dtype=FP8)
    g = torch.Generator().manual_seed(31)
    fill(arena, g)
    cu_q, used, table = sequences(g, [n], [n], pages)
    q = torch.randn(n, hq, d, generator=g).to(torch.bfloat16).to(DEV)
    plan = attention_plan(*(torch.from_numpy(a).to(DEV) for a in (cu_q, used, table)),
                          heads=(hq, hk, d))
    out, lse = engine_of(arena, hq).read_pages(q, plan, 0)
    assert bool(torch.isfinite(out).all())
    last = np.asarray([0, 3], dtype=np.int32)
    check_rows(out[-3:], lse[:, -3:], q[-3:], arena, last, used, table, True)


def test_read_pages_refuses_pages_that_the_arena_does_not_have():
    from quail_amd.chunk import attention_plan
    arena = engine_arena(4)
    fill(arena, torch.Generator().manual_seed(5))    # a new arena holds any bytes, NaN codes too
    eng = engine_of(arena, 32)
    ints = lambda *a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    q = torch.zeros(1, 32, 128, dtype=torch.bfloat16, device=DEV)
    plan = attention_plan(ints(0, 1), ints(20), ints(3, 4).view(1, 2), heads=(32, 8, 128))
    with pytest.raises(ValueError, match="page 4"):
        eng.read_pages(q, plan, 0)
    plan = attention_plan(ints(0, 1), ints(16), ints(3, 4).view(1, 2), heads=(32, 8, 128))
    assert bool(torch.isfinite(eng.read_pages(q, plan, 0)[0]).all())


@pytest.mark.parametrize("v_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (4, 2, 64)])
@pytest.mark.parametrize("q_lens,used,causal", [((1, 1, 3), (300, 17, 64), True),
                                                ((40, 21, 1), (90, 500, 33), True),
                                                ((70, 2), (40, 1100), False)])
def test_read_pages_of_a_16_bit_arena(v_dtype, hq, hk, d, q_lens, used, causal):
    """The same call over bf16 K and 16-bit V: the oracle's codes are the
    values, its scales 1; P is rounded to V's type (2^-8 at most)."""
    from types import SimpleNamespace

    from quail_amd.chunk import attention_plan
    g = torch.Generator().manual_seed(41)
    pages = sum(-(-u // PAGE) for u in used) + 3
    arena = KVArena(1, pages, PAGE, hk, d, v_dtype=v_dtype)
    for pool in arena.layer_kv(0):
        pool.copy_(torch.randn(pool.shape, generator=g))
    cu_q, used, table = sequences(g, q_lens, used, pages)
    q = torch.randn(int(cu_q[-1]), hq, d, generator=g).to(torch.bfloat16).to(DEV)
    plan = attention_plan(*(torch.from_numpy(a).to(DEV) for a in (cu_q, used, table)),
                          heads=(hq, hk, d), causal=causal, eight_bit=False)
    out, lse = engine_of(arena, hq).read_pages(q, plan, 0)
    ones = torch.full((pages, hk, 2), 127, dtype=torch.uint8, device=DEV)
    same = SimpleNamespace(layer_kv=arena.layer_kv, layer_scales=lambda layer: ones)
    check_rows(out, lse, q, same, cu_q, used, table, causal)
