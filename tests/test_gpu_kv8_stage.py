"""A stage's own calls on an 8-bit arena at head_dim 128: K and V written
without q, then attention with q normed as it is loaded and its output
quantized, in packs as the stage lays them out."""

from dataclasses import replace

import numpy as np
import pytest
import torch

from oracle import kv8_ref as ref
from quail_amd.arena import FP8, KVArena
from tests.test_gpu_kv8 import (DEV, PAGE, _Attn, engine_arena, engine_of, fill, plan_of,
                                rope_cache)

pytestmark = pytest.mark.gpu


def packed(arena, groups, hq):
    from quail_amd.chunk import InputStaging, pack_chunk, upload
    hk, d = arena.kv_shape
    chunk = upload(pack_chunk(arena, groups, attention_heads=(hq, hk, d)), InputStaging())
    chunk.meta["layer"] = 0
    return chunk


def pack_of(kind, arena, rng, hq):
    """Documents with their questions (query tiles, several questions on a copied
    partial page among them), or a few rows each on kept documents."""
    groups = []
    sizes = dict(tiles=((130, (3,)), (47, (20, 9, 33)), (16, (1,)), (1, (40,))),
                 few=((300, (1,)), (1500, (2,)), (17, (1,)), (64, (2,))))[kind]
    for key, (f, suffixes) in enumerate(sizes):
        extra = suffixes[0] if len(suffixes) == 1 else 0
        assert arena.activate(key, f, capacity_tokens=f + extra) is not None
        groups.append(dict(key=key, prefix=rng.integers(0, 99, f) if kind == "tiles" else None, f=f,
                           suffixes=[rng.integers(0, 99, n) for n in suffixes]))
    return packed(arena, groups, hq)


@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["tiles", "few"])
@pytest.mark.parametrize("hq,hk", [(8, 8), (16, 8), (6, 2), (32, 8), (64, 8)])
def test_kv_norm_rope_then_attention_is_the_pass_then_attention_then_quant(hq, hk, kind, cache_dtype):
    """Pages bit for bit; over query tiles the quantized rows too. Over few
    rows q's sum of squares adds in another order: a q may be the next bf16
    (2^-7 of a score's products, and so of the weights), then a code is off
    by half a step of e4m3 on either side (2^-4, or 2^-10 of the scale)."""
    g = torch.Generator().manual_seed(61)
    d = 128
    arenas = [engine_arena(200, hk, d) for _ in range(2)]
    attn, cache = _Attn(d, g), rope_cache(4096, d, cache_dtype)
    got, want = [], []
    for arena, fused in zip(arenas, (True, False)):
        fill(arena, torch.Generator().manual_seed(62))
        chunk = pack_of(kind, arena, np.random.default_rng(1), hq)
        meta, n = chunk.meta, chunk.tokens
        assert (meta["unified"]["work_rows"] > 0) == (kind == "few")
        eng = engine_of(arena, hq, cache)
        gen = torch.Generator().manual_seed(63)
        qkv = torch.randn(n, (hq + 2 * hk) * d, generator=gen).to(torch.bfloat16).to(DEV)
        if fused:
            q = eng.kv_norm_rope(qkv, chunk.positions, attn, meta)
            assert q.data_ptr() == qkv.data_ptr()
            got = eng.attention_unified(q.view(n, hq, d), None, None, meta)
        else:
            q = eng.qk_norm_rope_kv(qkv, chunk.positions, attn, meta).view(n, hq, d)
            rows = eng.attention_bf16(q, meta, 0)
            want = eng.quant(rows)
        assert meta["layer"] == (1 if fused else 0)
    for a, b in zip((*arenas[0].layer_kv(0), arenas[0].layer_scales(0)),
                    (*arenas[1].layer_kv(0), arenas[1].layer_scales(0))):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    if kind == "tiles":
        assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))
        assert torch.equal(got[1], want[1])
        return
    u = chunk.meta["unified"]
    k, v = arenas[1].layer_kv(0)
    exact, _, size, reach = ref.attend(q, k, v, arenas[1].layer_scales(0), u["cu_q"].tolist(),
                                       u["used"].tolist(), u["table"].cpu().numpy(), True)
    scale = got[1].double()[:, :, None]
    values = got[0].double().view(n, hq, d) * scale
    off = 2.0 ** -7 * reach + 2 * (d + 8) * 2.0 ** -24 * reach
    row = (2.0 ** -8 + 2.0 ** -16 + torch.expm1(2 * off))[..., None] * size + 2.0 ** -8 * exact.abs()
    bound = row + 2.0 ** -4 * (exact.abs() + row) + 2.0 ** -10 * scale
    assert bool(((values - exact).abs() <= bound).all())


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (6, 2, 128), (24, 8, 64)])
@pytest.mark.parametrize("q_lens,used", [((1, 2, 1), (900, 20, 3000)), ((40, 70, 3), (90, 2000, 64))])
def test_rows_by_index_are_the_rows_in_order(hq, hk, d, q_lens, used):
    """Call B of tree packs reads its query rows through an index, not
    causally: bit for bit the rows in order."""
    g = torch.Generator().manual_seed(64)
    arena = engine_arena(sum(-(-u // PAGE) for u in used) + 3, hk, d)
    fill(arena, g)
    plan, cu_q, _, _ = plan_of(arena, hq, q_lens, used, g, causal=False)
    n = int(cu_q[-1])
    q = torch.randn(n + 9, hq, d, generator=g).to(torch.bfloat16).to(DEV)
    index = torch.randperm(n + 9, generator=g)[:n].to(DEV)
    eng = engine_of(arena, hq)
    want, want_lse = eng.read_pages(q[index], plan, 0)
    out, lse = torch.empty_like(want), torch.empty_like(want_lse)
    eng._attend8(q, plan, 0, d ** -0.5, q_index=index, out=out, lse=lse)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


def stage(model, wl, fuse_q_norm):
    from quail_amd import readout as ro
    from quail_amd.executor import StageRun
    from quail_amd.model import retain_answer_head
    from quail_amd.qwen3 import Qwen3Pipeline
    cfg = model.config
    arena = KVArena(cfg.layers, 3 * wl.chunk_budget // PAGE + 64, PAGE, cfg.kv_heads, cfg.head_dim,
                    dtype=FP8)
    arena.storage.view(torch.uint8).zero_()
    labels = list(wl.label_ids[:2])
    retain_answer_head(model, labels)
    pipe = Qwen3Pipeline(model, arena)
    assert pipe.fuse_q_norm
    pipe.fuse_q_norm = fuse_q_norm
    prefixes, suffixes = wl.groups_input()
    run = StageRun(pipe, arena, ro.AsyncMargins(ro.AnswerRows(model, labels[:1], labels[1:])),
                   prefixes, suffixes, wl.chunk_budget // 4)
    results = run.run()
    torch.cuda.synchronize()
    assert run.stats["chunks"] > 1 and run.stats["borrowed_tokens"] > 0
    return arena, np.array([y - n for y, n in results])


@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (8, 2), (2, 2)])
def test_a_head_dim_128_stage_with_q_norm_on_load(heads, kv_heads):
    """The whole stage with q normed on load against the stage whose pass
    norms it: every page of every layer bit for bit (layer 1's rows come out
    of layer 0's attention), and margins apart by less than the bound that
    every stage is held to against the oracle (only the last layer's
    few rows can differ, in a bf16 step of q)."""
    from quail_amd.model import CONFIGS, build_synthetic
    from quail_amd.workload import make_workload
    wl = make_workload("tiny", seed=0)
    cfg = replace(CONFIGS["tiny"], head_dim=128, heads=heads, kv_heads=kv_heads)
    model = build_synthetic(cfg, seed=0, device="cuda", gen_device="cpu", norm_init="random")
    (a, on_load), (b, by_pass) = (stage(model, wl, fuse) for fuse in (True, False))
    assert torch.equal(a.storage.view(torch.uint8), b.storage.view(torch.uint8))
    assert torch.equal(a.scales, b.scales)
    assert np.isfinite(on_load).all() and float(np.abs(on_load - by_pass).max()) <= 0.05
