"""The operators of a KV arena that keeps K and V in 8 bits, as cases to measure.

Pages hold 16 tokens. A page's codes are e4m3, with one power-of-two scale
per (page, KV head), K's and V's apart, held as an E8M0 byte b that stands
for 2^(b - 127). Three operators:

  write   the qkv projection's rows: q through its norm and RoPE, K through its
          norm and RoPE into pages, V into pages. Each item is one page:
          (destination page, source page, kept rows, first row, rows); the
          kept rows are the source page's first ones, the fresh rows follow.
  attend  varlen grouped-query attention over such pages through a block
          table, bf16 rows and their log-sum-exps.
  pages   pages copied to other pages in every layer's pools.

With `own` false each runs in its plain form, elementary torch operations in
32 bits; with `own` true through the framework's Engine and KVArena.
"""

import math
import random
from types import SimpleNamespace

import numpy as np
import torch

own = False

PAGE = 16
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # one more token for each of 8 sequences whose last pages are part full
        dict(name="write-append-8", kind="write", hq=32, hk=8, d=128, seqs=8, lo=1, hi=1,
             median=1, at="ragged", lengths=1),
        # a small model's pack of short documents, head_dim 64
        dict(name="write-tiny-pack", kind="write", hq=4, hk=2, d=64, seqs=16, lo=16, hi=128,
             median=60, at="pages", lengths=3),
        # a whole AI.IF pack of Qwen3-4B: lognormal documents behind a 64-token prefix
        dict(name="write-if-pack", kind="write", hq=32, hk=8, d=128, seqs=46, lo=32, hi=2048,
             median=256, at="pages", lengths=4),
        # the last layer's one row of a short document
        dict(name="attend-one-row", kind="attend", hq=32, hk=8, d=128, seqs=1, q=1, lo=300, hi=300,
             median=300, prefix=64, causal=True, lengths=5),
        # the last layer's final rows of a pack of AI.IF documents
        dict(name="attend-final-46", kind="attend", hq=32, hk=8, d=128, seqs=46, q=1, lo=32, hi=2048,
             median=256, prefix=64, causal=True, lengths=4),
        # final rows of long AI.CLASSIFY documents
        dict(name="attend-final-200-long", kind="attend", hq=32, hk=8, d=128, seqs=200, q=1, lo=256,
             hi=8192, median=1500, prefix=96, causal=True, lengths=6),
        # two whole contexts, 64 heads, a few rows each
        dict(name="attend-contexts", kind="attend", hq=64, hk=8, d=128, seqs=2, q=3, lo=39999,
             hi=39999, median=39999, prefix=0, causal=True, lengths=7),
        # questions on kept documents, the tree path's reads
        dict(name="attend-questions", kind="attend", hq=32, hk=8, d=128, seqs=60, q=21, lo=200,
             hi=2000, median=900, prefix=64, causal=False, lengths=8),
        # every row of an AI.IF pack
        dict(name="attend-if-pack", kind="attend", hq=32, hk=8, d=128, seqs=46, q=0, lo=32, hi=2048,
             median=256, prefix=64, causal=True, lengths=4),
        # two long documents, every row
        dict(name="attend-long-rows", kind="attend", hq=32, hk=8, d=128, seqs=2, q=0, lo=7999,
             hi=8003, median=8001, prefix=96, causal=True, lengths=9),
        # forks' last pages, and half of an arena moved, in 36 layers
        dict(name="pages-fork-37", kind="pages", layers=36, hk=8, d=128, pages=512, moved=37,
             lengths=10),
        dict(name="pages-compact-1000", kind="pages", layers=36, hk=8, d=128, pages=2048, moved=1000,
             lengths=11),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "write", "attend", "attend", "attend", "attend", "pages"])
    seed = rng.randrange(1 << 30)
    if kind == "pages":
        pages = _spread(rng, 40, 2000)
        return dict(kind=kind, layers=rng.choice([2, 7, 36]), hk=rng.choice([2, 4, 8]),
                    d=rng.choice([64, 128]), pages=pages, moved=rng.randint(1, pages // 2),
                    lengths=seed)
    hq, hk, d = rng.choice([(32, 8, 128), (32, 8, 128), (64, 8, 128), (16, 8, 128), (8, 8, 128),
                            (4, 2, 64), (24, 8, 64)])
    if kind == "write":
        rows = _spread(rng, 1, 7000)
        seqs = _spread(rng, 1, min(rows, 400))
        median = max(1, rows // seqs)
        return dict(kind=kind, hq=hq, hk=hk, d=d, seqs=seqs, lo=max(1, median // 4),
                    hi=min(2 * median, 4000), median=median, at=rng.choice(["ragged", "pages"]),
                    lengths=seed)
    shape = rng.choice(["few", "few", "questions", "rows"])
    prefix = rng.choice([0, 16, 64, 96])
    if shape == "few":
        median = _spread(rng, 1, 20000)
        seqs = _spread(rng, 1, max(1, min(256, 200000 // median)))
        q = rng.choice([1, 1, 1, 2, 5])
    elif shape == "questions":
        median, seqs, q = _spread(rng, 30, 2000), _spread(rng, 1, 60), _spread(rng, 6, 100)
    else:
        median = _spread(rng, 1, 2700)
        seqs, q = _spread(rng, 1, max(1, min(40, 5400 // median))), 0
    return dict(kind="attend", hq=hq, hk=hk, d=d, seqs=seqs, q=q, lo=max(1, median // 4),
                hi=min(2 * median, 39000), median=median, prefix=prefix,
                causal=True if q == 0 else rng.choice([True, False]), lengths=seed)


def _lengths(case):
    """Tokens of each sequence: lognormal about the median, within [lo, hi]."""
    rng = random.Random(case["lengths"])
    return [min(case["hi"], max(case["lo"], int(rng.lognormvariate(math.log(case["median"]), 0.8))))
            for _ in range(case["seqs"])]


def _write_items(case):
    """The page items of a write, and the position of each row."""
    rng = random.Random(case["lengths"] + 1)
    items, positions, row, page = [], [], 0, 0
    for n in _lengths(case):
        start = 64 if case["at"] == "pages" else rng.randint(0, 500)
        positions += range(start, start + n)
        at, end = start, start + n
        while at < end:
            count = min(PAGE - at % PAGE, end - at)
            items.append((page, page, at % PAGE, row, count))
            page, row, at = page + 1, row + count, at + count
    order = list(range(page))
    rng.shuffle(order)
    return [(order[p], order[p], k, r, c) for p, _, k, r, c in items], positions


def _sequences(case):
    """(query rows, keys) of each sequence of an attention."""
    return [(n if case["q"] == 0 else case["q"],
             case["prefix"] + (n if case["q"] == 0 else max(n, case["q"])))
            for n in _lengths(case)]


def work(case):
    if case["kind"] == "pages":
        page = 2 * case["layers"] * case["hk"] * (PAGE * case["d"] + 1)
        return {"bytes": 2 * case["moved"] * page, "flops": 0}
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["kind"] == "write":
        items, positions = _write_items(case)
        rows = len(positions)
        kept = sum(k for _, _, k, _, _ in items)
        return {"bytes": rows * d * (2 * (2 * hq + 2 * hk) + 2 * hk) + kept * 2 * hk * d
                + 2 * hk * len(items) + 16 * len(items), "flops": 12 * rows * (hq + hk) * d}
    pairs = keys = rows = 0
    shared = case["prefix"] // PAGE * PAGE
    for q, used in _sequences(case):
        pairs += q * used - (q * (q - 1) // 2 if case["causal"] else 0)
        keys, rows = keys + used - shared, rows + q
    keys += shared
    return {"bytes": rows * hq * (4 * d + 4) + keys * 2 * hk * d + 2 * hk * (keys // PAGE),
            "flops": 4 * hq * d * pairs}


def _byte(amax):
    """The least E8M0 byte b with amax <= 448 * 2^(b - 127), at least 1."""
    mantissa, exponent = torch.frexp(amax)          # amax = mantissa * 2^exponent, in [0.5, 1)
    b = exponent + 127 - 9 + (mantissa > 0.875).to(exponent.dtype)
    return torch.where(amax > 0, b, torch.ones_like(b)).clamp(min=1)


def _quantized(x, dims):
    b = _byte(x.abs().amax(dims, keepdim=True))
    return (x * torch.exp2((127 - b).to(x.dtype))).clamp(-FP8_MAX, FP8_MAX).to(FP8), b


def _rotary(rows, d, device):
    inv = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).to(torch.bfloat16).to(device)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    state = dict(case=case)

    def pages(n, hk, d):
        """Codes (n * 16, hk, d) and scale bytes (n, hk) of normed K- or V-like rows, each head
        of a size of its own."""
        size = 2.0 ** (2 * randn(1, 1, hk, 1))
        x = randn(n, PAGE, hk, d) * size * (1 + 0.2 * randn(1, 1, hk, d))
        codes, b = _quantized(x, (1, 3))
        return codes.view(n * PAGE, hk, d), b.view(n, hk).to(torch.uint8)

    if case["kind"] == "pages":
        n, layers, hk, d = case["pages"], case["layers"], case["hk"], case["d"]
        order = torch.randperm(n, generator=g, device=dev).cpu().tolist()
        state["src"], state["dst"] = order[:case["moved"]], order[case["moved"]:2 * case["moved"]]
        codes = torch.randint(0, 120, (2 * layers, n, PAGE * hk * d), generator=g, device=dev,
                              dtype=torch.uint8)
        state["codes"] = codes.view(FP8)
        state["scales"] = torch.randint(100, 140, (layers, n, hk, 2), generator=g, device=dev,
                                        dtype=torch.uint8)
        return state

    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["kind"] == "write":
        items, positions = _write_items(case)
        n_pages = len(items)
        state["items"] = torch.tensor(items, dtype=torch.int32, device=dev).view(-1, 5)
        state["positions"] = torch.tensor(positions, dtype=torch.int64, device=dev)
        state["qkv"] = randn(len(positions), (hq + 2 * hk) * d).to(torch.bfloat16)
        state["q_w"], state["k_w"] = ((1 + 0.2 * randn(d)).to(torch.bfloat16) for _ in range(2))
        state["cos_sin"] = _rotary(max(positions) + 1, d, dev)
        state["k"], kb = pages(n_pages, hk, d)
        state["v"], vb = pages(n_pages, hk, d)
        state["scales"] = torch.stack([kb, vb], -1).contiguous()
        return state

    seqs = _sequences(case)
    shared = case["prefix"] // PAGE
    need = [-(-used // PAGE) - shared for _, used in seqs]
    n_pages = shared + sum(need)
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32).cpu().numpy()
    table = np.zeros((len(seqs), shared + max(need)), dtype=np.int32)
    table[:, :shared] = order[:shared]
    at = shared
    for s, count in enumerate(need):
        table[s, shared:shared + count] = order[at:at + count]
        at += count
    rows = [q for q, _ in seqs]
    state["cu_q"] = torch.tensor([0, *np.cumsum(rows)], dtype=torch.int32, device=dev)
    state["used"] = torch.tensor([u for _, u in seqs], dtype=torch.int32, device=dev)
    state["table"] = torch.from_numpy(table).to(dev)
    state["max_q"], state["max_used"] = max(rows), max(u for _, u in seqs)
    state["q"] = randn(sum(rows), hq, d).to(torch.bfloat16)
    state["k"], kb = pages(n_pages, hk, d)
    state["v"], vb = pages(n_pages, hk, d)
    state["scales"] = torch.stack([kb, vb], -1).contiguous()
    return state


def _norm_rope(x, w, cos, sin):
    """RMS norm of the last dimension and neox RoPE; x (rows, heads, d), cos and sin (rows, 1, d/2)."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _write(state, dtype, pools):
    """(q rows, and the pools' codes and scales with the items' pages written), in `dtype`.
    pools: (k, v, scales), written in place."""
    case = state["case"]
    hq, hk, d = case["hq"], case["hk"], case["d"]
    x = state["qkv"].to(dtype).view(-1, hq + 2 * hk, d)
    cs = state["cos_sin"][state["positions"]].to(dtype)[:, None]
    cos, sin = cs.chunk(2, -1)
    q = _norm_rope(x[:, :hq], state["q_w"].to(dtype), cos, sin)
    rows = {0: _norm_rope(x[:, hq:hq + hk], state["k_w"].to(dtype), cos, sin), 1: x[:, hq + hk:]}
    dst, src, keep, row0, count = (c[:, None] for c in state["items"].long().unbind(1))
    slot = torch.arange(PAGE, device=dst.device)[None]
    fresh = ((slot >= keep) & (slot < keep + count))[..., None, None]
    kept = (slot < keep)[..., None, None]
    at = (row0 + slot - keep).clamp(0, x.shape[0] - 1)
    scales = pools[2]

    def one(which):
        pool = pools[which].view(-1, PAGE, hk, d)
        new = rows[which][at]
        old_b = scales[src[:, 0], :, which].long()[:, None, :, None]
        old = pool[src[:, 0]].to(dtype) * torch.exp2((old_b - 127).to(dtype))
        b = _byte((new * fresh).abs().amax((1, 3), keepdim=True))
        b = torch.where(keep[..., None, None] > 0, torch.maximum(b, old_b), b)
        value = torch.where(fresh, new, old) * torch.exp2((127 - b).to(dtype))
        code = value.clamp(-FP8_MAX, FP8_MAX).to(FP8)
        here = pool[dst[:, 0]].view(torch.uint8)
        pool.view(torch.uint8)[dst[:, 0]] = torch.where(fresh | kept, code.view(torch.uint8), here)
        scales[dst[:, 0], :, which] = b[:, 0, :, 0].to(torch.uint8)

    one(0)
    one(1)
    return q


def _standing_for(scales):
    """The scales that E8M0 bytes stand for."""
    return scales.view(torch.float8_e8m0fnu)


def _attend(state):
    """Every sequence as one of a padded batch, in 32 bits."""
    case = state["case"]
    hq, hk, d = case["hq"], case["hk"], case["d"]
    cu, used = state["cu_q"].long(), state["used"].long()
    n = state["q"].shape[0]
    row = torch.arange(state["max_q"], device=cu.device)
    key = torch.arange(state["max_used"], device=cu.device)
    q_len = cu[1:] - cu[:-1]
    q = state["q"][(cu[:-1, None] + row).clamp(max=n - 1)].float()
    q = q.view(*q.shape[:2], hk, hq // hk, d)
    page = state["table"].long()[:, key // PAGE]
    scale = torch.exp2(state["scales"].float() - 127)[page]
    k = state["k"].view(-1, PAGE, hk, d).float()[page, key % PAGE] * scale[..., :1]
    v = state["v"].view(-1, PAGE, hk, d).float()[page, key % PAGE] * scale[..., 1:]
    seen = used[:, None] - (q_len[:, None] - row - 1 if case["causal"] else 0 * row)
    visible = key < seen[..., None]                                   # (seqs, rows, keys)
    score = torch.matmul(q.permute(0, 2, 3, 1, 4).flatten(2, 3).contiguous(),
                         k.permute(0, 2, 3, 1).contiguous()) * d ** -0.5
    score = score.view(len(used), hk, hq // hk, len(row), len(key))
    score.masked_fill_(~visible[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)     # a row that sees no key: 0, not nan
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), v.permute(0, 2, 1, 3).contiguous()).view(*p.shape[:4], d)
    out = torch.where(total > 0, out / total, 0 * out)
    lse = (torch.log(total) + top)[..., 0]
    live = (row < q_len[:, None]).nonzero()
    out = out.permute(0, 3, 1, 2, 4)[live[:, 0], live[:, 1]].reshape(n, hq * d)
    lse = lse.permute(0, 3, 1, 2)[live[:, 0], live[:, 1]].reshape(n, hq)
    return {"out": out.to(torch.bfloat16), "lse": lse.t()}


def _kept(state):
    """The arena, engine and plan that a program keeps, made on the first pass."""
    if "kept" not in state:
        from quail_amd.arena import KVArena
        from quail_amd.chunk import attention_plan
        from quail_amd.engine import Engine
        case = state["case"]
        hk, d = case["hk"], case["d"]
        if case["kind"] == "pages":
            arena = KVArena(case["layers"], case["pages"], PAGE, hk, d, dtype=FP8)
            for layer in range(case["layers"]):
                k, v = arena.layer_kv(layer)
                k.copy_(state["codes"][2 * layer].view(k.shape))
                v.copy_(state["codes"][2 * layer + 1].view(v.shape))
                arena.layer_scales(layer).copy_(state["scales"][layer])
            state["kept"] = (arena, None, None)
            return state["kept"]
        arena = KVArena(1, state["k"].shape[0] // PAGE, PAGE, hk, d, dtype=FP8)
        k, v = arena.layer_kv(0)
        k.copy_(state["k"])
        v.copy_(state["v"])
        arena.layer_scales(0).copy_(state["scales"])
        rotary = SimpleNamespace(cos_sin_cache=state.get("cos_sin"))
        engine = Engine(arena, num_q_heads=case["hq"], num_kv_heads=hk, head_dim=d, rotary=rotary)
        if case["kind"] == "write":
            norm = lambda w: SimpleNamespace(weight=w, variance_epsilon=EPS)  # noqa: E731
            plan = SimpleNamespace(q_norm=norm(state["q_w"]), k_norm=norm(state["k_w"]))
        else:
            plan = attention_plan(state["cu_q"], state["used"], state["table"],
                                  heads=(case["hq"], hk, d), causal=case["causal"])
        state["kept"] = (arena, engine, plan)
    return state["kept"]


def run(state):
    kind = state["case"]["kind"]
    if own:
        arena, engine, plan = _kept(state)
        if kind == "pages":
            arena.copy_pages(state["src"], state["dst"])
            return {"codes": arena.storage.view(state["codes"].shape),
                    "scales": _standing_for(arena.scales)}
        if kind == "write":
            meta = dict(layer=0, unified=dict(page_writes=(state["items"],)))
            q = engine.qk_norm_rope_kv(state["qkv"], state["positions"], plan, meta)
            k, v = arena.layer_kv(0)
            return {"q": q, "k": k, "v": v, "scales": _standing_for(arena.layer_scales(0))}
        out, lse = engine.read_pages(state["q"], plan, 0)
        return {"out": out, "lse": lse}
    if kind == "pages":
        src, dst = torch.tensor([state["src"], state["dst"]], device=state["codes"].device)
        codes = state["codes"].view(torch.uint8)
        codes[:, dst] = codes[:, src]
        state["scales"][:, dst] = state["scales"][:, src]
        return {"codes": state["codes"], "scales": _standing_for(state["scales"])}
    if kind == "write":
        q = _write(state, torch.float32, (state["k"], state["v"], state["scales"]))
        return {"q": q.to(torch.bfloat16).flatten(1), "k": state["k"], "v": state["v"],
                "scales": _standing_for(state["scales"])}
    return _attend(state)


def exact(case, seed):
    """The definition in 64 bits, a sequence or a set of rows at a time. A fresh code stands
    unrounded: the clamped row over its page's scale."""
    state = prepare(case, seed)
    if case["kind"] == "pages":
        codes, scales = state["codes"], state["scales"]
        for src, dst in zip(state["src"], state["dst"]):
            codes[:, dst].copy_(codes[:, src])
            scales[:, dst].copy_(scales[:, src])
        return {"codes": codes.double(), "scales": torch.exp2(scales.double() - 127)}
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["kind"] == "write":
        return _exact_write(state, hq, hk, d)
    value = {}
    for which, name in enumerate("kv"):
        scale = torch.exp2(state["scales"][:, :, which].double() - 127)
        value[name] = state[name].double() * scale.repeat_interleave(PAGE, 0)[..., None]
    out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(out.shape[:2], dtype=torch.float64, device="cuda")
    cu, used, table = (state[n].cpu().tolist() for n in ("cu_q", "used", "table"))
    for s, keys in enumerate(used):
        rows = slice(cu[s], cu[s + 1])
        pages = torch.tensor(table[s][:-(-keys // PAGE)], device="cuda")
        at = (pages[:, None] * PAGE + torch.arange(PAGE, device="cuda")).view(-1)[:keys]
        back = torch.arange(cu[s + 1] - cu[s], 0, -1, device="cuda")
        last = keys - back if case["causal"] else torch.full_like(back, keys - 1)
        hidden = torch.arange(keys, device="cuda") > last[:, None]
        for h in range(hq):
            w = state["q"][rows, h].double() @ value["k"][at, h * hk // hq].t() / math.sqrt(d)
            w[hidden] = -math.inf
            lse[rows, h] = w.logsumexp(-1)
            out[rows, h] = (w - lse[rows, h, None]).exp() @ value["v"][at, h * hk // hq]
    return {"out": out.flatten(1), "lse": lse.t()}


def _exact_write(state, hq, hk, d):
    qkv = state["qkv"].double().view(-1, hq + 2 * hk, d)
    angle = state["cos_sin"].double()[state["positions"]]
    c, s = angle[:, None, :d // 2], angle[:, None, d // 2:]

    def turned(x, w):
        x = x / ((x ** 2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        lo, hi = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)

    row = torch.arange(qkv.shape[0], device="cuda")
    item = torch.bucketize(row, state["items"][:, 3].long(), right=True) - 1
    dst, src, keep, row0, _ = state["items"].long().t()
    pool_row = dst[item] * PAGE + keep[item] + row - row0[item]
    found = {"q": turned(qkv[:, :hq], state["q_w"]).flatten(1)}
    scales = state["scales"].double()
    fresh = {"k": turned(qkv[:, hq:hq + hk], state["k_w"]), "v": qkv[:, hq + hk:]}
    slot = torch.arange(PAGE, device="cuda")
    for which, name in enumerate("kv"):
        old = state["scales"][:, :, which].double()
        most = torch.zeros(len(dst), hk, dtype=torch.float64, device="cuda")
        most.scatter_reduce_(0, item[:, None].expand(-1, hk), fresh[name].abs().amax(-1), "amax")
        need = 127 + torch.ceil(torch.log2((most / FP8_MAX).clamp(min=2.0 ** -126)))
        new = torch.where(keep[:, None] > 0, torch.maximum(need, old[src]), need)
        values = state[name].double().view(-1, PAGE, hk, d)
        grown = torch.exp2(old[src] - new)[:, None, :, None]
        kept = (slot < keep[:, None])[..., None, None]
        values[dst] = torch.where(kept, values[src] * grown, values[dst])
        values = values.view(-1, hk, d)
        values[pool_row] = fresh[name] * torch.exp2(127 - new[item])[..., None]
        found[name] = values
        scales[dst, :, which] = new
    return {**found, "scales": torch.exp2(scales - 127)}
