"""Long documents in a bounded KV arena, as cases to measure.

Pages hold 16 tokens of 16-bit rows, or of e4m3 codes with one power-of-two
scale per (page, KV head), an E8M0 byte b that stands for 2^(b - 127), K's and
V's apart. Three operators:

  weights  the attention weight that each key has gathered: for every KV head
           the softmax probabilities summed over the query rows that see the
           key and the query heads of its group, on top of earlier sums.
  thin     of each (layer, sequence, KV head) the first `sinks` rows, the last
           `recent` ones and the heaviest of the others are kept, `keep` in
           all; kept rows past `keep` move into the places of dropped ones.
  rotary   rows of q and k turned by their positions: half or interleaved
           pairs, all of the head or its first part, frequencies scaled for
           long contexts.

With `own` false each runs in its plain form, elementary torch operations in
32 bits (angles in 64); with `own` true through the framework's Engine,
KVArena and RotaryEmbedding.
"""

import math
import random
from types import SimpleNamespace

import numpy as np
import torch

own = False

PAGE = 16
FP8 = torch.float8_e4m3fn
BASE = 1e6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one more token for each of 8 sequences, weights gathered as they go
        dict(name="weights-one-token", kind="weights", bits=16, hq=32, hk=8, d=128, seqs=8, q=1, lo=300,
             hi=1100, median=700, prefix=64, prior=True, lengths=1),
        # a token on each of two whole contexts, 64 heads
        dict(name="weights-token-contexts", kind="weights", bits=16, hq=64, hk=8, d=128, seqs=2, q=1,
             lo=39990, hi=39990, median=39990, prefix=0, prior=True, lengths=2),
        # the last rows of kept documents stand for the questions to come
        dict(name="weights-window-8bit", kind="weights", bits=8, hq=32, hk=8, d=128, seqs=8, q=64, lo=2000,
             hi=8000, median=4000, prefix=64, prior=False, lengths=3),
        # every row of an AI.IF pack of Qwen3-4B behind a 64-token prefix
        dict(name="weights-if-pack", kind="weights", bits=16, hq=32, hk=8, d=128, seqs=46, q=0, lo=32,
             hi=2048, median=256, prefix=64, prior=False, lengths=4),
        # every row of a long document
        dict(name="weights-long-rows", kind="weights", bits=16, hq=32, hk=8, d=128, seqs=1, q=0, lo=8003,
             hi=8003, median=8003, prefix=0, prior=False, lengths=5),
        # a small model's documents, thinned as they are kept
        dict(name="thin-tiny", kind="thin", bits=16, layers=2, hk=2, d=64, seqs=5, lo=60, hi=300, median=200,
             keep=77, sinks=4, recent=16, lengths=6),
        # sequences that grow by 64 tokens between thinnings, all layers
        dict(name="thin-step", kind="thin", bits=16, layers=36, hk=8, d=128, seqs=8, lo=1088, hi=1088,
             median=1088, keep=1024, sinks=4, recent=64, lengths=7),
        # a long document thinned to a quarter before its questions, all layers
        dict(name="thin-document", kind="thin", bits=16, layers=36, hk=8, d=128, seqs=1, lo=8003, hi=8003,
             median=8003, keep=2000, sinks=4, recent=64, lengths=8),
        # a whole context in 8 bits thinned to a quarter, all layers
        dict(name="thin-context-8bit", kind="thin", bits=8, layers=36, hk=8, d=128, seqs=1, lo=39990,
             hi=39990, median=39990, keep=10000, sinks=16, recent=128, lengths=9),
        # a few tokens far past the trained positions
        dict(name="rotary-one-token", kind="rotary", rows=8, hq=32, hk=8, d=128, rd=128, pairs="half",
             scaling="yarn", factor=4.0, trained=32768, at=120000, type="bf16", lengths=10),
        # a whole pack of Qwen3-4B rows, context scaled by 4
        dict(name="rotary-if-pack", kind="rotary", rows=15654, hq=32, hk=8, d=128, rd=128, pairs="half",
             scaling="yarn", factor=4.0, trained=32768, at=0, type="bf16", lengths=11),
        # half of each head turned in interleaved pairs
        dict(name="rotary-part-pairs", kind="rotary", rows=4001, hq=32, hk=8, d=128, rd=64,
             pairs="interleaved", scaling="linear", factor=8.0, trained=4096, at=20000, type="fp16",
             lengths=12),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["weights", "weights", "weights", "thin", "thin", "thin", "rotary", "rotary"])
    seed = rng.randrange(1 << 30)
    if kind == "rotary":
        d = rng.choice([64, 128, 128])
        return dict(kind=kind, rows=_spread(rng, 1, 15000), hq=rng.choice([4, 32, 32]), hk=rng.choice([2, 8]),
                    d=d, rd=rng.choice([d, d, d // 2, 20]), pairs=rng.choice(["half", "half", "interleaved"]),
                    scaling=rng.choice(["yarn", "yarn", "linear", "none"]),
                    factor=rng.choice([2.0, 4.0, 6.5]), trained=rng.choice([4096, 32768]),
                    at=_spread(rng, 1, 1000000), type=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    lengths=seed)
    bits = rng.choice([16, 16, 8])
    if kind == "thin":
        layers, hk, d = rng.choice([(2, 2, 64), (36, 8, 128), (36, 8, 128), (9, 4, 128)])
        seqs = _spread(rng, 1, 12)
        median = _spread(rng, 40, (22000 if bits == 8 else 10000) // seqs)
        keep = max(16, int(median * rng.uniform(0.1, 0.95)))
        keep = keep // PAGE * PAGE if bits == 8 else keep
        return dict(kind=kind, bits=bits, layers=layers, hk=hk, d=d, seqs=seqs, lo=max(1, median // 3),
                    hi=min(39999, 3 * median // 2), median=median, keep=keep,
                    sinks=rng.choice([0, 1, 4]), recent=rng.randrange(0, min(200, keep - 4)), lengths=seed)
    hq, hk, d = rng.choice([(4, 2, 64), (32, 8, 128), (32, 8, 128), (64, 8, 128), (20, 4, 128)])
    shape = rng.choice(["token", "window", "rows"])
    if shape == "token":
        seqs = _spread(rng, 1, 60)
        median = _spread(rng, 20, 60000 // seqs if seqs > 2 else 30000)
        q = 1
    elif shape == "window":
        seqs = _spread(rng, 1, 12)
        median, q = _spread(rng, 100, 20000 // seqs), _spread(rng, 2, 100)
    else:
        seqs = _spread(rng, 1, 40)
        median, q = _spread(rng, 20, 5000 // seqs if seqs > 1 else 4000), 0
    return dict(kind=kind, bits=bits, hq=hq, hk=hk, d=d, seqs=seqs, q=q, lo=max(1, median // 4),
                hi=min(39900, 2 * median), median=median, prefix=rng.choice([0, 16, 64]),
                prior=rng.random() < 0.5, lengths=seed)


def _lengths(case):
    """Tokens of each sequence: lognormal about the median, within [lo, hi]."""
    rng = random.Random(case["lengths"])
    return [min(case["hi"], max(case["lo"], int(rng.lognormvariate(math.log(case["median"]), 0.6))))
            for _ in range(case["seqs"])]


def _sequences(case):
    """(query rows, keys) of each sequence of a weights case."""
    return [(n if case["q"] == 0 else case["q"],
             case["prefix"] + (n if case["q"] == 0 else max(n, case["q"])))
            for n in _lengths(case)]


def work(case):
    if case["kind"] == "rotary":
        item = 4 if case["type"] == "fp32" else 2
        heads = case["rows"] * (case["hq"] + case["hk"])
        return {"bytes": 2 * item * heads * case["d"] + 8 * case["rows"], "flops": 3 * heads * case["rd"]}
    hk, d = case["hk"], case["d"]
    if case["kind"] == "thin":
        # rows that move, where any of the unprotected ones is as likely to be kept as another
        keep, sinks, recent = case["keep"], case["sinks"], case["recent"]
        lengths, moved = _lengths(case), 0
        columns = _cols(max(lengths)) + keep
        for used in lengths:
            if used > keep:
                share = (keep - sinks - recent) / (used - sinks - recent)
                late = max(0, used - recent - keep)
                moved += share * late + min(recent, used - keep)
        return {"bytes": int(case["layers"] * hk * (4 * (sum(lengths) + columns * len(lengths))
                                                    + moved * 4 * d * case["bits"] // 8)), "flops": 0}
    hq = case["hq"]
    pairs = keys = rows = longest = 0
    shared = case["prefix"] // PAGE * PAGE
    for q, used in _sequences(case):
        pairs += q * used - q * (q - 1) // 2
        keys, rows, longest = keys + used - shared, rows + q, max(longest, used)
    keys += shared
    out = case["seqs"] * hk * _cols(longest) * 4 * (2 if case["prior"] else 1)
    return {"bytes": rows * hq * (2 * d + 4) + keys * hk * d * case["bits"] // 8
            + (hk * (keys // PAGE) if case["bits"] == 8 else 0) + out, "flops": 2 * hq * d * pairs}


def _cols(tokens):
    return -(-int(tokens) // PAGE) * PAGE


def _tables(needs, shared, g):
    """Block tables (numpy int32) over a random order of pages, the first `shared` of each row the
    same ones, and the number of pages."""
    n_pages = shared + sum(n - shared for n in needs)
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu().numpy()
    table = np.zeros((len(needs), max(needs)), dtype=np.int32)
    table[:, :shared] = order[:shared]
    at = shared
    for s, n in enumerate(needs):
        table[s, shared:n] = order[at:at + n - shared]
        at += n - shared
    return table, n_pages


def _coded(x):
    """e4m3 codes and scale bytes of rows (pages, 16, heads, d): the least power of two that brings
    a page's largest value of a head to 448 or below."""
    top = x.abs().amax((1, 3))
    b = (127 + torch.ceil(torch.log2(top / 448))).clamp(min=1)
    codes = (x * torch.exp2(127 - b)[:, None, :, None]).clamp(-448, 448).to(FP8)
    return codes, b.to(torch.uint8)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    state = dict(case=case)
    if case["kind"] == "rotary":
        dtype = TYPES[case["type"]]
        hq, hk, d, n = case["hq"], case["hk"], case["d"], case["rows"]
        qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g, device="cuda", dtype=dtype)
        state["q"], state["k"], _ = qkv.split([hq * d, hk * d, hk * d], 1)
        # documents one after another, each from a position of its own
        rng = random.Random(seed)
        positions = []
        while len(positions) < n:
            first = case["at"] + rng.randrange(2000)
            positions += range(first, first + rng.randrange(1, 1200))
        state["positions"] = torch.tensor(positions[:n], dtype=torch.int64, device="cuda")
        return state
    hk, d, bits = case["hk"], case["d"], case["bits"]
    if case["kind"] == "thin":
        lengths, layers = _lengths(case), case["layers"]
        table, n_pages = _tables([-(-n // PAGE) for n in lengths], 0, g)
        kv = torch.empty(layers, 2, n_pages * PAGE, hk, d, dtype=FP8 if bits == 8 else torch.bfloat16,
                         device="cuda")
        scales = torch.empty(layers, n_pages, hk, 2, dtype=torch.uint8, device="cuda")
        for layer in range(layers):
            for side in range(2):
                x = randn(n_pages, PAGE, hk, d) * torch.exp2(2 * randn(n_pages, 1, hk, 1))
                if bits == 8:
                    codes, scales[layer, :, :, side] = _coded(x)
                    kv[layer, side] = codes.view(-1, hk, d)
                else:
                    kv[layer, side] = x.view(-1, hk, d).to(kv.dtype)
        state["kv"] = kv
        if bits == 8:
            state["scales"] = scales
        # gathered weights: a few keys hold most, and some never had any
        w = torch.exp(2.5 * randn(layers, len(lengths), hk, table.shape[1] * PAGE))
        state["weights"] = torch.where(w < 0.05, torch.zeros_like(w), w)
        used = lengths
    else:
        seqs, hq = _sequences(case), case["hq"]
        used = [u for _, u in seqs]
        table, n_pages = _tables([-(-u // PAGE) for u in used], case["prefix"] // PAGE, g)
        size = torch.exp2(0.5 * randn(1, 1, hk, 1))
        k = randn(n_pages, PAGE, hk, d) * size * (1 + 0.2 * randn(1, 1, hk, d))
        if bits == 8:
            codes, state["scales"] = _coded(k)
            state["k"] = codes.view(-1, hk, d)
        else:
            state["k"] = k.to(torch.bfloat16).view(-1, hk, d)
        rows = [q for q, _ in seqs]
        state["cu_q"] = torch.tensor([0, *np.cumsum(rows)], dtype=torch.int32, device="cuda")
        state["q"] = randn(sum(rows), hq, d).to(torch.bfloat16)
        state["max_q"] = max(rows)
        if case["prior"]:
            state["prior"] = torch.exp(2 * randn(len(seqs), hk, table.shape[1] * PAGE))
    state["max_used"] = max(used)
    state["used"] = torch.tensor(used, dtype=torch.int32, device="cuda")
    state["table"] = torch.from_numpy(table).to("cuda")
    if case["kind"] == "weights":
        # the log-sum-exps that the attention over these keys has left, a sequence's head at a time
        state["lse"] = torch.empty(case["hq"], sum(rows), device="cuda")
        first = 0
        for s, (n, keys) in enumerate(seqs):
            x = _keys(state, s, keys).float()
            last = keys - n + torch.arange(n, device="cuda")
            hidden = torch.arange(keys, device="cuda") > last[:, None]
            for h in range(case["hq"]):
                score = state["q"][first:first + n, h].float() @ x[:, h * hk // case["hq"]].t() * d ** -0.5
                state["lse"][h, first:first + n] = score.masked_fill_(hidden, -math.inf).logsumexp(-1)
            first += n
    return state


def _keys(state, s, keys, dtype=torch.float32):
    """A sequence's keys (keys, hk, d)."""
    j = torch.arange(keys, device="cuda")
    page = state["table"][s].long()[j // PAGE]
    x = state["k"].view(-1, PAGE, *state["k"].shape[1:])[page, j % PAGE].to(dtype)
    if "scales" in state:
        x = x * torch.exp2(state["scales"][page].to(dtype) - 127)[..., None]
    return x


def _plain_weights(state):
    """Every sequence as one of a padded batch, in 32 bits."""
    case = state["case"]
    hq, hk, d = case["hq"], case["hk"], case["d"]
    cu, used, table = state["cu_q"].long(), state["used"].long(), state["table"].long()
    n = state["q"].shape[0]
    row = torch.arange(state["max_q"], device=cu.device)
    key = torch.arange(state["max_used"], device=cu.device)
    q_len = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + row).clamp(max=n - 1)
    q = state["q"][at].float().view(*at.shape, hk, hq // hk, d)
    lse = state["lse"].t()[at].view(*at.shape, hk, hq // hk)
    page = table[:, key // PAGE]
    k = state["k"].view(-1, PAGE, hk, d)[page, key % PAGE].float()
    if "scales" in state:
        k = k * torch.exp2(state["scales"].float() - 127)[page][..., None]
    seen = used[:, None] - (q_len[:, None] - row - 1)
    visible = (key < seen[..., None]) & (row < q_len[:, None])[..., None]     # (seqs, rows, keys)
    score = torch.matmul(q.permute(0, 2, 3, 1, 4).flatten(2, 3).contiguous(),
                         k.permute(0, 2, 3, 1).contiguous()) * d ** -0.5
    score = score.view(len(used), hk, hq // hk, len(row), len(key))
    p = score.sub_(lse.permute(0, 2, 3, 1)[..., None]).exp_().masked_fill_(~visible[:, None, None], 0.0)
    total = p.sum((2, 3))
    out = state["prior"].clone() if case["prior"] else \
        torch.zeros(len(used), hk, table.shape[1] * PAGE, device=cu.device)
    out[..., :len(key)] += total
    return {"weights": out}


def _plain_thin(state):
    case, w, kv = state["case"], state["weights"], state["kv"]
    keep, table = case["keep"], state["table"].long()
    used = state["used"].long()[:, None, None]                 # against (layers, seqs, heads, columns)
    i = torch.arange(w.shape[-1], device=w.device)
    k = used.clamp(max=keep)
    live = i < used
    safe = live & ((i < case["sinks"]) | (i >= used - case["recent"]))
    # heaviest first, then the protected ones before the others; ties stay in order
    by_weight = torch.where(live, w, -math.inf).sort(dim=-1, descending=True, stable=True)[1]
    safe_first = safe.expand(w.shape).gather(-1, by_weight).to(torch.uint8).sort(dim=-1, descending=True,
                                                                               stable=True)[1]
    order = by_weight.gather(-1, safe_first)
    rank = torch.empty_like(order).scatter_(-1, order, i.expand(order.shape).contiguous())
    kept = live & (rank < k)
    hole, mover = (i < k) & ~kept, (i >= k) & kept
    movers = mover.to(torch.uint8).sort(dim=-1, descending=True, stable=True)[1]
    source = torch.where(hole, movers.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), i)
    out = torch.where(i < k, w.gather(-1, source), torch.zeros_like(w))
    left = torch.where(i < k, source, -1)[..., :keep].to(torch.int32)
    found = {"kept": left, "weights": out}
    if case["bits"] == 16:
        layer, s, h, slot = hole.nonzero(as_tuple=True)
        src = source[layer, s, h, slot]
        at, of = table[s, slot // PAGE] * PAGE + slot % PAGE, table[s, src // PAGE] * PAGE + src % PAGE
        rows = kv.permute(0, 2, 3, 1, 4)                       # (layers, rows, heads, K and V, d)
        rows[layer, at, h] = rows[layer, of, h]
        return {**found, "kv": kv}
    # pages that a row moves into are written anew, at the largest scale their rows come with
    pages = min(keep, w.shape[-1]) // PAGE
    layer, s, h, page = hole[..., :pages * PAGE].unflatten(-1, (pages, PAGE)).any(-1).nonzero(as_tuple=True)
    src = source[..., :pages * PAGE].unflatten(-1, (pages, PAGE))[layer, s, h, page]
    of = table[s[:, None], src // PAGE]
    b = state["scales"][layer[:, None], of, h[:, None]].float()               # (pages, 16, K and V)
    top = b.amax(1)
    rows = kv.view(torch.uint8).permute(0, 2, 3, 1, 4)
    old = rows[layer[:, None], of * PAGE + src % PAGE, h[:, None]].view(FP8).float()
    new = (old * torch.exp2(b - top[:, None])[..., None]).to(FP8)
    at = table[s, page]
    to = at[:, None] * PAGE + torch.arange(PAGE, device=at.device)
    rows[layer[:, None], to, h[:, None]] = new.view(torch.uint8)
    state["scales"][layer, at, h] = top.to(torch.uint8)
    return {**found, "kv": kv, "scales": _standing_for(state["scales"])}


def _standing_for(scales):
    """The scales that E8M0 bytes stand for."""
    return scales.view(torch.float8_e8m0fnu)


def _frequencies(case):
    """The angle per position of each pair, and the factor on cos and sin, in 64 bits."""
    rd, factor = case["rd"], case["factor"]
    i = torch.arange(rd // 2, dtype=torch.float64, device="cuda")
    f = BASE ** (-2 * i / rd)
    if case["scaling"] == "none":
        return f, 1.0
    if case["scaling"] == "linear":
        return f / factor, 1.0
    # pairs that turn more than 32 times over the trained positions stay, those that turn less
    # than once are slowed by the factor, a ramp between
    where = lambda turns: rd * math.log(case["trained"] / (turns * 2 * math.pi)) / (2 * math.log(BASE))  # noqa: E731
    low, high = max(0, math.floor(where(32))), min(rd - 1, math.ceil(where(1)))
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1


def _turned(x, cos, sin, case, dtype):
    rd = case["rd"]
    x = x.to(dtype).view(x.shape[0], -1, case["d"])
    turn, rest = x[..., :rd], x[..., rd:]
    if case["pairs"] == "half":
        a, b = turn.chunk(2, -1)
        turn = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = turn[..., ::2], turn[..., 1::2]
        turn = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turn, rest], -1).flatten(1)


def _plain_rotary(state):
    case = state["case"]
    f, factor = _frequencies(case)
    angle = state["positions"].double()[:, None, None] * f
    cos, sin = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    return {n: _turned(state[n], cos, sin, case, torch.float32).to(state[n].dtype) for n in "qk"}


def _kept(state):
    """The arena, engine, tables or rotary module that a program keeps, made on the first pass."""
    if "kept" in state:
        return state["kept"]
    case = state["case"]
    if case["kind"] == "rotary":
        from quail_amd.rotary import RotaryEmbedding
        scaling = None
        if case["scaling"] != "none":
            scaling = dict(rope_type=case["scaling"], factor=case["factor"],
                           original_max_position_embeddings=case["trained"])
        state["kept"] = RotaryEmbedding(case["d"], rotary_dim=case["rd"], base=BASE, scaling=scaling,
                                        interleaved=case["pairs"] == "interleaved")
        return state["kept"]
    from quail_amd.arena import KVArena
    layers, hk, d = case.get("layers", 1), case["hk"], case["d"]
    dtype = FP8 if case["bits"] == 8 else torch.bfloat16
    rows = state["kv"].shape[2] if case["kind"] == "thin" else state["k"].shape[0]
    arena = KVArena(layers, rows // PAGE, PAGE, hk, d, dtype=dtype, v_dtype=dtype)
    if case["kind"] == "thin":
        arena.storage.view(torch.uint8).copy_(state["kv"].view(torch.uint8).view(-1))
        if case["bits"] == 8:
            arena.scales.copy_(state["scales"])
        tables = dict(used=state["used"], table=state["table"], max_used=state["max_used"])
        state["kept"] = arena, tables, None
        return state["kept"]
    from quail_amd.chunk import attention_plan
    from quail_amd.engine import Engine
    arena.layer_kv(0)[0].copy_(state["k"])
    if case["bits"] == 8:
        arena.layer_scales(0)[..., 0].copy_(state["scales"])
    engine = Engine(arena, num_q_heads=case["hq"], num_kv_heads=hk, head_dim=d,
                    rotary=SimpleNamespace(cos_sin_cache=None))
    plan = attention_plan(state["cu_q"], state["used"], state["table"], heads=(case["hq"], hk, d),
                          causal=True, eight_bit=case["bits"] == 8)
    state["kept"] = arena, plan, engine
    return state["kept"]


def run(state):
    case = state["case"]
    if not own:
        return {"weights": _plain_weights, "thin": _plain_thin, "rotary": _plain_rotary}[case["kind"]](state)
    if case["kind"] == "rotary":
        q, k = _kept(state)(state["positions"], state["q"], state["k"])
        return {"q": q, "k": k}
    arena, tables, engine = _kept(state)
    if case["kind"] == "weights":
        return {"weights": engine.key_weights(state["q"], state["lse"], tables, 0,
                                              weights=state.get("prior"))}
    kept, weights = arena.thin_rows(tables, state["weights"], case["keep"], sinks=case["sinks"],
                                    recent=case["recent"])
    found = {"kept": kept, "weights": weights, "kv": arena.storage.view(state["kv"].shape)}
    if case["bits"] == 8:
        found["scales"] = _standing_for(arena.scales)
    return found


def exact(case, seed):
    """The definition in 64 bits, a head at a time. Rows that move are not computed and have no
    value here."""
    state = prepare(case, seed)
    if case["kind"] == "rotary":
        f, factor = _frequencies(case)
        turn = torch.polar(torch.full_like(f, factor), torch.zeros_like(f)) * \
            torch.exp(1j * state["positions"].double()[:, None] * f)
        found = {}
        for name in "qk":
            x = state[name].double().reshape(case["rows"], -1, case["d"])
            rd = case["rd"]
            first, second = (x[..., :rd // 2], x[..., rd // 2:rd]) if case["pairs"] == "half" else \
                (x[..., 0:rd:2], x[..., 1:rd:2])
            z = torch.complex(first.contiguous(), second.contiguous()) * turn[:, None]
            y = x.clone()
            if case["pairs"] == "half":
                y[..., :rd // 2], y[..., rd // 2:rd] = z.real, z.imag
            else:
                y[..., 0:rd:2], y[..., 1:rd:2] = z.real, z.imag
            found[name] = y.flatten(1)
        return found
    if case["kind"] == "thin":
        w = state["weights"].double()
        out = torch.zeros_like(w)
        for s, used in enumerate(_lengths(case)):
            k = min(used, case["keep"])
            if used <= case["keep"]:
                out[:, s, :, :k] = w[:, s, :, :k]
                continue
            free = slice(case["sinks"], used - case["recent"])
            rest = k - case["sinks"] - case["recent"]
            stay = torch.zeros(*w.shape[:1], w.shape[2], used, dtype=torch.bool, device="cuda")
            stay[..., :case["sinks"]] = True
            stay[..., used - case["recent"]:] = True
            # of the border's equal weights the first ones
            middle = w[:, s, :, free]
            if rest:
                border = middle.topk(rest, -1)[0][..., -1:]
                above, equal = middle > border, middle == border
                spare = rest - above.sum(-1, keepdim=True)
                stay[..., free] |= above | (equal & (equal.cumsum(-1) <= spare))
            for layer in range(w.shape[0]):
                for h in range(w.shape[2]):
                    row = w[layer, s, h, :used]
                    flags = stay[layer, h]
                    new = row[:k].clone()
                    new[~flags[:k]] = row[k:][flags[k:]]
                    out[layer, s, h, :k] = new
        found = {"kept": None, "weights": out, "kv": None}
        return {**found, "scales": None} if case["bits"] == 8 else found
    hq, hk, d = case["hq"], case["hk"], case["d"]
    seqs = _sequences(case)
    cols = state["table"].shape[1] * PAGE
    out = state["prior"].double() if case["prior"] else \
        torch.zeros(len(seqs), hk, cols, dtype=torch.float64, device="cuda")
    first = 0
    for s, (n, keys) in enumerate(seqs):
        x = _keys(state, s, keys, torch.float64)
        last = keys - n + torch.arange(n, device="cuda")
        hidden = torch.arange(keys, device="cuda") > last[:, None]
        for h in range(hq):
            g = h * hk // hq
            score = state["q"][first:first + n, h].double() @ x[:, g].t() / math.sqrt(d)
            p = (score - state["lse"][h, first:first + n, None].double()).exp()
            out[s, g, :keys] += p.masked_fill(hidden, 0.0).sum(0)
        first += n
    return {"weights": out}
