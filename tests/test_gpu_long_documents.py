"""Long documents in an arena of bounded pages, on the GPU: positions past the
trained ones (RotaryEmbedding), rows written, read (read_pages) and their
attention gathered by key (key_weights), the lightest rows dropped (thin) and
further tokens appended (append_rows), over and over. Each step against plain
definitions in 64 bits over the rows that the pages hold.

Bounds of the attention rows as in tests/test_gpu_kv8.py (its P, rounded to bf16,
is the coarser one of the two arenas), of the weights as in
tests/test_gpu_key_weights.py, of the rotation as in tests/test_gpu_rotary.py. A
row as written: K of 16 bits as it is, V in fp16 from bf16 exact down to 2^-14 and
off by at most 2^-25 below; 8 bits off by 2^-4 of a value or half the smallest
code's step, 2^-10, of the page's scale. Moved rows are the same values, in 8
bits off by that half step of their new page's scale.
"""

import numpy as np
import pytest
import torch

from oracle.thin_ref import kept_slots
from quail_amd.arena import FP8, KVArena
from quail_amd.chunk import attention_plan, page_writes
from quail_amd.rotary import RotaryEmbedding, frequencies
from tests.test_gpu_key_weights import check as check_weights
from tests.test_gpu_kv8 import engine_of
from tests.test_gpu_rotary import check as check_rotation

pytestmark = pytest.mark.gpu

DEV = "cuda"
PAGE = 16
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}


def write(eng, k3, v3, rows, layer):
    n = len(rows)
    unified = dict(src=torch.arange(n, device=DEV), dst=torch.from_numpy(rows).to(DEV), tail_src=None)
    if eng.arena.eight_bit:
        unified = dict(page_writes=tuple(torch.from_numpy(p).to(DEV) for p in page_writes(np.arange(n), rows)))
    eng.write_kv(k3, v3, dict(layer=layer, unified=unified))


def held(arena, rows, layer):
    """K and V of pool rows in 64 bits, and their scales (1 without)."""
    rows = torch.from_numpy(np.asarray(rows))
    k, v = (p.cpu()[rows].double() for p in arena.layer_kv(layer))
    scale = torch.ones(2, len(rows), arena.kv_shape[0], 1, dtype=torch.float64)
    if arena.eight_bit:
        s = torch.exp2(arena.layer_scales(layer).cpu().double() - 127)[rows // PAGE]
        scale = torch.stack([s[..., 0], s[..., 1]])[..., None]
        k, v = k * scale[0], v * scale[1]
    return torch.stack([k, v]), scale


def check_attention(out, lse, q, cu_q, kv):
    """Causal rows of each sequence over its K and V, (2, keys, hk, d)."""
    n, hq, d = q.shape
    out, lse, q = out.cpu().double().view(n, hq, d), lse.cpu().double(), q.cpu().double()
    for s, (k, v) in enumerate(kv):
        g = hq // k.shape[1]
        k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
        rows = slice(int(cu_q[s]), int(cu_q[s + 1]))
        count, keys = rows.stop - rows.start, len(k)
        score = torch.stack([q[rows, h] @ k[:, h].t() for h in range(hq)]) * d ** -0.5
        reach = torch.stack([q[rows, h].abs() @ k[:, h].abs().t() for h in range(hq)]).amax(-1) * d ** -0.5
        hidden = torch.arange(keys) > keys - count + torch.arange(count)[:, None]
        score.masked_fill_(hidden, -torch.inf)
        p = score.softmax(-1)
        want = torch.stack([p[h] @ v[:, h] for h in range(hq)], 1)
        size = torch.stack([p[h] @ v[:, h].abs() for h in range(hq)], 1)
        off = (d + 8) * 2.0 ** -24 * reach
        bound = 2.0 ** -8 * (size + want.abs()) + (2 * off.t()[..., None] + 2.0 ** -20 + 2.0 ** -16) * size
        assert bool(((out[rows] - want).abs() <= bound).all())
        want = score.logsumexp(-1)
        # (the weights' sum is of P before its rounding, or of what it is rounded to: 2^-8)
        assert bool(((lse[:, rows] - want).abs() <= 2 * off + 2.0 ** -20 * (1 + want.abs()) + 2.0 ** -8).all())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 64), (32, 8, 128)])
def test_documents_are_read_thinned_and_continued(bits, hq, hk, d):
    g = torch.Generator().manual_seed(bits + d)
    layers, keep, sinks, recent = 2, 64, 4, 16
    arena = KVArena(layers, 60, PAGE, hk, d, dtype=FP8 if bits == 8 else torch.bfloat16)
    eng = engine_of(arena, hq)
    rot = RotaryEmbedding(d, scaling=YARN, max_positions=131072)
    inv, factor = frequencies(d, 1e6, YARN)
    assert torch.equal(rot.inv_freq, inv) and rot.factor == factor
    keys, new, at = ["long", "short", "one"], [300, 77, 1], [130000, 40000, 0]
    weights = None                 # (layers, sequences, heads, columns)
    for step in range(5):
        rows = []
        for key, n in zip(keys, new):
            if step == 0:
                assert arena.activate(key, n, capacity_tokens=n) is not None
                rows.append(arena.capacity_rows(key)[:n])
            else:
                rows.append(arena.append_rows(key, n))
        table, used = arena.block_table(keys)
        cu_q = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        tables = attention_plan(*(torch.from_numpy(a).to(DEV) for a in (cu_q, used, table)),
                                heads=(hq, hk, d), causal=True, eight_bit=bits == 8)
        positions = torch.cat([torch.arange(p, p + n) for p, n in zip(at, new)]).to(DEV)
        at = [p + n for p, n in zip(at, new)]
        cols = table.shape[1] * PAGE
        gathered = torch.zeros(layers, len(keys), hk, cols, device=DEV)
        if weights is not None:
            width = min(cols, weights.shape[-1])
            gathered[..., :width] = weights[..., :width]
        prior = gathered.clone()
        for layer in range(layers):
            qkv = torch.randn(len(positions), (hq + 2 * hk) * d, generator=g).to(torch.bfloat16).to(DEV)
            x = qkv[:, :hq * d], qkv[:, hq * d:(hq + hk) * d]
            q, k = rot(positions, *x)
            check_rotation(q, x[0], positions, rot, d)
            check_rotation(k, x[1], positions, rot, d)
            v = qkv[:, (hq + hk) * d:].reshape(-1, hk, d)
            q, k = q.view(-1, hq, d), k.view(-1, hk, d)
            write(eng, k, v, np.concatenate(rows), layer)
            # the rows as they were written
            got, scale = held(arena, np.concatenate(rows), layer)
            want = torch.stack([k.cpu().double(), v.cpu().double()])
            off = 2.0 ** -4 * want.abs() + 2.0 ** -10 * scale if bits == 8 else \
                torch.tensor([0.0, 2.0 ** -25], dtype=torch.float64).view(2, 1, 1, 1)
            assert bool(((got - want).abs() <= off).all())
            out, lse = eng.read_pages(q, tables, layer)
            kv = [held(arena, arena.capacity_rows(key)[:n], layer)[0] for key, n in zip(keys, used)]
            check_attention(out, lse, q, cu_q, kv)
            eng.key_weights(q, lse, tables, layer, weights=gathered[layer], out=gathered[layer])
            check_weights(gathered[layer], q, lse, arena, cu_q, used.tolist(), table, True, prior[layer],
                          layer=layer)
        before = {(key, layer): held(arena, arena.capacity_rows(key)[:n], layer)[0]
                  for key, n in zip(keys, used) for layer in range(layers)}
        kept, weights = arena.thin(keys, gathered, keep, sinks=sinks, recent=recent)
        left = [min(int(n), keep) for n in used]
        assert [arena.tokens(key) for key in keys] == left
        for layer in range(layers):
            for s, (key, n) in enumerate(zip(keys, used)):
                got, scale = held(arena, arena.capacity_rows(key)[:left[s]], layer)
                for h in range(hk):
                    w = gathered[layer, s, h].tolist()
                    slots = kept_slots(w, int(n), keep, sinks, recent)
                    assert kept[layer, s, h, :left[s]].tolist() == slots
                    assert weights[layer, s, h].tolist() == [w[i] for i in slots] + [0.0] * (cols - left[s])
                    off = 2.0 ** -10 * scale[:, :, h] if bits == 8 else 0
                    assert bool(((got[:, :, h] - before[key, layer][:, slots, h]).abs() <= off).all())
        assert [arena.is_thinned(key) for key in keys] == [True, True, step == 4]
        new = [[1, 1, 1], [20, 3, 40], [17, 33, 5], [2, 0, 19]][step % 4]


def test_tokens_of_a_captured_step():
    """One graph that rotates a token of each sequence, writes, reads and gathers
    it and thins, replayed with lengths and positions as they then are; the same
    steps run eagerly over an arena of their own give the same bits."""
    g = torch.Generator().manual_seed(3)
    hq, hk, d, keep = 8, 2, 64, 48
    rot = RotaryEmbedding(d, scaling=YARN, max_positions=131072)
    table = torch.randperm(12, generator=g).to(torch.int32).view(3, 4)[:, :4].to(DEV)
    qkv = torch.empty(3, (hq + 2 * hk) * d, dtype=torch.bfloat16, device=DEV)

    class Side:
        def __init__(self):
            self.arena = KVArena(1, 12, PAGE, hk, d)
            self.eng = engine_of(self.arena, hq)
            self.used = torch.tensor([40, 48, 9], dtype=torch.int32, device=DEV)
            self.positions = torch.tensor([90000, 131071, 9], device=DEV)
            self.w = torch.zeros(1, 3, hk, 64, device=DEV)
            self.tables = dict(cu_q=torch.arange(4, dtype=torch.int32, device=DEV), used=self.used,
                               table=table, causal=True, max_q=1, max_used=keep + 1)

        def step(self):
            q, k = rot(self.positions, qkv[:, :hq * d], qkv[:, hq * d:(hq + hk) * d])
            at = self.used.long()
            rows = table.gather(1, (at // PAGE)[:, None])[:, 0].long() * PAGE + at % PAGE
            self.used.add_(1)
            self.eng.kv_row_scatter(k.view(3, hk, d), qkv[:, (hq + hk) * d:].view(3, hk, d),
                                    torch.arange(3, device=DEV), rows, 0)
            out, lse = self.eng.read_pages(q.view(3, hq, d), self.tables, 0)
            self.eng.key_weights(q.view(3, hq, d), lse, self.tables, 0, weights=self.w[0], out=self.w[0])
            kept, w = self.arena.thin_rows(self.tables, self.w, keep, sinks=2, recent=4)
            self.w.copy_(w)
            self.used.clamp_(max=keep)
            self.positions.add_(1)
            return out, lse, kept

    start = (torch.randn(12 * PAGE, hk, d, generator=g).to(DEV), torch.randn(12 * PAGE, hk, d, generator=g).to(DEV))
    captured, eager = Side(), Side()
    for side in (captured, eager):
        for pool, x in zip(side.arena.layer_kv(0), start):
            pool.copy_(x)
    qkv.copy_(torch.randn(qkv.shape, generator=g))
    saved = [t.clone() for t in (captured.used, captured.positions, captured.w)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        captured.step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = captured.step()
    for t, x in zip((captured.used, captured.positions, captured.w), saved):
        t.copy_(x)
    for pool, x in zip(captured.arena.layer_kv(0), start):
        pool.copy_(x)
    for _ in range(12):
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        graph.replay()
        want = eager.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(captured.w, eager.w) and captured.used.tolist() == eager.used.tolist()
        for a, b in zip(captured.arena.layer_kv(0), eager.arena.layer_kv(0)):
            assert torch.equal(a, b)
    assert captured.used.tolist() == [48, 48, 21] and captured.positions.tolist() == [90012, 131083, 21]
