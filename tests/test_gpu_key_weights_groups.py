"""Accumulated key weights of wide head groups and far rows on the GPU: groups that
take a step of columns by themselves (33 to 64 heads, and more), and items of more
rows than their bytes are counted for at once. Bounds as in
tests/test_gpu_key_weights.py; the log-sum-exps are the definition's, rounded to
fp32."""

import numpy as np
import pytest
import torch

from tests.test_gpu_key_weights import check, keys_of, make
from tests.test_gpu_kv8 import engine_of, sequences

pytestmark = pytest.mark.gpu

DEV = "cuda"


def lse_of(q, arena, cu_q, used, table, causal):
    """(hq, rows) fp32 from scores in 64 bits; -inf of rows that see no key."""
    n, hq, d = q.shape
    hk = arena.kv_shape[0]
    lse = torch.full((hq, n), -torch.inf)
    for s, keys in enumerate(used):
        rows = slice(int(cu_q[s]), int(cu_q[s + 1]))
        count = rows.stop - rows.start
        if not keys or not count:
            continue
        k = keys_of(arena, table[s], int(keys))
        last = keys - count + torch.arange(count) if causal else torch.full((count,), keys - 1)
        hidden = torch.arange(int(keys)) > last[:, None]
        for h in range(hq):
            score = q[rows, h].double() @ k[:, h * hk // hq].t() * d ** -0.5
            lse[h, rows] = score.masked_fill(hidden, -torch.inf).logsumexp(-1).float()
    return lse


HEADS = [(40, 1, 64), (64, 1, 128), (65, 1, 64), (130, 1, 64), (80, 2, 128), (260, 2, 64), (192, 3, 64)]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("hq,hk,d", HEADS)
@pytest.mark.parametrize("q_lens,used,causal", [
    ((1, 1), (1, 290), True), ((2, 5, 0), (129, 40, 7), True), ((5, 3), (130, 2), True), ((4,), (300,), False),
    ((70, 33), (300, 90), True), ((70, 33), (300, 20), True), ((40, 3), (513, 90), False), ((300,), (300,), True)])
def test_wide_groups(bits, hq, hk, d, q_lens, used, causal):
    g = torch.Generator().manual_seed(hq + sum(used))
    pages = sum(-(-u // 16) for u in used) + 2
    arena = make(pages, hk, d, bits, g)
    eng = engine_of(arena, hq)
    cu_q, used, table = sequences(g, q_lens, used, pages, 1)
    q = torch.randn(int(cu_q[-1]), hq, d, generator=g).to(torch.bfloat16)
    lse = lse_of(q, arena, cu_q, used, table, causal).to(DEV)
    tables = dict(cu_q=torch.from_numpy(cu_q).to(DEV), used=torch.from_numpy(used).to(DEV),
                  table=torch.from_numpy(table).to(DEV), causal=causal, max_q=max(q_lens), max_used=int(used.max()))
    prior = torch.rand(len(used), hk, table.shape[1] * 16, generator=g).to(DEV)
    q = q.to(DEV)
    got = eng.key_weights(q, lse, tables, 0, weights=prior)
    check(got, q, lse, arena, cu_q, used.tolist(), table, causal, prior)
    assert torch.equal(eng.key_weights(q, lse, tables, 0, weights=prior), got)


@pytest.mark.parametrize("bits", [16, 8])
def test_items_of_more_rows_than_are_counted_at_once(bits):
    """Rows 2^18 elements apart: 32 bits of bytes reach 4096 of them, and a tile that all
    5000 rows see is one item for the workgroup that has it whole (64 heads of a group of
    one: 64 x 24 tiles of up to 87 groups in shares of 204 and 123, 256 such items)."""
    g = torch.Generator().manual_seed(9)
    hq, d, n, keys = 64, 64, 5000, 6000
    pages = keys // 16 + 3
    arena = make(pages, hq, d, bits, g)
    eng = engine_of(arena, hq)
    cu_q, used, table = sequences(g, (n,), (keys,), pages, 0)
    wide = torch.empty(n, 2 ** 18, dtype=torch.bfloat16, device=DEV)
    part = wide[:, 512:512 + hq * d]
    part.copy_(torch.randn(n, hq * d, generator=g))
    q = part.unflatten(1, (hq, d))
    tables = dict(cu_q=torch.from_numpy(cu_q).to(DEV), used=torch.from_numpy(used).to(DEV),
                  table=torch.from_numpy(table).to(DEV), causal=True, max_q=n, max_used=keys)
    near = q.contiguous()
    _, lse = eng.read_pages(near, tables, 0)
    got = eng.key_weights(q, lse, tables, 0)
    # (the rows side by side: one item a tile, the same groups, the sums in another order)
    again = eng.key_weights(near, lse, tables, 0)
    assert torch.allclose(got, again, rtol=(2 * n / 32 + 40) * 2.0 ** -24, atol=0)
    one = got[:, :1]
    for h in (0, 17, 63):
        class Head:
            eight_bit, kv_shape = arena.eight_bit, (1, d)

            @staticmethod
            def layer_kv(layer):
                return (arena.layer_kv(layer)[0][:, h:h + 1],)

            @staticmethod
            def layer_scales(layer):
                return arena.layer_scales(layer)[:, h:h + 1]

        one = got[:, h:h + 1]
        check(one, near[:, h:h + 1], lse[h:h + 1], Head, cu_q, used.tolist(), table, True)
    assert np.isfinite(float(one.sum()))
