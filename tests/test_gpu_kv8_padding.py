"""The 8-bit page write of a padded batch: rows that go to no page."""

import numpy as np
import pytest
import torch

from quail_amd.chunk import page_writes
from tests.test_gpu_kv8 import DEV, _Attn, engine_arena, engine_of, fill, rope_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hk,d", [(32, 8, 128), (6, 2, 128), (24, 8, 64)])
def test_padding_rows_get_their_q_and_touch_no_page(hq, hk, d):
    """q of every row as the pass without pages writes it; the pages as the
    batch without its padding leaves them."""
    g = torch.Generator().manual_seed(81)
    n = 40
    dst = np.arange(n) + 19
    dst[[3, 4, 17, 30]] = -1
    dst[36:] = -1
    qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g).to(torch.bfloat16).to(DEV)
    pos = torch.arange(n, device=DEV)
    attn, cache = _Attn(d, g), rope_cache(n, d, torch.bfloat16)
    arenas = [engine_arena(5, hk, d) for _ in range(2)]
    for arena, rows in zip(arenas, (n, None)):
        fill(arena, torch.Generator().manual_seed(82))
        eng = engine_of(arena, hq, cache)
        items = tuple(torch.from_numpy(p).to(DEV) for p in page_writes(np.arange(n), dst, rows=rows))
        meta = dict(layer=0, unified=dict(page_writes=items))
        if rows is None:
            eng.kv_norm_rope(qkv, pos, attn, meta) if d == 128 else \
                eng.qk_norm_rope_kv(qkv, pos, attn, meta)
        else:
            q = eng.qk_norm_rope_kv(qkv, pos, attn, meta)
            eng.write_kv(None, None, meta)      # nothing left to write
    want, _ = eng.qk_norm_rope(qkv, pos, attn)
    assert torch.equal(q, want.view_as(q))
    for a, b in zip((*arenas[0].layer_kv(0), arenas[0].layer_scales(0)),
                    (*arenas[1].layer_kv(0), arenas[1].layer_scales(0))):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    # from K and V rows the items of page -1 write nothing
    eng = engine_of(arenas[0], hq, cache)
    items = torch.tensor([(-1, -1, 0, 0, 16)], dtype=torch.int32, device=DEV)
    x = torch.ones(16, hk, d, dtype=torch.bfloat16, device=DEV)
    eng._write_page_rows(x, x, (items,), 0)
    for a, b in zip(arenas[0].layer_kv(0), arenas[1].layer_kv(0)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
