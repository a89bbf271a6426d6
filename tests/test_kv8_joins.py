"""What joining the splits of an 8-bit call costs: scratch rows and joins of
packs that mix a few rows over long keys with many rows. No GPU."""

import numpy as np
import pytest

from quail_amd import _lib
from quail_amd.chunk import _work_list8


def plan(q_lens, used, heads=(32, 8, 128), causal=True):
    cu_q = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    used = np.asarray(used, dtype=np.int32)
    work, n, unit, (n_joins, rows) = _work_list8(dict(cu_q=cu_q, used=used, causal=causal), heads)
    assert len(work) == 3 * n + 4 * n_joins
    return cu_q, work[:2 * n].reshape(-1, 2), work[2 * n:3 * n], work[3 * n:].reshape(-1, 4), unit, rows


def documents(n, seed=4):
    rng = np.random.default_rng(seed)
    return np.clip(np.rint(rng.lognormal(np.log(256), 0.8, n)), 32, 2048).astype(int).tolist()


MIXED = [  # (query rows, keys) of each sequence, heads, the rows that are split
    ([*documents(46), 21], [*(d + 64 for d in documents(46)), 8000], (32, 8, 128), 21),
    ([*documents(46), 21], [*(d + 64 for d in documents(46)), 40000], (32, 8, 128), 21),
    ([*documents(46), 21], [*(d + 64 for d in documents(46)), 40000], (64, 8, 128), 21),
    ([16] * 900 + [2000, 21], [80] * 900 + [2000, 40000], (32, 8, 128), 21),
    ([250] * 60 + [21], [250] * 60 + [40000], (32, 8, 128), 21),
    ([12] * 1000 + [500], [64] * 1000 + [40000], (32, 8, 128), 500),
]


@pytest.mark.parametrize("case", range(len(MIXED)))
def test_scratch_and_joins_follow_what_is_split(case):
    q_lens, used, heads, split_rows = MIXED[case]
    cu_q, items, slots, joins, unit, rows = plan(q_lens, used, heads)
    assert unit < 0
    bytes_ = rows * heads[0] * (heads[2] + 2) * 4
    print(unit, len(joins), rows, bytes_ / 1e6, "MB")
    first = int(cu_q[-1]) - q_lens[-1]
    long = joins[joins[:, 0] >= first]
    assert long[:, 1].sum() == split_rows
    # only tiles of more keys than a split holds; their splits' rows, nothing else
    assert rows == int((joins[:, 1] * joins[:, 3]).sum())
    assert bytes_ <= 128 << 20


@pytest.mark.parametrize("hq,hk", [(32, 8), (16, 8), (8, 8), (24, 8), (64, 8)])
@pytest.mark.parametrize("q_lens,used,causal", [
    ([1, 2, 3, 0, 1], [300, 0, 8192, 5, 40000], True),
    ([1, 1], [100, 50], True),
    ([40, 21, 21, 0], [20000, 900, 70, 10], True),
    ([70, 33, 1], [9000, 6000, 40000], False),
    ([130, 3], [100, 20000], True),
    ([100, 1, 33], [150, 40, 33], True),
    ([], [], True)])
def test_every_part_of_a_split_tile_has_rows_of_its_own(hq, hk, q_lens, used, causal):
    cu_q, items, slots, joins, unit, rows = plan(q_lens, used, (hq, hk, 128), causal)
    g = hq // hk
    height = 32 if g % 4 == 0 else 64 if g % 2 == 0 else 128
    taken, want_joins = np.zeros(rows, dtype=int), set()
    for (s, part), slot in zip(items.tolist(), slots.tolist()):
        q = q_lens[s]
        tile, split = (0, part) if unit > 0 else (part & 0xffff, part >> 16)
        row0, here = (0, q) if unit > 0 else (tile * height, min(height, q - tile * height))
        keys = used[s]
        if unit <= 0 and causal:
            keys = min(keys, max(0, used[s] - q + row0 + here))
        if not unit or keys <= abs(unit):
            assert slot == -1 and split == 0
            continue
        parts = -(-keys // abs(unit))
        taken[slot:slot + here] += 1
        want_joins.add((int(cu_q[s]) + row0, here, slot - split * here, parts))
    assert (taken == 1).all()
    assert {tuple(j) for j in joins.tolist()} == want_joins and len(joins) == len(want_joins)


def test_joins_refuse_lists_of_another_call_and_too_little_room():
    cu_q, items, slots, joins, unit, rows = plan([40, 21], [20000, 900])
    used = np.asarray([20000, 900], dtype=np.int32)
    out, found = np.zeros(len(items), dtype=np.int32), np.zeros(1, dtype=np.int64)
    room = np.zeros((len(items), 4), dtype=np.int32)

    def call(work, cap=len(items), seqs=2, unit=unit, hk=8):
        work = np.ascontiguousarray(work, dtype=np.int32)
        return _lib.count("qx_paged_attention8_joins", cu_q.ctypes.data, used.ctypes.data, seqs, 32,
                          hk, 1, unit, work.ctypes.data, len(work), out.ctypes.data,
                          room.ctypes.data, cap, found.ctypes.data)

    assert call(items) == len(joins) and found[0] == rows
    with pytest.raises(_lib.QxError, match="room"):
        call(items, cap=len(joins) - 1)
    for bad in ([2, 0], [-1, 0], [0, 7], [0, 300 << 16]):
        with pytest.raises(_lib.QxError, match="none of this call"):
            call([bad])
    with pytest.raises(_lib.QxError, match="arguments"):
        call(items, hk=5)

    def attend(**kw):
        a = dict(work=16, n_work=2, unit=-64, slots=16, joins=16, n_joins=1, rows=2, ws=16,
                 size=2 * 32 * 130 * 4)
        a.update(kw)
        _lib.call("qx_paged_attention8_joined", 16, 4096, None, 16, 16, 16, 16, 16, 16, 8, 1, 1, 1,
                  256, 32, 8, 128, 16, 0.1, 1, 16, None, 4096, None, 0, None, 0, a["work"],
                  a["n_work"], a["unit"], a["slots"], a["joins"], a["n_joins"], a["rows"], a["ws"],
                  a["size"], None, None, 0, None, 1e-6, None)

    for kw, match in ((dict(work=None), "null"), (dict(slots=None), "null"), (dict(joins=None), "joins"),
                      (dict(n_joins=65536), "joins"), (dict(n_joins=-1), "joins"),
                      (dict(rows=0), "joins"), (dict(rows=1 << 31), "joins"),
                      (dict(n_joins=0), "joins"), (dict(ws=None), "workspace"),
                      (dict(size=2 * 32 * 130 * 4 - 1), "workspace"), (dict(unit=-100), "items")):
        with pytest.raises(_lib.QxError, match=match):
            attend(**kw)


@pytest.mark.parametrize("hq,hk,unit,most", [(64, 8, 128, 1 << 21), (32, 8, 0, 1 << 21), (8, 8, 0, 1 << 21),
                                             (128, 8, -64, 1 << 19)])
def test_items_are_refused_where_a_launch_ends_and_not_before(hq, hk, unit, most):
    """2^24 workgroups of 256 threads; what comes next in the checks, the
    missing scratch memory or joins, says that the items were taken."""
    def attend(n_work):
        _lib.call("qx_paged_attention8_joined", 16, 16384, None, 16, 16, 16, 16, 16, 16, 8, 1, 1, 1,
                  256, hq, hk, 128, 16, 0.1, 1, 16, None, 16384, None, 0, None, 0, 16, n_work, unit,
                  16, None, 1, 1, None, 0, None, None, 0, None, 1e-6, None)

    with pytest.raises(_lib.QxError, match="joins"):
        attend(most - 1)
    for n in (most, 1 << 60, -1):
        with pytest.raises(_lib.QxError, match="work items"):
            attend(n)
