"""The 8-bit KV arena's host side: page items of a pack's writes, compaction
and forks in the page accounting, and what the entry points refuse. No GPU."""

import numpy as np
import pytest
import torch

from oracle import kv8_ref as ref
from quail_amd import _lib
from quail_amd.arena import FP8, KVArena
from quail_amd.chunk import attention_plan, pack_chunk, page_writes
from quail_amd.pages import PageArena

PAGE = 16


def apply_items(phases, pool):
    """The pool rows (row -> content) after the items, by their definition;
    each page is a destination once per phase and no source of that phase."""
    for items in phases:
        dst = items[:, 0].tolist()
        assert len(set(dst)) == len(dst)
        assert not {s for d, s in items[:, :2].tolist() if s != d} & set(dst)
        before = dict(pool)
        for d, s, keep, row0, count in items.tolist():
            assert 0 <= keep and 0 < count and keep + count <= PAGE
            for r in range(keep):
                if s != d:
                    pool[d * PAGE + r] = before.get(s * PAGE + r)
            for r in range(count):
                pool[d * PAGE + keep + r] = ("row", row0 + r)
    return pool


def apply_scatter(src, dst, tail_src, tail_dst, pool):
    for s, d in zip(src, dst):
        if d >= 0:
            pool[int(d)] = ("row", int(s))
    if tail_src is not None:
        got = {int(d): pool.get(int(s)) for s, d in zip(tail_src, tail_dst)}
        pool.update(got)
    return pool


def test_page_writes_of_runs_that_share_pages_go_in_order():
    # rows 0..9 at slots 3..12 of page 4, rows 10..12 at 13..15, rows 20.. into page 2
    dst = np.r_[67:77, 77:80, 32:40]
    src = np.r_[0:10, 10:13, 20:28]
    phases = page_writes(src, dst)
    assert [p.tolist() for p in phases] == [[[4, 4, 3, 0, 13], [2, 2, 0, 20, 8]]]
    # the second run of page 4 comes from other rows: a phase of its own
    src[10:13] = [15, 16, 17]
    phases = page_writes(src, dst)
    assert [p.tolist() for p in phases] == [[[4, 4, 3, 0, 10], [2, 2, 0, 20, 8]],
                                            [[4, 4, 13, 15, 3]]]
    assert page_writes([], []) == ()
    assert page_writes([1, 2], [-1, -1]) == ()
    # unwritten rows break no run of the others
    assert page_writes([0, 1, 2], [5, -1, 6])[0].tolist() == [[0, 0, 5, 0, 1]]


def test_page_writes_refuse_what_a_page_scale_cannot_hold():
    with pytest.raises(ValueError, match="rising order"):
        page_writes([5, 6, 0], [8, 9, 0])          # slot 0 would drop slots 8 and 9
    with pytest.raises(ValueError, match="slots"):
        page_writes([0], [33], [2, 3], [32, 34])
    with pytest.raises(ValueError, match="one run"):
        page_writes([0], [40], [2], [82])           # a copied page no row follows
    with pytest.raises(ValueError, match="one run"):
        page_writes([0], [40], [2], [34])           # slots 3 to 7 of the copy are missing


@pytest.mark.parametrize("seed", range(6))
def test_packs_page_items_write_what_their_scatter_writes(seed):
    """Seeded packs (prefixes, several questions with copied partial pages,
    kept documents): the items, applied by their definition, leave the rows
    that the scatter and the tail copy leave."""
    rng = np.random.default_rng(seed)
    arena = KVArena(1, 400, PAGE, 2, 64, dtype=FP8, device="cpu")
    groups, kept = [], {}
    for d in range(8):
        f = int(rng.integers(1, 90))
        n_suf = int(rng.integers(1, 4))
        suf = [rng.integers(0, 99, int(rng.integers(1, 30))) for _ in range(n_suf)]
        extra = len(suf[0]) if n_suf == 1 else 0
        start = 0
        if d % 3 == 2:      # a document whose first rows an earlier pass wrote
            start = int(rng.integers(0, f))
        assert arena.activate(d, f, capacity_tokens=f + extra) is not None
        for row in arena.capacity_rows(d)[:start]:
            kept[int(row)] = ("kept", d, int(row))
        prefix = None if d % 3 == 1 else rng.integers(0, 99, f - start)
        if prefix is None:
            for row in arena.capacity_rows(d)[:f]:
                kept[int(row)] = ("kept", d, int(row))
        groups.append(dict(key=d, prefix=prefix, f=f, start=start, suffixes=suf))
    chunk = pack_chunk(arena, groups)
    u = chunk.meta["unified"]
    want = apply_scatter(u["src"], u["dst"], u["tail_src"], u["tail_dst"], dict(kept))
    got = apply_items(u["page_writes"], dict(kept))
    assert {r: v for r, v in got.items() if v is not None} == want
    rows = np.concatenate([np.arange(r, r + c) for p in u["page_writes"]
                           for _, _, _, r, c in p.tolist()])
    assert sorted(rows.tolist()) == list(range(chunk.tokens))
    # a 16-bit arena's packs carry none
    plain = KVArena(1, 400, PAGE, 2, 64, device="cpu")
    for g in groups:
        plain.activate(g["key"], g["f"])
    assert "page_writes" not in pack_chunk(plain, groups).meta["unified"]


def test_attention_items_cover_every_key_of_every_tile():
    import ctypes

    def items(q_lens, used, hq=32, hk=8, causal=1):
        cu_q = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        used = np.asarray(used, dtype=np.int32)
        unit = ctypes.c_int64()
        _lib.call("qx_paged_attention8_unit", cu_q.ctypes.data, used.ctypes.data, len(used), hq, hk,
                  causal, ctypes.byref(unit))
        work = np.zeros(2 * 8192, dtype=np.int32)

        def fill(cap):
            return _lib.count("qx_paged_attention8_work", cu_q.ctypes.data, used.ctypes.data,
                              len(used), hq, hk, causal, unit.value, work.ctypes.data, cap)
        n = fill(8192)
        with pytest.raises(_lib.QxError, match="room"):
            fill(n - 1)
        return unit.value, [(int(s), int(p) & 0xffff, int(p) >> 16)
                            for s, p in work[:2 * n].reshape(-1, 2)]

    # few rows a sequence: splits of their keys
    used = [300, 0, 8192, 5, 40000]
    unit, got = items([1, 2, 3, 0, 1], used)
    assert unit and unit % 128 == 0
    assert sorted(got) == [(s, i, 0) for s, u in enumerate(used) if s != 3
                           for i in range(max(1, -(-u // unit)))]
    load = [min(unit, used[s] - i * unit) for s, i, _ in got]
    assert load == sorted(load, reverse=True)
    # whole query tiles
    unit, got = items([100, 1, 33], [150, 40, 33])
    assert unit == 0
    assert sorted(got) == [(s, t, 0) for s, t in ((0, 0), (0, 1), (0, 2), (0, 3), (1, 0), (2, 0),
                                                  (2, 1))]
    unit, got = items([100, 1], [150, 40], hq=16)       # two heads a KV head: 64 rows
    assert unit == 0 and sorted(got) == [(0, 0, 0), (0, 1, 0), (1, 0, 0)]
    # tiles whose keys are split: one long sequence among short ones
    q_lens, used = [40, 21, 21, 0], [20000, 900, 70, 10]
    unit, got = items(q_lens, used)
    assert unit < 0 and unit % 64 == 0
    want = []
    for s, (q, u) in enumerate(zip(q_lens, used)):
        for t in range(-(-q // 32)):
            keys = u - q + min(32 * t + 32, q)
            want += [(s, t, i) for i in range(-(-keys // -unit))]
    assert sorted(got) == sorted(want)
    # many rows of equal length: nothing to even out
    assert items([8000, 8000], [8100, 8100])[0] == 0


def test_scale_bytes_and_codes_of_the_oracle():
    assert [ref.scale_byte(a) for a in (0.0, 448.0, 448.1, 1.75, 1.76, 3.5e-38)] == \
        [1, 127, 128, 119, 120, 1]
    table = torch.arange(256, dtype=torch.uint8).view(FP8).double()
    table = table[torch.isfinite(table)]
    assert torch.equal(ref.codes_of(table, torch.tensor(127)).double(), table)
    x = torch.tensor([17.0, 19.0, 2.0 ** -10, 1.5 * 2.0 ** -9, 500.0, -23.0])
    assert ref.codes_of(x.double(), torch.tensor(127)).float().tolist() == \
        x.clamp(-448, 448).to(FP8).float().tolist()


def test_arena_types_and_sizes():
    arena = KVArena(3, 5, PAGE, 2, 64, dtype=FP8, device="cpu")
    assert arena.eight_bit and arena.v_dtype == FP8
    k, v = arena.layer_kv(2)
    assert k.dtype == v.dtype == FP8 and k.shape == (80, 2, 64)
    assert arena.layer_scales(1).shape == (5, 2, 2)
    plain = KVArena(1, 5, PAGE, 2, 64, device="cpu")
    assert not plain.eight_bit and plain.scales is None and plain.v_dtype == torch.float16
    for bad in (dict(dtype=torch.float16), dict(dtype=FP8, v_dtype=torch.bfloat16),
                dict(v_dtype=FP8)):
        with pytest.raises(ValueError):
            KVArena(1, 5, PAGE, 2, 64, device="cpu", **bad)
    with pytest.raises(ValueError, match="16 rows"):
        KVArena(1, 5, 32, 2, 64, dtype=FP8, device="cpu")
    with pytest.raises(ValueError, match="16 rows"):
        KVArena(1, 5, PAGE, 2, 96, dtype=FP8, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        arena.copy_pages([0], [1])
    with pytest.raises(ValueError, match="GPU"):
        arena.compact()
    with pytest.raises(ValueError, match="destinations"):
        arena.copy_pages([0], [1, 2])


def test_compaction_gives_the_lowest_ids_and_keeps_every_table():
    """Tables name the same contents after the moves; borrowed pages move
    once for all their holders; the free stack goes on in rising order."""
    rng = np.random.default_rng(3)
    acct = PageArena(60, PAGE)
    for k in range(12):
        acct.alloc(k, int(rng.integers(1, 60)))
    acct.alloc("child", 40, borrowed=acct.shared_pages(7, 16) if acct.key_tokens(7) >= 16 else ())
    for k in (0, 3, 4, 8, 11):
        acct.free_key(k)
    acct.retain(5)
    content = {p: ("page", p) for p in range(60)}
    want = {k: [content[p] for p in acct.table_pages(k)] for k in acct.resident_keys()}
    free, retained = acct.free_pages, acct.retained_pages
    src, dst = acct.compact()
    assert len(src) == len(dst) == len(set(dst)) and not set(src) & set(dst)
    for s, d in zip(src, dst):
        assert d < s
        content[d] = content[s]
    assert {k: [content[p] for p in acct.table_pages(k)] for k in acct.resident_keys()} == want
    live = {p for k in acct.resident_keys() for p in acct.table_pages(k)}
    assert live == set(range(60 - free))
    assert acct.free_pages == free and acct.retained_pages == retained
    assert acct.alloc("new", 3 * PAGE) == [60 - free, 61 - free, 62 - free]
    assert acct.compact() == ([], [])
    # the moved pages are freed as any
    for k in list(acct.resident_keys()):
        acct.free_key(k)
    assert acct.free_pages == 60


def test_compaction_is_refused_while_packs_name_the_pages():
    acct = PageArena(10, PAGE)
    acct.alloc("a", 20)
    acct.pin("a")
    with pytest.raises(ValueError, match="pinned"):
        acct.compact()
    arena = KVArena(1, 10, PAGE, 2, 64, dtype=FP8, device="cpu")
    arena.hold("a", 2)
    with pytest.raises(ValueError, match="held"):
        arena.compact()


def test_fork_shares_full_pages_and_refuses_what_it_cannot_hold():
    arena = KVArena(1, 8, PAGE, 2, 64, dtype=FP8, device="cpu")
    arena.alloc("doc", 32)
    pages = arena.fork("doc", ["a", "b"], capacity_tokens=50)
    assert arena.owned_pages("a")[:2] == arena.owned_pages("doc")[:2] == arena.owned_pages("b")[:2]
    assert len(pages[0]) == len(pages[1]) == 2 and not set(pages[0]) & set(pages[1])
    assert arena.tokens("a") == 32
    assert arena.fork("doc", ["c"], capacity_tokens=100) is None     # 2 pages left
    assert not arena.is_resident("c")
    assert arena.fork("doc", []) == []
    assert arena.fork("doc", ["whole"], tokens=16)[0] == [] and arena.tokens("whole") == 16
    with pytest.raises(ValueError, match="once"):
        arena.fork("doc", ["x", "x"])
    with pytest.raises(ValueError, match="holds 32"):
        arena.fork("doc", ["x"], tokens=33)
    with pytest.raises(ValueError, match="capacity"):
        arena.fork("doc", ["x"], capacity_tokens=31)
    with pytest.raises(KeyError):
        arena.fork("doc", ["a"])
    with pytest.raises(KeyError):
        arena.fork("nobody", ["x"])
    # the parent's pages outlive it while a child reads them
    arena.free_key("doc")
    arena.free_key("whole")
    assert arena.free_pages == 8 - 6
    arena.free_key("a")
    arena.free_key("b")
    assert arena.free_pages == 8


def test_entry_points_refuse_bad_arguments():
    def attend(**kw):
        a = dict(q=16, q_ld=4096, k=16, v=16, s=16, cu=16, used=16, table=16, tld=8, seqs=1, rows=1,
                 mq=1, mu=64, hq=32, hk=8, d=128, page=16, out=16, out8=None, o_ld=4096, os=None,
                 os_ld=0, lse=None, lse_ld=0, work=None, n_work=0, unit=0, ws=None,
                 wsb=0, pos=None, cs=16, qw=16)
        a.update(kw)
        _lib.call("qx_paged_attention8", a["q"], a["q_ld"], None, a["k"], a["v"], a["s"], a["cu"],
                  a["used"], a["table"], a["tld"], a["seqs"], a["rows"], a["mq"], a["mu"], a["hq"],
                  a["hk"], a["d"], a["page"], 0.1, 1, a["out"], a["out8"], a["o_ld"], a["os"],
                  a["os_ld"], a["lse"], a["lse_ld"], a["work"], a["n_work"], a["unit"], a["ws"],
                  a["wsb"], a["pos"], a["cs"], 0, a["qw"], 1e-6, None)

    for kw, match in ((dict(q=None), "null"), (dict(table=None), "null"), (dict(out=None), "output"),
                      (dict(out8=16), "output"), (dict(d=96), "head_dim"), (dict(hk=5), "heads"),
                      (dict(page=32), "page"), (dict(mu=40961), "at most"), (dict(seqs=-1), "seq"),
                      (dict(out=None, out8=16), "e4m3"),
                      (dict(out=None, out8=16, os=16, os_ld=1, d=64), "e4m3"),
                      (dict(q_ld=4095), "strides"), (dict(lse=16, lse_ld=0), "strides"),
                      (dict(q=18), "alignment"), (dict(k=17), "alignment"),
                      (dict(seqs=65536), "grid"), (dict(mu=40000), "workspace"),
                      (dict(mu=40000, ws=16, wsb=100), "workspace"),
                      (dict(work=16, n_work=-1), "work"), (dict(work=16, n_work=1 << 24), "work"),
                      (dict(pos=16, d=64), "q-norm"),
                      (dict(pos=16, cs=None), "q-norm"), (dict(pos=16, qw=8), "q-norm"),
                      (dict(unit=128), "items"), (dict(work=16, n_work=1, unit=100), "items"),
                      (dict(work=16, n_work=1, unit=8192), "items"),
                      (dict(work=16, n_work=1, unit=-100), "items"),
                      (dict(work=16, n_work=1, unit=-64, mu=256), "workspace"),
                      (dict(work=16, n_work=1, unit=128, mu=256), "workspace")):
        with pytest.raises(_lib.QxError, match=match):
            attend(**kw)
    space = lambda *a: _lib.count("qx_paged_attention8_workspace", 1, 1, *a)  # noqa: E731
    assert space(1, 40000, 32, 8, 128, 0, 0) > 0
    assert space(1, 64, 32, 8, 128, 0, 0) == 0
    assert space(1, 512, 32, 8, 128, 1, 128) == 4 * 32 * 130 * 4
    assert space(1000, 40000, 32, 8, 128, 1, 0) == 0
    attend(seqs=0)
    attend(rows=0)

    def write(*, k=16, k_ld=1024, items=16, n=1, hk=8, d=128):
        _lib.call("qx_kv8_write", k, k_ld, 16, 1024, 16, 16, 16, items, n, hk, d, None)

    for kw, match in ((dict(k=None), "null"), (dict(items=None), "null"), (dict(k_ld=1022), "strides"),
                      (dict(k=12), "alignment"), (dict(d=80), "head_dim"), (dict(hk=0), "heads"),
                      (dict(n=1 << 26), "one launch")):
        with pytest.raises(_lib.QxError, match=match):
            write(**kw)
    write(n=0)
    with pytest.raises(_lib.QxError, match="null"):
        _lib.call("qx_qk_norm_rope_kv8", 16, 8, None, 0, 16, 16, 16, 16, 1, None, 0, 16, 16, 16, 4,
                  2, 64, 1e-6, None)

    def copy(src, dst, *, pages=8, page_bytes=256, n_scales=0, scales=None, scale_bytes=0):
        ids = lambda x: np.asarray(x, dtype=np.int32)  # noqa: E731
        s, d = ids(src), ids(dst)
        _lib.call("qx_copy_pages", 16, 2, 4096, page_bytes, scales, n_scales, 64, scale_bytes,
                  s.ctypes.data, d.ctypes.data, len(s), pages, None)

    for args, kw, match in ((([0], [8]), {}, "of 8"), (([-1], [2]), {}, "of 8"),
                            (([1, 2], [3, 3]), {}, "twice"), (([1, 2], [2, 3]), {}, "source"),
                            (([2, 1], [3, 2]), {}, "source"), (([4], [4]), {}, "page 4"),
                            (([0], [1]), dict(page_bytes=24), "sizes"),
                            (([0], [1]), dict(n_scales=1), "null"),
                            (([0], [1]), dict(n_scales=1, scales=16, scale_bytes=3), "sizes")):
        with pytest.raises(_lib.QxError, match=match):
            copy(*args, **kw)
    copy([], [])


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("inf")])
def test_attention_refuses_scales_that_are_not_positive(scale):
    with pytest.raises(_lib.QxError, match="scale"):
        _lib.call("qx_paged_attention8", 16, 4096, None, 16, 16, 16, 16, 16, 16, 8, 1, 1, 1, 64, 32, 8,
                  128, 16, scale, 1, 16, None, 4096, None, 0, None, 0, None, 0, 0, None, 0, None, None,
                  0, None, 1e-6, None)


def test_what_a_cpu_arena_cannot_copy_changes_nothing():
    arena = KVArena(1, 8, PAGE, 2, 64, dtype=FP8, device="cpu")
    arena.alloc("doc", 20)
    with pytest.raises(ValueError, match="CPU"):
        arena.fork("doc", ["a", "b"])                # the partial page needs a copy
    assert not arena.is_resident("a") and not arena.is_resident("b") and arena.free_pages == 6
    for src, dst in (([0], [1 << 32]), ([(1 << 32) + 1], [2]), ([-1], [2])):
        with pytest.raises(ValueError, match="of 8|CPU"):
            arena.copy_pages(src, dst)


def test_an_attention_plan_names_what_it_was_made_for():
    ints = lambda *a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    plan = attention_plan(ints(0, 1, 3), ints(20, 5), ints(1, 2, 3, 0).view(2, 2), heads=(4, 2, 64))
    assert plan["made_for"] == (3, 4, 2, 64, True)


def test_an_attention_plan_checks_the_pages_that_are_read():
    ints = lambda *a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    table = ints(1, 7, -1, 3, 99, -5).view(2, 3)
    plan = attention_plan(ints(0, 1, 2), ints(32, 16), table, heads=(4, 2, 64))
    assert plan["pages"] == 8                        # entries past a sequence's keys are not read
    with pytest.raises(ValueError, match="page -1"):
        attention_plan(ints(0, 1, 2), ints(33, 16), table, heads=(4, 2, 64))
    assert attention_plan(ints(0, 1, 2), ints(0, 0), table, heads=(4, 2, 64))["pages"] == 0
