"""Thinning by token on the CPU: the oracle against its definition, keys that are
thinned after every few tokens, and what the calls refuse."""

import random
import warnings

import pytest
import torch

from oracle.thin_ref import kept_slots, kept_slots_by_token
from quail_amd.arena import KVArena

GROWTHS = [1, 7, 8, 9]      # about a newest of 8


def test_the_oracles_slots_hold_the_protected_tokens_and_the_heaviest_others():
    rng = random.Random(2)
    for _ in range(400):
        used, keep = rng.randrange(0, 30), rng.randrange(0, 30)
        sinks = rng.randrange(0, keep + 1)
        newest = rng.randrange(0, keep - sinks + 1)
        total = used + rng.randrange(0, 40)
        fresh = rng.randrange(0, used + 1)          # rows appended since
        older = rng.sample(range(total - fresh), used - fresh)
        tokens = older + [-1] * fresh
        w = [rng.choice([0.0, 1.0, 2.5, rng.random(), float("nan")]) for _ in range(used)]
        slots, numbers = kept_slots_by_token(w, tokens, total, used, keep, sinks, newest)
        all_numbers = older + list(range(total - fresh, total))
        k = min(used, keep)
        assert len(slots) == len(set(slots)) == k and numbers == [all_numbers[i] for i in slots]
        assert all(i == slot or i >= k for slot, i in enumerate(slots))
        moved = [i for slot, i in enumerate(slots) if i != slot]
        assert moved == sorted(moved)
        safe = {i for i, t in enumerate(all_numbers) if t < sinks or t >= total - newest}
        assert used <= keep or safe <= set(slots)
        key = lambda i: (w[i] != w[i], w[i] if w[i] == w[i] else 0.0, -i)  # noqa: E731
        dropped = set(range(used)) - set(slots)
        for i in set(slots) - safe:
            assert all(key(j) < key(i) for j in dropped)


def test_sequences_not_thinned_before_lose_the_same_rows_either_way():
    rng = random.Random(3)
    for _ in range(200):
        used, keep = rng.randrange(0, 40), rng.randrange(0, 30)
        sinks = rng.randrange(0, keep + 1)
        recent = rng.randrange(0, keep - sinks + 1)
        w = [rng.choice([0.0, 1.0, rng.random()]) for _ in range(used)]
        slots, numbers = kept_slots_by_token(w, [-1] * used, used, used, keep, sinks, recent)
        assert slots == numbers == kept_slots(w, used, keep, sinks, recent)


def thin_on_paper(self, tables, weights, keep, *, sinks=0, recent=0, newest=None, tokens=None):
    """thin_rows after the oracle, without the rows themselves."""
    kept = torch.full((*weights.shape[:3], min(keep, weights.shape[3])), -1, dtype=torch.int32)
    out, left = torch.zeros_like(weights), torch.full_like(weights, -1, dtype=torch.int32)
    for layer, s, h in torch.cartesian_prod(*(torch.arange(n) for n in weights.shape[:3])).tolist():
        w, used = weights[layer, s, h], int(tables["used"][s])
        if newest is None:
            slots = kept_slots(w.tolist(), used, keep, sinks, recent)
        else:
            slots, numbers = kept_slots_by_token(w.tolist(), tokens[layer, s, h].tolist(),
                                                 int(tables["tokens"][s]), used, keep, sinks, newest)
            left[layer, s, h, :len(slots)] = torch.tensor(numbers, dtype=torch.int32)
        kept[layer, s, h, :len(slots)] = torch.tensor(slots, dtype=torch.int32)
        out[layer, s, h, :len(slots)] = w[slots]
    return (kept, out) if newest is None else (kept, out, left)


@pytest.fixture
def arena(monkeypatch):
    monkeypatch.setattr(KVArena, "thin_rows", thin_on_paper)
    return KVArena(2, 40, 16, 2, 64, device="cpu")


def gathered(w, cols, g):
    """Weights after a step: those of the slots and some on every row, the newest least."""
    wide = torch.zeros(*w.shape[:3], cols)
    wide[..., :min(cols, w.shape[3])] = w[..., :cols]
    return wide + torch.rand(wide.shape, generator=g)


@pytest.mark.parametrize("growth", GROWTHS)
def test_the_newest_tokens_of_keys_that_grow_stay(arena, growth):
    """By token number, each row's followed through `kept`: after every thinning a
    head holds the first tokens and the last ones."""
    g = torch.Generator().manual_seed(growth)
    keep, sinks, newest = 32, 3, 8
    keys, totals = ["a", "b"], [50, 20]
    for key, n in zip(keys, totals):
        assert arena.activate(key, n) is not None
    held = {(key, layer, h): list(range(n)) for key, n in zip(keys, totals)
            for layer in range(2) for h in range(2)}
    w = torch.zeros(2, 2, 2, 64)
    for step in range(25):
        if step:
            for s, key in enumerate(keys):
                assert len(arena.append_rows(key, growth)) == growth
                for layer in range(2):
                    for h in range(2):
                        held[key, layer, h] += range(totals[s], totals[s] + growth)
                totals[s] += growth
        w = gathered(w, 64, g)
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            kept, w = arena.thin(keys, w, keep, sinks=sinks, newest=newest)
        for (key, layer, h), numbers in held.items():
            s = keys.index(key)
            slots = kept[layer, s, h]
            numbers[:] = [numbers[i] for i in slots[slots >= 0].tolist()]
            assert len(numbers) == len(set(numbers)) == arena.tokens(key) == min(totals[s], keep)
            assert set(numbers) >= set(range(sinks)) | set(range(totals[s] - newest, totals[s]))
    assert arena.is_thinned("a") and arena.is_thinned("b")


def test_places_are_not_tokens_and_a_thinning_that_counts_them_says_so(arena):
    g = torch.Generator().manual_seed(5)
    arena.activate("a", 40)
    held, total, w = list(range(40)), 40, torch.zeros(2, 1, 2, 64)
    for step in range(12):
        w = gathered(w, 64, g)
        if step == 0:
            with warnings.catch_warnings():
                warnings.simplefilter("error")
                kept, w = arena.thin(["a"], w, 32, recent=8)
        else:
            with pytest.warns(RuntimeWarning, match="grew by 1 rows"):
                kept, w = arena.thin(["a"], w, 32, recent=8)
        held = [held[i] for i in kept[0, 0, 0].tolist()]
        arena.append_rows("a", 1)
        held.append(total)
        total += 1
    assert len(set(range(total - 8, total)) & set(held)) < 8
    # growth of as many rows needs no word
    arena.append_rows("a", 7)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        arena.thin(["a"], gathered(w, 64, g), 32, recent=8)
    # the tokens of its rows were not kept
    arena.append_rows("a", 1)
    with pytest.raises(ValueError, match="without newest"):
        arena.thin(["a"], gathered(w, 64, g), 32, newest=8)


def test_forks_and_keys_that_came_later_have_numbers_of_their_own(arena):
    g = torch.Generator().manual_seed(6)
    arena.activate("a", 60)
    w = gathered(torch.zeros(2, 1, 2, 64), 64, g)
    kept, w = arena.thin(["a"], w, 32, sinks=1, newest=4)
    before = kept[0, 0, 0].tolist()
    arena.fork("a", ["x"])
    arena.free_key("a")
    assert arena.is_thinned("x") and not arena.is_thinned("a")
    # (the child's rows are those of the key, which is gone)
    record = arena._thinned["x"]
    assert record.numbers[0, 0].tolist() == before and record.dropped == 28
    # another key of the old name starts anew
    arena.activate("a", 40)
    kept, _ = arena.thin(["a"], gathered(torch.zeros(2, 1, 2, 64), 64, g), 32, sinks=1, newest=4)
    assert set(kept[0, 0, 0].tolist()) >= {0, 36, 37, 38, 39}
    # nothing to drop: the numbers stay as they are
    record = arena._thinned["a"]
    arena.thin(["a"], gathered(torch.zeros(2, 1, 2, 64), 64, g), 48, newest=4)
    assert arena._thinned["a"] is record and arena.tokens("a") == 32
    assert [t.shape for t in arena.thin([], torch.zeros(2, 0, 2, 64), 16, newest=2)] == [
        (2, 0, 2, 16), (2, 0, 2, 64)]


def call(**kw):
    arena = KVArena(2, 16, 16, 2, 64, device="cpu")
    tables = dict(used=torch.tensor([5, 20], dtype=torch.int32), table=torch.zeros(2, 2, dtype=torch.int32),
                  max_used=20, tokens=torch.tensor([5, 30], dtype=torch.int32))
    tables.update(kw.pop("tables", {}))
    args = dict(dict(newest=4, tokens=torch.full((2, 2, 2, 32), -1, dtype=torch.int32)), **kw)
    return arena.thin_rows(tables, torch.zeros(2, 2, 2, 32), 16, **args)


@pytest.mark.parametrize("kw,match", [
    (dict(tokens=None), "newest"), (dict(newest=None), "newest"), (dict(recent=1), "newest"),
    (dict(newest=-1), "stay"), (dict(newest=10, sinks=7), "stay"),
    (dict(tokens=torch.zeros(2, 2, 2, 32)), "tokens"), (dict(tokens=torch.zeros(2, 2, 2, 31).int()), "tokens"),
    (dict(tokens=torch.zeros(2, 2, 2, 64).int()[..., ::2]), "tokens"),
    (dict(tables=dict(tokens=None)), "one for each"), (dict(tables=dict(tokens=30)), "one for each"), (dict(tables=dict(tokens=torch.zeros(2))), "one for each"),
    (dict(tables=dict(tokens=torch.zeros(3).int())), "one for each"),
    (dict(tables=dict(tokens=torch.zeros(4).int()[::2])), "one for each"), (dict(), "on the CPU")])
def test_calls_that_are_refused(kw, match):
    with pytest.raises(ValueError, match=match):
        call(**kw)


@pytest.mark.parametrize("weights", [torch.zeros(2, 2, 2, 8), torch.zeros(2, 1, 2, 64), torch.zeros(2, 2, 64),
                                     torch.zeros(())])
def test_weights_of_another_shape_change_no_key(weights):
    arena = KVArena(2, 16, 16, 2, 64, device="cpu")
    for key in "ab":
        arena.activate(key, 40)
    with pytest.raises(ValueError, match="weights"):
        arena.thin(["a", "b"], weights, 16, newest=2)
    assert arena.tokens("a") == 40 and not arena.is_thinned("a")


def test_c_entry_refuses_what_the_kernels_do_not_take():
    from quail_amd import _lib
    ok = dict(pools=16, pool_stride=1 << 20, element_bytes=2, scales=None, scale_stride=0, weights=16,
              w_layer=0, w_seq=0, w_head=0, tokens=16, t_layer=0, t_seq=0, t_head=0, total=16, used=16,
              table=16, table_ld=4, layers=1, seqs=1, HK=2, D=64, page=16, max_used=64, cols=64, keep=32,
              sinks=0, newest=0, kept=16, out=16, left=16, stream=None)
    for name, value, match in [("D", 96, "head_dim"), ("max_used", 65, "columns"), ("newest", 33, "stay"),
                               ("tokens", None, "null"), ("total", None, "null"), ("left", None, "null"),
                               ("weights", None, "null"), ("layers", 1 << 21, "launch")]:
        with pytest.raises(_lib.QxError, match=match):
            _lib.call("qx_thin_rows_by_token", *dict(ok, **{name: value}).values())
