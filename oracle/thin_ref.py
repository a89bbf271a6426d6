"""Thinning of kept keys and accumulated key weights in plain Python and 64 bits."""

import math

import torch

PAGE = 16


def kept_slots(weights, used, keep, sinks, recent):
    """The row that each of min(used, keep) slots holds afterwards, for one
    head's weights (a list)."""
    if used <= keep:
        return list(range(used))
    safe = set(range(sinks)) | set(range(used - recent, used))

    def heavier_first(i):
        w = weights[i]
        return (0, 0.0, i) if math.isnan(w) else (1, -w, i)

    others = sorted((i for i in range(used) if i not in safe), key=heavier_first)
    stay = safe | set(others[:keep - sinks - recent])
    movers = iter(sorted(i for i in stay if i >= keep))
    return [i if i in stay else next(movers) for i in range(keep)]


def kept_slots_by_token(weights, tokens, total, used, keep, sinks, newest):
    """The same where the tokens numbered below `sinks` and the last `newest` of
    `total` stay, and each row's number goes with it (negative: appended since
    the last thinning, numbered on to the end): the slots' rows and their numbers."""
    number = [total - used + i if tokens[i] < 0 else tokens[i] for i in range(used)]
    slots = list(range(used))
    if used > keep:
        safe = {i for i, t in enumerate(number) if t < sinks or t >= total - newest}

        def first_out_last(i):
            w = weights[i]
            return (0, 0.0, i) if i in safe else (1, 0.0, i) if math.isnan(w) else (2, -w, i)

        stay = set(sorted(range(used), key=first_out_last)[:keep])
        movers = iter(sorted(i for i in stay if i >= keep))
        slots = [i if i in stay else next(movers) for i in range(keep)]
    return slots, [number[i] for i in slots]


def key_weights(q, lse, keys, first, count, causal, scale, hk):
    """Accumulated weights (hk, keys) of one sequence: rows [first, first +
    count) of q (n, hq, d) and lse (hq, n) over keys (keys, hk, d), float64,
    and the sums of |weight| times the score's size that their roundings scale
    with."""
    hq, n = q.shape[1], keys.shape[0]
    out = torch.zeros(hk, n, dtype=torch.float64)
    off = torch.zeros_like(out)
    last = (n - count + torch.arange(count)) if causal else torch.full((count,), n - 1)
    hidden = torch.arange(n) > last[:, None]
    for h in range(hq):
        g = h * hk // hq
        rows = q[first:first + count, h].double()
        score = scale * (rows @ keys[:, g].double().t())
        size = abs(scale) * (rows.abs() @ keys[:, g].double().abs().t())
        row_lse = lse[h, first:first + count].double()[:, None]
        p = (score - row_lse).exp().masked_fill(hidden, 0.0)
        out[g] += p.sum(0)
        off[g] += (p * (size + row_lse.abs() + 1)).masked_fill(hidden, 0.0).sum(0)
    return out, off
