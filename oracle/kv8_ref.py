"""The 8-bit KV arena's operators from their definitions, in float64.

Test infrastructure (see oracle/__init__.py). A page of 16 tokens of one KV
head holds e4m3 codes and an E8M0 byte b; a value is code * 2^(b - 127).
"""

import numpy as np
import torch

from oracle.fp8 import FP8_MAX

PAGE = 16
FP8 = torch.float8_e4m3fn
LAST_SCALE = 247    # of the largest float


def scale_byte(amax: float) -> int:
    """The least b >= 1 with amax <= 448 * 2^(b - 127)."""
    b = 1
    while amax > FP8_MAX * 2.0 ** (b - 127):
        b += 1
    return b


def codes_of(x: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """e4m3 codes of float64 values under scale bytes b (broadcast). The
    scaled value is rounded once: float64 -> float32 would round first, so
    values are moved to the e4m3 grid in float64."""
    y = (x * torch.exp2(127.0 - b.double())).clamp(-FP8_MAX, FP8_MAX)
    # under the last scale 256 would stand for 2^128: the codes end at 240
    y = torch.where(b == LAST_SCALE, y.clamp(-240.0, 240.0), y)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(y / step) * step).float().to(FP8)     # round half to even


def write_items(k_pool, v_pool, scales, k_rows, v_rows, items):
    """Write page items (destination, source, keep, row0, count) into codes
    (rows, HK, D) and bytes (pages, HK, 2), in place. k_rows and v_rows:
    float64 (n, HK, D)."""
    for dst, src, keep, row0, count in items:
        for side, (pool, rows) in enumerate(((k_pool, k_rows), (v_pool, v_rows))):
            fresh = rows[row0:row0 + count]
            finite = torch.nan_to_num(fresh, nan=0.0, posinf=3.4028234663852886e38,
                                      neginf=-3.4028234663852886e38)
            for h in range(pool.shape[1]):
                amax = float(finite[:, h].abs().max()) if count else 0.0
                need = scale_byte(amax)
                old = int(scales[src, h, side])
                b = max(old, need) if keep else need
                kept = pool[src * PAGE:src * PAGE + keep, h].double()
                bt = torch.tensor(b)
                if keep:
                    pool[dst * PAGE:dst * PAGE + keep, h] = codes_of(
                        kept * 2.0 ** (old - 127), bt)
                at = dst * PAGE + keep
                codes = codes_of(finite[:, h], bt)
                codes = torch.where(torch.isnan(fresh[:, h]), torch.full_like(
                    codes.float(), float("nan")), codes.float()).to(FP8)
                pool[at:at + count, h] = codes
                scales[dst, h, side] = b


def values(codes, scales, side):
    """float64 (rows, HK, D) of a pool's codes and bytes."""
    s = torch.exp2(scales[:, :, side].double() - 127)
    return codes.double() * s.repeat_interleave(PAGE, 0)[..., None]


def _rows(pool, rows):
    if pool.dtype == FP8:       # indexed as bytes
        return pool.view(torch.uint8)[rows].view(FP8).double()
    return pool[rows].double()


def attend(q, k_pool, v_pool, scales, cu_q, used, table, causal, scale=None):
    """Over codes and their scales (or 16-bit rows and scales of 1):
    attention rows (n, HQ, D), log-sum-exps (n, HQ), and for error bounds
    sum_j p_j |v_j| (n, HQ, D) and max_j scale * sum |q||k_j| (n, HQ)."""
    n, hq, d = q.shape
    hk = k_pool.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(n, hq, d, dtype=torch.float64, device=q.device)
    size, lse = torch.zeros_like(out), torch.full((n, hq), -np.inf, dtype=torch.float64,
                                                  device=q.device)
    reach = torch.zeros_like(lse)
    for s, keys in enumerate(used):
        r0, r1 = cu_q[s], cu_q[s + 1]
        if r1 == r0 or keys == 0:
            continue
        pages = torch.as_tensor(table[s][:-(-keys // PAGE)], device=q.device).long()
        rows = (pages[:, None] * PAGE + torch.arange(PAGE, device=q.device)).view(-1)[:keys]
        sc = torch.exp2(scales[pages].double() - 127).repeat_interleave(PAGE, 0)[:keys]
        k, v = (_rows(pool, rows) * sc[..., i:i + 1] for i, pool in enumerate((k_pool, v_pool)))
        for i in range(r0, r1):
            seen = min(keys, keys - (r1 - r0) + (i - r0) + 1) if causal else keys
            if seen <= 0:
                continue
            for h in range(hq):
                kh, vh, qi = k[:seen, h * hk // hq], v[:seen, h * hk // hq], q[i, h].double()
                z = kh @ qi * scale
                lse[i, h] = torch.logsumexp(z, 0)
                p = torch.exp(z - lse[i, h])
                out[i, h] = p @ vh
                size[i, h] = p @ vh.abs()
                reach[i, h] = (kh.abs() @ qi.abs()).max() * scale
    return out, lse, size, reach
