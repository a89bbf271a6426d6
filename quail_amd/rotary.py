"""Rotary positions past the checkpoint's own: scaled frequencies, half or
interleaved pairs, all of a head or its first part.

A `RotaryEmbedding` is a model's rotary module. Called, it rotates rows of q
and k by their positions (qx_rotary: angles from the positions themselves, so
no table bounds them; they are off by up to 3 2^-53 of themselves, less than
fp32 does to cos and sin at positions up to about 2^29). Its `cos_sin_cache` is
the table that the engine's own passes read (`Engine(rotary=...)`, a layer's
`rotary_emb`), where the head is rotated whole in half pairs, as Qwen3's is.

Frequencies are base^(-2i / rotary_dim), or `inv_freq`, and with `scaling`:
  linear  all divided by `factor`;
  yarn    pair i divided by `factor` where it turns less than beta_slow (1)
          times over the trained positions, as it is where it turns more than
          beta_fast (32) times, a linear ramp over i between; cos and sin times
          attention_factor, 0.1 ln(factor) + 1 by default.
The dictionary has the names of a checkpoint's rope_scaling. Frequencies and
angles are formed in 64 bits.
"""

import math

import torch

from quail_amd.engine import _launch

_KNOWN = {"default": set(), "linear": {"factor"},
          "yarn": {"factor", "original_max_position_embeddings", "beta_fast", "beta_slow",
                   "attention_factor", "truncate"}}
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def scaling_type(scaling):
    """The type that a checkpoint's rope_scaling (or rope_parameters) names;
    "default" for none. ValueError where one that says how to scale names none."""
    scaling = scaling or {}
    kind = scaling.get("rope_type") or scaling.get("type")
    if kind:
        return kind
    left = sorted(k for k, v in scaling.items() if v is not None and k not in ("rope_type", "type", "rope_theta"))
    if left:
        raise ValueError(f"a rope scaling with {left} and no rope_type")
    return "default"


def frequencies(rotary_dim, base, scaling=None, max_positions=None):
    """(angle per position of each pair, float64 on the CPU; factor of cos and
    sin) for `scaling` as a checkpoint's rope_scaling names it."""
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    inv = float(base) ** (-2 * i / rotary_dim)
    scaling = dict(scaling or {})
    kind = scaling_type(scaling)
    for name in ("rope_type", "type", "rope_theta"):
        scaling.pop(name, None)
    if kind not in _KNOWN:
        raise ValueError(f"rope_type {kind!r}: one of {sorted(_KNOWN)}")
    if kind == "default":
        return inv, 1.0
    left = {k for k, v in scaling.items() if v is not None} - _KNOWN[kind]
    if kind == "linear":
        left.discard("original_max_position_embeddings")   # says where, changes nothing
    if left:
        raise ValueError(f"{kind} scaling with {sorted(left)} is not supported")
    factor = float(scaling.get("factor") or 0)
    if not 1 <= factor < math.inf:
        raise ValueError(f"a scaling factor of {scaling.get('factor')!r} (1 or more)")
    if kind == "linear":
        return inv / factor, 1.0
    trained = scaling.get("original_max_position_embeddings") or max_positions
    if not trained or trained <= 0:
        raise ValueError("yarn scaling needs original_max_position_embeddings")
    if scaling.get("truncate") not in (None, True):
        raise ValueError("yarn scaling with truncate false is not supported")
    fast = 32.0 if scaling.get("beta_fast") is None else float(scaling["beta_fast"])
    slow = 1.0 if scaling.get("beta_slow") is None else float(scaling["beta_slow"])
    if not 0 < slow <= fast:
        raise ValueError(f"beta_slow {slow} and beta_fast {fast}")

    def pair_of(turns):    # the pair (not whole) that turns so often over the trained positions
        return rotary_dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(0, math.floor(pair_of(fast))), min(rotary_dim - 1, math.ceil(pair_of(slow)))
    slowed = ((i - low) / (high - low if high != low else 0.001)).clamp(0, 1)
    attention = scaling.get("attention_factor")
    attention = 0.1 * math.log(factor) + 1 if attention is None else float(attention)
    return inv * (1 - slowed) + inv / factor * slowed, attention


class RotaryEmbedding:
    """Rotary positions of q and k rows.

    Args:
        head_dim: columns of a head.
        rotary_dim: the head's first columns that are rotated (all by default).
        base: of the frequencies, where inv_freq does not give them.
        max_positions: rows of cos_sin_cache (calls take any position).
        interleaved: pairs are columns (2i, 2i + 1), not (i, i + rotary_dim / 2).
        scaling: a checkpoint's rope_scaling.
        inv_freq: the angle per position of each of rotary_dim / 2 pairs.
        dtype: of cos_sin_cache, bf16 or fp32.
    """

    def __init__(self, head_dim, *, rotary_dim=None, base=1e6, max_positions=40960,
                 interleaved=False, scaling=None, inv_freq=None, dtype=torch.bfloat16,
                 device="cuda"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if rotary_dim <= 0 or rotary_dim % 2 or rotary_dim > min(head_dim, 512):
            raise ValueError(f"{rotary_dim} rotated columns of a head of {head_dim}: an even "
                             "number, at most the head and 512")
        if inv_freq is None:
            if not 1 < base < math.inf:
                raise ValueError(f"base {base}")
            inv_freq, factor = frequencies(rotary_dim, base, scaling, max_positions)
        else:
            if scaling:
                raise ValueError("frequencies are given as inv_freq or by scaling, not both")
            inv_freq, factor = torch.as_tensor(inv_freq, dtype=torch.float64, device="cpu"), 1.0
            if inv_freq.shape != (rotary_dim // 2,):
                raise ValueError(f"inv_freq of {tuple(inv_freq.shape)} for {rotary_dim // 2} pairs")
        if dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"cos_sin_cache in bf16 or fp32, not {dtype}")
        self.head_size = head_dim
        self.rotary_dim = rotary_dim
        self.base = base
        self.max_positions = max_positions
        self.is_neox_style = not interleaved
        self.inv_freq = inv_freq
        self.factor = factor
        self.dtype = dtype
        self.device = torch.device(device)
        self._turns = (inv_freq / (2 * math.pi)).to(device)
        self._cache = None

    @property
    def cos_sin_cache(self):
        """(max_positions, head_dim): [cos | sin] of every position."""
        if self._cache is None:
            if self.rotary_dim != self.head_size or not self.is_neox_style:
                raise ValueError("the engine's passes rotate whole heads in half pairs; rows of "
                                 "other layouts are rotated by calling the module")
            on_gpu = self.device.type == "cuda"
            if on_gpu and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("cos_sin_cache is made at its first use, which a graph cannot "
                                   "capture; read it once before")
            turns = torch.arange(self.max_positions, dtype=torch.float64,
                                 device=self.device)[:, None] * self._turns
            angle = (turns - turns.round()) * (2 * math.pi)
            cache = (torch.cat([angle.cos(), angle.sin()], 1) * self.factor).to(self.dtype)
            if on_gpu:   # other streams read it too
                torch.cuda.current_stream(cache.device).synchronize()
            self._cache = cache
        return self._cache

    def _rows(self, name, x, n):
        """(heads, row stride) of rows (n, heads * head_dim) or (n, heads, head_dim)."""
        d = self.head_size
        shape, stride = x.shape, x.stride()
        if len(shape) == 2:
            heads, rest = divmod(shape[1], d)
            ok = not rest and stride[1] == 1
        else:
            ok = len(shape) == 3 and shape[2] == d and stride[2] == 1
            heads = shape[1] if ok else 0
            ok = ok and (heads == 1 or stride[1] == d)
        if not ok or shape[0] != n or heads == 0:
            raise ValueError(f"{name}: {n} rows of contiguous heads of {d}, not {tuple(shape)} "
                             f"with strides {stride}")
        if n <= 1:
            return heads, heads * d
        if stride[0] < heads * d:
            raise ValueError(f"{name}: rows overlap (strides {stride})")
        return heads, stride[0]

    def _result(self, x, heads, ld, y, n):
        """(result, its row stride) for rows x: a new tensor, or y."""
        if y is None:
            return torch.empty_like(x, memory_format=torch.contiguous_format), heads * self.head_size
        if y is x:
            return x, ld
        if y.dtype != x.dtype or y.shape != x.shape:
            raise ValueError(f"out of {tuple(y.shape)} {y.dtype} for {tuple(x.shape)} {x.dtype}")
        return y, self._rows("out", y, n)[1]

    def __call__(self, positions, q, k=None, *, out=None):
        """q and k (n rows, bf16, fp16 or fp32) rotated by `positions` (n,
        int64, any value), as new tensors or into out = (q's, k's), which may
        be the rows themselves and overlap them in no other way. With q alone, `out` and the result are q's."""
        n = q.shape[0]
        if positions.shape != (n,) or positions.dtype != torch.int64 or \
                not (n == 1 or positions.is_contiguous()):
            raise ValueError(f"{n} rows need as many contiguous int64 positions")
        kind = _TYPES.get(q.dtype)
        if kind is None or (k is not None and k.dtype != q.dtype):
            raise ValueError(f"rows of {q.dtype}{'' if k is None else f' and {k.dtype}'}: one of "
                             "bf16, fp16 and fp32")
        q_to, k_to = (None, None) if out is None else (out, None) if k is None else out
        hq, q_ld = self._rows("q", q, n)
        qo, qo_ld = self._result(q, hq, q_ld, q_to, n)
        tensors = (positions, self._turns, qo)
        hk = k_ld = ko_ld = 0
        kp = kop = None
        if k is not None:
            hk, k_ld = self._rows("k", k, n)
            ko, ko_ld = self._result(k, hk, k_ld, k_to, n)
            tensors += (k, ko)
            kp, kop = k.data_ptr(), ko.data_ptr()
        device = q.get_device()
        if device < 0 or any(t.get_device() != device for t in tensors):
            raise ValueError("rows, results, positions and the module are on one GPU, not "
                             f"{q.device}, {', '.join(str(t.device) for t in tensors)}")
        if n:
            args = (q.data_ptr(), q_ld, kp, k_ld, qo.data_ptr(), qo_ld, kop, ko_ld,
                    positions.data_ptr(), self._turns.data_ptr(), self.factor, n, hq, hk,
                    self.head_size, self.rotary_dim, int(not self.is_neox_style), kind)
            _launch(device, "qx_rotary", *args)
        return qo if k is None else (qo, ko)
