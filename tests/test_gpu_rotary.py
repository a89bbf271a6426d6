"""Rotary rows on the GPU against the definition in 64 bits, and through the
engine's own passes with a scaled table.

Bounds: cos and sin are off by at most 2^-22 (the angle's fraction of a turn
rounded to fp32 and the functions' own 2 ulp), times the pair's size and the
factor; products and sum 3 roundings of 2^-24 of the same; then half a step of
the rows' type.
"""

from types import SimpleNamespace

import pytest
import torch

from quail_amd.rotary import RotaryEmbedding, frequencies

pytestmark = pytest.mark.gpu

DEV = "cuda"
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def definition(x, positions, inv, factor, rotary_dim, interleaved, d):
    """Rows (n, heads * d) in 64 bits, and the size of each value's pair."""
    x = x.double().cpu().reshape(x.shape[0], -1, d)
    angle = positions.cpu().double()[:, None, None] * inv
    c, s = angle.cos() * factor, angle.sin() * factor
    y, size = x.clone(), torch.zeros_like(x)
    i = torch.arange(rotary_dim // 2)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = factor * (a.abs() + b.abs())
    return y, size


def check(got, x, positions, rot, d):
    want, size = definition(x, positions, rot.inv_freq, rot.factor, rot.rotary_dim,
                            not rot.is_neox_style, d)
    got = got.double().cpu().reshape(want.shape)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0      # half a step of fp16's subnormals
    bound = HALF[x.dtype] * want.abs() + (2.0 ** -22 + 2.0 ** -22) * size * (1 + HALF[x.dtype]) + tiny
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / (bound + 1e-30)).max())


def positions_of(n, g, far):
    p = torch.randint(0, far, (n,), generator=g)
    p[0] = 0
    p[-1] = far
    return p.to(DEV)


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotary_dim", [(64, 64), (128, 128), (128, 64), (128, 20), (64, 2), (80, 80),
                                          (96, 48), (512, 512), (33, 14)])
@pytest.mark.parametrize("n,hq,hk", [(1, 4, 2), (5, 32, 8), (67, 3, 1)])
def test_rows_against_the_definition(dtype, interleaved, d, rotary_dim, n, hq, hk):
    g = torch.Generator().manual_seed(n * d + rotary_dim)
    rot = RotaryEmbedding(d, rotary_dim=rotary_dim, interleaved=interleaved, scaling=YARN)
    qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g).to(dtype).to(DEV)
    q, k, _ = qkv.split([hq * d, hk * d, hk * d], 1)
    p = positions_of(n, g, 131071)
    before = qkv.clone()
    got_q, got_k = rot(p, q, k)
    assert torch.equal(qkv, before) and got_q.shape == q.shape and got_k.shape == k.shape
    check(got_q, q, p, rot, d)
    check(got_k, k, p, rot, d)


@pytest.mark.parametrize("far", [40960, 10 ** 6, 2 ** 31 + 5, 2 ** 40])
def test_far_and_negative_positions(far):
    """The product that gives the turns is rounded in 64 bits, by at most 2^-53
    of itself here and as much in the kernel (none where it is fused with the
    subtraction): the angles differ by at most 2 pi 2^-52 |turns|, 2^-12 of a
    pair's size at 2^40 and nothing to speak of at 2^31."""
    g = torch.Generator().manual_seed(3)
    rot = RotaryEmbedding(128)
    x = torch.randn(64, 2 * 128, generator=g).to(DEV)
    p = positions_of(64, g, far)
    for sign in (1, -1):
        got = rot(sign * p, x)
        inv = rot.inv_freq
        turns = (sign * p).cpu().double()[:, None] * (inv / (2 * torch.pi))
        angle = (turns - turns.round()) * (2 * torch.pi)
        a, b = x.cpu().double().view(64, 2, 2, 64).unbind(2)
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        want = torch.cat([a * c - b * s, b * c + a * s], -1)
        size = torch.cat([a.abs() + b.abs()] * 2, -1)
        angle_off = torch.cat([turns.abs()] * 2, 1)[:, None] * (2 * torch.pi * 2.0 ** -52)
        over = (got.cpu().double().view(64, 2, 128) - want).abs() - \
            (2.0 ** -24 * want.abs() + (2.0 ** -21 + angle_off) * size)
        assert float(over.max()) <= 0


def test_in_place_strided_rows_and_heads_of_q_alone():
    g = torch.Generator().manual_seed(4)
    rot = RotaryEmbedding(128, rotary_dim=96, interleaved=True)
    wide = torch.randn(9, 7 * 128 + 4, generator=g).to(torch.bfloat16).to(DEV)
    q = wide[:, 4:4 + 512]                                  # 8 bytes past 16: one value at a time
    p = positions_of(9, g, 5000)
    before = wide.clone()
    out = rot(p, q)
    assert torch.equal(wide, before)
    check(out, before[:, 4:516], p, rot, 128)
    three = wide[:, 4:516].unflatten(1, (4, 128))
    again = rot(p, three, out=three)
    assert again is three
    assert torch.equal(wide[:, 4:516], out) and torch.equal(wide[:, 516:], before[:, 516:]) \
        and torch.equal(wide[:, :4], before[:, :4])


def test_in_place_q_and_k_of_a_projection():
    g = torch.Generator().manual_seed(5)
    rot = RotaryEmbedding(128, scaling=YARN)
    qkv = torch.randn(33, 48 * 128, generator=g).to(torch.bfloat16).to(DEV)
    q, k, v = qkv.split([32 * 128, 8 * 128, 8 * 128], 1)
    p = positions_of(33, g, 100000)
    kept, want = v.clone(), rot(p, q, k)
    rot(p, q, k, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, kept)


def test_no_rows_and_values_that_are_not_numbers():
    rot = RotaryEmbedding(64)
    none = rot(torch.zeros(0, dtype=torch.int64, device=DEV), torch.zeros(0, 128, device=DEV))
    assert none.shape == (0, 128)
    x = torch.ones(2, 128, device=DEV)
    x[0, 3], x[1, 64] = float("nan"), float("inf")
    y = rot(torch.tensor([5, 7], device=DEV), x).cpu()
    assert torch.isnan(y[0, [3, 35]]).all() and int(torch.isfinite(y[0]).sum()) == 126
    assert not torch.isfinite(y[1, [64, 96]]).any() and int(torch.isfinite(y[1]).sum()) == 126


def test_replays_of_a_captured_call_read_positions_as_they_are():
    g = torch.Generator().manual_seed(6)
    rot = RotaryEmbedding(128, scaling=YARN)
    q = torch.randn(8, 32 * 128, generator=g).to(torch.bfloat16).to(DEV)
    k = torch.randn(8, 8 * 128, generator=g).to(torch.bfloat16).to(DEV)
    p = torch.arange(8, device=DEV) + 1000
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rot(p, q, k)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rot(p, q, k)
    for step in range(4):
        p.add_(37)
        q.mul_(-1)
        graph.replay()
        want = rot(p, q, k)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_the_engines_table_is_not_made_inside_a_graph():
    rot = RotaryEmbedding(64, max_positions=100)
    x = torch.zeros(1, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="first use"):
            rot.cos_sin_cache
    assert rot.cos_sin_cache.shape == (100, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_engines_pass_with_a_scaled_table_rotates_as_the_module(dtype):
    """Norm weights 1: the qk-norm-rope pass is the norm, then the rotation
    (there with the table's rounding, here with none)."""
    from quail_amd.arena import KVArena
    from quail_amd.engine import Engine
    g = torch.Generator().manual_seed(7)
    rot = RotaryEmbedding(128, scaling=YARN, max_positions=131072, dtype=dtype)
    eng = Engine(KVArena(1, 4, 16, 8, 128), num_q_heads=32, num_kv_heads=8, head_dim=128, rotary=rot)
    n = 40
    qkv = torch.randn(n, 48 * 128, generator=g).to(torch.bfloat16).to(DEV)
    p = positions_of(n, g, 131071)
    ones = SimpleNamespace(weight=torch.ones(128, dtype=torch.bfloat16, device=DEV), variance_epsilon=1e-6)
    q, k = eng.qk_norm_rope(qkv, p, SimpleNamespace(q_norm=ones, k_norm=ones))
    x = qkv[:, :40 * 128].double().view(n, 40, 128)
    x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
    want, size = definition(x.view(n, -1), p, *frequencies(128, 1e6, YARN), 128, False, 128)
    got = torch.cat([q, k], 1).double().cpu().view(n, 40, 128)
    table = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -22
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + (1.01 * table + 2.0 ** -20) * size).all())
