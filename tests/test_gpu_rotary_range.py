"""Rotary angles of far positions on the GPU against decimal arithmetic.

The frequency is taken as the module's fp64 value; its turns are off by 2 2^-53 of
themselves (2 pi as a number of 64 bits, the division) and position times turns by
2^-53 more: 3 2^-53 of the angle. Dropping whole turns is exact. The rest as in
tests/test_gpu_rotary.py: 2^-21 of the pair's size for the fraction of a turn, cos,
sin and the products in fp32, and half a step of the result.
"""

from decimal import Decimal, localcontext

import pytest
import torch

from quail_amd.rotary import RotaryEmbedding

pytestmark = pytest.mark.gpu

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


def angle(position, inv):
    """position * inv less whole turns, to 40 digits and more (inv: a float as it is)."""
    with localcontext() as ctx:
        ctx.prec = 75
        a = Decimal(position) * Decimal(inv)
        turns = (a / (2 * PI)).to_integral_value()
        return float(a - turns * 2 * PI)


@pytest.mark.parametrize("far", [2 ** 20, 2 ** 29, 2 ** 31 + 5, 2 ** 40, 2 ** 46 + 3])
def test_far_positions_against_decimal_angles(far):
    g = torch.Generator().manual_seed(1)
    rot = RotaryEmbedding(128, base=1e6)
    p = torch.cat([torch.tensor([far, -far, far - 1, 1 - far]), torch.randint(far // 2, far, (12,), generator=g)])
    x = torch.randn(16, 128, generator=g)
    got = rot(p.to("cuda"), x.to("cuda")).cpu().double()
    inv = rot.inv_freq.tolist()
    theta = torch.tensor([[angle(n, f) for f in inv] for n in p.tolist()], dtype=torch.float64)
    a, b = x.double().chunk(2, 1)
    want = torch.cat([a * theta.cos() - b * theta.sin(), b * theta.cos() + a * theta.sin()], 1)
    size = torch.cat([a.abs() + b.abs()] * 2, 1)
    off = torch.cat([p.abs().double()[:, None] * rot.inv_freq] * 2, 1) * (3 * 2.0 ** -53)
    assert far > 2 ** 29 or float(off.max()) < 2.0 ** -22       # what the module promises there
    assert bool(((got - want).abs() <= 2.0 ** -24 * want.abs() + (2.0 ** -21 + off) * size).all())
