"""Rotation by positions so far on that the digits of double precision count, and none at all."""
import math
from decimal import Decimal, getcontext

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,base", [(128, 1.5), (128, 10000.), (64, 2.), (22, 1.0625)])
def test_far_positions(cuda, dim, base, interleaved):
    """Against angles worked out with 60 digits.  The turns of a position are off by (5 + ln base) 2^-53 of them: 1 for each of the constant, the
    product and the fraction, 2 for the power, ln base for the rounding of its exponent, which is at most one.  An angle is off by 2 pi
    as much, a turned value by (D + 16) 2^-24 of its pair besides (see test_norm_rotate_gpu)."""
    from hgcalml_b200.norm_rotate_op import NormRotate
    getcontext().prec = 60
    pairs, places = dim // 2, [2 ** 41 + 12345, -(2 ** 43) + 7, 2 ** 36 + 1, 10 ** 6 + 3, 5]
    x = torch.randn((len(places), 2, dim), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda)
    y, _ = NormRotate(x, None, None, None, torch.tensor(places, device=cuda), base=base, interleaved=interleaved, eps=0.)
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    n = x.double() / x.double().square().mean(-1, keepdim=True).sqrt()
    first = torch.arange(pairs, device=cuda) * (2 if interleaved else 1)
    second = first + (1 if interleaved else pairs)
    for row, place in enumerate(places):
        turns = [Decimal(place) * (Decimal(base) ** (Decimal(-i) / Decimal(pairs))) / (2 * pi) for i in range(pairs)]
        angle = torch.tensor([float((t - t.to_integral_value()) * 2 * pi) for t in turns], dtype=torch.float64, device=cuda)
        off = 2 * 3.1416 * (5 + math.log(base)) * 2. ** -53 * torch.tensor([float(abs(t)) for t in turns], dtype=torch.float64, device=cuda)
        a, b = n[row][:, first], n[row][:, second]
        size = a.abs() + b.abs()
        bound = size * (off + (dim + 16) * 2. ** -24)
        assert ((y[row][:, first].double() - (a * angle.cos() - b * angle.sin())).abs() <= bound).all()
        assert ((y[row][:, second].double() - (b * angle.cos() + a * angle.sin())).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [1, 8, 22, 33, 64, 100, 128])
def test_no_column_turns(cuda, dtype, dim):
    """``rotary_dim`` of zero is no rotation, whatever the positions are, forward and backward."""
    from hgcalml_b200.norm_rotate_op import NormRotate
    g = torch.Generator(device=cuda).manual_seed(dim)
    x, grad = (torch.randn((37, 3, dim), generator=g, device=cuda).to(dtype) for _ in range(2))
    w = torch.randn(dim, generator=g, device=cuda).to(dtype)
    results = []
    for pos in (None, torch.arange(37, device=cuda), torch.full((37, 2), float("nan"), device=cuda)):
        leaves = [t.clone().requires_grad_(True) for t in (x, w)]
        y, _ = NormRotate(leaves[0], None, leaves[1], None, pos, rotary_dim=0)
        results.append((y, *torch.autograd.grad(y, leaves, grad)))
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(r, results[0])) and results[0][0].isfinite().all()
