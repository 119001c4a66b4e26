"""The 64-bit restatement of the 8-bit path (oracle/fp8.py) against torch's own casts and gradients."""
from __future__ import annotations

import pytest
import torch

from oracle import fp8 as o
from tests.util import gen


@pytest.mark.parametrize("fmt", [o.E4M3, o.E5M2])
def test_rounding_is_the_cast_within_range(fmt):
    g = gen(1)
    v = torch.cat([torch.randn(4000, generator=g) * 10.0 ** k for k in range(-9, 3)])
    v = v[v.abs() <= o.LARGEST[fmt]]
    assert torch.equal(o.round8(v.double(), fmt), v.to(fmt).double())
    every = torch.arange(256, dtype=torch.uint8).view(fmt).double()
    every = every[torch.isfinite(every)]
    assert torch.equal(o.round8(every, fmt), every)
    # halfway between neighbours: to the even one
    s = torch.sort(every.unique()).values
    mid = (s[1:] + s[:-1]) / 2
    assert torch.equal(o.round8(mid, fmt), mid.float().to(fmt).double())


@pytest.mark.parametrize("fmt", [o.E4M3, o.E5M2])
def test_scale_is_the_smallest_power_that_fits(fmt):
    x = torch.tensor([[1.75 * 2.0 ** 3, 0.0], [0.0, 0.0], [float("inf"), 2.0], [1e-30, float("nan")]])
    x[0, 1] = o.LARGEST[fmt]
    e = o.exponents(x, fmt, 1, 128)
    assert e.shape == (4, 1) and e[0, 0] == 0 and e[1, 0] == 0
    for row, a in ((2, 2.0), (3, float(torch.tensor(1e-30)))):
        assert a <= o.LARGEST[fmt] * 2.0 ** int(e[row, 0]) and a > o.LARGEST[fmt] * 2.0 ** (int(e[row, 0]) - 1)
    x[0, 1] = torch.nextafter(x[0, 1], torch.tensor(float("inf")))
    assert o.exponents(x, fmt, 1, 128)[0, 0] == 1
    # tiles and columns share the same rule
    y = torch.randn(130, 260, generator=gen(2))
    assert o.exponents(y, fmt, 128, 128).shape == (2, 3)
    assert torch.equal(o.exponents(y.t().contiguous(), fmt, 1, 128), o.exponents(y, fmt, 128, 1).t())


def test_dequantised_values_are_within_half_a_step():
    x = torch.randn(40, 300, generator=gen(3))
    for fmt in (o.E4M3, o.E5M2):
        q, s = o.quantize(x, fmt)
        back = q * o.spread(s, 1, 128, *x.shape)
        step = 2.0 ** (o.LOWEST_EXPONENT[fmt] - o.MANTISSA[fmt]) * o.spread(s, 1, 128, *x.shape)
        assert ((back - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -(o.MANTISSA[fmt] + 1), step / 2)).all()


@pytest.mark.parametrize("with_w,with_dh", [(True, True), (False, True), (True, False)])
def test_norm_gradients_are_the_derivatives(with_w, with_dh):
    g = gen(4)
    x = torch.randn(5, 12, generator=g, dtype=torch.float64, requires_grad=True)
    r = torch.randn(5, 12, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True) if with_w else None
    dy, dh = torch.randn(5, 12, generator=g, dtype=torch.float64), torch.randn(5, 12, generator=g, dtype=torch.float64)

    def outputs(x, r):
        h, _, y = o.add_rmsnorm(x, r, w, 1e-5)
        return (h, y) if with_dh else y

    assert torch.autograd.gradcheck(outputs, (x, r), eps=1e-6, atol=1e-8)
    h, _, y = o.add_rmsnorm(x, r, w, 1e-5)
    ((y * dy).sum() + ((h * dh).sum() if with_dh else 0)).backward()
    dx, dw = o.add_rmsnorm_bwd(dy, h.detach(), None if w is None else w.detach(), dh if with_dh else None, 1e-5)
    torch.testing.assert_close(dx, x.grad, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(dx, r.grad, rtol=1e-12, atol=1e-12)
    if with_w:
        torch.testing.assert_close(dw, w.grad, rtol=1e-12, atol=1e-12)
