"""Residual addition + RMSNorm with an 8-bit (or the input's) output, and its backward, against the 64-bit oracle.

Tolerances.  h is one addition rounded once: equal.  rstd: a sum of n squares in fp32 by a tree (relative error below
``2**-20`` for the widths here) and one reciprocal root.  An 8-bit value is y rounded once: half a step of its
binade, ``2**-4`` (e4m3) / ``2**-3`` (e5m2) relative, or half its smallest step times the scale, plus the fp32 error of
y.  Gradients: fp32 arithmetic (``2**-18`` of the magnitudes that are added) and one rounding to the type."""
from __future__ import annotations

import pytest
import torch

from oracle import fp8 as o
from tests.test_gpu_fp8 import same, values
from tests.util import gen

from flextrain_amd import ops

pytestmark = pytest.mark.gpu

EPS = 1e-5
SHAPES = [(1, 1), (1, 4096), (3, 7), (5, 128), (9, 136), (4, 256), (7, 520), (3, 1024), (2, 2048), (300, 72), (2, 3000), (3, 8192), (1, 16384), (2, 1000), (2, 16392)]


def check8(q, s, y, fmt):
    """8-bit values and scales against 64-bit y; a scale may be off by one binade only where y's block maximum lies within
    fp32 error of the border."""
    e = o.exponents(y, fmt, 1, 128)
    got_e = s.contiguous().cpu().view(torch.uint8).to(torch.int64) - 127
    lo, hi = o.exponents(y * (1 - 2.0 ** -18), fmt, 1, 128), o.exponents(y * (1 + 2.0 ** -18), fmt, 1, 128)
    assert ((got_e == lo) | (got_e == hi)).all(), (got_e - e).abs().max()
    scale = o.spread(o.pow2(got_e), 1, 128, *y.shape)
    got = q.cpu().float().double() * scale
    half = 2.0 ** -(o.MANTISSA[fmt] + 1)
    tol = (half + 2.0 ** -18) * y.abs() + 0.5 * 2.0 ** (o.LOWEST_EXPONENT[fmt] - o.MANTISSA[fmt]) * scale
    assert ((got - y).abs() <= tol).all(), float(((got - y).abs() / tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(dev, rows, cols, dtype):
    g = gen(rows + cols)
    x, r = values(g, rows, cols, dtype), values(g, rows, cols, dtype, 2.0)
    for w in (None, (1 + 0.1 * torch.randn(cols, generator=g)).to(dtype), 1 + 0.1 * torch.randn(cols, generator=g)):
        wd = None if w is None else w.to(dev)
        for res in (r, None):
            rd = None if res is None else res.to(dev)
            h, rstd, y = o.add_rmsnorm(x, res, w, EPS)
            for fmt in (o.E4M3, o.E5M2):
                q, s, H, R = ops.flextrain_add_rmsnorm_fwd(x.to(dev), rd, wd, output_dtype=fmt)
                assert torch.equal(H.cpu(), h) and q.dtype == fmt and q.shape == x.shape
                torch.testing.assert_close(R.cpu().double(), rstd, rtol=2.0 ** -20, atol=0)
                check8(q, s, y, fmt)
            Y, none, H, R = ops.flextrain_add_rmsnorm_fwd(x.to(dev), rd, wd)
            assert none is None and torch.equal(H.cpu(), h)
            torch.testing.assert_close(Y.cpu().double(), y, rtol=1.5 * torch.finfo(dtype).eps + 2.0 ** -18, atol=1e-30 if dtype != torch.float16 else 2.0 ** -24)


# 64-bit statistics and one rounding: every 8-bit value and scale is that of the exact y
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(64, 4096), (300, 1001), (1000, 128), (3, 16390)])
def test_8_bit_values_are_rounded_once(dev, rows, cols, dtype):
    g = gen(rows)
    x, r, w = values(g, rows, cols, dtype), values(g, rows, cols, dtype), (1 + 0.1 * torch.randn(cols, generator=g)).to(dtype)
    for fmt in (o.E4M3, o.E5M2):
        for weight in (w, None):
            q, s, _, rstd = ops.flextrain_add_rmsnorm_fwd(x.to(dev), r.to(dev), None if weight is None else weight.to(dev), output_dtype=fmt)
            _, root, y = o.add_rmsnorm(x, r, weight, float(torch.tensor(EPS)))
            want, scale = o.quantize(y, fmt)
            same(q, want, "values")
            same(s, scale, "scales")
            assert ((rstd.cpu().double() - root).abs() <= 2.0 ** -24 * root).all()


# a last pack of 1 .. 7 values at every width of the kernel, and rows at every address
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(33, 121), (18, 129), (9, 257), (9, 511), (5, 1023), (3, 2047), (2, 3001), (2, 4101), (2, 8191), (2, 8195), (1, 16383), (2, 16387)])
def test_forward_at_odd_widths(dev, rows, cols, dtype):
    test_forward(dev, rows, cols, dtype)


@pytest.mark.parametrize("rows,cols", [(5, 128), (3, 4096), (2, 1000), (3, 7)])
def test_same_dtype_output_is_the_norm_of_the_sum(dev, rows, cols):
    g = gen(2)
    x, r = values(g, rows, cols), values(g, rows, cols)
    w = (1 + 0.1 * torch.randn(cols, generator=g)).to(torch.bfloat16).to(dev)
    Y, _, H, R = ops.flextrain_add_rmsnorm_fwd(x.to(dev), r.to(dev), w)
    want, rstd = ops.flextrain_rmsnorm_fwd(H, w)
    if cols % 8 == 0:
        assert torch.equal(Y, want) and torch.equal(R, rstd)
    else:                       # that op's kernel for odd widths adds the squares in another order
        torch.testing.assert_close(R, rstd, rtol=2.0 ** -20, atol=0)
        torch.testing.assert_close(Y.float(), want.float(), rtol=2.0 ** -7, atol=0)


@pytest.mark.parametrize("cols", [256, 100])
def test_sum_in_place(dev, cols):
    g = gen(3)
    x, r = values(g, 6, cols), values(g, 6, cols)
    q, s, H, _ = ops.flextrain_add_rmsnorm_fwd(x.to(dev), r.to(dev), None, output_dtype=o.E4M3)
    for which in (0, 1):
        a, b = x.to(dev).clone(), r.to(dev).clone()
        q2, s2, H2, _ = ops.flextrain_add_rmsnorm_fwd(a, b, None, output_dtype=o.E4M3, sum_out=(a, b)[which])
        assert H2 is (a, b)[which] and torch.equal(H2, H)
        assert torch.equal(q2.contiguous().view(torch.uint8), q.contiguous().view(torch.uint8)) and torch.equal(s2.float(), s.float())


def test_nan_and_infinity_stay_in_their_row(dev):
    g = gen(4)
    for cols in (384, 130):
        x = values(g, 4, cols)
        x[1, 3], x[2, cols - 1] = float("nan"), float("inf")
        q, s, _, rstd = ops.flextrain_add_rmsnorm_fwd(x.to(dev), None, None, output_dtype=o.E4M3)
        _, _, y = o.add_rmsnorm(x, None, None, EPS)
        assert torch.isnan(q.cpu().float()[1]).all()
        assert float(rstd.cpu()[2]) == 0.0 and torch.isnan(q.cpu().float()[2, -1]) and (q.cpu().float()[2, :-1] == 0).all()
        keep = [0, 3]
        check8(q[keep], s[keep], y[keep], o.E4M3)


def test_zero_rows_and_rows_of_zeros(dev):
    q, s, H, R = ops.flextrain_add_rmsnorm_fwd(torch.empty(0, 256, dtype=torch.bfloat16, device=dev), None, None, output_dtype=o.E4M3)
    assert q.shape == (0, 256) and s.shape == (0, 2) and R.shape == (0, 1)
    x = torch.zeros(2, 300, dtype=torch.bfloat16).to(dev)
    q, s, H, R = ops.flextrain_add_rmsnorm_fwd(x, None, None, output_dtype=o.E5M2)
    assert (q.float() == 0).all() and (s.float() == 1).all()
    dx, dw = ops.flextrain_add_rmsnorm_bwd(torch.empty(0, 8, dtype=torch.bfloat16, device=dev), torch.empty(0, 8, dtype=torch.bfloat16, device=dev),
                                           torch.ones(8, device=dev), torch.empty(0, 1, device=dev))
    assert dx.shape == (0, 8) and (dw == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 7), (9, 136), (300, 72), (70, 1000), (1000, 33), (2, 8192), (2, 3001), (1, 16392)])
def test_backward(dev, rows, cols, dtype):
    g = gen(rows * 3 + cols)
    h, dy, dh = values(g, rows, cols, dtype), values(g, rows, cols, dtype, 0.5), values(g, rows, cols, dtype, 0.5)
    w = (1 + 0.1 * torch.randn(cols, generator=g)).to(dtype)
    _, _, H, rstd = ops.flextrain_add_rmsnorm_fwd(h.to(dev), None, None)
    for past in (dh, None):
        dx_want, dw_want = o.add_rmsnorm_bwd(dy, h, w, past, EPS)
        pd = None if past is None else past.to(dev)
        dx, dw = ops.flextrain_add_rmsnorm_bwd(dy.to(dev), H, w.to(dev), rstd, dH=pd)
        n = h.double() * rstd.cpu().double()
        g_ = dy.double() * w.double()
        mag = rstd.cpu().double() * (g_.abs() + n.abs() * (g_ * n).abs().mean(1, keepdim=True)) + (0 if past is None else past.double().abs())
        tol = torch.finfo(dtype).eps / 2 * dx_want.abs() + 2.0 ** -18 * mag + (2.0 ** -25 if dtype == torch.float16 else 1e-30)
        assert ((dx.cpu().double() - dx_want).abs() <= tol).all()
        assert dw.dtype == torch.float32
        assert ((dw.cpu().double() - dw_want).abs() <= 2.0 ** -18 * (dy.double() * n).abs().sum(0) + 1e-30).all()
        if past is not None:
            assert torch.equal(pd.cpu(), past)          # left as it was
            same, _ = ops.flextrain_add_rmsnorm_bwd(dy.to(dev), H, w.to(dev), rstd, dH=pd, dX=pd)
            assert same is pd and torch.equal(pd, dx)
    start = torch.randn(cols, generator=g)
    acc = start.to(dev).clone()
    dx, got = ops.flextrain_add_rmsnorm_bwd(dy.to(dev), H, w.to(dev), rstd, dW=acc)
    assert got is acc
    assert ((acc.cpu().double() - start.double() - dw_want).abs() <= 2.0 ** -18 * ((dy.double() * n).abs().sum(0) + start.double().abs()) + 1e-30).all()
    dx, none = ops.flextrain_add_rmsnorm_bwd(dy.to(dev), H, None, rstd)
    assert none is None


# a last pack of 1 .. 7 values at every width of the kernel, rows at every address, and one that is too long for it
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(600, 1), (33, 121), (700, 129), (300, 257), (40, 511), (900, 1023), (3, 2047), (520, 3001), (2, 4101), (2, 8191), (1, 8195), (1, 16383), (30, 16387)])
def test_backward_at_odd_widths(dev, rows, cols, dtype):
    test_backward(dev, rows, cols, dtype)


@pytest.mark.parametrize("cols", [256, 100])
def test_rows_at_any_address(dev, cols):
    """Contiguous tensors that start inside a larger one, one element further each."""
    g = gen(11)
    n = 5 * cols
    x, r, dy, w = values(g, 5, cols), values(g, 5, cols), values(g, 5, cols), (1 + 0.1 * torch.randn(cols, generator=g)).to(torch.bfloat16)
    put = lambda t, k: torch.cat([torch.zeros(k, dtype=t.dtype), t.flatten()]).to(dev)[k:].view(t.shape)
    first = ops.flextrain_add_rmsnorm_fwd(x.to(dev), r.to(dev), w.to(dev), output_dtype=o.E4M3)
    back = ops.flextrain_add_rmsnorm_bwd(dy.to(dev), first[2], w.to(dev), first[3], dH=x.to(dev))
    for k in (1, 3):
        X, R, DY, W = put(x, k), put(r, k + 1), put(dy, k + 2), put(w, k)
        got = ops.flextrain_add_rmsnorm_fwd(X, R, W, output_dtype=o.E4M3, sum_out=X)
        for a, b in zip(got, first):
            assert torch.equal(a.float(), b.float())
        dx, dw = ops.flextrain_add_rmsnorm_bwd(DY, X, W, got[3], dH=put(x, k))
        assert torch.equal(dx, back[0]) and torch.equal(dw, back[1])


def test_backward_against_differences(dev):
    """sum(c * y) of the fp32 forward, differenced: a step of 2^-6 leaves a curvature error of its square and an fp32
    error of 2^-22 / 2^-6 of the sum's magnitude."""
    g = gen(11)
    rows, cols, step = 2, 24, 2.0 ** -6
    x, c = torch.randn(rows, cols, generator=g), torch.randn(rows, cols, generator=g)
    w = 1 + 0.1 * torch.randn(cols, generator=g)
    r = torch.randn(rows, cols, generator=g)
    f = lambda x_, w_: (ops.flextrain_add_rmsnorm_fwd(x_.to(dev), r.to(dev), w_.to(dev))[0].cpu().double() * c.double()).sum()
    _, _, H, rstd = ops.flextrain_add_rmsnorm_fwd(x.to(dev), r.to(dev), w.to(dev))
    dx, dw = ops.flextrain_add_rmsnorm_bwd(c.to(dev), H, w.to(dev), rstd)
    for i in range(rows):
        for j in range(0, cols, 5):
            d = torch.zeros(rows, cols)
            d[i, j] = step
            assert abs(float((f(x + d, w) - f(x - d, w)) / (2 * step)) - float(dx[i, j])) < 5e-3
    for j in range(0, cols, 5):
        d = torch.zeros(cols)
        d[j] = step
        assert abs(float((f(x, w + d) - f(x, w - d)) / (2 * step)) - float(dw[j])) < 5e-3


def test_refusals(dev):
    x = torch.randn(4, 128).to(torch.bfloat16).to(dev)
    for bad in (dict(residual=x[:, :64]), dict(residual=x.float()), dict(W=torch.ones(64, device=dev)), dict(sum_out=x[:2])):
        with pytest.raises((ValueError, TypeError)):
            ops.flextrain_add_rmsnorm_fwd(x, **bad)
    with pytest.raises(TypeError):
        ops.flextrain_add_rmsnorm_fwd(x, output_dtype=torch.float32)
    with pytest.raises(ValueError):
        ops.flextrain_add_rmsnorm_fwd(x[:, ::2])
    _, _, H, rstd = ops.flextrain_add_rmsnorm_fwd(x)
    for bad in (dict(dH=x[:2]), dict(dX=x.float()), dict(dW=torch.zeros(128, device=dev)), ):
        with pytest.raises((ValueError, TypeError)):
            ops.flextrain_add_rmsnorm_bwd(x, H, None, rstd, **bad)
    with pytest.raises(ValueError):
        ops.flextrain_add_rmsnorm_bwd(x, H, None, rstd[:2])


# one width for every split of a row over lanes and packs
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("cols", [8, 128, 136, 256, 512, 1000, 1024, 2048, 4096, 8192, 16384])
def test_same_dtype_output_has_the_bits_of_the_norm(dev, cols, dtype):
    """In fp16 a product may be rounded to fp32 on its way to fp16, or not: each of the two roundings of Y then falls to one
    of two neighbours, at most two steps in all (2^-24 each among the subnormals)."""
    g = gen(cols)
    x, r = values(g, 3, cols, dtype).to(dev), values(g, 3, cols, dtype).to(dev)
    weight = (1 + 0.1 * torch.randn(cols, generator=g)).to(dev)
    for w in (None, weight, weight.to(dtype)):
        for res in (r, None):
            Y, _, H, R = ops.flextrain_add_rmsnorm_fwd(x, res, w)
            want, rstd = ops.flextrain_rmsnorm_fwd(H, w)
            assert torch.equal(R, rstd)
            if dtype == torch.float16:
                torch.testing.assert_close(Y.double(), want.double(), rtol=2 * torch.finfo(dtype).eps, atol=2.0 ** -23)
            else:
                assert torch.equal(Y, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("cols,first", [(7, 0), (1001, 0), (16392, 0), (16391, 0), (256, 1), (4096, 3)])
def test_same_dtype_output_of_other_rows_differs_by_the_order_of_a_sum(dev, cols, first, dtype):
    """Two orders of at most 16392 squares: 65 a lane and 8 levels of a tree at most, each addition off by 2^-24, so the
    means are 146 * 2^-24 apart and rstd half of that and two roots' roundings (below 2^-17).  Y is rounded twice, and either
    rounding may fall to the other side: two steps of the type."""
    g = gen(cols)
    flat = torch.cat([torch.zeros(first, dtype=dtype), values(g, 3, cols, dtype).flatten()]).to(dev)
    x, w = flat[first:].view(3, cols), (1 + 0.1 * torch.randn(cols, generator=g)).to(dev)
    Y, _, H, R = ops.flextrain_add_rmsnorm_fwd(x, None, w)
    assert H is x
    want, rstd = ops.flextrain_rmsnorm_fwd(x, w)
    torch.testing.assert_close(R.double(), rstd.double(), rtol=2.0 ** -17, atol=0)
    torch.testing.assert_close(Y.double(), want.double(), rtol=2 * torch.finfo(dtype).eps + 2.0 ** -16, atol=2.0 ** -23 if dtype == torch.float16 else 0)


@pytest.mark.parametrize("cols", [120, 128, 16400])
def test_8_bit_values_are_those_of_the_given_eps(dev, cols):
    """Rows whose mean square is about eps, and weights that put every y as near to the middle between two e4m3 values as fp32
    weights can (2^-25 of it): eps rounded to fp32 moves y by 6e-9 of itself, across the middle in every tenth place."""
    for seed in range(3):
        g = gen(20 + seed)
        h = torch.randn(1, cols, generator=g) * 3e-3
        rstd = 1 / torch.sqrt((h.double() ** 2).mean() + EPS)
        middle = (1 + torch.randint(0, 8, (cols,), generator=g) / 8 + 1 / 16).double() * 2.0 ** torch.randint(-3, 0, (cols,), generator=g)
        middle[::16] = 1.5                     # a block's largest: its scale is 2^-8
        w = (middle / (h[0].double() * rstd)).float()
        q, s, _, _ = ops.flextrain_add_rmsnorm_fwd(h.to(dev), None, w.to(dev), output_dtype=o.E4M3, rms_norm_eps=EPS)
        _, _, y = o.add_rmsnorm(h, None, w, EPS)
        want, scale = o.quantize(y, o.E4M3)
        same(s, scale, "scales")
        same(q, want, "values")


@pytest.mark.parametrize("rows,cols", [(9, 136), (40, 511), (3, 4096), (30, 16387), (5, 16392)])
def test_backward_with_one_gradient_for_everything(dev, rows, cols):
    """The gradient that reaches h past the norm may be the norm's own (h used twice), and take the result in its place."""
    g = gen(rows + cols)
    h, d = values(g, rows, cols), values(g, rows, cols, sigma=0.5)
    w = (1 + 0.1 * torch.randn(cols, generator=g)).to(torch.bfloat16).to(dev)
    _, _, H, rstd = ops.flextrain_add_rmsnorm_fwd(h.to(dev), None, None)
    dx, dw = ops.flextrain_add_rmsnorm_bwd(d.to(dev), H, w, rstd, dH=d.to(dev))
    one = d.to(dev)
    got, dw2 = ops.flextrain_add_rmsnorm_bwd(one, H, w, rstd, dH=one, dX=one)
    assert got is one and torch.equal(got, dx)
    assert torch.equal(dw2, dw)
