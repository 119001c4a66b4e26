"""Plain 64-bit restatement of the 8-bit path (flextrain_amd/csrc/fp8.h): block scales, quantisation, block-scaled
products and the residual RMSNorm.  Written from the definitions; CPU tensors only.  Test infrastructure."""
from __future__ import annotations

import torch

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
LARGEST = {E4M3: 448.0, E5M2: 57344.0}
MANTISSA = {E4M3: 3, E5M2: 2}
LOWEST_EXPONENT = {E4M3: -6, E5M2: -14}


def pow2(e):
    """2**e in 64 bits for integer tensors e (by the bits of the result)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def exponents(x, fmt, rows, cols):
    """Smallest e with amax <= LARGEST * 2**e for every block of ``rows`` x ``cols`` (0 for blocks of zeros)."""
    x = x.double()
    x = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    r, c = x.shape
    pad = torch.zeros(-(-r // rows) * rows, -(-c // cols) * cols, dtype=torch.float64)
    pad[:r, :c] = x
    amax = pad.reshape(pad.shape[0] // rows, rows, pad.shape[1] // cols, cols).amax(dim=(1, 3))
    out = torch.zeros(amax.shape, dtype=torch.int64)
    for i in range(amax.shape[0]):
        for j in range(amax.shape[1]):
            a = float(amax[i, j])
            if a == 0.0:
                continue
            e = -127
            while a > LARGEST[fmt] * 2.0 ** e:
                e += 1
            out[i, j] = e
    return out


def round8(v, fmt):
    """64-bit values (at most LARGEST, infinite or NaN) rounded to the 8-bit type, ties to even."""
    _, p = torch.frexp(torch.where(torch.isfinite(v), v, torch.zeros_like(v)))
    step = pow2(torch.clamp(p - 1, min=LOWEST_EXPONENT[fmt]) - MANTISSA[fmt])
    out = torch.round(v / step) * step
    if fmt is E4M3:
        out = torch.where(torch.isinf(v), torch.full_like(out, float("nan")), out)
    return out


def spread(s, rows, cols, r, c):
    return s.repeat_interleave(rows, 0).repeat_interleave(cols, 1)[:r, :c]


def quantize(x, fmt, rows=1, cols=128):
    """(values as numbers, scales as numbers) in 64 bits."""
    s = pow2(exponents(x, fmt, rows, cols))
    return round8(x.double() / spread(s, rows, cols, *x.shape), fmt), s


def dequantize(q, s, rows=1):
    """What 8-bit values with scales (torch float8 tensors) stand for, in 64 bits."""
    e = s.contiguous().view(torch.uint8).to(torch.int64) - 127
    return q.float().double() * spread(pow2(e), rows, 128, *q.shape)


def add_rmsnorm(x, residual, w, eps):
    """(h rounded to x's dtype, rstd, y in 64 bits)."""
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    hd = h.double()
    rstd = 1.0 / torch.sqrt((hd * hd).mean(1, keepdim=True) + eps)
    y = hd * rstd
    return h, rstd, y if w is None else y * w.double()


def add_rmsnorm_bwd(dy, h, w, dh, eps):
    """(dx, dw) in 64 bits."""
    h, dy = h.double(), dy.double()
    rstd = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    n = h * rstd
    g = dy if w is None else dy * w.double()
    dx = rstd * (g - n * (g * n).mean(1, keepdim=True))
    return (dx if dh is None else dh.double() + dx), (dy * n).sum(0)
