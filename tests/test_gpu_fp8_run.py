"""The 8-bit operators together, as a training step and a routed layer use them, and under the conditions that a program
puts them in: captured graphs, several streams, operands and outputs past 32-bit offsets and past the caches.

Every stage is compared with the 64-bit oracle applied to what the stage was given (the tolerances of test_gpu_fp8.py).
The whole run is compared with the unquantised mathematics in 64 bits.  A rounding to e4m3 is off by at most ``h = 2**-4``
of the value, ``h / sqrt(6)`` of it in the mean square over a binade (uniform in the step, values uniform in the binade:
``1/sqrt(3) * sqrt(1/2)``), so 0.0255; e5m2 0.051.  Independent roundings add in squares: the up product is off by
0.036 of its norm, the gated activation by twice that at most, the down product by ``sqrt(0.072**2 + 2 * 0.0255**2) = 0.08``;
backward, the gradient of the activations by 0.057, of the gate's inputs by ``0.057 + 0.072``, of a weight by ``sqrt(0.13**2 +
0.051**2 + 0.0255**2) = 0.14``.  Twice these figures are allowed; an operand that is transposed, shifted or scaled by the
wrong block is off by the whole norm."""
from __future__ import annotations

import pytest
import torch

from oracle import fp8 as o
from tests.test_gpu_add_rmsnorm import check8
from tests.test_gpu_fp8 import E4M3, E5M2, check, largest_of_groups, operand, same, some_rows, values
from tests.util import gen

from flextrain_amd import ops

pytestmark = pytest.mark.gpu

EPS = 1e-5


def number(q, s, rows=1):
    return o.dequantize(q.cpu(), s.cpu(), rows)


def quantised_both(x, fmt, tiles=False):
    """flextrain_fp8_quantize_both, checked."""
    q, s, qt, st = ops.flextrain_fp8_quantize_both(x, dtype=fmt, tiles=tiles)
    n = 128 if tiles else 1
    want, scale = o.quantize(x.cpu(), fmt, n, 128)
    same(q, want, "values")
    same(s, scale, "scales")
    want, scale = o.quantize(x.cpu().t().contiguous(), fmt, n, 128)
    same(qt, want, "transposed values")
    same(st, scale, "transposed scales")
    return q, s, qt, st


def product(a, sa, b, sb, C=None, b_tiles=False):
    """flextrain_fp8_matmul, checked."""
    out = ops.flextrain_fp8_matmul(a, sa, b, sb, C=C)
    av, bv = number(a, sa), number(b, sb, 128 if b_tiles else 1)
    c = None if C is None else C.cpu()
    check(out, av @ bv.t() + (0 if c is None else c.double()), av, bv, c)
    return out


def off(got, want):
    return float((got.cpu().double() - want).norm() / want.norm())


@pytest.mark.parametrize("T,D,F", [(1, 128, 64), (70, 264, 200), (200, 256, 328)])
def test_dense_block_forward_and_backward(dev, T, D, F):
    g = gen(T + D)
    x = torch.randn(T, D, generator=g).to(torch.bfloat16)
    res = torch.randn(T, D, generator=g).to(torch.bfloat16)
    wn = (1 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16)
    w1 = (torch.randn(2 * F, D, generator=g) * D ** -0.5).to(torch.bfloat16)
    w2 = (torch.randn(D, F, generator=g) * F ** -0.5).to(torch.bfloat16)
    dout = torch.randn(T, D, generator=g).to(torch.bfloat16)

    W1, S1, W1t, S1t = quantised_both(w1.to(dev), E4M3, tiles=True)
    W2, S2, W2t, S2t = quantised_both(w2.to(dev), E4M3, tiles=True)
    # forward
    y8, ys, h, rstd = ops.flextrain_add_rmsnorm_fwd(x.to(dev), res.to(dev), wn.to(dev), output_dtype=E4M3, rms_norm_eps=EPS)
    check8(y8, ys, o.add_rmsnorm(x, res, wn, EPS)[2], E4M3)
    u = product(y8, ys, W1, S1, b_tiles=True)
    gate, up = u[:, :F].contiguous(), u[:, F:].contiguous()
    a = ops.flextrain_swiglu_fwd(gate, up)
    aq, as_, at, ats = quantised_both(a, E4M3)
    out = product(aq, as_, W2, S2, C=h, b_tiles=True)
    # backward
    dq, ds, dqt, dst = quantised_both(dout.to(dev), E5M2)
    da = product(dq, ds, W2t, S2t, b_tiles=True)
    dw2 = product(dqt, dst, at, ats)
    dgate, dup = ops.flextrain_swiglu_bwd(gate, up, da)[:2]
    du = torch.cat([dgate, dup], 1)
    uq, us, uqt, ust = quantised_both(du, E5M2)
    dy = product(uq, us, W1t, S1t, b_tiles=True)
    y = ops.flextrain_rmsnorm_fwd_recompute(h, wn.to(dev), rstd)
    _, _, yt, yts = quantised_both(y, E4M3)
    dw1 = product(uqt, ust, yt, yts)
    dx, dwn = ops.flextrain_add_rmsnorm_bwd(dy, h, wn.to(dev), rstd, dH=dout.to(dev))

    # the unquantised mathematics
    X, R, WN, A1, A2 = (t.double().requires_grad_() for t in (x, res, wn, w1, w2))
    H = X + R
    U = (H * torch.rsqrt((H * H).mean(1, keepdim=True) + EPS) * WN) @ A1.t()
    O = H + (torch.nn.functional.silu(U[:, :F]) * U[:, F:]) @ A2.t()
    O.backward(dout.double())
    assert off(out.cpu().double() - h.cpu().double(), (O - H).detach()) < 0.16
    assert off(dw2, A2.grad) < 2 * (0.072 ** 2 + 0.051 ** 2 + 0.0255 ** 2) ** 0.5
    assert off(dw1, A1.grad) < 0.28 and off(dwn, WN.grad) < 0.28
    through = X.grad - dout.double()
    assert torch.equal(X.grad, R.grad) and off(dx.cpu().double() - dout.double(), through) < 0.28


@pytest.mark.parametrize("T,K,E,D,F", [(3, 2, 8, 128, 64), (90, 2, 5, 264, 200)])
def test_routed_block_forward_and_backward(dev, T, K, E, D, F):
    g = gen(T + E)
    x = torch.randn(T, D, generator=g).to(torch.bfloat16).to(dev)
    ids = torch.stack([torch.randperm(E - 1, generator=g)[:K] for _ in range(T)]).to(torch.int32).to(dev)       # the last expert is idle
    weights = torch.rand(T, K, generator=g).to(dev)
    w1 = (torch.randn(E, 2 * F, D, generator=g) * D ** -0.5).to(torch.bfloat16).to(dev)
    w2 = (torch.randn(E, D, F, generator=g) * F ** -0.5).to(torch.bfloat16).to(dev)
    dout = torch.randn(T, D, generator=g).to(torch.bfloat16).to(dev)

    indices, counts = ops.flextrain_moe_sort(ids, E)
    sources = ops.flextrain_moe_row_sources(indices)
    n, src = counts.tolist(), sources.cpu().long()
    assert n[-1] == 0 and sum(n) == T * K
    W1, S1, W1t, S1t = ops.flextrain_fp8_quantize_both(w1, tiles=True)
    W2, S2, W2t, S2t = ops.flextrain_fp8_quantize_both(w2, tiles=True)

    def rows(out, a, b, sb):
        at = 0
        for e, m in enumerate(n):
            if m:
                bv = number(b[e], sb[e], 128)
                check(out[at:at + m], a[at:at + m] @ bv.t(), a[at:at + m], bv, what=f"expert {e}")
            at += m

    def grads(out, a, sa, b, sb):
        av, bv, at = number(a, sa), number(b, sb), 0
        for e, m in enumerate(n):
            p = -(-m // 128) * 128
            check(out[e], av[:, at:at + p] @ bv[:, at:at + p].t(), av[:, at:at + p], bv[:, at:at + p], what=f"expert {e}")
            at += p

    xq, xs = ops.flextrain_fp8_quantize(x)
    u = ops.flextrain_fp8_grouped_matmul(xq, xs, W1, S1, counts, row_sources=sources)
    rows(u, number(xq, xs)[src], W1, S1)
    a = ops.flextrain_swiglu_moe_fwd(u)
    aq, as_ = ops.flextrain_fp8_quantize(a)
    y = ops.flextrain_fp8_grouped_matmul(aq, as_, W2, S2, counts)
    rows(y, number(aq, as_), W2, S2)
    out = ops.flextrain_moe_gather(y, indices, weights)

    dy = ops.flextrain_moe_scatter(dout, indices, weights)
    dq, ds = ops.flextrain_fp8_quantize(dy, dtype=E5M2)
    da = ops.flextrain_fp8_grouped_matmul(dq, ds, W2t, S2t, counts)
    rows(da, number(dq, ds), W2t, S2t)
    ct, cts = ops.flextrain_fp8_quantize_grouped_cols(dy, counts, dtype=E5M2)
    at, ats = ops.flextrain_fp8_quantize_grouped_cols(a, counts)
    dw2 = ops.flextrain_fp8_grouped_wgrad(ct, cts, at, ats, counts)
    grads(dw2, ct, cts, at, ats)
    du = ops.flextrain_swiglu_moe_bwd(da, u, torch.ones(T * K, device=dev))[0]
    ut, uts = ops.flextrain_fp8_quantize_grouped_cols(du, counts, dtype=E5M2)
    xt, xts = ops.flextrain_fp8_quantize_grouped_cols(x, counts, row_sources=sources)
    dw1 = ops.flextrain_fp8_grouped_wgrad(ut, uts, xt, xts, counts)
    grads(dw1, ut, uts, xt, xts)
    uq, us = ops.flextrain_fp8_quantize(du, dtype=E5M2)
    dx = ops.flextrain_moe_gather(ops.flextrain_fp8_grouped_matmul(uq, us, W1t, S1t, counts), indices)
    assert (dw1[-1] == 0).all() and (dw2[-1] == 0).all()

    # the unquantised mathematics (packed rows hold [value | gate])
    X, A1, A2 = (t.cpu().double().requires_grad_() for t in (x, w1, w2))
    total = torch.zeros(T, D, dtype=torch.float64)
    for t in range(T):
        for k in range(K):
            e = int(ids[t, k])
            v = X[t] @ A1[e].t()
            total[t] = total[t] + weights.cpu().double()[t, k] * ((torch.nn.functional.silu(v[F:]) * v[:F]) @ A2[e].t())
    total.backward(dout.cpu().double())
    assert off(out, total.detach()) < 0.16
    assert off(dw2, A2.grad) < 2 * (0.072 ** 2 + 0.051 ** 2 + 0.0255 ** 2) ** 0.5
    assert off(dw1, A1.grad) < 0.28 and off(dx, X.grad) < 0.28


def test_one_source_row_for_every_expert_row(dev):
    g = gen(5)
    x = values(g, 3, 136)
    counts = torch.tensor([40, 0, 90], dtype=torch.int32).to(dev)
    sources = torch.full((130,), 2, dtype=torch.int32).to(dev)
    a, sa, av = operand(dev, x)
    w = torch.randn(3, 24, 136, generator=g).to(torch.bfloat16)
    b, sb = ops.flextrain_fp8_quantize(w.to(dev), tiles=True)
    out = ops.flextrain_fp8_grouped_matmul(a, sa, b, sb, counts, row_sources=sources)
    assert torch.equal(out[:40], out[:1].expand(40, -1)) and torch.equal(out[40:], out[40:41].expand(90, -1))
    av = av[2:3]
    for row, e in ((0, 0), (129, 2)):
        bv = number(b[e], sb[e], 128)
        check(out[row:row + 1], av @ bv.t(), av, bv)
    qt, st = ops.flextrain_fp8_quantize_grouped_cols(x.to(dev), counts, row_sources=sources)
    same(qt[:, :40], o.quantize(x[2:3].expand(40, -1).t().contiguous(), E4M3)[0], "columns")


def bits(t):
    return t.contiguous().view(torch.uint8) if t.dtype in (E4M3, E5M2, torch.float8_e8m0fnu) else t


class Step:
    """One call of every operator over buffers that stay where they are."""

    def __init__(self, dev, seed):
        g = gen(seed)
        put = lambda *shape, std=1.0, dtype=torch.bfloat16: (torch.randn(*shape, generator=g) * std).to(dtype).to(dev)
        self.x, self.res, self.wn = put(16, 512), put(16, 512), put(512)
        self.w = put(640, 512, std=0.05)
        self.long = put(520, 9000), put(500, 9000)                                  # sliced contraction: a workspace
        self.many = put(1300, 300, std=0.1), put(2100, 300)
        self.ew = put(4, 200, 512, std=0.05)
        self.counts = torch.tensor([7, 0, 5, 4], dtype=torch.int32).to(dev)
        self.inputs = [self.x, self.res, *self.long, *self.many]

    def run(self):
        q = ops.flextrain_fp8_quantize
        y, ys, h, rstd = ops.flextrain_add_rmsnorm_fwd(self.x, self.res, self.wn, output_dtype=E4M3)
        w = q(self.w, tiles=True)
        u = ops.flextrain_fp8_matmul(y, ys, *w)
        split = ops.flextrain_fp8_matmul(*q(self.long[0], dtype=E5M2), *q(self.long[1]))
        many = ops.flextrain_fp8_matmul(*q(self.many[0]), *q(self.many[1]))
        rows = ops.flextrain_fp8_grouped_matmul(y, ys, *q(self.ew, tiles=True), self.counts)
        cols = ops.flextrain_fp8_quantize_grouped_cols(rows, self.counts, dtype=E5M2)
        dw = ops.flextrain_fp8_grouped_wgrad(*cols, *ops.flextrain_fp8_quantize_grouped_cols(h, self.counts), self.counts)
        dx, dwn = ops.flextrain_add_rmsnorm_bwd(self.res, h, self.wn, rstd, dH=self.x)
        return [bits(t) for t in (y, ys, h, rstd, u, split, many, rows, *cols, dw, dx, dwn)]


def test_captured_and_replayed(dev):
    """Two graphs of one memory pool, replayed in turn with new inputs and eager work between them."""
    steps = [Step(dev, 1), Step(dev, 2)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for s in steps:
            s.run()
    side.synchronize()
    pool, graphs = torch.cuda.graph_pool_handle(), []
    for s in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = s.run()
        graphs.append((graph, out))
    g = gen(9)
    for _ in range(4):
        for s, (graph, out) in zip(steps, graphs):
            for t in s.inputs:
                t.copy_(torch.randn(t.shape, generator=g))
            want = [t.clone() for t in s.run()]
            graph.replay()
            torch.cuda.synchronize()
            for i, (got, w) in enumerate(zip(out, want)):
                assert torch.equal(got, w), f"output {i}"
            ops.flextrain_fp8_matmul(*ops.flextrain_fp8_quantize(s.long[0]), *ops.flextrain_fp8_quantize(s.long[1]))


def test_two_streams_at_once(dev):
    """Calls on other streams than the default one, overlapping, each with what it allocates for itself."""
    steps = [Step(dev, 3), Step(dev, 4)]
    want = [[t.clone() for t in s.run()] for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(steps):
            with torch.cuda.stream(streams[i]):
                got[i].append(s.run())
    torch.cuda.synchronize()
    for i in (0, 1):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_quantize_past_32_bit_offsets(dev):
    """More than 2**32 elements, and (16-bit inputs above 96 MB) the loads that pass the caches."""
    rows, cols = 70000, 65536
    g = gen(6)
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=dev)
    last = values(g, 300, cols)
    x[rows - 300:] = last.to(dev)
    q, s, qt, st = ops.flextrain_fp8_quantize_both(x)
    a, b = cols - 500, cols - 200
    want, scale = o.quantize(last[-40:, :1280], E4M3)
    same(q[rows - 40:, :1280], want, "values")
    same(s[rows - 40:, :10], scale, "scales")
    # the row blocks of the transposed output start at multiples of 128
    start = rows // 128 * 128 - 128
    want, scale = o.quantize(last[start - (rows - 300):, a:b].t().contiguous(), E4M3)
    same(qt[a:b, start:], want, "transposed values")
    same(st[a:b, start // 128:], scale, "transposed scales")
    assert not q[: rows - 300].contiguous().view(torch.uint8).any() and not qt[a:b, : rows - 300].contiguous().view(torch.uint8).any()
    del qt, st
    # as the rows of a product, with its output past 32 bits in the second
    w, sw, wv = operand(dev, values(g, 17, cols, sigma=0.01))
    av = number(q[rows - 6:], s[rows - 6:])
    check(ops.flextrain_fp8_matmul(q, s, w, sw)[rows - 6:], av @ wv.t(), av, wv)
    k = 136
    w, sw, wv = operand(dev, values(g, cols, k, sigma=0.1))
    out = ops.flextrain_fp8_matmul(q[:, :k], s[:, :2], w, sw)
    av = number(q[rows - 6:, :k], s[rows - 6:, :2])
    check(out[rows - 6:, cols - 100:], av @ wv[cols - 100:].t(), av, wv[cols - 100:])
    check(out[rows - 6:, :100], av @ wv[:100].t(), av, wv[:100])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_expert_columns_larger_than_the_caches(dev, dtype):
    g = gen(7)
    counts = torch.tensor([20000, 0, 129, 30000, 1], dtype=torch.int32)
    rows, cols = 50137, 1000 + 8 * (dtype == torch.bfloat16)
    x = torch.randn(rows, cols, generator=g).to(dtype).to(dev)
    qt, st = ops.flextrain_fp8_quantize_grouped_cols(x, counts.to(dev))
    at = to = 0
    for c in counts.tolist():
        if c:
            _, _, q, s = ops.flextrain_fp8_quantize_both(x[at:at + c])
            assert torch.equal(bits(qt[:, to:to + c]), bits(q)), c
            assert torch.equal(bits(st[:, to // 128:(to + c + 127) // 128]), bits(s)), c
        at, to = at + c, to + -(-c // 128) * 128


@pytest.mark.parametrize("m,n,t", [(16500, 8200, torch.bfloat16), (8300, 8200, torch.float32)])
def test_outputs_larger_than_the_caches(dev, m, n, t):
    g = gen(8)
    k = 200
    a, sa, av = operand(dev, values(g, m, k, sigma=1e-3), E5M2)
    b, sb, bv = operand(dev, values(g, n, k, sigma=k ** -0.5), tiles=True)
    some = some_rows(g, m)
    av = av[some]
    ref = av @ bv.t()
    check(ops.flextrain_fp8_matmul(a, sa, b, sb, out_dtype=t)[some], ref, av, bv)
    c = torch.randn(m, n, generator=g).mul_(float(ref.std())).to(t)
    acc = c.to(dev)
    ops.flextrain_fp8_matmul(a, sa, b, sb, C=acc, out=acc)
    check(acc[some], ref + c[some].double(), av, bv, c[some])


def test_expert_outputs_larger_than_the_caches(dev):
    g = gen(10)
    k, n, counts = 200, 3000, torch.tensor([9000, 0, 30000, 301, 10000], dtype=torch.int32)
    rows, cd = int(counts.sum()), counts.to(dev)
    x = values(g, rows, k)
    a, sa, av = operand(dev, x)
    b, sb = ops.flextrain_fp8_quantize((torch.randn(5, n, k, generator=g) * k ** -0.5).to(torch.bfloat16).to(dev), tiles=True)
    out = ops.flextrain_fp8_grouped_matmul(a, sa, b, sb, cd)
    at = 0
    for e, c in enumerate(counts.tolist()):
        if c:
            some = at + some_rows(g, c)
            bv = number(b[e], sb[e], 128)
            check(out[some], av[some] @ bv.t(), av[some], bv, what=f"expert {e}")
        at += c
    # weight gradients: 40 experts of 2000 x 1800
    counts = torch.randint(0, 60, (40,), generator=g, dtype=torch.int32)
    counts[7] = 0
    rows, cd = int(counts.sum()), counts.to(dev)
    dy, x = values(g, rows, 2000, sigma=1e-3), values(g, rows, 1800)
    a, sa = ops.flextrain_fp8_quantize_grouped_cols(dy.to(dev), cd, dtype=E5M2)
    b, sb = ops.flextrain_fp8_quantize_grouped_cols(x.to(dev), cd)
    acc = torch.full((40, 2000, 1800), 0.5, dtype=torch.bfloat16, device=dev)
    dw = ops.flextrain_fp8_grouped_wgrad(a, sa, b, sb, cd)
    ops.flextrain_fp8_grouped_wgrad(a, sa, b, sb, cd, C=acc, out=acc)
    to = 0
    for e, c in enumerate(counts.tolist()):
        p = -(-c // 128) * 128
        if e in (0, 7, 8, 39):
            some = some_rows(g, 2000)
            ae, be = number(a[some, to:to + p], sa[some, to // 128:(to + p) // 128]), number(b[:, to:to + p], sb[:, to // 128:(to + p) // 128])
            check(dw[e][some], ae @ be.t(), ae, be, what=f"expert {e}")
            half = torch.full((len(some), 1800), 0.5)
            check(acc[e][some], ae @ be.t() + 0.5, ae, be, half, what=f"expert {e} with C")
        to += p


def test_outputs_that_overlap_are_refused(dev):
    counts = torch.tensor([1, 1], dtype=torch.int32).to(dev)
    x = torch.ones(2, 16, dtype=torch.bfloat16, device=dev)
    a, sa = ops.flextrain_fp8_quantize_grouped_cols(x, counts, dtype=E5M2)
    b, sb = ops.flextrain_fp8_quantize_grouped_cols(x, counts)
    one = torch.zeros(16, 16, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError, match="overlap"):
        ops.flextrain_fp8_grouped_wgrad(a, sa, b, sb, counts, out=one.expand(2, 16, 16))
    # the experts' matrices side by side
    wide = torch.zeros(16, 2, 16, dtype=torch.bfloat16, device=dev)
    ops.flextrain_fp8_grouped_wgrad(a, sa, b, sb, counts, C=one.expand(2, 16, 16), out=wide.transpose(0, 1))
    assert (wide == 1.0).all()


@pytest.mark.parametrize("rows,cols", [(384, 200), (300, 136), (5, 64)])
def test_columns_alone_are_those_of_one_expert(dev, rows, cols):
    """A weight gradient reads the columns of the norm's output and nothing of its rows: all rows as one expert's."""
    g = gen(rows)
    y, dout = values(g, rows, cols).to(dev), values(g, rows, 72, sigma=1e-3).to(dev)
    all_rows = torch.tensor([rows], dtype=torch.int32).to(dev)
    yt, yts = ops.flextrain_fp8_quantize_grouped_cols(y, all_rows)
    _, _, want, want_s = ops.flextrain_fp8_quantize_both(y)
    same(yt[:, :rows], want.cpu().float().double(), "values")
    same(yts, want_s.cpu().float().double(), "scales")
    assert (yt.float()[:, rows:] == 0).all()
    _, _, dt, dts = ops.flextrain_fp8_quantize_both(dout, dtype=E5M2)
    dw = torch.randn(72, cols, generator=g).to(torch.bfloat16).to(dev)
    got = ops.flextrain_fp8_matmul(dt, dts, yt[:, :rows], yts, C=dw)
    assert torch.equal(got, ops.flextrain_fp8_matmul(dt, dts, want, want_s, C=dw))
