"""8-bit operands that are a part of a wider matrix: nothing behind the end of a row counts, whatever stands there.

Rows of an operand start at 16-byte addresses and the tile kernels load whole 16-byte chunks, so the bytes from K to the next
multiple of 16 are loaded and have to be dropped.  K takes every way its last 128 can end: inside its last chunk (241 .. 255:
no step back is needed, 383), inside an earlier one, at a chunk's end and at a block's.  Tolerances: test_gpu_fp8.py."""
from __future__ import annotations

import pytest
import torch

from oracle import fp8 as o
from tests.test_gpu_fp8 import E4M3, E5M2, check, operand, some_rows, values
from tests.util import gen

from flextrain_amd import ops

pytestmark = pytest.mark.gpu


def inside(dev, q, junk, g):
    """The values of ``q (.., rows, K)`` with the same bytes in rows that go on behind K: NaN, or finite numbers of the type."""
    k = q.shape[-1]
    ld = -(-k // 16) * 16 + 16
    if junk == "nan":
        wide = torch.full(q.shape[:-1] + (ld,), 0x7F, dtype=torch.uint8)
    else:
        wide = torch.randint(0, 0x78, q.shape[:-1] + (ld,), generator=g).to(torch.uint8)
    wide[..., :k] = q.cpu().contiguous().view(torch.uint8)
    return wide.to(dev).view(q.dtype)[..., :k]


# 128 x 128 tiles: outputs of a few hundred thousand values (the kernel of few rows is the faster one below)
@pytest.mark.parametrize("junk", ["nan", "finite"])
@pytest.mark.parametrize("k", [113, 127, 128, 129, 240, 241, 250, 255, 256, 300, 383])
def test_tiles(dev, k, junk):
    g = gen(k)
    m, n, fmt = 700, 520, E5M2 if k % 2 else E4M3
    a, sa, av = operand(dev, values(g, m, k, sigma=1e-3 if fmt is E5M2 else 1.0), fmt)
    b, sb, bv = operand(dev, values(g, n, k, sigma=k ** -0.5), tiles=fmt is E4M3)
    check(ops.flextrain_fp8_matmul(inside(dev, a, junk, g), sa, inside(dev, b, junk, g), sb), av @ bv.t(), av, bv)


# few tiles and a long contraction: slices, of which only the last ends with the row; and the kernel of few rows
@pytest.mark.parametrize("junk", ["nan", "finite"])
@pytest.mark.parametrize("m,n", [(1, 16), (40, 130)])
@pytest.mark.parametrize("k", [14322, 14330, 14335, 14337, 1009, 2041])
def test_long_contractions(dev, m, n, k, junk):
    g = gen(k + m)
    a, sa, av = operand(dev, values(g, m, k))
    b, sb, bv = operand(dev, values(g, n, k, sigma=k ** -0.5))
    out = ops.flextrain_fp8_matmul(inside(dev, a, junk, g), sa, inside(dev, b, junk, g), sb, out_dtype=torch.float32)
    check(out, av @ bv.t(), av, bv)
    assert torch.equal(out, ops.flextrain_fp8_matmul(a, sa, b, sb, out_dtype=torch.float32))


# one contiguous row, and rows of which the last ends where its memory does: the other bytes of the last 16 are another tensor's
@pytest.mark.parametrize("m,n,k", [(1, 16, 14330), (1, 300, 1003), (1, 1, 5), (20, 16, 14321), (3, 1, 250)])
def test_memory_that_ends_with_the_last_row(dev, m, n, k):
    def last(q):
        rows, ld = q.shape[0], -(-k // 16) * 16
        memory = torch.full((rows * ld,), 0x7F, dtype=torch.uint8, device=dev)
        memory[:(rows - 1) * ld + k].as_strided((rows, k), (ld, 1)).copy_(q.view(torch.uint8))
        if rows == 1:
            return memory[:k].view(1, k).view(q.dtype)
        return memory[:(rows - 1) * ld + k].as_strided((rows, k), (ld, 1)).view(q.dtype)

    g = gen(k)
    a, sa, av = operand(dev, values(g, m, k))
    b, sb, bv = operand(dev, values(g, n, k, sigma=k ** -0.5))
    out = ops.flextrain_fp8_matmul(last(a), sa, last(b), sb, out_dtype=torch.float32)
    check(out, av @ bv.t(), av, bv)
    assert torch.equal(out, ops.flextrain_fp8_matmul(a, sa, b, sb, out_dtype=torch.float32))


# 256 x 256 tiles, several to a workgroup
@pytest.mark.parametrize("junk", ["nan", "finite"])
@pytest.mark.parametrize("k", [241, 250, 255, 383, 1148])
def test_large_outputs(dev, k, junk):
    g = gen(k)
    m, n = 4200, 3700
    some = some_rows(g, m)
    a, sa, av = operand(dev, values(g, m, k))
    b, sb, bv = operand(dev, values(g, n, k, sigma=k ** -0.5), tiles=True)
    out = ops.flextrain_fp8_matmul(inside(dev, a, junk, g), sa, inside(dev, b, junk, g), sb)
    check(out[some], av[some] @ bv.t(), av[some], bv)
    assert torch.equal(out, ops.flextrain_fp8_matmul(a, sa, b, sb))


# by expert: the kernel of few rows, 128-row tiles, 256-row tiles
@pytest.mark.parametrize("junk", ["nan", "finite"])
@pytest.mark.parametrize("k", [113, 241, 250, 255, 300, 383])
@pytest.mark.parametrize("counts,n", [([3, 0, 1, 9], 72), ([130, 0, 300, 51], 512)], ids=["few", "tiles"])
def test_experts(dev, counts, n, k, junk):
    experts(dev, counts, n, k, junk)


@pytest.mark.parametrize("junk", ["nan", "finite"])
@pytest.mark.parametrize("k", [250, 383])
def test_experts_large(dev, k, junk):
    experts(dev, [700, 0, 513] * 5 + [900], 2000, k, junk)


def experts(dev, counts, n, k, junk):
    g = gen(n + k)
    E, rows = len(counts), sum(counts)
    c = torch.tensor(counts, dtype=torch.int32).to(dev)
    b, sb = ops.flextrain_fp8_quantize((torch.randn(E, n, k, generator=g) * k ** -0.5).to(torch.bfloat16).to(dev), tiles=True)
    bj = inside(dev, b, junk, g)
    source = torch.randint(0, 21, (rows,), generator=g, dtype=torch.int32)
    for gathered in (False, True):
        a, sa, av = operand(dev, values(g, 21 if gathered else rows, k))
        kw = {"row_sources": source.to(dev)} if gathered else {}
        out = ops.flextrain_fp8_grouped_matmul(inside(dev, a, junk, g), sa, bj, sb, c, **kw)
        # the quantiser's own operands have zeros there
        assert torch.equal(out, ops.flextrain_fp8_grouped_matmul(a, sa, b, sb, c, **kw))
        av = av[source.long()] if gathered else av
        at = 0
        for e, m in enumerate(counts):
            if m:
                some = some_rows(g, m)
                bv = o.dequantize(b[e].cpu(), sb[e].cpu(), 128)
                check(out[at:at + m][some], av[at:at + m][some] @ bv.t(), av[at:at + m][some], bv, what=f"expert {e}")
            at += m
