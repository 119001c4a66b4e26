"""Argument checks of the 8-bit entry points of the C ABI, on the CPU: every refused call returns -1 before anything is
enqueued, so the pointers are never dereferenced.  Each case breaks one rule of a valid call, which the GPU tests launch;
calls with nothing to do return 0."""
from __future__ import annotations

import pytest
import torch

from flextrain_amd._lib import fp8_enum, lib

F32, F16, BF16, E4M3, E5M2 = 0, 1, 2, 3, 4
P = 0x7F0000001000          # a 16-byte-aligned, never-dereferenced address
ODD = P + 2


def _norm(**kw):
    a = dict(x=P, r=P, w=P, h=P, y=P, ldy=128, s=P, lds=4, rstd=P, rows=4, cols=128, x_dt=BF16, w_dt=BF16, y_dt=E4M3)
    a.update(kw)
    return lib().fx_add_rmsnorm_fwd(a["x"], a["r"], a["w"], a["h"], a["y"], a["ldy"], a["s"], a["lds"], a["rstd"], a["rows"], a["cols"],
                                    1e-5, a["x_dt"], a["w_dt"], a["y_dt"], None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(cols=0), dict(x=None), dict(y=None), dict(rstd=None), dict(s=None), dict(h=None), dict(x_dt=3),
                                dict(w_dt=9), dict(y_dt=F16), dict(y_dt=7), dict(ldy=120), dict(ldy=144), dict(cols=120, ldy=120), dict(lds=3),
                                dict(y=ODD), dict(y_dt=BF16, ldy=136), dict(rows=1 << 24, lds=1 << 24)])
def test_add_rmsnorm_fwd_refuses(kw):
    assert _norm(**kw) == -1


def test_add_rmsnorm_of_no_rows_is_a_no_op():
    assert _norm(rows=0, x=None, r=None, h=None, y=None, s=None, rstd=None) == 0
    assert lib().fx_add_rmsnorm_bwd(None, None, None, None, None, None, None, 0, 0, 0, 128, BF16, BF16, None, 0, None) == 0


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(cols=0), dict(dy=None), dict(h=None), dict(rstd=None), dict(dx=None), dict(ws=None), dict(nbytes=0),
                                dict(rows=1 << 24)])
def test_add_rmsnorm_bwd_refuses(kw):
    a = dict(dy=P, h=P, rstd=P, dx=P, rows=4, cols=128, ws=P, nbytes=int(lib().fx_add_rmsnorm_bwd_ws_bytes(4, 128)))
    assert a["nbytes"] > 0
    a.update(kw)
    assert lib().fx_add_rmsnorm_bwd(a["dy"], P, a["h"], P, a["rstd"], a["dx"], P, F32, 0, a["rows"], a["cols"], BF16, BF16, a["ws"], a["nbytes"], None) == -1


def _quant(**kw):
    a = dict(x=P, ldx=200, xb=0, batch=1, rows=300, cols=200, x_dt=BF16, q_dt=E4M3, tiles=0, q=P, ldq=208, qb=0, s=P, lds=300, sb=0, qt=P, ldt=304, tb=0,
             st=P, ldst=200, stb=0)
    a.update(kw)
    return lib().fx_fp8_quantize(a["x"], a["ldx"], a["xb"], a["batch"], a["rows"], a["cols"], a["x_dt"], a["q_dt"], a["tiles"], a["q"], a["ldq"], a["qb"],
                                 a["s"], a["lds"], a["sb"], a["qt"], a["ldt"], a["tb"], a["st"], a["ldst"], a["stb"], None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(cols=0), dict(x=None), dict(q=None), dict(s=None), dict(st=None), dict(qt=None), dict(x_dt=E4M3),
                                dict(q_dt=BF16), dict(ldx=199), dict(ldq=200), dict(ldq=224), dict(ldq=192), dict(lds=299), dict(q=ODD), dict(qt=ODD),
                                dict(ldt=300), dict(ldt=320), dict(ldst=199), dict(tiles=1, lds=2), dict(tiles=1, ldst=1), dict(batch=-1), dict(batch=65536),
                                dict(batch=2, qb=8), dict(batch=2, qb=300 * 208, tb=24),
                                dict(rows=1 << 33, cols=8, ldx=8, ldq=16, lds=1 << 33, qt=None, st=None)])
def test_quantize_refuses(kw):
    assert _quant(**kw) == -1


def test_quantize_of_nothing_is_a_no_op():
    assert _quant(rows=0) == 0 and _quant(batch=0) == 0


def _columns(**kw):
    cap = int(lib().fx_fp8_grouped_capacity(300, 4))
    a = dict(x=P, ldx=200, src=300, rows=300, cols=200, x_dt=BF16, q_dt=E5M2, counts=P, E=4, map=None, qt=P, ldt=cap, st=P, ldst=200)
    a.update(kw)
    return lib().fx_fp8_quantize_grouped_cols(a["x"], a["ldx"], a["src"], a["rows"], a["cols"], a["x_dt"], a["q_dt"], a["counts"], a["E"], a["map"],
                                              a["qt"], a["ldt"], a["st"], a["ldst"], None)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(E=0), dict(cols=0), dict(src=-1), dict(x=None), dict(counts=None), dict(qt=None), dict(st=None),
                                dict(src=299), dict(src=0, map=P), dict(rows=(1 << 24) + 1, src=1 << 25), dict(map=P, src=1 << 31), dict(ldt=300),
                                dict(ldt=1024), dict(qt=ODD), dict(ldst=199), dict(ldx=8), dict(x_dt=9), dict(q_dt=F32)])
def test_quantize_grouped_columns_refuses(kw):
    assert _columns(**kw) == -1


def test_capacity_holds_every_split():
    cap = lib().fx_fp8_grouped_capacity
    assert cap(-1, 4) == -1 and cap(4, 0) == -1 and cap(0, 4) == 384
    for rows, counts in [(5, [1] * 5), (300, [1, 1, 1, 297]), (129, [129]), (1000, [125] * 8), (260, [129, 131, 0])]:
        assert cap(rows, len(counts)) >= sum(-(-c // 128) * 128 for c in counts) and cap(rows, len(counts)) % 128 == 0


def _gemm(**kw):
    a = dict(A=P, lda=512, a_dt=E5M2, SA=P, sar=1, sak=300, at=0, B=P, ldb=512, SB=P, sbr=1, sbk=3, bt=1, C=None, ldc=0, D=P, ldd=400, M=300, N=400, K=500,
             d_dt=BF16, ws=P, nbytes=1 << 40)
    a.update(kw)
    return lib().fx_fp8_gemm(a["A"], a["lda"], a["a_dt"], a["SA"], a["sar"], a["sak"], a["at"], a["B"], a["ldb"], a["SB"], a["sbr"], a["sbk"], a["bt"],
                             a["C"], a["ldc"], a["D"], a["ldd"], a["M"], a["N"], a["K"], a["d_dt"], a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("kw", [dict(M=-1), dict(N=-1), dict(K=-1), dict(a_dt=BF16), dict(d_dt=E4M3), dict(D=None), dict(A=None), dict(B=None), dict(SA=None),
                                dict(SB=None), dict(A=ODD), dict(B=ODD), dict(lda=500), dict(ldb=504), dict(lda=496), dict(ldd=399), dict(C=P, ldc=399),
                                dict(lda=1 << 23), dict(sar=-1), dict(sbk=-1), dict(sar=1 << 28), dict(M=0x7FFFFFFF, sar=0), dict(N=0x7FFFFFFF, ldd=1 << 31, sbr=0),
                                dict(ws=ODD)])
def test_matmul_refuses(kw):
    assert _gemm(**kw) == -1


def test_matmul_workspace_is_checked():
    ws = lib().fx_fp8_gemm_ws_bytes
    assert ws(0, 8, 8) == 0 and ws(8, 8, 0) == 0 and ws(1, 4096, 4096) == 0
    # few tiles and a long contraction, which is cut into slices
    shape = dict(M=520, N=500, K=9000, lda=9008, ldb=9008, ldd=500, bt=0, sbk=500, sak=520)
    need = int(ws(520, 500, 9000))
    assert need >= 2 * 4 * 520 * 500
    assert _gemm(**shape, nbytes=need - 1) == -1 and _gemm(**shape, ws=None) == -1


def test_matmul_of_nothing_is_a_no_op():
    assert _gemm(M=0, A=None, D=None) == 0 and _gemm(N=0, B=None, D=None) == 0


def _rows(**kw):
    a = dict(A=P, lda=512, a_dt=E4M3, SA=P, sar=1, sak=300, map=None, arows=300, B=P, ldb=512, be=400 * 512, SB=P, sbr=1, sbk=3, sbe=12, bt=1, counts=P, E=4,
             rows=300, D=P, ldd=400, N=400, K=500, d_dt=BF16)
    a.update(kw)
    return lib().fx_fp8_grouped_gemm(a["A"], a["lda"], a["a_dt"], a["SA"], a["sar"], a["sak"], a["map"], a["arows"], a["B"], a["ldb"], a["be"], a["SB"], a["sbr"],
                                     a["sbk"], a["sbe"], a["bt"], a["counts"], a["E"], a["rows"], a["D"], a["ldd"], a["N"], a["K"], a["d_dt"], None)


@pytest.mark.parametrize("kw", [dict(E=0), dict(rows=-1), dict(N=-1), dict(K=-1), dict(a_dt=F16), dict(d_dt=8), dict(rows=(1 << 24) + 1, arows=1 << 25),
                                dict(counts=None), dict(D=None), dict(A=None), dict(SB=None), dict(A=ODD), dict(lda=500), dict(be=400 * 512 + 8), dict(ldb=496),
                                dict(ldd=399), dict(ldb=1 << 23), dict(arows=299), dict(map=P, arows=0), dict(map=P, arows=1 << 24), dict(sak=-1), dict(sbe=-1),
                                dict(be=-16), dict(sar=1 << 28), dict(N=0x7FFFFFFF, ldd=1 << 31, sbr=0)])
def test_grouped_matmul_refuses(kw):
    assert _rows(**kw) == -1


def test_grouped_matmul_of_nothing_is_a_no_op():
    assert _rows(rows=0, A=None, D=None) == 0 and _rows(N=0, B=None, D=None) == 0


def _wgrad(**kw):
    a = dict(A=P, lda=768, a_dt=E5M2, SA=P, sar=1, sak=200, B=P, ldb=768, SB=P, sbr=1, sbk=264, counts=P, E=4, cap=768, C=None, ldc=0, ce=0, D=P, ldd=264,
             de=200 * 264, M=200, N=264, d_dt=BF16)
    a.update(kw)
    return lib().fx_fp8_grouped_wgrad(a["A"], a["lda"], a["a_dt"], a["SA"], a["sar"], a["sak"], a["B"], a["ldb"], a["SB"], a["sbr"], a["sbk"], a["counts"], a["E"],
                                      a["cap"], a["C"], a["ldc"], a["ce"], a["D"], a["ldd"], a["de"], a["M"], a["N"], a["d_dt"], None)


@pytest.mark.parametrize("kw", [dict(E=0), dict(cap=-128), dict(cap=700), dict(M=-1), dict(N=-1), dict(a_dt=BF16), dict(d_dt=5), dict(cap=1 << 23), dict(counts=None),
                                dict(D=None), dict(A=None), dict(SB=None), dict(A=ODD), dict(ldb=776), dict(lda=640), dict(ldd=263), dict(C=P, ldc=263),
                                dict(lda=1 << 23), dict(sar=-1), dict(sbr=1 << 28), dict(M=0x7FFFFFFF, sar=0)])
def test_grouped_wgrad_refuses(kw):
    assert _wgrad(**kw) == -1


def test_grouped_wgrad_of_nothing_is_a_no_op():
    assert _wgrad(M=0, A=None, D=None) == 0 and _wgrad(N=0, B=None, D=None) == 0


def test_dimensions_past_32_bits_are_refused_by_the_wrappers():
    """(The C ABI takes them as int; tensors without storage show it.)"""
    from flextrain_amd import ops

    big = 1 << 31
    fp8 = lambda *shape: torch.empty(shape, dtype=torch.float8_e4m3fn, device="meta")
    scales = lambda *shape: torch.empty(shape, dtype=torch.float8_e8m0fnu, device="meta")
    counts = torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="larger than"):
        ops.flextrain_fp8_matmul(fp8(big, 16), scales(big, 1), fp8(8, 16), scales(8, 1))
    with pytest.raises(ValueError, match="larger than"):
        ops.flextrain_fp8_grouped_matmul(fp8(8, 16), scales(8, 1), fp8(2, big, 16), scales(2, big, 1), counts)
    with pytest.raises(ValueError, match="larger than"):
        ops.flextrain_fp8_grouped_wgrad(fp8(big, 128), scales(big, 1), fp8(8, 128), scales(8, 1), counts)
    x = torch.empty(1, big, dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="larger than"):
        ops.flextrain_add_rmsnorm_fwd(x)
    with pytest.raises(ValueError, match="larger than"):
        ops.flextrain_add_rmsnorm_bwd(x, x, None, torch.empty(1, 1, device="meta"))
    with pytest.raises(ValueError, match="65535"):
        ops.flextrain_fp8_quantize(torch.empty(1 << 16, 1, 16, dtype=torch.bfloat16, device="meta"))


def test_only_the_two_8_bit_types_have_an_enum():
    assert fp8_enum(torch.float8_e4m3fn) == E4M3 and fp8_enum(torch.float8_e5m2) == E5M2
    for t in (torch.bfloat16, torch.float8_e4m3fnuz, torch.float8_e5m2fnuz, torch.uint8):
        with pytest.raises(TypeError):
            fp8_enum(t)


def test_expert_columns_that_no_weight_gradient_takes_are_refused():
    """Rows of the quantised columns are operands of the expert weight gradient, whose strides are below 2^23."""
    from flextrain_amd import ops

    cap = lambda rows, E: (rows + 127 * E) // 128 * 128
    for rows, E in (((1 << 23) - 127, 1), ((1 << 23) - 4 * 127, 4), (1 << 24, 2), (5, 1 << 17)):
        assert cap(rows, E) >= 1 << 23
        assert _columns(rows=rows, src=rows, E=E, ldt=cap(rows, E)) == -1
        with pytest.raises(ValueError, match="capacity"):
            ops.flextrain_fp8_quantize_grouped_cols(torch.empty(rows, 1, dtype=torch.bfloat16, device="meta"), torch.ones(E, dtype=torch.int32))
    # the largest that both take: refused only for what is broken beside it
    rows = (1 << 23) - 128
    assert cap(rows, 1) < 1 << 23 and _columns(rows=rows, src=rows, E=1, ldt=cap(rows, 1), counts=None) == -1
    with pytest.raises(ValueError, match="on the GPU"):
        ops.flextrain_fp8_quantize_grouped_cols(torch.empty(rows, 1, dtype=torch.bfloat16, device="meta"), torch.ones(1, dtype=torch.int32))


def test_lanes_exchange_through_lds_by_a_fence():
    """The epilogue of the 8-bit tiles hands values from lane to lane through LDS with no workgroup barrier: a fence of the
    wave's scope orders them in the program (in the host simulation it is what brings the lanes together)."""
    import os

    import flextrain_amd

    text = open(os.path.join(os.path.dirname(flextrain_amd.__file__), "csrc", "fp8_core.h")).read()
    assert "// lockstep:" not in text                                       # an order that only a comment claims
    body = text[text.index("FX_DEV void wave_exchange()"):][:400]
    assert body.index("__ATOMIC_RELEASE") < body.index("wave_barrier()") < body.index("__ATOMIC_ACQUIRE")
    epilogue = text[text.index("FX_DEV void fp8_epilogue"):text.index("kernels over a list of tiles")]
    assert epilogue.count("wave_exchange();") == 3                          # band free, C staged, band staged
