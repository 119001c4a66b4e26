"""8-bit matrix products with a power-of-two scale per block of 128 values: the quantiser that makes the operands,
the products that read them, and the products grouped by expert.  The reference's ops are 16-bit and wider; these
have no counterpart there.

Values are ``torch.float8_e4m3fn`` or ``torch.float8_e5m2``, scales ``torch.float8_e8m0fnu`` (``2**e``).  A scale
tensor has one entry per block, indexed like the values it belongs to: ``(rows, ceil(cols / 128))`` for blocks of one
row, ``(ceil(rows / 128), ceil(cols / 128))`` for 128 x 128 tiles.  The quantiser stores scales with the block index
outermost and pads rows of values to multiples of 16 bytes; the products take scales of any strides and values whose
rows start at 16-byte addresses.

=================  ==========================================  =====================================================
 product            operands                                    made by
=================  ==========================================  =====================================================
 ``x @ W.T``        ``x`` by rows, ``W (N, K)`` in tiles        :func:`flextrain_fp8_quantize` /
                                                                :func:`flextrain_fp8_quantize_both` (``tiles=True``)
 ``dy @ W``         ``dy`` by rows, ``W`` transposed in tiles   the transposed pair of the same two calls
 ``dy.T @ x``       both by columns (transposed)                :func:`flextrain_fp8_quantize_both`
 per expert         the same                                    :func:`flextrain_fp8_quantize_grouped_cols`
=================  ==========================================  =====================================================
"""
from __future__ import annotations

import torch

from .._lib import check, dtype_enum, fp8_enum, lib, on_device, ptr, require_same_device, stream_ptr

_E8M0 = torch.float8_e8m0fnu


def _round_up(n: int, m: int) -> int:
    return (n + m - 1) // m * m


def _blocks(n: int) -> int:
    return (n + 127) // 128


def _fp8_rows(lead, rows, cols, dtype, device):
    """Uninitialised 8-bit values ``(*lead, rows, cols)`` whose rows start at multiples of 16 bytes."""
    return torch.empty(*lead, rows, _round_up(cols, 16), dtype=dtype, device=device)[..., :cols]


def _scale_store(lead, rows, blocks, device):
    """Uninitialised scales ``(*lead, rows, blocks)``, the block index outermost in memory."""
    return torch.empty(*lead, blocks, rows, dtype=_E8M0, device=device).transpose(-1, -2)


def _input_matrix(X, op):
    if X.dim() not in (2, 3):
        raise ValueError(f"{op}: X must be (rows, cols) or (batch, rows, cols), got {X.dim()} dims")
    if X.shape[-1] == 0:
        raise ValueError(f"{op}: X has no columns")
    if X.shape[-1] > 1 and X.stride(-1) != 1:
        raise ValueError(f"{op}: X must have unit column stride")
    # a dimension of one has no stride of its own
    ldx = X.stride(-2) if X.shape[-2] > 1 else X.shape[-1]
    if ldx < X.shape[-1] or (X.dim() == 3 and X.shape[0] > 1 and X.stride(0) < 0):
        raise ValueError(f"{op}: the rows of X overlap")
    return ldx, X.stride(0) if X.dim() == 3 else 0


def _quantize(X, dtype, tiles, both, op):
    ldx, x_batch = _input_matrix(X, op)
    require_same_device(X, op=op)
    lead, (rows, cols) = X.shape[:-2], X.shape[-2:]
    batch = X.shape[0] if X.dim() == 3 else 1
    q = _fp8_rows(lead, rows, cols, dtype, X.device)
    s = _scale_store(lead, _blocks(rows) if tiles else rows, _blocks(cols), X.device)
    qt = st = None
    if both:
        qt = _fp8_rows(lead, cols, rows, dtype, X.device)
        st = _scale_store(lead, _blocks(cols) if tiles else cols, _blocks(rows), X.device)
    if rows == 0 or batch == 0:
        return q, s, qt, st
    ldq, ldt = _round_up(cols, 16), _round_up(rows, 16)
    with on_device(X):
        rc = lib().fx_fp8_quantize(
            ptr(X), ldx, x_batch, batch, rows, cols, dtype_enum(X.dtype), fp8_enum(dtype), 1 if tiles else 0,
            ptr(q), ldq, rows * ldq, ptr(s), s.shape[-2], s.shape[-2] * s.shape[-1],
            ptr(qt), ldt, cols * ldt, ptr(st), st.shape[-2] if both else 0, st.shape[-2] * st.shape[-1] if both else 0,
            stream_ptr(X.device))
    check(rc, "fx_fp8_quantize")
    return q, s, qt, st


def flextrain_fp8_quantize(X, dtype=torch.float8_e4m3fn, tiles=False):
    """``(q, scales)`` of a matrix ``X (rows, cols)`` (or a batch of them): blocks of one row and 128 columns, or with
    ``tiles`` of 128 x 128.

    A block's scale is ``2**e`` with the smallest ``e`` that brings its largest finite magnitude to at most the
    dtype's largest number (448 / 57344); a block of zeros has scale 1.  Infinities and NaN do not count and stay
    (e4m3, which has no infinity: NaN).  ``X`` may be bf16, fp16 or fp32 with any row stride."""
    q, s, _, _ = _quantize(X, dtype, tiles, False, "flextrain_fp8_quantize")
    return q, s


def flextrain_fp8_quantize_both(X, dtype=torch.float8_e4m3fn, tiles=False):
    """``(q, scales, qt, scales_t)``: ``X`` as :func:`flextrain_fp8_quantize` gives it, and ``X.T`` in blocks along the
    rows of ``X``, from one read of ``X``.  With ``tiles`` both hold the same values and scales, transposed."""
    return _quantize(X, dtype, tiles, True, "flextrain_fp8_quantize_both")


def _counts_of(counts, op):
    if counts.dtype != torch.int32 or counts.dim() != 1 or not counts.is_contiguous() or counts.numel() == 0:
        raise ValueError(f"{op}: expert counts must be a contiguous int32 vector")
    return counts.numel()


def _sources_of(row_sources, op):
    if row_sources.dtype != torch.int32 or row_sources.dim() != 1 or not row_sources.is_contiguous():
        raise ValueError(f"{op}: row sources must be a contiguous int32 vector")
    return row_sources.numel()


def flextrain_fp8_quantize_grouped_cols(X, counts, dtype=torch.float8_e4m3fn, row_sources=None):
    """``(qt, scales_t)`` of expert-sorted rows ``X (rows, cols)`` for the expert weight gradients: the transposed
    matrix, quantised per expert in blocks of 128 rows of one column.

    ``qt`` is ``(cols, capacity)`` with every expert's rows starting at a multiple of 128 (capacity: room for any
    split of the rows); places without a row hold 0 with scale 1.  ``counts (E,)`` int32 on the GPU.  With
    ``row_sources`` (int32, one entry per expert-sorted row) ``X`` is the unsorted matrix and sorted row ``r`` is its
    row ``row_sources[r]``."""
    op = "flextrain_fp8_quantize_grouped_cols"
    if X.dim() != 2:
        raise ValueError(f"{op}: X must be (rows, cols)")
    ldx, _ = _input_matrix(X, op)
    E = _counts_of(counts, op)
    rows = X.shape[0] if row_sources is None else _sources_of(row_sources, op)
    require_same_device(X, counts, row_sources, op=op)
    if rows > 0 and X.shape[0] == 0:
        raise ValueError(f"{op}: X has no rows")
    if rows > 1 << 24:
        raise ValueError(f"{op}: at most 2**24 expert rows")
    cols = X.shape[1]
    cap = int(lib().fx_fp8_grouped_capacity(rows, E))
    qt = torch.empty(cols, cap, dtype=dtype, device=X.device)
    st = _scale_store((), cols, cap // 128, X.device)
    q_dt = fp8_enum(dtype)
    if cap > 0:
        with on_device(X):
            rc = lib().fx_fp8_quantize_grouped_cols(ptr(X), ldx, X.shape[0], rows, cols, dtype_enum(X.dtype), q_dt,
                                                    ptr(counts), E, ptr(row_sources), ptr(qt), cap, ptr(st), cols,
                                                    stream_ptr(X.device))
        check(rc, "fx_fp8_quantize_grouped_cols")
    return qt, st


def _values(t, name, op):
    """Row stride of an 8-bit operand ``(..., rows, cols)``."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{op}: {name} must have unit stride along the contraction")
    ld = t.stride(-2) if t.shape[-2] > 1 else _round_up(t.shape[-1], 16)
    if t.numel() and (ld % 16 or ld < t.shape[-1] or t.data_ptr() % 16):
        raise ValueError(f"{op}: the rows of {name} must start at 16-byte addresses (they are {ld} bytes apart)")
    return ld


def _scales(s, rows, blocks, tiles_allowed, name, op):
    """(row stride, block stride, 1 for 128-row tiles) of an operand's scales ``(..., rows | row blocks, blocks)``."""
    if s.dtype != _E8M0:
        raise TypeError(f"{op}: {name} must be {_E8M0}, got {s.dtype}")
    got = tuple(s.shape[-2:])
    if got == (rows, blocks):
        return s.stride(-2), s.stride(-1), 0
    if tiles_allowed and got == (_blocks(rows), blocks):
        return s.stride(-2), s.stride(-1), 1
    raise ValueError(f"{op}: {name} has shape {tuple(s.shape)}, expected {(rows, blocks)}"
                     + (f" or {(_blocks(rows), blocks)}" if tiles_allowed else ""))


def _operand_dtypes(A, B, op):
    a_dt = fp8_enum(A.dtype)
    if B.dtype != torch.float8_e4m3fn:
        raise TypeError(f"{op}: B must be torch.float8_e4m3fn (a gradient in e5m2 is the first operand), got {B.dtype}")
    return a_dt


def _output(out, shape, out_dtype, C, device, op):
    """The output tensor; C and out have its shape, its dtype and unit column stride."""
    for t, name in ((C, "C"), (out, "out")):
        if t is None:
            continue
        if tuple(t.shape) != tuple(shape):
            raise ValueError(f"{op}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{op}: {name} must have unit column stride")
        if t.shape[-2] > 1 and t.stride(-2) < t.shape[-1]:
            raise ValueError(f"{op}: the rows of {name} overlap")
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else C.dtype if C is not None else torch.bfloat16
    dtype_enum(out_dtype)
    for t, name in ((C, "C"), (out, "out")):
        if t is not None and t.dtype != out_dtype:
            raise TypeError(f"{op}: {name} is {t.dtype}, the output {out_dtype}")
    return out if out is not None else torch.empty(shape, dtype=out_dtype, device=device)


def _ld(t):
    return 0 if t is None else t.stride(-2) if t.shape[-2] > 1 else t.shape[-1]


def flextrain_fp8_matmul(A, A_scales, B, B_scales, C=None, out=None, out_dtype=None):
    """``out = A @ B.T (+ C)`` of 8-bit operands ``A (M, K)``, ``B (N, K)`` with block scales, accumulated in fp32.

    ``A`` is e4m3 or e5m2, ``B`` e4m3; each has scales per row and 128 k or per 128 x 128 tile (told apart by their
    shape).  ``C`` has the output's shape and dtype and may be ``out`` (a gradient accumulated in place).  Output
    dtype: ``out_dtype``, else that of ``out`` or ``C``, else bf16."""
    op = "flextrain_fp8_matmul"
    if A.dim() != 2 or B.dim() != 2 or A.shape[1] != B.shape[1]:
        raise ValueError(f"{op}: A {tuple(A.shape)} and B {tuple(B.shape)} must be (M, K) and (N, K)")
    a_dt = _operand_dtypes(A, B, op)
    (M, K), N = A.shape, B.shape[0]
    lda, ldb = _values(A, "A", op), _values(B, "B", op)
    sa = _scales(A_scales, M, _blocks(K), True, "A_scales", op)
    sb = _scales(B_scales, N, _blocks(K), True, "B_scales", op)
    require_same_device(A, A_scales, B, B_scales, C, out, op=op)
    D = _output(out, (M, N), out_dtype, C, A.device, op)
    if M == 0 or N == 0:
        return D
    L = lib()
    with on_device(A):
        nbytes = int(L.fx_fp8_gemm_ws_bytes(M, N, K))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=A.device) if nbytes else None
        rc = L.fx_fp8_gemm(ptr(A), lda, a_dt, ptr(A_scales), *sa, ptr(B), ldb, ptr(B_scales), *sb, ptr(C), _ld(C), ptr(D),
                           _ld(D), M, N, K, dtype_enum(D.dtype), ptr(ws), nbytes, stream_ptr(A.device))
    check(rc, "fx_fp8_gemm")
    return D


def flextrain_fp8_grouped_matmul(A, A_scales, B, B_scales, counts, row_sources=None, out=None, out_dtype=None):
    """``out[rows of e] = A[rows of e] @ B[e].T`` for every expert, in one launch that reads the counts on the GPU.

    ``A (rows, K)`` expert-sorted, e4m3 or e5m2, scales per row; ``B (E, N, K)`` e4m3, scales ``(E, ceil(N / 128),
    ceil(K / 128))`` (tiles) or ``(E, N, ceil(K / 128))``; ``counts (E,)`` int32 with the sum ``rows``.  With
    ``row_sources`` (int32, one entry per expert-sorted row) ``A`` is the unsorted matrix and its rows are gathered by
    the tile loads.  Rows of ``out`` behind the last expert's are left as they were."""
    op = "flextrain_fp8_grouped_matmul"
    if A.dim() != 2 or B.dim() != 3 or A.shape[1] != B.shape[2]:
        raise ValueError(f"{op}: A {tuple(A.shape)} and B {tuple(B.shape)} must be (rows, K) and (E, N, K)")
    a_dt = _operand_dtypes(A, B, op)
    E, N, K = B.shape
    if _counts_of(counts, op) != E:
        raise ValueError(f"{op}: {counts.numel()} counts for {E} experts")
    rows = A.shape[0] if row_sources is None else _sources_of(row_sources, op)
    if rows > 1 << 24:
        raise ValueError(f"{op}: at most 2**24 expert rows")
    if rows > 0 and A.shape[0] == 0:
        raise ValueError(f"{op}: A has no rows")
    lda, ldb = _values(A, "A", op), _values(B, "B", op)
    if E > 1 and B.numel() and B.stride(0) % 16:
        raise ValueError(f"{op}: every expert's matrix must start at a 16-byte address")
    sa_row, sa_k, _ = _scales(A_scales, A.shape[0], _blocks(K), False, "A_scales", op)
    if B_scales.dim() != 3 or B_scales.shape[0] != E:
        raise ValueError(f"{op}: B_scales has shape {tuple(B_scales.shape)}, expected {E} experts")
    sb_row, sb_k, b_tiles = _scales(B_scales, N, _blocks(K), True, "B_scales", op)
    require_same_device(A, A_scales, B, B_scales, counts, row_sources, out, op=op)
    D = _output(out, (rows, N), out_dtype, None, A.device, op)
    if rows == 0 or N == 0:
        return D
    with on_device(A):
        rc = lib().fx_fp8_grouped_gemm(ptr(A), lda, a_dt, ptr(A_scales), sa_row, sa_k, ptr(row_sources), A.shape[0], ptr(B),
                                       ldb, B.stride(0), ptr(B_scales), sb_row, sb_k, B_scales.stride(0), b_tiles,
                                       ptr(counts), E, rows, ptr(D), _ld(D), N, K, dtype_enum(D.dtype), stream_ptr(A.device))
    check(rc, "fx_fp8_grouped_gemm")
    return D


def flextrain_fp8_grouped_wgrad(A, A_scales, B, B_scales, counts, C=None, out=None, out_dtype=None):
    """``out[e] = A_e @ B_e.T (+ C[e])`` for every expert: the weight gradient ``dy_e.T @ x_e`` of operands made by
    :func:`flextrain_fp8_quantize_grouped_cols` with the same ``counts``.

    ``A (M, capacity)`` e4m3 or e5m2, ``B (N, capacity)`` e4m3, scales ``(M | N, capacity / 128)``; ``out`` / ``C``
    ``(E, M, N)`` of one dtype (``C`` may be ``out``).  An expert without rows gives ``C[e]``, or zeros."""
    op = "flextrain_fp8_grouped_wgrad"
    if A.dim() != 2 or B.dim() != 2 or A.shape[1] != B.shape[1]:
        raise ValueError(f"{op}: A {tuple(A.shape)} and B {tuple(B.shape)} must be (M, capacity) and (N, capacity)")
    a_dt = _operand_dtypes(A, B, op)
    E = _counts_of(counts, op)
    (M, cap), N = A.shape, B.shape[0]
    if cap % 128:
        raise ValueError(f"{op}: the capacity {cap} is not a multiple of 128")
    if cap > 1 << 24:
        raise ValueError(f"{op}: at most 2**24 expert rows")
    lda, ldb = _values(A, "A", op), _values(B, "B", op)
    sa_row, sa_k, _ = _scales(A_scales, M, cap // 128, False, "A_scales", op)
    sb_row, sb_k, _ = _scales(B_scales, N, cap // 128, False, "B_scales", op)
    require_same_device(A, A_scales, B, B_scales, counts, C, out, op=op)
    D = _output(out, (E, M, N), out_dtype, C, A.device, op)
    if M == 0 or N == 0:
        return D
    with on_device(A):
        rc = lib().fx_fp8_grouped_wgrad(ptr(A), lda, a_dt, ptr(A_scales), sa_row, sa_k, ptr(B), ldb, ptr(B_scales), sb_row, sb_k,
                                        ptr(counts), E, cap, ptr(C), _ld(C), C.stride(0) if C is not None else 0, ptr(D), _ld(D),
                                        D.stride(0), M, N, dtype_enum(D.dtype), stream_ptr(A.device))
    check(rc, "fx_fp8_grouped_wgrad")
    return D
