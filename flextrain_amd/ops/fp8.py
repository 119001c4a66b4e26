"""8-bit matrix products with a power-of-two scale per block of 128 values: the quantiser that makes the operands,
the products that read them, and the products grouped by expert.  The reference's ops are 16-bit and wider; these
have no counterpart there.

Values are ``torch.float8_e4m3fn`` or ``torch.float8_e5m2``, scales ``torch.float8_e8m0fnu`` (``2**e``).  A scale
tensor has one entry per block, indexed like the values it belongs to: ``(rows, ceil(cols / 128))`` for blocks of one
row, ``(ceil(rows / 128), ceil(cols / 128))`` for 128 x 128 tiles.  The quantiser stores scales with the block index
outermost and pads rows of values to multiples of 16 bytes; the products take scales of any strides and values whose
rows start at 16-byte addresses.

An operand may be a part of a wider matrix: the products load rows in whole 16-byte pieces, and bytes of a row's last
piece that lie behind its end do not count, whatever they are (NaN too).  Such a piece starts inside the row at a
16-byte address, so the up to 15 bytes read behind a tensor's last row, or behind a single one, lie in its own memory
page; they need not be the tensor's.

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

from functools import lru_cache

import torch

from .._lib import check, dtype_enum, fp8_enum, lib, on_device, raw_stream, require_same_device

_E8M0 = torch.float8_e8m0fnu


def _round_up(n: int, m: int) -> int:
    return (n + m - 1) // m * m


def _blocks(n: int) -> int:
    return (n + 127) // 128


def _fp8_rows(like, batch, rows, cols, dtype):
    """Uninitialised 8-bit values ``(rows, cols)``, or ``(batch, rows, cols)`` when ``batch`` is not None, on the device of
    ``like``, whose rows start at multiples of 16 bytes.  (``new_empty`` takes 0.4 us less than ``torch.empty`` with a
    device.)"""
    ld = _round_up(cols, 16)
    if batch is None:
        if ld == cols:
            return like.new_empty((rows, cols), dtype=dtype)
        return like.new_empty((rows, ld), dtype=dtype)[:, :cols]
    return like.new_empty((batch, rows, ld), dtype=dtype)[..., :cols]


def _scale_store(like, batch, rows, blocks):
    """Uninitialised scales ``(rows, blocks)`` / ``(batch, rows, blocks)``, the block index outermost in memory."""
    if batch is None:
        return like.new_empty_strided((rows, blocks), (1, rows), dtype=_E8M0)
    return like.new_empty((batch, blocks, rows), dtype=_E8M0).transpose(1, 2)


def _extents(op, *sizes):
    """Sizes that the C ABI takes as 32-bit integers."""
    if max(sizes) > 0x7FFFFFFF:
        raise ValueError(f"{op}: a dimension is larger than 2**31 - 1")


def _input_matrix(X, op):
    """(batch or None, rows, cols, row stride, batch stride) of a matrix to quantise."""
    shape, stride = X.shape, X.stride()
    if len(shape) not in (2, 3):
        raise ValueError(f"{op}: X must be (rows, cols) or (batch, rows, cols), got {len(shape)} dims")
    rows, cols = shape[-2:]
    if cols == 0:
        raise ValueError(f"{op}: X has no columns")
    if cols > 1 and stride[-1] != 1:
        raise ValueError(f"{op}: X must have unit column stride")
    # a dimension of one has no stride of its own
    ldx = stride[-2] if rows > 1 else cols
    if ldx < cols:
        raise ValueError(f"{op}: the rows of X overlap")
    if len(shape) == 2:
        return None, rows, cols, ldx, 0
    if shape[0] > 65535:
        raise ValueError(f"{op}: a batch holds at most 65535 matrices")
    return shape[0], rows, cols, ldx, stride[0]


def _quantize(X, dtype, tiles, both, op):
    batch, rows, cols, ldx, x_batch = _input_matrix(X, op)
    require_same_device(X, op=op)
    x_dt, q_dt = dtype_enum(X.dtype), fp8_enum(dtype)
    rb, cb = _blocks(rows), _blocks(cols)
    s_rows = rb if tiles else rows
    q, s = _fp8_rows(X, batch, rows, cols, dtype), _scale_store(X, batch, s_rows, cb)
    qt = st = None
    t_rows = 0
    if both:
        t_rows = cb if tiles else cols
        qt, st = _fp8_rows(X, batch, cols, rows, dtype), _scale_store(X, batch, t_rows, rb)
    if rows == 0 or batch == 0:
        return q, s, qt, st
    ldq, ldt = _round_up(cols, 16), _round_up(rows, 16)
    with on_device(X):
        rc = lib().fx_fp8_quantize(
            X.data_ptr(), ldx, x_batch, 1 if batch is None else batch, rows, cols, x_dt, q_dt, 1 if tiles else 0,
            q.data_ptr(), ldq, rows * ldq, s.data_ptr(), s_rows, s_rows * cb,
            qt.data_ptr() if both else None, ldt, cols * ldt, st.data_ptr() if both else None, t_rows, t_rows * rb,
            raw_stream(X))
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
    split of the rows, ``(rows + 127 E) // 128 * 128``, which has to be below 2**23); places without a row hold 0 with
    scale 1.  ``counts (E,)`` int32 on the GPU.  With ``row_sources`` (int32, one entry per expert-sorted row) ``X`` is
    the unsorted matrix and sorted row ``r`` is its row ``row_sources[r]``."""
    op = "flextrain_fp8_quantize_grouped_cols"
    if X.dim() != 2:
        raise ValueError(f"{op}: X must be (rows, cols)")
    _, x_rows, cols, ldx, _ = _input_matrix(X, op)
    E = _counts_of(counts, op)
    rows = x_rows if row_sources is None else _sources_of(row_sources, op)
    cap = (rows + 127 * E) // 128 * 128          # fx_fp8_grouped_capacity
    if cap >= 1 << 23:
        raise ValueError(f"{op}: the capacity {cap} of {rows} rows and {E} experts is not below 2**23")
    require_same_device(X, counts, row_sources, op=op)
    if rows > 0 and x_rows == 0:
        raise ValueError(f"{op}: X has no rows")
    x_dt, q_dt = dtype_enum(X.dtype), fp8_enum(dtype)
    qt = X.new_empty((cols, cap), dtype=dtype)
    st = _scale_store(X, None, cols, cap // 128)
    if cap > 0:
        with on_device(X):
            rc = lib().fx_fp8_quantize_grouped_cols(X.data_ptr(), ldx, x_rows, rows, cols, x_dt, q_dt, counts.data_ptr(), E,
                                                    None if row_sources is None else row_sources.data_ptr(),
                                                    qt.data_ptr(), cap, st.data_ptr(), cols, raw_stream(X))
        check(rc, "fx_fp8_quantize_grouped_cols")
    return qt, st


def _values(t, rows, cols, stride, name, op):
    """Row stride of an 8-bit operand ``(.., rows, cols)``."""
    if cols > 1 and stride[-1] != 1:
        raise ValueError(f"{op}: {name} must have unit stride along the contraction")
    ld = stride[-2] if rows > 1 else _round_up(cols, 16)
    if rows and cols and (ld % 16 or ld < cols or t.data_ptr() % 16):
        raise ValueError(f"{op}: the rows of {name} must start at 16-byte addresses (they are {ld} bytes apart)")
    return ld


def _scales(s, rows, blocks, tiles_allowed, name, op):
    """(row stride, block stride, 1 for 128-row tiles) of an operand's scales ``(.., rows | row blocks, blocks)``."""
    if s.dtype != _E8M0:
        raise TypeError(f"{op}: {name} must be {_E8M0}, got {s.dtype}")
    got, stride = s.shape, s.stride()
    if got[-1] == blocks:
        if got[-2] == rows:
            return stride[-2], stride[-1], 0
        if tiles_allowed and got[-2] == _blocks(rows):
            return stride[-2], stride[-1], 1
    raise ValueError(f"{op}: {name} has shape {tuple(got)}, expected {(rows, blocks)}"
                     + (f" or {(_blocks(rows), blocks)}" if tiles_allowed else ""))


def _operand_dtypes(A, B, op):
    a_dt = fp8_enum(A.dtype)
    if B.dtype != torch.float8_e4m3fn:
        raise TypeError(f"{op}: B must be torch.float8_e4m3fn (a gradient in e5m2 is the first operand), got {B.dtype}")
    return a_dt


def _addend(t, shape, dtype, name, op):
    """Row stride (and batch stride) of C or out: the output's shape and dtype, unit column stride."""
    got, stride = t.shape, t.stride()
    if got != shape:
        raise ValueError(f"{op}: {name} has shape {tuple(got)}, expected {tuple(shape)}")
    if got[-1] > 1 and stride[-1] != 1:
        raise ValueError(f"{op}: {name} must have unit column stride")
    if got[-2] > 1 and stride[-2] < got[-1]:
        raise ValueError(f"{op}: the rows of {name} overlap")
    if t.dtype != dtype:
        raise TypeError(f"{op}: {name} is {t.dtype}, the output {dtype}")
    return stride[-2] if got[-2] > 1 else got[-1], stride[0]


def _output(like, out, shape, out_dtype, C, op):
    """(output, its dtype's enum, its row and batch strides, those of C): C and out have the output's shape and dtype."""
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else C.dtype if C is not None else torch.bfloat16
    d_dt = dtype_enum(out_dtype)
    shape = torch.Size(shape)
    ldc = c_batch = 0
    if C is not None:
        ldc, c_batch = _addend(C, shape, out_dtype, "C", op)
    if out is not None:
        ldd, d_batch = _addend(out, shape, out_dtype, "out", op)
        if len(shape) == 3 and shape[0] > 1 and not (
                d_batch >= (shape[1] - 1) * ldd + shape[2]                                       # one behind the other
                or (d_batch >= shape[2] and ldd >= (shape[0] - 1) * d_batch + shape[2])):        # side by side
            raise ValueError(f"{op}: the experts' matrices in out overlap")
        return out, d_dt, ldd, d_batch, ldc, c_batch
    D = like.new_empty(shape, dtype=out_dtype)
    return D, d_dt, shape[-1], shape[-1] * shape[-2], ldc, c_batch


@lru_cache(maxsize=4096)
def _gemm_ws_bytes(M, N, K):
    return int(lib().fx_fp8_gemm_ws_bytes(M, N, K))


def flextrain_fp8_matmul(A, A_scales, B, B_scales, C=None, out=None, out_dtype=None):
    """``out = A @ B.T (+ C)`` of 8-bit operands ``A (M, K)``, ``B (N, K)`` with block scales.

    ``A`` is e4m3 or e5m2, ``B`` e4m3; each has scales per row and 128 k or per 128 x 128 tile (told apart by their
    shape).  ``C`` has the output's shape and dtype and may be ``out`` (a gradient accumulated in place).  Output
    dtype: ``out_dtype``, else that of ``out`` or ``C``, else bf16.  Rows of ``A`` and ``B`` are less than 2**23 bytes
    apart, and a scale tensor spans less than 2 GB.

    The matrix unit sums the products.  Before it adds the products of 8 consecutive k it cuts them to multiples of
    ``2**(E - 13)``, ``E`` being the largest sum of two exponents among the 8: a product below that is lost, where an
    fp32 sum would hold it to ``2**(E - 23)``.  Those sums of 8, and ``C``, are added in fp32.  The same holds for the
    products by expert below."""
    op = "flextrain_fp8_matmul"
    a_shape, b_shape = A.shape, B.shape
    if len(a_shape) != 2 or len(b_shape) != 2 or a_shape[1] != b_shape[1]:
        raise ValueError(f"{op}: A {tuple(a_shape)} and B {tuple(b_shape)} must be (M, K) and (N, K)")
    a_dt = _operand_dtypes(A, B, op)
    (M, K), N = a_shape, b_shape[0]
    _extents(op, M, N, K)
    kb = _blocks(K)
    lda, ldb = _values(A, M, K, A.stride(), "A", op), _values(B, N, K, B.stride(), "B", op)
    sa_row, sa_k, a_tiles = _scales(A_scales, M, kb, True, "A_scales", op)
    sb_row, sb_k, b_tiles = _scales(B_scales, N, kb, True, "B_scales", op)
    require_same_device(A, A_scales, B, B_scales, C, out, op=op)
    D, d_dt, ldd, _, ldc, _ = _output(A, out, (M, N), out_dtype, C, op)
    if M == 0 or N == 0:
        return D
    with on_device(A):
        nbytes = _gemm_ws_bytes(M, N, K)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=A.device) if nbytes else None
        rc = lib().fx_fp8_gemm(A.data_ptr(), lda, a_dt, A_scales.data_ptr(), sa_row, sa_k, a_tiles, B.data_ptr(), ldb,
                               B_scales.data_ptr(), sb_row, sb_k, b_tiles, None if C is None else C.data_ptr(), ldc,
                               D.data_ptr(), ldd, M, N, K, d_dt, None if ws is None else ws.data_ptr(), nbytes, raw_stream(A))
    check(rc, "fx_fp8_gemm")
    return D


def flextrain_fp8_grouped_matmul(A, A_scales, B, B_scales, counts, row_sources=None, out=None, out_dtype=None):
    """``out[rows of e] = A[rows of e] @ B[e].T`` for every expert, in one launch that reads the counts on the GPU.

    ``A (rows, K)`` expert-sorted, e4m3 or e5m2, scales per row; ``B (E, N, K)`` e4m3, scales ``(E, ceil(N / 128),
    ceil(K / 128))`` (tiles) or ``(E, N, ceil(K / 128))``; ``counts (E,)`` int32 with the sum ``rows``.  With
    ``row_sources`` (int32, one entry per expert-sorted row) ``A`` is the unsorted matrix and its rows are gathered by
    the tile loads (it is then smaller than 4 GB).  At most 2**24 expert-sorted rows.  Rows of ``out`` behind the last
    expert's are left as they were."""
    op = "flextrain_fp8_grouped_matmul"
    a_shape, b_shape = A.shape, B.shape
    if len(a_shape) != 2 or len(b_shape) != 3 or a_shape[1] != b_shape[2]:
        raise ValueError(f"{op}: A {tuple(a_shape)} and B {tuple(b_shape)} must be (rows, K) and (E, N, K)")
    a_dt = _operand_dtypes(A, B, op)
    E, N, K = b_shape
    a_rows, kb = a_shape[0], _blocks(K)
    _extents(op, N, K)
    if _counts_of(counts, op) != E:
        raise ValueError(f"{op}: {counts.numel()} counts for {E} experts")
    rows = a_rows if row_sources is None else _sources_of(row_sources, op)
    if rows > 1 << 24:
        raise ValueError(f"{op}: at most 2**24 expert rows")
    if rows > 0 and a_rows == 0:
        raise ValueError(f"{op}: A has no rows")
    b_stride = B.stride()
    lda, ldb = _values(A, a_rows, K, A.stride(), "A", op), _values(B, N, K, b_stride, "B", op)
    b_expert = b_stride[0] if E > 1 else 0          # (a dimension of one has no stride of its own)
    if N and K and b_expert % 16:
        raise ValueError(f"{op}: every expert's matrix must start at a 16-byte address")
    sa_row, sa_k, _ = _scales(A_scales, a_rows, kb, False, "A_scales", op)
    if B_scales.dim() != 3 or B_scales.shape[0] != E:
        raise ValueError(f"{op}: B_scales has shape {tuple(B_scales.shape)}, expected {E} experts")
    sb_row, sb_k, b_tiles = _scales(B_scales, N, kb, True, "B_scales", op)
    require_same_device(A, A_scales, B, B_scales, counts, row_sources, out, op=op)
    D, d_dt, ldd, _, _, _ = _output(A, out, (rows, N), out_dtype, None, op)
    if rows == 0 or N == 0:
        return D
    with on_device(A):
        rc = lib().fx_fp8_grouped_gemm(A.data_ptr(), lda, a_dt, A_scales.data_ptr(), sa_row, sa_k,
                                       None if row_sources is None else row_sources.data_ptr(), a_rows, B.data_ptr(), ldb,
                                       b_expert, B_scales.data_ptr(), sb_row, sb_k, B_scales.stride(0), b_tiles,
                                       counts.data_ptr(), E, rows, D.data_ptr(), ldd, N, K, d_dt, raw_stream(A))
    check(rc, "fx_fp8_grouped_gemm")
    return D


def flextrain_fp8_grouped_wgrad(A, A_scales, B, B_scales, counts, C=None, out=None, out_dtype=None):
    """``out[e] = A_e @ B_e.T (+ C[e])`` for every expert: the weight gradient ``dy_e.T @ x_e`` of operands made by
    :func:`flextrain_fp8_quantize_grouped_cols` with the same ``counts``.

    ``A (M, capacity)`` e4m3 or e5m2, ``B (N, capacity)`` e4m3, scales ``(M | N, capacity / 128)``; ``out`` / ``C``
    ``(E, M, N)`` of one dtype (``C`` may be ``out``).  An expert without rows gives ``C[e]``, or zeros."""
    op = "flextrain_fp8_grouped_wgrad"
    a_shape, b_shape = A.shape, B.shape
    if len(a_shape) != 2 or len(b_shape) != 2 or a_shape[1] != b_shape[1]:
        raise ValueError(f"{op}: A {tuple(a_shape)} and B {tuple(b_shape)} must be (M, capacity) and (N, capacity)")
    a_dt = _operand_dtypes(A, B, op)
    E = _counts_of(counts, op)
    (M, cap), N = a_shape, b_shape[0]
    _extents(op, M, N)
    if cap % 128:
        raise ValueError(f"{op}: the capacity {cap} is not a multiple of 128")
    if cap >= 1 << 23:
        raise ValueError(f"{op}: at most 2**23 expert rows")
    lda, ldb = _values(A, M, cap, A.stride(), "A", op), _values(B, N, cap, B.stride(), "B", op)
    sa_row, sa_k, _ = _scales(A_scales, M, cap // 128, False, "A_scales", op)
    sb_row, sb_k, _ = _scales(B_scales, N, cap // 128, False, "B_scales", op)
    require_same_device(A, A_scales, B, B_scales, counts, C, out, op=op)
    D, d_dt, ldd, d_batch, ldc, c_batch = _output(A, out, (E, M, N), out_dtype, C, op)
    if M == 0 or N == 0:
        return D
    with on_device(A):
        rc = lib().fx_fp8_grouped_wgrad(A.data_ptr(), lda, a_dt, A_scales.data_ptr(), sa_row, sa_k, B.data_ptr(), ldb,
                                        B_scales.data_ptr(), sb_row, sb_k, counts.data_ptr(), E, cap,
                                        None if C is None else C.data_ptr(), ldc, c_batch, D.data_ptr(), ldd, d_batch, M, N,
                                        d_dt, raw_stream(A))
    check(rc, "fx_fp8_grouped_wgrad")
    return D
