"""RMSNorm forward / recompute / backward behind the reference signatures
(flextrain/ops/_kernels/rmsnorm.py:419-832).

Same argument names, shape/contiguity errors, return tuples and in-place
rules: ``output`` may be ``X``; a caller-provided ``dX``/``dW`` is accumulated
into, a missing one is allocated and overwritten.
"""
from __future__ import annotations

from functools import lru_cache

import torch

from .._lib import check, dtype_enum, fp8_enum, lib, on_device, ptr, raw_stream, require_gpu, require_same_device, stream_ptr
from .fp8 import _blocks, _extents, _fp8_rows, _round_up, _scale_store


def _norm_config(X, W, head_dim):
    # flextrain/ops/_kernels/rmsnorm.py:419-454
    if X.dim() != 2:
        raise ValueError(f"Input tensor X must be 2D, got {X.dim()} dims")
    T, D = X.shape
    if head_dim is None:
        n_cols, n_heads = D, 1
    else:
        if D % head_dim != 0:
            raise ValueError(f"Input dimension D ({D}) must be divisible by head_dim ({head_dim})")
        n_cols, n_heads = head_dim, D // head_dim
    if W is not None:
        expected = (n_cols,)
        if tuple(W.shape) != expected:
            raise ValueError(f"Weight tensor has incorrect shape. Expected {expected}, got {tuple(W.shape)}")
    if not X.is_contiguous():
        raise ValueError("Input tensor X must be contiguous")
    if W is not None and not W.is_contiguous():
        raise ValueError("Weight tensor W must be contiguous")
    return T, D, n_cols, n_heads


def _check_like(t, X, name):
    if t.shape != X.shape:
        raise ValueError(f"{name} shape {tuple(t.shape)} must match input shape {tuple(X.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.dtype != X.dtype:
        raise TypeError(f"{name} dtype {t.dtype} must match input dtype {X.dtype}")


def _fwd(X, W, head_dim, output, rstd, eps, saved):
    T, D, n_cols, n_heads = _norm_config(X, W, head_dim)
    require_gpu(X, W, output, rstd, op="flextrain_rmsnorm_fwd")
    if output is None:
        Y = torch.empty_like(X)
    else:
        _check_like(output, X, "Output tensor")
        Y = output
    if rstd is None:
        if saved:
            raise ValueError("rstd is required")
        rstd = torch.empty(T, n_heads, dtype=torch.float32, device=X.device)
    else:
        if tuple(rstd.shape) != (T, n_heads):
            raise ValueError(f"rstd tensor shape {tuple(rstd.shape)} must match (T, N_HEADS) {(T, n_heads)}")
        if not rstd.is_contiguous():
            raise ValueError("rstd tensor must be contiguous")
        if rstd.dtype != torch.float32:
            raise TypeError("rstd tensor must be float32")
    rc = lib().fx_rmsnorm_fwd(
        ptr(X), ptr(W), ptr(Y), ptr(rstd), T * n_heads, n_cols, float(eps),
        dtype_enum(X.dtype), dtype_enum(W.dtype) if W is not None else 0, 1 if saved else 0,
        stream_ptr(X.device))
    check(rc, "fx_rmsnorm_fwd")
    return Y, rstd


def flextrain_rmsnorm_fwd(X, W=None, head_dim=None, output=None, rstd=None, rms_norm_eps=1e-5):
    """``(Y, rstd)``; flextrain/ops/_kernels/rmsnorm.py:456-530."""
    return _fwd(X, W, head_dim, output, rstd, rms_norm_eps, saved=False)


def flextrain_rmsnorm_fwd_recompute(X, W, rstd, head_dim=None, output=None):
    """``Y`` from the saved ``rstd``; flextrain/ops/_kernels/rmsnorm.py:532-583."""
    Y, _ = _fwd(X, W, head_dim, output, rstd, 0.0, saved=True)
    return Y


def flextrain_rmsnorm_bwd(dY, X, W, rstd, head_dim=None, dX=None, dW=None,
                          recompute_output=False, recomputed_output_tensor=None):
    """``(dX, dW, Y_or_None)``; flextrain/ops/_kernels/rmsnorm.py:585-832.

    ``dW`` is None when ``W`` is None; with ``W`` given and ``dW=None`` a fresh
    fp32 gradient is returned (the reference computes it in that case too,
    rmsnorm.py:690-704).  Unlike the reference's atomics the reduction order is
    fixed, so results are reproducible run to run.
    """
    T, D, n_cols, n_heads = _norm_config(X, W, head_dim)
    require_gpu(dY, X, W, rstd, dX, dW, recomputed_output_tensor, op="flextrain_rmsnorm_bwd")
    _check_like(dY, X, "dY")
    if tuple(rstd.shape) != (T, n_heads) or not rstd.is_contiguous() or rstd.dtype != torch.float32:
        raise ValueError(f"rstd must be a contiguous float32 tensor of shape {(T, n_heads)}")
    y_out = None
    if recompute_output:
        if recomputed_output_tensor is None:
            y_out = torch.empty_like(X)
        else:
            _check_like(recomputed_output_tensor, X, "recomputed_output_tensor")
            y_out = recomputed_output_tensor
    if dX is None:
        dX = torch.empty_like(X)
        acc_dx = 0
    else:
        _check_like(dX, X, "dX")
        acc_dx = 1
    dw_buf, acc_dw = None, 0
    if W is not None:
        if dW is None:
            dw_buf = torch.empty((n_cols,), dtype=torch.float32, device=X.device)
        else:
            if tuple(dW.shape) != (n_cols,):
                raise ValueError(f"dW shape {tuple(dW.shape)} mismatch. Expected {(n_cols,)}")
            if not dW.is_contiguous():
                raise ValueError("dW tensor must be contiguous")
            dw_buf, acc_dw = dW, 1
    rows = T * n_heads
    L = lib()
    ws, ws_bytes = None, 0
    if dw_buf is not None:
        ws_bytes = int(L.fx_rmsnorm_bwd_ws_bytes(rows, n_cols))
        if ws_bytes:
            ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=X.device)
    rc = L.fx_rmsnorm_bwd(
        ptr(dY), ptr(X), ptr(W), ptr(rstd), ptr(dX), acc_dx, ptr(dw_buf),
        dtype_enum(dw_buf.dtype) if dw_buf is not None else 0, acc_dw, ptr(y_out), rows, n_cols,
        dtype_enum(X.dtype), dtype_enum(W.dtype) if W is not None else 0, ptr(ws), ws_bytes,
        stream_ptr(X.device))
    check(rc, "fx_rmsnorm_bwd")
    return dX, dw_buf, y_out


def flextrain_add_rmsnorm_fwd(X, residual=None, W=None, output_dtype=None, sum_out=None, rms_norm_eps=1e-5):
    """Residual addition and RMSNorm in one pass: ``(Y, scales, H, rstd)``.  The reference runs the addition, the norm
    and any cast as separate passes; this op has no counterpart there.

    ``H = X + residual`` rounded to ``X``'s dtype (``X`` itself without a residual), ``rstd (T, 1)`` fp32 of ``H``,
    ``Y = H * rstd * W``.  ``output_dtype``: ``torch.float8_e4m3fn`` / ``torch.float8_e5m2`` give ``Y`` in 8 bits with
    ``scales (T, ceil(D / 128))`` as :func:`flextrain_fp8_quantize` defines them (``Y`` is formed exactly and rounded
    once); ``None`` gives ``Y`` in ``X``'s dtype, with the roundings of ``flextrain_rmsnorm_fwd(H, W)``, and no scales.
    ``sum_out`` receives ``H`` and may be ``X`` or ``residual``.

    Against ``flextrain_rmsnorm_fwd(H, W)``: the same ``rstd``, and in bf16 and fp32 the same ``Y``, bit for bit, where
    ``D`` is a multiple of 8 and at most 16384 and all tensors start at 16-byte addresses.  Elsewhere that op adds the
    squares in another order and ``rstd`` may differ in its last bits; in fp16 either op may round a product to fp32
    before it rounds it to fp16."""
    op = "flextrain_add_rmsnorm_fwd"
    shape, dtype = X.shape, X.dtype
    if len(shape) != 2 or not X.is_contiguous() or (W is not None and (W.shape != shape[1:] or not W.is_contiguous())):
        _norm_config(X, W, None)            # raises
    T, D = shape
    if D == 0:
        raise ValueError(f"{op}: X has no columns")
    _extents(op, D)
    if residual is not None:
        _check_like(residual, X, "residual")
    if sum_out is not None:
        _check_like(sum_out, X, "sum_out")
    require_same_device(X, residual, W, sum_out, op=op)
    x_dt = dtype_enum(dtype)
    y_dt = x_dt if output_dtype is None or output_dtype == dtype else fp8_enum(output_dtype)
    H = sum_out
    if H is None:
        H = torch.empty_like(X) if residual is not None else X
    rstd = X.new_empty((T, 1), dtype=torch.float32)
    if y_dt == x_dt:
        Y, scales, ldy = torch.empty_like(X), None, D
    else:
        Y, scales = _fp8_rows(X, None, T, D, output_dtype), _scale_store(X, None, T, _blocks(D))
        ldy = _round_up(D, 16)
    with on_device(X):
        rc = lib().fx_add_rmsnorm_fwd(X.data_ptr(), None if residual is None else residual.data_ptr(),
                                      None if W is None else W.data_ptr(), None if H is X and residual is None else H.data_ptr(),
                                      Y.data_ptr(), ldy, None if scales is None else scales.data_ptr(), T, rstd.data_ptr(), T, D,
                                      rms_norm_eps, x_dt, 0 if W is None else dtype_enum(W.dtype), y_dt, raw_stream(X))
    check(rc, "fx_add_rmsnorm_fwd")
    return Y, scales, H, rstd


@lru_cache(maxsize=4096)
def _bwd_ws_bytes(T, D):
    return int(lib().fx_add_rmsnorm_bwd_ws_bytes(T, D))


def flextrain_add_rmsnorm_bwd(dY, H, W, rstd, dH=None, dX=None, dW=None):
    """``(dX, dW)`` of :func:`flextrain_add_rmsnorm_fwd`: ``dX = dH + (gradient of the norm)`` is the gradient of ``X``
    and of ``residual`` alike.

    ``dH`` is the gradient that reaches ``H`` past the norm (the residual stream's; ``None``: zero) and is left as it is
    unless it is given as ``dX`` too; ``dY``, ``dH`` and ``dX`` may be one tensor.  ``dY`` is the gradient of the
    unquantised output (the 8-bit rounding is passed straight through).  ``dW``: accumulated into when given, else a
    fresh fp32 gradient; ``None`` without ``W``."""
    op = "flextrain_add_rmsnorm_bwd"
    shape, dtype = H.shape, H.dtype
    if len(shape) != 2 or not H.is_contiguous() or (W is not None and (W.shape != shape[1:] or not W.is_contiguous())):
        _norm_config(H, W, None)            # raises
    T, D = shape
    _extents(op, D)
    _check_like(dY, H, "dY")
    if dH is not None:
        _check_like(dH, H, "dH")
    if dX is not None:
        _check_like(dX, H, "dX")
    if rstd.numel() != T or not rstd.is_contiguous() or rstd.dtype != torch.float32:
        raise ValueError(f"rstd must be a contiguous float32 tensor of shape {(T, 1)}")
    if W is None and dW is not None:
        raise ValueError(f"{op}: dW without W")
    if dW is not None and (dW.shape != shape[1:] or not dW.is_contiguous()):
        raise ValueError(f"dW must be contiguous of shape {(D,)}")
    require_same_device(dY, H, W, rstd, dH, dX, dW, op=op)
    x_dt = dtype_enum(dtype)
    if dX is None:
        dX = torch.empty_like(H)
    accumulate = dW is not None
    if W is not None and dW is None:
        dW = H.new_empty((D,), dtype=torch.float32)
        if T == 0:
            dW.zero_()
    if T == 0:
        return dX, dW
    with on_device(H):
        nbytes = _bwd_ws_bytes(T, D) if dW is not None else 0
        ws = H.new_empty((nbytes // 4,), dtype=torch.float32) if nbytes else None
        rc = lib().fx_add_rmsnorm_bwd(dY.data_ptr(), None if dH is None else dH.data_ptr(), H.data_ptr(),
                                      None if W is None else W.data_ptr(), rstd.data_ptr(), dX.data_ptr(),
                                      None if dW is None else dW.data_ptr(), 0 if dW is None else dtype_enum(dW.dtype),
                                      1 if accumulate else 0, T, D, x_dt, 0 if W is None else dtype_enum(W.dtype),
                                      None if ws is None else ws.data_ptr(), nbytes, raw_stream(H))
    check(rc, "fx_add_rmsnorm_bwd")
    return dX, dW
