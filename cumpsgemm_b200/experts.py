"""Products of a mixture-of-experts layer on row-major torch CUDA tensors.

The rows of ``x`` (tokens) are sorted by the expert they go to; ``group_ends``, an int32 tensor on the
same device, holds the running total of rows after each expert, so expert e has the rows
``x[group_ends[e - 1]:group_ends[e]]``.  It stays on the device: nothing here waits for it.  Rows behind
the last total belong to no expert; their results are zero.

    ends = torch.bincount(expert_of_row, minlength=E).cumsum(0).to(torch.int32)
    y = grouped_linear(handle, x, w, ends)              # training: has a backward pass
    q, s = quantize_rows(handle, x, row_index=tokens)   # serving: gather and quantise in one pass
    y = i8_matmul(handle, q, s, wq, w_scale, ends)

Everything goes through the C ABI (``cuMpSGEMM_grouped_gemm`` and its neighbours in
``cumpsgemm_ext.h``) on the handle's stream; there is no other implementation behind it.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import api

_DATA_TYPES = {torch.float16: api.CUDA_R_16F, torch.bfloat16: api.CUDA_R_16BF,
               torch.float32: api.CUDA_R_32F}


def _data_type(dtype) -> int:
    try:
        return _DATA_TYPES[dtype]
    except KeyError:
        raise ValueError(f"expected float16, bfloat16 or float32, got {dtype}") from None


def _rows_of(t, what: str, cols: Optional[int] = None):
    """(rows, columns, leading dimension) of a matrix whose rows are contiguous."""
    if t.dim() != 2:
        raise ValueError(f"{what} must have two dimensions, got {tuple(t.shape)}")
    rows, n = t.shape
    if cols is not None and n != cols:
        raise ValueError(f"{what} has {n} columns where {cols} are needed")
    if n > 1 and t.stride(1) != 1:
        raise ValueError(f"the rows of {what} must be contiguous")
    if rows > 1 and t.stride(0) < n:
        raise ValueError(f"the rows of {what} overlap")
    return rows, n, t.stride(0) if rows > 1 else n


def _matrices_of(t, what: str):
    """(matrices, rows, columns, leading dimension, stride) of a stack of such matrices."""
    if t.dim() != 3:
        raise ValueError(f"{what} must have three dimensions, got {tuple(t.shape)}")
    e, rows, n = t.shape
    if n > 1 and t.stride(2) != 1:
        raise ValueError(f"the rows of {what} must be contiguous")
    ld = t.stride(1) if rows > 1 else n
    if ld < n or (e > 1 and t.stride(0) < (rows - 1) * ld + n):
        raise ValueError(f"the matrices of {what} overlap")
    return e, rows, n, ld, t.stride(0) if e > 1 else rows * ld


def _check(tensors, group_ends, groups: int) -> None:
    device = tensors[0].device
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("operands must live in device memory")
        if t.device != device:
            raise ValueError("operands are on different devices")
    if group_ends is None:
        if groups != 1:
            raise ValueError("group_ends is needed for more than one expert")
        return
    if group_ends.dtype != torch.int32 or group_ends.dim() != 1 or not group_ends.is_contiguous():
        raise ValueError("group_ends must be a contiguous int32 vector")
    if group_ends.device != device:
        raise ValueError("group_ends is on another device")
    if group_ends.numel() != groups:
        raise ValueError(f"{group_ends.numel()} group_ends for {groups} experts")


def _output(out, beta, shape, dtype, device):
    if out is None:
        if beta != 0.0:
            raise ValueError("beta needs an out to read")
        return torch.empty(shape, dtype=dtype, device=device)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != device:
        raise ValueError(f"out must be {dtype} of shape {tuple(shape)} on {device}")
    return out


def grouped_matmul(handle: api.Handle, x, w, group_ends=None, transpose_w: bool = False, *,
                   mode: int = api.ComputeMode.FP16TCEC, alpha: float = 1.0, beta: float = 0.0,
                   out=None):
    """``out[r] = alpha * x[r] @ w[e] + beta * out[r]`` for the rows r of each expert e.

    x is (rows, k), w (experts, k, n), or (experts, n, k) with ``transpose_w``; all of float16, bfloat16
    or float32, which ``mode`` multiplies (FP16TCEC or FP16TCEC_SCALING).  The gradient of x is
    ``grouped_matmul(handle, dy, w, group_ends, not transpose_w)``.
    """
    groups, w_rows, w_cols, ldw, stridew = _matrices_of(w, "w")
    k, n = (w_cols, w_rows) if transpose_w else (w_rows, w_cols)
    rows, _, ldx = _rows_of(x, "x", k)
    _check((x, w), group_ends, groups)
    if x.dtype != w.dtype:
        raise ValueError(f"x is {x.dtype}, w is {w.dtype}")
    out = _output(out, beta, (rows, n), x.dtype, x.device)
    _, _, ldy = _rows_of(out, "out")
    handle.grouped_gemm(api.CUBLAS_OP_T if transpose_w else api.CUBLAS_OP_N, rows, n, k, groups,
                        group_ends, alpha, x, ldx, w, ldw, stridew, beta, out, ldy,
                        _data_type(x.dtype), mode)
    return out


def grouped_matmul_wgrad(handle: api.Handle, x, dy, group_ends=None, transpose_w: bool = False, *,
                         mode: int = api.ComputeMode.FP16TCEC, alpha: float = 1.0, beta: float = 0.0,
                         out=None):
    """``out[e] = alpha * x_e^T @ dy_e + beta * out[e]`` over the rows of each expert e, (experts, k, n);
    its transpose, (experts, n, k), with ``transpose_w``.  Experts without rows: ``beta * out[e]``."""
    rows, k, ldx = _rows_of(x, "x")
    dy_rows, n, lddy = _rows_of(dy, "dy")
    if dy_rows != rows:
        raise ValueError(f"x has {rows} rows, dy {dy_rows}")
    groups = 1 if group_ends is None else group_ends.numel()
    _check((x, dy), group_ends, groups)
    if x.dtype != dy.dtype:
        raise ValueError(f"x is {x.dtype}, dy is {dy.dtype}")
    shape = (groups, n, k) if transpose_w else (groups, k, n)
    out = _output(out, beta, shape, x.dtype, x.device)
    _, _, _, lddw, stridedw = _matrices_of(out, "out")
    handle.grouped_gemm_wgrad(api.CUBLAS_OP_T if transpose_w else api.CUBLAS_OP_N, rows, n, k, groups,
                              group_ends, alpha, x, ldx, dy, lddy, beta, out, lddw, stridedw,
                              _data_type(x.dtype), mode)
    return out


def quantize_rows(handle: api.Handle, x, row_index=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale): int8 rows and their float32 scales, ``scale[r] * q[r]`` being row r of x, or with
    ``row_index`` (int32) row ``row_index[r]``; an index outside x gives a row of zeros.

    q's rows start at multiples of 16 bytes, so that ``i8_matmul`` reads them in place; a weight of
    (experts, n, k) is quantised as (experts * n, k) rows."""
    src_rows, k, ldx = _rows_of(x, "x")
    if not x.is_cuda:
        raise ValueError("operands must live in device memory")
    rows = src_rows
    if row_index is not None:
        if row_index.dtype != torch.int32 or row_index.dim() != 1 or not row_index.is_contiguous():
            raise ValueError("row_index must be a contiguous int32 vector")
        if row_index.device != x.device:
            raise ValueError("row_index is on another device")
        rows = row_index.numel()
    ldq = (k + 15) // 16 * 16
    q = torch.empty((rows, ldq), dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    handle.quantize_rows_i8(rows, k, x, ldx, _data_type(x.dtype), row_index, src_rows, q, ldq, scale)
    return (q if ldq == k else q[:, :k]), scale


def i8_matmul(handle: api.Handle, xq, x_scale, wq, w_scale, group_ends=None, *, bias=None, out=None,
              out_dtype=torch.bfloat16):
    """``out[r] = x_scale[r] * w_scale[e] * (xq[r] @ wq[e]^T) + bias[e]`` for the rows r of each expert e.

    xq is (rows, k) and wq (experts, n, k), int8; x_scale (rows,), w_scale and bias (experts, n),
    float32.  A (n, k) wq with (n,) scales is one expert of all rows: a plain linear layer."""
    if wq.dim() == 2:
        wq = wq.unsqueeze(0)
    groups, n, k, ldw, stridew = _matrices_of(wq, "wq")
    rows, _, ldx = _rows_of(xq, "xq", k)
    _check((xq, x_scale, wq, w_scale) + (() if bias is None else (bias,)), group_ends, groups)
    if xq.dtype != torch.int8 or wq.dtype != torch.int8:
        raise ValueError(f"xq is {xq.dtype}, wq is {wq.dtype}: both must be int8")
    for t, what, count in ((x_scale, "x_scale", rows), (w_scale, "w_scale", groups * n),
                           (bias, "bias", groups * n)):
        if t is not None and (t.dtype != torch.float32 or t.numel() != count or not t.is_contiguous()):
            raise ValueError(f"{what} must be {count} contiguous float32 values")
    out = _output(out, 0.0, (rows, n), out_dtype if out is None else out.dtype, xq.device)
    _, _, ldy = _rows_of(out, "out")
    handle.i8_grouped_gemm(rows, n, k, groups, group_ends, xq, ldx, x_scale, wq, ldw, stridew, w_scale,
                           bias, out, ldy, _data_type(out.dtype))
    return out


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, group_ends, handle, transpose_w, mode):
        ctx.save_for_backward(x, w, group_ends)
        ctx.how = (handle, transpose_w, mode)
        return grouped_matmul(handle, x, w, group_ends, transpose_w, mode=mode)

    @staticmethod
    def backward(ctx, dy):
        x, w, group_ends = ctx.saved_tensors
        handle, transpose_w, mode = ctx.how
        if dy.stride(-1) != 1 or dy.stride(0) < dy.shape[1]:  # e.g. of a sum: one value for all rows
            dy = dy.contiguous()
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = grouped_matmul(handle, dy, w, group_ends, not transpose_w, mode=mode)
        if ctx.needs_input_grad[1]:
            dw = grouped_matmul_wgrad(handle, x, dy, group_ends, transpose_w, mode=mode)
        return dx, dw, None, None, None, None


def grouped_linear(handle: api.Handle, x, w, group_ends=None, transpose_w: bool = False, *,
                   mode: int = api.ComputeMode.FP16TCEC):
    """``grouped_matmul`` with a backward pass: gradients of x and w.  Forward and backward run on the
    handle's stream, which has to be the one that autograd runs on."""
    return _GroupedLinear.apply(x, w, group_ends, handle, transpose_w, mode)
