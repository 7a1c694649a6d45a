"""Products of a mixture-of-experts layer on row-major torch CUDA tensors.

The rows of ``x`` (tokens) are sorted by the expert they go to; ``group_ends``, an int32 tensor on the
same device, holds the running total of rows after each expert, so expert e has the rows
``x[group_ends[e - 1]:group_ends[e]]``.  It stays on the device: nothing here waits for it.  Rows behind
the last total belong to no expert; their results are zero.

    ends = torch.bincount(expert_of_row, minlength=E).cumsum(0).to(torch.int32)
    y = grouped_linear(handle, x, w, ends)              # training: gradients of x and w
    q, s = quantize_rows(handle, x, row_index=tokens)   # serving: gather and quantise in one pass
    y = i8_matmul(handle, q, s, wq, w_scale, ends)

Everything goes through the C ABI (``cuMpSGEMM_grouped_gemm`` and its neighbours in
``cumpsgemm_ext.h``); there is no other implementation behind it.  Results are allocated on the current
stream and written on the handle's, so the two have to be one: ``handle.use_current_torch_stream()``
wherever the current stream changes, or the call is refused.  The 8-bit calls have no gradients.
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


# A call with few rows takes as long as its checks: they ask a tensor for each thing once.
def _rows_of(t, what: str, cols: Optional[int] = None):
    """(rows, columns, leading dimension) of a matrix whose rows are contiguous."""
    shape = t.shape
    if len(shape) != 2:
        raise ValueError(f"{what} must have two dimensions, got {tuple(shape)}")
    rows, n = shape
    ld, step = t.stride()
    if cols is not None and n != cols:
        raise ValueError(f"{what} has {n} columns where {cols} are needed")
    if step != 1 and n > 1 and rows > 0:
        raise ValueError(f"the rows of {what} must be contiguous")
    if rows <= 1:
        return rows, n, n
    if ld < n:
        raise ValueError(f"the rows of {what} overlap")
    return rows, n, ld


def _matrices_of(t, what: str):
    """(matrices, rows, columns, leading dimension, stride) of a stack of such matrices."""
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{what} must have three dimensions, got {tuple(shape)}")
    e, rows, n = shape
    stride, ld, step = t.stride()
    if step != 1 and n > 1:
        raise ValueError(f"the rows of {what} must be contiguous")
    if rows <= 1:
        ld = n
    if e <= 1:
        stride = rows * ld
    if ld < n or stride < (rows - 1) * ld + n:
        raise ValueError(f"the matrices of {what} overlap")
    return e, rows, n, ld, stride


def _stream_of(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _stream_of)  # the first is 1 us shorter


def _check_place(handle, device: int) -> None:
    if device < 0:
        raise ValueError("operands must live in device memory")
    if device != handle.device:
        raise ValueError(f"operands are on device {device}, the handle is on {handle.device}")
    if _current_stream(device) != handle.stream:
        raise ValueError("the handle's stream is not the current one; call handle.use_current_torch_stream()")


def _check(handle, device: int, others, group_ends, groups: int) -> None:
    _check_place(handle, device)
    for t in others:
        if t.get_device() != device:
            raise ValueError("operands are on different devices")
    if group_ends is None:
        if groups != 1:
            raise ValueError("group_ends is needed for more than one expert")
        return
    if group_ends.dtype is not torch.int32 or group_ends.dim() != 1 or not group_ends.is_contiguous():
        raise ValueError("group_ends must be a contiguous int32 vector")
    if group_ends.get_device() != device:
        raise ValueError("group_ends is on another device")
    if group_ends.shape[0] != groups:
        raise ValueError(f"{group_ends.shape[0]} group_ends for {groups} experts")


def _check_scales(t, what: str, count: int) -> None:
    if t.dtype is not torch.float32 or t.numel() != count or not t.is_contiguous():
        raise ValueError(f"{what} must be {count} contiguous float32 values")


def _output(out, beta, shape, dtype, like):
    if out is None:
        if beta != 0.0:
            raise ValueError("beta needs an out to read")
        return like.new_empty(shape, dtype=dtype)
    if tuple(out.shape) != shape or out.dtype is not dtype or out.get_device() != like.get_device():
        raise ValueError(f"out must be {dtype} of shape {shape} on {like.device}")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out requires a gradient, which what is written to it has not: use torch.no_grad()")
    torch.autograd.graph.increment_version(out)  # a backward pass that needs what stood there says so
    return out


_BACKWARD_MODE = api.ComputeMode.FP16TCEC_SCALING  # FP32 gradients may have any magnitude


def _no_graph_through(out, beta) -> None:
    if out is not None:
        raise ValueError("an operand requires a gradient, and what is written to out has none: use torch.no_grad()")
    if beta != 0.0:
        raise ValueError("beta needs an out to read")


def grouped_matmul(handle: api.Handle, x, w, group_ends=None, transpose_w: bool = False, *,
                   mode: int = api.ComputeMode.FP16TCEC, alpha: float = 1.0, beta: float = 0.0,
                   out=None):
    """``out[r] = alpha * x[r] @ w[e] + beta * out[r]`` for the rows r of each expert e.

    x is (rows, k), w (experts, k, n), or (experts, n, k) with ``transpose_w``; all of float16, bfloat16
    or float32, which ``mode`` multiplies (FP16TCEC or FP16TCEC_SCALING).  The gradient of x is
    ``grouped_matmul(handle, dy, w, group_ends, not transpose_w)``; autograd's where x or w requires one,
    as with ``grouped_linear`` (without ``out``).
    """
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        _no_graph_through(out, beta)
        return _GroupedLinear.apply(x, w, group_ends, handle, transpose_w, mode, _BACKWARD_MODE, alpha)
    groups, w_rows, w_cols, ldw, stridew = _matrices_of(w, "w")
    k, n = (w_cols, w_rows) if transpose_w else (w_rows, w_cols)
    rows, _, ldx = _rows_of(x, "x", k)
    _check(handle, x.get_device(), (w,), group_ends, groups)
    dtype = x.dtype
    if dtype is not w.dtype:
        raise ValueError(f"x is {dtype}, w is {w.dtype}")
    data_type = _data_type(dtype)
    ldy = n
    if out is not None:
        _, _, ldy = _rows_of(out, "out")
    out = _output(out, beta, (rows, n), dtype, x)
    handle.grouped_gemm(api.CUBLAS_OP_T if transpose_w else api.CUBLAS_OP_N, rows, n, k, groups,
                        None if group_ends is None else group_ends.data_ptr(), alpha, x.data_ptr(), ldx,
                        w.data_ptr(), ldw, stridew, beta, out.data_ptr(), ldy, data_type, mode)
    return out


def grouped_matmul_wgrad(handle: api.Handle, x, dy, group_ends=None, transpose_w: bool = False, *,
                         mode: int = api.ComputeMode.FP16TCEC, alpha: float = 1.0, beta: float = 0.0,
                         out=None):
    """``out[e] = alpha * x_e^T @ dy_e + beta * out[e]`` over the rows of each expert e, (experts, k, n);
    its transpose, (experts, n, k), with ``transpose_w``.  Experts without rows: ``beta * out[e]``.  Has
    gradients as ``grouped_matmul`` does."""
    if torch.is_grad_enabled() and (x.requires_grad or dy.requires_grad):
        _no_graph_through(out, beta)
        return _WeightGradient.apply(x, dy, group_ends, handle, transpose_w, mode, _BACKWARD_MODE, alpha)
    rows, k, ldx = _rows_of(x, "x")
    dy_rows, n, lddy = _rows_of(dy, "dy")
    if dy_rows != rows:
        raise ValueError(f"x has {rows} rows, dy {dy_rows}")
    groups = 1 if group_ends is None else group_ends.numel()
    _check(handle, x.get_device(), (dy,), group_ends, groups)
    dtype = x.dtype
    if dtype is not dy.dtype:
        raise ValueError(f"x is {dtype}, dy is {dy.dtype}")
    data_type = _data_type(dtype)
    shape = (groups, n, k) if transpose_w else (groups, k, n)
    lddw, stridedw = shape[2], n * k
    if out is not None:
        _, _, _, lddw, stridedw = _matrices_of(out, "out")
    out = _output(out, beta, shape, dtype, x)
    handle.grouped_gemm_wgrad(api.CUBLAS_OP_T if transpose_w else api.CUBLAS_OP_N, rows, n, k, groups,
                              None if group_ends is None else group_ends.data_ptr(), alpha, x.data_ptr(),
                              ldx, dy.data_ptr(), lddy, beta, out.data_ptr(), lddw, stridedw, data_type,
                              mode)
    return out


def quantize_rows(handle: api.Handle, x, row_index=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale): int8 rows and their float32 scales, ``scale[r] * q[r]`` being row r of x, or with
    ``row_index`` (int32) row ``row_index[r]``; an index outside x gives a row of zeros.

    q's rows start at multiples of 16 bytes, so that ``i8_matmul`` reads them in place; a weight of
    (experts, n, k) is quantised as (experts * n, k) rows."""
    src_rows, k, ldx = _rows_of(x, "x")
    device = x.get_device()
    _check_place(handle, device)
    data_type = _data_type(x.dtype)
    rows = src_rows
    if row_index is not None:
        if row_index.dtype is not torch.int32 or row_index.dim() != 1 or not row_index.is_contiguous():
            raise ValueError("row_index must be a contiguous int32 vector")
        if row_index.get_device() != device:
            raise ValueError("row_index is on another device")
        rows = row_index.shape[0]
    ldq = (k + 15) // 16 * 16
    q = x.new_empty((rows, ldq), dtype=torch.int8)
    scale = x.new_empty(rows, dtype=torch.float32)
    handle.quantize_rows_i8(rows, k, x.data_ptr(), ldx, data_type,
                            None if row_index is None else row_index.data_ptr(), src_rows, q.data_ptr(),
                            ldq, scale.data_ptr())
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
    others = (x_scale, wq, w_scale) if bias is None else (x_scale, wq, w_scale, bias)
    _check(handle, xq.get_device(), others, group_ends, groups)
    if xq.dtype is not torch.int8 or wq.dtype is not torch.int8:
        raise ValueError(f"xq is {xq.dtype}, wq is {wq.dtype}: both must be int8")
    _check_scales(x_scale, "x_scale", rows)
    _check_scales(w_scale, "w_scale", groups * n)
    if bias is not None:
        _check_scales(bias, "bias", groups * n)
    ldy = n
    if out is not None:
        out_dtype = out.dtype
        _, _, ldy = _rows_of(out, "out")
    data_type = _data_type(out_dtype)
    out = _output(out, 0.0, (rows, n), out_dtype, xq)
    handle.i8_grouped_gemm(rows, n, k, groups, None if group_ends is None else group_ends.data_ptr(),
                           xq.data_ptr(), ldx, x_scale.data_ptr(), wq.data_ptr(), ldw, stridew,
                           w_scale.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(),
                           ldy, data_type)
    return out


def _dense_rows(t):
    """t, copied where its rows, or its matrices, do not lie one behind the other."""
    rows, cols = t.shape[-2:]
    dense = t.stride(-1) == 1 and t.stride(-2) >= cols and (
        t.dim() < 3 or t.stride(-3) >= (rows - 1) * t.stride(-2) + cols)
    return t if dense else t.contiguous()


# The gradients of either product are products of the same two kinds, so each backward pass is made of these
# functions again and can itself be differentiated, any number of times.
class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, group_ends, handle, transpose_w, mode, backward_mode, alpha):
        ctx.save_for_backward(x, w, group_ends)
        ctx.how = (handle, transpose_w, backward_mode, alpha)
        return grouped_matmul(handle, x, w, group_ends, transpose_w, mode=mode, alpha=alpha)

    @staticmethod
    def backward(ctx, dy):
        x, w, group_ends = ctx.saved_tensors
        handle, transpose_w, mode, alpha = ctx.how
        dy = _dense_rows(dy)  # the gradient of a sum, say, is one value for all of them
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = _linear(dy, w, group_ends, handle, not transpose_w, mode, alpha)
        if ctx.needs_input_grad[1]:
            dw = _weight_gradient(x, dy, group_ends, handle, transpose_w, mode, alpha)
        return dx, dw, None, None, None, None, None, None


class _WeightGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dy, group_ends, handle, transpose_w, mode, backward_mode, alpha):
        ctx.save_for_backward(x, dy, group_ends)
        ctx.how = (handle, transpose_w, backward_mode, alpha)
        return grouped_matmul_wgrad(handle, x, dy, group_ends, transpose_w, mode=mode, alpha=alpha)

    @staticmethod
    def backward(ctx, v):
        # dw_e = x_e^T dy_e: the gradient of x is dy v_e^T, that of dy is x v_e
        x, dy, group_ends = ctx.saved_tensors
        handle, transpose_w, mode, alpha = ctx.how
        v = _dense_rows(v)
        gx = gdy = None
        if ctx.needs_input_grad[0]:
            gx = _linear(dy, v, group_ends, handle, not transpose_w, mode, alpha)
        if ctx.needs_input_grad[1]:
            gdy = _linear(x, v, group_ends, handle, transpose_w, mode, alpha)
        return gx, gdy, None, None, None, None, None, None


# What backward passes are made of: without a graph to leave, which is the usual case, the products
# themselves (10 us each shorter).
def _linear(x, w, group_ends, handle, transpose_w, mode, alpha):
    if torch.is_grad_enabled():
        return _GroupedLinear.apply(x, w, group_ends, handle, transpose_w, mode, mode, alpha)
    return grouped_matmul(handle, x, w, group_ends, transpose_w, mode=mode, alpha=alpha)


def _weight_gradient(x, dy, group_ends, handle, transpose_w, mode, alpha):
    if torch.is_grad_enabled():
        return _WeightGradient.apply(x, dy, group_ends, handle, transpose_w, mode, mode, alpha)
    return grouped_matmul_wgrad(handle, x, dy, group_ends, transpose_w, mode=mode, alpha=alpha)


def grouped_linear(handle: api.Handle, x, w, group_ends=None, transpose_w: bool = False, *,
                   mode: int = api.ComputeMode.FP16TCEC,
                   backward_mode: int = _BACKWARD_MODE):
    """``grouped_matmul`` with a backward pass: gradients of x and w, which have gradients in turn
    (``create_graph=True``).  Autograd runs the backward pass on the stream of the forward pass.

    ``mode`` multiplies FP32 operands of the forward pass, ``backward_mode`` those of the backward pass.
    FP16TCEC knows an element to 2^-36 and none above 65504: enough for activations and weights of order one,
    not for gradients, which FP16TCEC_SCALING takes at any magnitude.  16-bit operands look at neither."""
    return _GroupedLinear.apply(_dense_rows(x), _dense_rows(w), group_ends, handle, transpose_w, mode,
                                backward_mode, 1.0)
