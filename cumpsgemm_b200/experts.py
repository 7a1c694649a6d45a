"""Products of a mixture-of-experts layer on row-major torch CUDA tensors.

The rows of ``x`` (tokens) are sorted by the expert they go to; ``group_ends``, an int32 tensor on the
same device, holds the running total of rows after each expert, so expert e has the rows
``x[group_ends[e - 1]:group_ends[e]]``.  It stays on the device: nothing here waits for it.  Rows behind
the last total belong to no expert; their results are zero.

    ends = torch.bincount(expert_of_row, minlength=E).cumsum(0).to(torch.int32)
    y = grouped_linear(handle, x, w, ends)              # training: gradients of x and w
    y = gated_feed_forward(handle, x, gate_up, down, ends)  # a gated block: gradients of all three
    q, s = quantize_rows(handle, x, row_index=tokens)   # serving: gather and quantise in one pass
    y = i8_matmul(handle, q, s, wq, w_scale, ends)
    q, s = quantize_blocks(handle, x, row_index=tokens)  # the same in 8-bit floating point
    y = f8_matmul(handle, q, s, wq, w_scale, ends)

Everything goes through the C ABI (``cuMpSGEMM_grouped_gemm`` and its neighbours in
``cumpsgemm_ext.h``); there is no other implementation behind it.  Results are allocated on the current
stream and written on the handle's, so the two have to be one: ``handle.use_current_torch_stream()``
wherever the current stream changes, or the call is refused.  The 8-bit calls have no gradients.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import api

_F8_TYPES = {torch.float8_e4m3fn: api.CUDA_R_8F_E4M3, torch.float8_e5m2: api.CUDA_R_8F_E5M2}
_ACTIVATIONS = {"silu": api.Activation.SILU, "gelu": api.Activation.GELU, "gelu_tanh": api.Activation.GELU_TANH,
                "relu": api.Activation.RELU}
_BLOCK = 128  # columns, or rows and columns, that share a scale in 8-bit floating point

_DATA_TYPES = {torch.float16: api.CUDA_R_16F, torch.bfloat16: api.CUDA_R_16BF,
               torch.float32: api.CUDA_R_32F}


def _data_type(dtype) -> int:
    try:
        return _DATA_TYPES[dtype]
    except KeyError:
        raise ValueError(f"expected float16, bfloat16 or float32, got {dtype}") from None


def _f8_type(dtype, what: str) -> int:
    try:
        return _F8_TYPES[dtype]
    except KeyError:
        raise ValueError(f"{what} must be float8_e4m3fn or float8_e5m2, got {dtype}") from None


def _activation(name) -> int:
    try:
        return _ACTIVATIONS[name]
    except KeyError:
        raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}, got {name!r}") from None


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
    if t.is_contiguous():
        return t
    shape, strides = t.shape, t.stride()
    rows, cols = shape[-2:]
    step, ld = strides[-1], strides[-2]
    dense = step == 1 and ld >= cols and (len(shape) < 3 or strides[-3] >= (rows - 1) * ld + cols)
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


# ---------------------------------------------------------------- gated feed-forward blocks
def _gated_shapes(handle, x, gate_up, group_ends):
    """What a gated product checks; (rows, hidden, width, groups, leading dimensions ..., data type)."""
    groups, both, width, ldw, stridew = _matrices_of(gate_up, "gate_up")
    if both % 2:
        raise ValueError(f"gate_up has {both} rows: as many of the gate as of what it gates are needed")
    rows, _, ldx = _rows_of(x, "x", width)
    _check(handle, x.get_device(), (gate_up,), group_ends, groups)
    if x.dtype is not gate_up.dtype:
        raise ValueError(f"x is {x.dtype}, gate_up is {gate_up.dtype}")
    return rows, both // 2, width, groups, ldx, ldw, stridew, _data_type(x.dtype)


def _gated(handle, x, gate_up, group_ends, act, mode, out=None, keep=False):
    """(act(gate) * up, both in front of that if they are to be kept)."""
    rows, hidden, width, groups, ldx, ldw, stridew, data_type = _gated_shapes(handle, x, gate_up, group_ends)
    ldy = hidden
    if out is not None:
        _, _, ldy = _rows_of(out, "out")
    out = _output(out, 0.0, (rows, hidden), x.dtype, x)
    pre = x.new_empty((rows, 2 * hidden)) if keep or data_type == api.CUDA_R_32F else None
    handle.grouped_gemm_gated(rows, hidden, width, groups, None if group_ends is None else group_ends.data_ptr(),
                              x.data_ptr(), ldx, gate_up.data_ptr(), ldw, stridew, act, out.data_ptr(), ldy,
                              None if pre is None else pre.data_ptr(), 2 * hidden, data_type, mode)
    return out, pre


def _as_kept(fits: bool) -> None:
    if not fits:
        raise ValueError("a saved tensor has come back on another device, or with another type or size")


def _gated_rows_grad(handle, pre, dh, act):
    rows, both, ldpre = _rows_of(pre, "pre")
    _, _, lddh = _rows_of(dh, "the gradient", both // 2)
    _check_place(handle, dh.get_device())
    if dh.dtype is not pre.dtype:
        raise ValueError(f"the gradient is {dh.dtype}, the operands are {pre.dtype}")
    _as_kept(pre.get_device() == dh.get_device() and rows == dh.shape[0])
    dpre = pre.new_empty((rows, both))
    handle.gated_rows(rows, both // 2, pre.data_ptr(), ldpre, dh.data_ptr(), lddh, act, dpre.data_ptr(), both,
                      _data_type(pre.dtype))
    return dpre


def _composed(handle, x, gate_up, down, group_ends, act, mode):
    """The same made of products that have gradients of any order, for those of gradients."""
    f = torch.nn.functional
    x, gate_up = _dense_rows(x), _dense_rows(gate_up)
    gate, up = _linear(x, gate_up, group_ends, handle, True, mode, 1.0).float().chunk(2, -1)
    gate = {api.Activation.SILU: f.silu, api.Activation.GELU: f.gelu, api.Activation.RELU: f.relu,
            api.Activation.GELU_TANH: lambda v: f.gelu(v, approximate="tanh")}[act](gate)
    h = (gate * up).to(x.dtype)
    return h if down is None else _linear(h, _dense_rows(down), group_ends, handle, True, mode, 1.0)


def _composed_gradients(ctx, dy, operands, handle, group_ends, act, mode):
    wanted = [t for t, need in zip(operands, ctx.needs_input_grad) if need]
    x, gate_up, down = operands if len(operands) == 3 else (*operands, None)
    grads = iter(torch.autograd.grad(_composed(handle, x, gate_up, down, group_ends, act, mode), wanted, dy,
                                     create_graph=True))
    return [next(grads) if need else None for _, need in zip(operands, ctx.needs_input_grad)]


# Hooks on saved tensors may have moved what the forward pass kept, or changed it: order and strides are asked for anew, and
# what the kernels could not read is refused.
class _GatedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_up, group_ends, handle, act, mode, backward_mode):
        h, pre = _gated(handle, x, gate_up, group_ends, act, mode, keep=True)
        ctx.save_for_backward(x, gate_up, group_ends, pre)
        ctx.how = (handle, act, backward_mode)
        return h

    @staticmethod
    def backward(ctx, dh):
        x, gate_up, group_ends, pre = ctx.saved_tensors
        handle, act, mode = ctx.how
        if torch.is_grad_enabled():
            return (*_composed_gradients(ctx, dh, (x, gate_up), handle, group_ends, act, mode), *(None,) * 5)
        x, gate_up = _dense_rows(x), _dense_rows(gate_up)
        _as_kept(x.shape[1] == gate_up.shape[2])
        dpre = _gated_rows_grad(handle, _dense_rows(pre), _dense_rows(dh), act)
        dx = dgate_up = None
        if ctx.needs_input_grad[0]:
            dx = grouped_matmul(handle, dpre, gate_up, group_ends, mode=mode)
        if ctx.needs_input_grad[1]:
            dgate_up = grouped_matmul_wgrad(handle, x, dpre, group_ends, True, mode=mode)
        return dx, dgate_up, None, None, None, None, None


class _GatedFeedForward(torch.autograd.Function):
    # (The checks of `gated_feed_forward` are those of every product in here: a small block's time is the calls'.)
    @staticmethod
    def forward(ctx, x, gate_up, down, group_ends, handle, act, mode, backward_mode):
        h, pre, y = _feed_forward(handle, x, gate_up, down, group_ends, act, mode, True)
        ctx.save_for_backward(x, gate_up, down, group_ends, pre, h)
        ctx.how = (handle, act, backward_mode)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, gate_up, down, group_ends, pre, h = ctx.saved_tensors
        handle, act, mode = ctx.how
        if torch.is_grad_enabled():
            return (*_composed_gradients(ctx, dy, (x, gate_up, down), handle, group_ends, act, mode), *(None,) * 5)
        x, gate_up, down, dy = _dense_rows(x), _dense_rows(gate_up), _dense_rows(down), _dense_rows(dy)
        pre, h = pre.contiguous(), h.contiguous()
        groups, both, width, ldw, stridew = _matrices_of(gate_up, "gate_up")
        matrices, out_width, hidden, ldd, strided = _matrices_of(down, "down")
        rows, _, ldx = _rows_of(x, "x", width)
        dy_rows, _, lddy = _rows_of(dy, "the gradient", out_width)
        _check(handle, dy.get_device(), (x, gate_up, down, pre, h), group_ends, groups)
        _as_kept(x.dtype is gate_up.dtype is down.dtype is pre.dtype is h.dtype is dy.dtype and both == 2 * hidden and
                 matrices == groups and dy_rows == rows and pre.shape == (rows, both) and h.shape == (rows, hidden))
        ends, data_type = None if group_ends is None else group_ends.data_ptr(), _data_type(x.dtype)
        need_x, need_gate_up, need_down = ctx.needs_input_grad[:3]
        dx = dgate_up = ddown = None
        if need_x or need_gate_up:
            dpre = torch.empty_like(pre)
            dpre_at = dpre.data_ptr()
            handle.grouped_gemm_gated_grad(api.CUBLAS_OP_N, rows, hidden, out_width, groups, ends, dy.data_ptr(), lddy,
                                           down.data_ptr(), ldd, strided, act, pre.data_ptr(), both, dpre_at, both,
                                           data_type, mode)
        if need_x:
            dx = x.new_empty((rows, width))
            handle.grouped_gemm(api.CUBLAS_OP_N, rows, width, both, groups, ends, 1.0, dpre_at, both, gate_up.data_ptr(),
                                ldw, stridew, 0.0, dx.data_ptr(), width, data_type, mode)
        if need_gate_up:
            dgate_up = x.new_empty((groups, both, width))
            handle.grouped_gemm_wgrad(api.CUBLAS_OP_T, rows, both, width, groups, ends, 1.0, x.data_ptr(), ldx, dpre_at,
                                      both, 0.0, dgate_up.data_ptr(), width, both * width, data_type, mode)
        if need_down:
            ddown = x.new_empty((groups, out_width, hidden))
            handle.grouped_gemm_wgrad(api.CUBLAS_OP_T, rows, out_width, hidden, groups, ends, 1.0, h.data_ptr(), hidden,
                                      dy.data_ptr(), lddy, 0.0, ddown.data_ptr(), hidden, out_width * hidden, data_type,
                                      mode)
        return dx, dgate_up, ddown, None, None, None, None, None


def _feed_forward(handle, x, gate_up, down, group_ends, act, mode, keep=False):
    """(h, what is in front of its activation, the block's result)."""
    groups, out_width, hidden, ldd, strided = _matrices_of(down, "down")
    if hidden * 2 != gate_up.shape[1] or groups != gate_up.shape[0]:
        raise ValueError(f"down {tuple(down.shape)} does not fit gate_up {tuple(gate_up.shape)}")
    if down.dtype is not x.dtype:
        raise ValueError(f"x is {x.dtype}, down is {down.dtype}")
    if down.get_device() != x.get_device():
        raise ValueError("operands are on different devices")
    h, pre = _gated(handle, x, gate_up, group_ends, act, mode, keep=keep)
    rows = h.shape[0]
    y = x.new_empty((rows, out_width))
    handle.grouped_gemm(api.CUBLAS_OP_T, rows, out_width, hidden, groups,
                        None if group_ends is None else group_ends.data_ptr(), 1.0, h.data_ptr(), hidden,
                        down.data_ptr(), ldd, strided, 0.0, y.data_ptr(), out_width, _data_type(x.dtype), mode)
    return h, pre, y


def gated_matmul(handle: api.Handle, x, gate_up, group_ends=None, *, activation: str = "silu",
                 mode: int = api.ComputeMode.FP16TCEC, backward_mode: int = _BACKWARD_MODE, out=None):
    """``out[r] = act(x[r] @ gate_e^T) * (x[r] @ up_e^T)`` for the rows r of each expert e; rows of none: 0.

    x is (rows, width), gate_up (experts, 2 * hidden, width) with the rows of the gate first; all of float16,
    bfloat16 or float32 (``mode``).  activation: "silu", "gelu" (by the error function), "gelu_tanh" or
    "relu".  Products, activation and their product are FP32, rounded once.  Differentiable in x and
    gate_up (without ``out``), any number of times; ``backward_mode`` as in ``grouped_linear``."""
    act = _activation(activation)
    x, gate_up = _dense_rows(x), _dense_rows(gate_up)
    if torch.is_grad_enabled() and (x.requires_grad or gate_up.requires_grad):
        _no_graph_through(out, 0.0)
        return _GatedMatmul.apply(x, gate_up, group_ends, handle, act, mode, backward_mode)
    return _gated(handle, x, gate_up, group_ends, act, mode, out)[0]


def gated_feed_forward(handle: api.Handle, x, gate_up, down, group_ends=None, *, activation: str = "silu",
                       mode: int = api.ComputeMode.FP16TCEC, backward_mode: int = _BACKWARD_MODE):
    """``gated_matmul(handle, x, gate_up, ...) @ down_e^T`` for the rows of each expert e: a gated feed-forward
    block, or one for each expert.  down is (experts, width, hidden).

    Differentiable in x, gate_up and down, any number of times.  The block in between is rounded to the
    operands' type, as is the gradient in front of the activation.  One expert without ``group_ends`` is a
    dense block."""
    act = _activation(activation)
    x, gate_up, down = _dense_rows(x), _dense_rows(gate_up), _dense_rows(down)
    if torch.is_grad_enabled() and (x.requires_grad or gate_up.requires_grad or down.requires_grad):
        return _GatedFeedForward.apply(x, gate_up, down, group_ends, handle, act, mode, backward_mode)
    return _feed_forward(handle, x, gate_up, down, group_ends, act, mode)[2]


# ---------------------------------------------------------------- 8-bit floating point
def _blocks(n: int) -> int:
    return (n + _BLOCK - 1) // _BLOCK


def _f8_rows(like, rows: int, k: int, dtype):
    """Room for such rows, which start at multiples of 16 bytes, and for their scales, rows side by side."""
    ldq = (k + 15) // 16 * 16
    q = like.new_empty((rows, ldq), dtype=dtype)
    scale = like.new_empty_strided((rows, _blocks(k)), (1, rows), dtype=torch.float32)
    return (q if ldq == k else q[:, :k]), ldq, scale


def quantize_blocks(handle: api.Handle, x, row_index=None, *, activation: Optional[str] = None,
                    dtype=torch.float8_e4m3fn) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale): 8-bit floating-point rows with a float32 scale for each 128 columns, (rows, ceil(k / 128)):
    ``scale[r, j // 128] * q[r, j]`` stands for ``x[r, j]``, or with ``row_index`` (int32) for
    ``x[row_index[r], j]``; an index outside x gives a row of zeros.  dtype: float8_e4m3fn or float8_e5m2.

    With an activation, x is (rows, 2 * k), and ``act(gate) * up`` of its halves is what is quantised.
    q's rows start at multiples of 16 bytes, and a block's scales of all rows lie side by side, which is
    what ``f8_matmul`` reads fastest.  No gradients."""
    act = api.Activation.NONE if activation is None else _activation(activation)
    src_rows, k, ldx = _rows_of(x, "x")
    if activation is not None:
        if k % 2:
            raise ValueError(f"x has {k} columns: as many of the gate as of what it gates are needed")
        k //= 2
    device = x.get_device()
    _check_place(handle, device)
    data_type, q_type = _data_type(x.dtype), _f8_type(dtype, "dtype")
    rows = src_rows
    if row_index is not None:
        if row_index.dtype is not torch.int32 or row_index.dim() != 1 or not row_index.is_contiguous():
            raise ValueError("row_index must be a contiguous int32 vector")
        if row_index.get_device() != device:
            raise ValueError("row_index is on another device")
        rows = row_index.shape[0]
    q, ldq, scale = _f8_rows(x, rows, k, dtype)
    handle.quantize_rows_f8(rows, k, x.data_ptr(), ldx, data_type,
                            None if row_index is None else row_index.data_ptr(), src_rows, act, q.data_ptr(), ldq,
                            q_type, scale.data_ptr(), 1, rows)
    return q, scale


def quantize_weight_blocks(handle: api.Handle, w, *, dtype=torch.float8_e4m3fn) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of weights (experts, n, k) or (n, k), with a float32 scale for each 128 x 128 of a matrix:
    (experts, ceil(n / 128), ceil(k / 128)), or without the first.  No gradients."""
    stack = w if w.dim() == 3 else w.unsqueeze(0)
    matrices, n, k, ldw, stridew = _matrices_of(stack, "w")
    _check_place(handle, w.get_device())
    ldq = (k + 15) // 16 * 16
    q = w.new_empty((matrices, n, ldq), dtype=dtype)
    scale = w.new_empty((matrices, _blocks(n), _blocks(k)), dtype=torch.float32)
    handle.quantize_blocks_f8(matrices, n, k, stack.data_ptr(), ldw, stridew, _data_type(w.dtype), q.data_ptr(), ldq,
                              n * ldq, _f8_type(dtype, "dtype"), scale.data_ptr())
    q = q if ldq == k else q[..., :k]
    return (q, scale) if w.dim() == 3 else (q[0], scale[0])


def _f8_operands(handle, xq, x_scale, wq, w_scale, group_ends, others=()):
    """What both products check: (rows, n, k, groups, ldx, ldw, stridew, types, steps of x_scale)."""
    groups, n, k, ldw, stridew = _matrices_of(wq, "wq")
    rows, _, ldx = _rows_of(xq, "xq", k)
    _check(handle, xq.get_device(), (x_scale, wq, w_scale, *others), group_ends, groups)
    x_type, w_type = _f8_type(xq.dtype, "xq"), _f8_type(wq.dtype, "wq")
    if x_scale.dtype is not torch.float32 or tuple(x_scale.shape) != (rows, _blocks(k)):
        raise ValueError(f"x_scale must be float32 of shape {(rows, _blocks(k))}")
    _check_scales(w_scale, "w_scale", groups * _blocks(n) * _blocks(k))
    return rows, n, k, groups, ldx, ldw, stridew, x_type, w_type, x_scale.stride()


def f8_matmul(handle: api.Handle, xq, x_scale, wq, w_scale, group_ends=None, *, bias=None, out=None,
              out_dtype=torch.bfloat16):
    """``out[r] = x[r] @ w_e^T + bias[e]`` for the rows r of each expert e, x and w being what 8-bit values and
    scales stand for; rows of none: 0.

    xq is (rows, k) and wq (experts, n, k), each of float8_e4m3fn or float8_e5m2; x_scale (rows, ceil(k / 128)),
    w_scale (experts, ceil(n / 128), ceil(k / 128)) and bias (experts, n), float32.  A (n, k) wq with
    its scales is one expert of all rows: a plain linear layer.  No gradients."""
    if wq.dim() == 2:
        wq = wq.unsqueeze(0)
    rows, n, k, groups, ldx, ldw, stridew, x_type, w_type, steps = _f8_operands(
        handle, xq, x_scale, wq, w_scale, group_ends, () if bias is None else (bias,))
    if bias is not None:
        _check_scales(bias, "bias", groups * n)
    ldy = n
    if out is not None:
        out_dtype = out.dtype
        _, _, ldy = _rows_of(out, "out")
    data_type = _data_type(out_dtype)
    out = _output(out, 0.0, (rows, n), out_dtype, xq)
    handle.f8_grouped_gemm(rows, n, k, groups, None if group_ends is None else group_ends.data_ptr(), xq.data_ptr(),
                           ldx, x_type, x_scale.data_ptr(), steps[0], steps[1], wq.data_ptr(), ldw, stridew, w_type,
                           w_scale.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), ldy,
                           data_type)
    return out


def f8_gated_matmul(handle: api.Handle, xq, x_scale, wq, w_scale, group_ends=None, *, activation: str = "silu",
                    dtype=torch.float8_e4m3fn) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scale) of ``act(x[r] @ gate_e^T) * (x[r] @ up_e^T)`` as ``quantize_blocks`` gives them, for ``f8_matmul``
    with the weights behind: operands as there, wq being (experts, 2 * hidden, k) with the rows of the gate
    first.  Products, activation and their product are FP32.  Where hidden is a multiple of 128 and the rows are
    many nothing else reaches memory; otherwise the products do, in FP32, and a pass over them.  Near the middle
    between two 8-bit values the two ways, and ``quantize_blocks``, may choose either of them.  No gradients."""
    act = _activation(activation)
    if wq.dim() == 2:
        wq = wq.unsqueeze(0)
    if wq.dim() == 3 and wq.shape[1] % 2:
        raise ValueError(f"wq has {wq.shape[1]} rows: as many of the gate as of what it gates are needed")
    if wq.dim() != 3 or (wq.shape[1] // 2) % _BLOCK:
        pre = f8_matmul(handle, xq, x_scale, wq, w_scale, group_ends, out_dtype=torch.float32)
        return quantize_blocks(handle, pre, activation=activation, dtype=dtype)
    rows, n, k, groups, ldx, ldw, stridew, x_type, w_type, steps = _f8_operands(handle, xq, x_scale, wq, w_scale, group_ends)
    q_type = _f8_type(dtype, "dtype")
    q, ldq, scale = _f8_rows(xq, rows, n // 2, dtype)
    handle.f8_grouped_gemm_gated(rows, n // 2, k, groups, None if group_ends is None else group_ends.data_ptr(),
                                 xq.data_ptr(), ldx, x_type, x_scale.data_ptr(), steps[0], steps[1], wq.data_ptr(), ldw,
                                 stridew, w_type, w_scale.data_ptr(), act, q.data_ptr(), ldq, q_type, scale.data_ptr(),
                                 1, rows)
    return q, scale
