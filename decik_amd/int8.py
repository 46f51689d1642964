"""Linear layers in 8-bit integers with a scale per token and per channel (dk_int8_*).

A frozen weight [N, K] is held as int8 rows with one fp32 scale each (quantize_int8), half the bytes of
fp16 and twice its matrix rate; activations are quantized per token on the way in:
  forward:  y = fp32(sum_k xq wq) * x_scale[m] * w_scale[n] + bias[n], rounded once
  backward: dX = fp32(sum_n gq wq) * g_scale[m], with gq, g_scale quantized per token from dY * w_scale
The integer sums are exact, so results depend neither on the number of tokens in a call nor on the
launch. The gradient is that of the dequantized linear (the rounding of x passes it on unchanged), its
own rounding at most half a step, max|dY * w_scale| / 254 of its row, a term.

Quantized rows are padded to 128 bytes; the tensors here are views of the padded rows.
"""

import ctypes

import torch
from torch.autograd.function import once_differentiable

from ._lib import DTYPES, call_on, check, gpu_input, lib, same_gpu


def _ptr(t):
    return None if t is None else t.data_ptr()


def _token_rows(x):
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1]) if x.numel() else x.reshape(0, x.shape[-1])
    return x2 if (x2.stride(1) == 1 or x2.shape[1] == 1) and x2.stride(0) >= 0 else x2.contiguous()


def _code(what, name, dtype):
    code = DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{what}: {name} must be fp16, bf16 or fp32")
    return code


def quantize_int8(x, col_scale=None):
    """(q int8 [rows, K], scale fp32 [rows]) of x [.., K] (fp16, bf16 or fp32) row by row: scale = absmax
    / 127, q = rint(x * (127 / absmax)); col_scale fp32 [K] multiplies x first. For a weight [N, K] the rows
    are its output channels. A row with an infinity or NaN gets the scale NaN."""
    what = "quantize_int8"
    dev = gpu_input(what, x)
    same_gpu(what, dev, col_scale)
    code = _code(what, "x", x.dtype)
    if x.dim() < 1:
        raise ValueError(f"{what}: x must be [.., K]")
    x2 = _token_rows(x)
    rows, k = x2.shape
    if col_scale is not None:
        if tuple(col_scale.shape) != (k,) or col_scale.dtype != torch.float32:
            raise ValueError(f"{what}: col_scale must be fp32 [{k}]")
        col_scale = col_scale.contiguous()
    ld = (k + 127) // 128 * 128
    q = x.new_empty(rows, ld, dtype=torch.int8)
    scale = x.new_empty(rows, dtype=torch.float32)
    call_on(dev, lib().dk_int8_quantize, x2.data_ptr(), code, x2.stride(0), _ptr(col_scale), q.data_ptr(), ld,
            scale.data_ptr(), rows, k)
    return q[:, :k], scale


def dequantize_int8(q, scale, dtype=torch.float32):
    """The values q stands for, [rows, K]."""
    return (q.to(torch.float32) * scale[:, None]).to(dtype)


def _int8_rows(what, name, q, zero_tail):
    """(q, its row stride), or a padded copy where its rows do not start at multiples of 16 bytes or its
    storage ends inside the last 16 (zero_tail: the padding must hold zeros, so only rows without any pass)."""
    if q.dim() != 2 or q.dtype != torch.int8:
        raise ValueError(f"{what}: {name} must be int8 [rows, columns]")
    rows, k = q.shape
    need = (k + 15) // 16 * 16
    ld = q.stride(0) if rows > 1 else need
    if ld % 16 == 0 and need <= ld < 2 ** 23 and (q.stride(1) == 1 or k == 1) and q.data_ptr() % 16 == 0 and \
            q.storage_offset() + max(rows - 1, 0) * ld + need <= q.untyped_storage().nbytes() and \
            (not zero_tail or k == need):
        return q, ld
    copy = torch.zeros((rows, need), dtype=torch.int8, device=q.device)
    copy[:, :k] = q
    return copy, need


def _channel_args(what, ws, bias, n):
    if ws.shape != (n,) or ws.dtype != torch.float32:
        raise ValueError(f"{what}: w_scale must be fp32 [{n}]")
    if bias is None:
        return ws.contiguous(), None, 0
    if bias.shape != (n,):
        raise ValueError(f"{what}: bias must be [{n}]")
    return ws.contiguous(), bias.contiguous(), _code(what, "bias", bias.dtype)


def _workspace(x, need):
    # a tensor of its own a call: graphs and streams share none
    return x.new_empty(need, dtype=torch.uint8) if need > 0 else None


def launch_plan(transposed, m, n, k):
    """What a product of these sizes runs as (dk_int8_linear_plan): dict of tile_tokens (0: the weight streams
    to registers), tile_channels, splits, fused (x quantized inside)."""
    out = (ctypes.c_int32 * 4)()
    check(lib().dk_int8_linear_plan(int(transposed), m, n, k, out))
    return dict(tile_tokens=out[0], tile_channels=out[1], splits=out[2], fused=bool(out[3]))


def int8_matmul(xq, x_scale, wq, w_scale, bias=None, dtype=torch.float16):
    """y [M, N] = (xq . wq^T) * x_scale * w_scale (+ bias) of int8 xq [M, K] and wq [N, K] with fp32 scales
    [M] and [N]; K <= 131071. Rows that do not start at multiples of 16 bytes, or of xq whose K is not one,
    are copied first."""
    what = "int8_matmul"
    dev = gpu_input(what, xq)
    same_gpu(what, dev, x_scale, wq, w_scale, bias)
    if xq.dim() != 2 or wq.dim() != 2 or xq.shape[1] != wq.shape[1]:
        raise ValueError(f"{what}: xq [M, K] and wq [N, K] must share K")
    m, k = xq.shape
    n = wq.shape[0]
    if x_scale.shape != (m,) or x_scale.dtype != torch.float32:
        raise ValueError(f"{what}: x_scale must be fp32 [{m}]")
    out = _code(what, "dtype", dtype)
    xq, ldx = _int8_rows(what, "xq", xq, True)
    wq, ldw = _int8_rows(what, "wq", wq, False)
    x_scale = x_scale.contiguous()
    ws, bias, bias_code = _channel_args(what, w_scale, bias, n)
    y = xq.new_empty(m, n, dtype=dtype)
    need = lib().dk_int8_linear_workspace(0, m, n, k)
    work = _workspace(xq, need)
    call_on(dev, lib().dk_int8_linear, 0, xq.data_ptr(), ldx, x_scale.data_ptr(), wq.data_ptr(), ldw, ws.data_ptr(),
            _ptr(bias), bias_code, y.data_ptr(), out, n, m, n, k, _ptr(work), max(need, 0))
    return y


def int8_linear_forward(x, wq, w_scale, bias=None, dtype=None):
    """y [.., N] (x's type, or dtype) = x . W^T + bias for W held as wq [N, K] int8 and w_scale [N], x [.., K]
    fp16, bf16 or fp32 quantized per token."""
    what = "int8_linear_forward"
    dev = gpu_input(what, x)
    same_gpu(what, dev, wq, w_scale, bias)
    if wq.dim() != 2 or x.dim() < 1 or x.shape[-1] != wq.shape[1]:
        raise ValueError(f"{what}: x [.., K] and wq [N, K] must share K")
    dtype = dtype or x.dtype
    code, out = _code(what, "x", x.dtype), _code(what, "dtype", dtype)
    wq, ldw = _int8_rows(what, "wq", wq, False)
    n, k = wq.shape[0], x.shape[-1]
    ws, bias, bias_code = _channel_args(what, w_scale, bias, n)
    x2 = _token_rows(x)
    m = x2.shape[0]
    y = x.new_empty(*x.shape[:-1], n, dtype=dtype)
    need = lib().dk_int8_linear_x_workspace(0, m, n, k)
    work = _workspace(x, need)
    call_on(dev, lib().dk_int8_linear_fwd, x2.data_ptr(), code, x2.stride(0), wq.data_ptr(), ldw, ws.data_ptr(),
            _ptr(bias), bias_code, y.data_ptr(), out, n, m, n, k, _ptr(work), max(need, 0))
    return y


def int8_linear_backward(dy, wq, w_scale, k=None, dtype=None):
    """dX [.., K] (dy's type, or dtype) = dY . W, dY * w_scale quantized per token. k, where given, must be
    the weight's K."""
    what = "int8_linear_backward"
    dev = gpu_input(what, dy)
    same_gpu(what, dev, wq, w_scale)
    if wq.dim() != 2 or dy.dim() < 1 or dy.shape[-1] != wq.shape[0] or (k is not None and k != wq.shape[1]):
        raise ValueError(f"{what}: dy [.., N] and wq [N, K] must share N")
    dtype = dtype or dy.dtype
    code, out = _code(what, "dy", dy.dtype), _code(what, "dtype", dtype)
    n, k = wq.shape
    wq, ldw = _int8_rows(what, "wq", wq, False)
    ws, _, _ = _channel_args(what, w_scale, None, n)
    dy2 = _token_rows(dy)
    m = dy2.shape[0]
    dx = dy.new_empty(*dy.shape[:-1], k, dtype=dtype)
    need = lib().dk_int8_linear_x_workspace(1, m, n, k)
    work = _workspace(dy, need)
    call_on(dev, lib().dk_int8_linear_bwd, dy2.data_ptr(), code, dy2.stride(0), wq.data_ptr(), ldw, ws.data_ptr(),
            dx.data_ptr(), out, k, m, n, k, _ptr(work), max(need, 0))
    return dx


class Int8Linear(torch.autograd.Function):
    """apply(x, wq, w_scale, bias) -> y: a linear whose int8 weight and bias are frozen; gradients reach x."""

    @staticmethod
    def forward(ctx, x, wq, w_scale, bias=None):
        if any(ctx.needs_input_grad[2:]):  # (three inputs where the call names no bias)
            raise ValueError("Int8Linear: the weight's scales and the bias are frozen (detach them)")
        ctx.save_for_backward(wq, w_scale)
        ctx.x_dtype = x.dtype
        return int8_linear_forward(x, wq, w_scale, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        wq, w_scale = ctx.saved_tensors
        return int8_linear_backward(grad, wq, w_scale, dtype=ctx.x_dtype), None, None, None
