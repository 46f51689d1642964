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

import torch

from ._lib import DTYPES, check, gpu_tensors, lib, on_device, ptr, stream_of


def _padded(rows, k, device):
    """int8 [rows, k] view of rows padded to a multiple of 128."""
    return torch.empty((rows, (k + 127) // 128 * 128), dtype=torch.int8, device=device)[:, :k]


def _token_rows(x):
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1]) if x.numel() else x.reshape(0, x.shape[-1])
    return x2 if (x2.stride(1) == 1 or x2.shape[1] == 1) and x2.stride(0) >= 0 else x2.contiguous()


def quantize_int8(x, col_scale=None):
    """(q int8 [rows, K], scale fp32 [rows]) of x [.., K] (fp16, bf16 or fp32) row by row: scale = absmax
    / 127, q = rint(x * (127 / absmax)); col_scale fp32 [K] multiplies x first. For a weight [N, K] the rows
    are its output channels. A row with an infinity or NaN gets the scale NaN."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("quantize_int8: needs GPU tensors")
    if x.dim() < 1 or x.dtype not in DTYPES:
        raise ValueError("quantize_int8: x must be fp16, bf16 or fp32 [.., K]")
    dev = x.device
    x2 = _token_rows(x)
    rows, k = x2.shape
    if col_scale is not None:
        gpu_tensors("quantize_int8", dev, col_scale=col_scale)
        if tuple(col_scale.shape) != (k,) or col_scale.dtype != torch.float32:
            raise ValueError(f"quantize_int8: col_scale must be fp32 [{k}]")
        col_scale = col_scale.contiguous()
    q = _padded(rows, k, dev)
    scale = torch.empty(rows, dtype=torch.float32, device=dev)
    with on_device(dev):
        check(lib().dk_int8_quantize(ptr(x2), DTYPES[x.dtype], x2.stride(0), ptr(col_scale), ptr(q), q.stride(0),
                                     ptr(scale), rows, k, stream_of(dev)))
    return q, scale


def dequantize_int8(q, scale, dtype=torch.float32):
    """The values q stands for, [rows, K]."""
    return (q.to(torch.float32) * scale[:, None]).to(dtype)


def _int8_rows(what, name, q, zero_tail):
    """q, or a padded copy where its rows do not start at multiples of 16 bytes or its storage ends inside
    the last 16 (zero_tail: the padding must hold zeros, so only quantize_int8's own rows pass)."""
    if q.dim() != 2 or q.dtype != torch.int8:
        raise ValueError(f"{what}: {name} must be int8 [rows, columns]")
    rows, k = q.shape
    ld, need = q.stride(0) if rows > 1 else (k + 15) // 16 * 16, (k + 15) // 16 * 16
    end = q.storage_offset() + max(rows - 1, 0) * q.stride(0) + need
    if (q.stride(1) == 1 or k == 1) and ld % 16 == 0 and need <= ld < 2 ** 23 and q.data_ptr() % 16 == 0 and \
            end <= q.untyped_storage().nbytes() and (not zero_tail or k == need):
        return q, ld
    copy = torch.zeros((rows, need), dtype=torch.int8, device=q.device)
    copy[:, :k] = q
    return copy, need


def _product(what, transposed, xq, ldx, xs, wq, ws, bias, dtype, m, n, k):
    dev = xq.device
    gpu_tensors(what, dev, x_scale=xs, wq=wq, w_scale=ws, bias=bias)
    if dtype not in DTYPES:
        raise ValueError(f"{what}: fp16, bf16 or fp32 outputs only")
    wq, ldw = _int8_rows(what, "wq", wq, False)
    if bias is not None and (tuple(bias.shape) != (n,) or bias.dtype not in DTYPES):
        raise ValueError(f"{what}: bias must be fp16, bf16 or fp32 [{n}]")
    if ws is not None and (tuple(ws.shape) != (n,) or ws.dtype != torch.float32):
        raise ValueError(f"{what}: w_scale must be fp32 [{n}]")
    bias = None if bias is None else bias.contiguous()
    ws = None if ws is None else ws.contiguous()
    y = torch.empty((m, n), dtype=dtype, device=dev)
    with on_device(dev):
        need = lib().dk_int8_linear_workspace(transposed, m, n, k)
        # a tensor of its own a call: graphs and streams share none
        work = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
        check(lib().dk_int8_linear(transposed, ptr(xq), ldx, ptr(xs), ptr(wq), ldw, ptr(ws), ptr(bias),
                                   0 if bias is None else DTYPES[bias.dtype], ptr(y), DTYPES[dtype], n, m, n, k,
                                   ptr(work), max(need, 0), stream_of(dev)))
    return y


def int8_matmul(xq, x_scale, wq, w_scale, bias=None, dtype=torch.float16):
    """y [M, N] = (xq . wq^T) * x_scale * w_scale (+ bias) of int8 xq [M, K] and wq [N, K] with fp32 scales
    [M] and [N]; K <= 131071. Rows that do not start at multiples of 16 bytes are copied first."""
    what = "int8_matmul"
    if not isinstance(xq, torch.Tensor) or not xq.is_cuda:
        raise ValueError(f"{what}: needs GPU tensors")
    gpu_tensors(what, xq.device, wq=wq)
    if xq.dim() != 2 or wq.dim() != 2 or xq.shape[1] != wq.shape[1]:
        raise ValueError(f"{what}: xq [M, K] and wq [N, K] must share K")
    m, k = xq.shape
    if tuple(x_scale.shape) != (m,) or x_scale.dtype != torch.float32:
        raise ValueError(f"{what}: x_scale must be fp32 [{m}]")
    xq, ldx = _int8_rows(what, "xq", xq, True)
    return _product(what, 0, xq, ldx, x_scale.contiguous(), wq, w_scale, bias, dtype, m, wq.shape[0], k)


def int8_linear_forward(x, wq, w_scale, bias=None, dtype=None):
    """y [.., N] (x's type, or dtype) = x . W^T + bias for W held as wq [N, K] int8 and w_scale [N], x [.., K]
    fp16, bf16 or fp32 quantized per token."""
    what = "int8_linear_forward"
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{what}: needs GPU tensors")
    gpu_tensors(what, x.device, wq=wq)
    if wq.dim() != 2 or x.shape[-1] != wq.shape[1]:
        raise ValueError(f"{what}: x [.., K] and wq [N, K] must share K")
    n, k = wq.shape
    xq, xs = quantize_int8(x)
    y = _product(what, 0, xq, xq.stride(0), xs, wq, w_scale, bias, x.dtype if dtype is None else dtype, xs.shape[0], n,
                 k)
    return y.reshape(*x.shape[:-1], n)


def int8_linear_backward(dy, wq, w_scale, k=None, dtype=None):
    """dX [.., K] (dy's type, or dtype) = dY . W, dY * w_scale quantized per token."""
    what = "int8_linear_backward"
    if not isinstance(dy, torch.Tensor) or not dy.is_cuda:
        raise ValueError(f"{what}: needs GPU tensors")
    gpu_tensors(what, dy.device, wq=wq, w_scale=w_scale)
    if wq.dim() != 2 or dy.shape[-1] != wq.shape[0] or (k is not None and k != wq.shape[1]):
        raise ValueError(f"{what}: dy [.., N] and wq [N, K] must share N")
    n, k = wq.shape
    gq, gs = quantize_int8(dy, w_scale)
    dx = _product(what, 1, gq, gq.stride(0), gs, wq, None, None, dy.dtype if dtype is None else dtype, gs.shape[0], k, n)
    return dx.reshape(*dy.shape[:-1], k)


class Int8Linear(torch.autograd.Function):
    """apply(x, wq, w_scale, bias) -> y: a linear with a frozen int8 weight; gradients reach x (and bias)."""

    @staticmethod
    def forward(ctx, x, wq, w_scale, bias=None):
        ctx.save_for_backward(wq, w_scale)
        ctx.x_dtype, ctx.bias_dtype = x.dtype, None if bias is None else bias.dtype
        return int8_linear_forward(x, wq, w_scale, bias)

    @staticmethod
    def backward(ctx, grad):
        wq, w_scale = ctx.saved_tensors
        dx = int8_linear_backward(grad, wq, w_scale, dtype=ctx.x_dtype) if ctx.needs_input_grad[0] else None
        db = None
        if ctx.needs_input_grad[3]:
            db = grad.reshape(-1, grad.shape[-1]).sum(0, dtype=torch.float32).to(ctx.bias_dtype)
        return dx, None, None, db
