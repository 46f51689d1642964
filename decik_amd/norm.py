"""The residual stream between two blocks of a decoder layer (dk_residual_norm_fwd / dk_residual_norm_bwd): the norm
after a block, its gate, the scaled residual and the norm before the next block in one pass.

  p = N(x) * post_weight, or x without a post weight     N(v) = v / sqrt(mean(v^2) + eps) over the last axis
  h = residual_scale * residual + gate * p               the stream, kept for the next block's join
  y = N(h) * weight                                      what the next block reads

x fp16, bf16 or fp32; the stream (residual, h) in x's type or fp32. Everything is computed in fp32 and rounded once: y
and the gradients follow from h before it is rounded, and the backward forms it again from x and residual, so nothing
else is kept. A gate has a value a channel [W], a token [.., 1] or an element [.., W]. The stored weights are taken as
they are: a checkpoint that keeps weight - 1 passes 1 + weight.
"""

import torch
from torch.autograd.function import once_differentiable

from ._lib import DTYPES, ResidualNorm, call_on, gpu_input, lib, same_gpu

MAX_WIDTH = 16384
_NONE, _CHANNEL, _TOKEN, _ELEMENT = range(4)  # DK_GATE_*


def _rows(t, width):
    """(t or a copy whose rows have one stride, that stride in elements)."""
    if t.is_contiguous():
        return t, width
    t2 = t if t.dim() == 2 else t.reshape(-1, width)
    if t2.stride(1) != 1 and width != 1 or t2.stride(0) < 0:
        t2 = t2.contiguous()
    return t2, t2.stride(0)


def _weight(what, name, w, width):
    """(contiguous weight, its address and type code)."""
    if w is None:
        return None, 0, 0
    code = DTYPES.get(w.dtype)
    if code is None or w.shape != (width,):
        raise ValueError(f"{what}: {name} must be [{width}], fp16, bf16 or fp32")
    w = w.contiguous()
    return w, w.data_ptr(), code


def _gate(what, gate, shape):
    """(gate, its address, type code, kind, row stride)."""
    if gate is None:
        return None, 0, 0, _NONE, 0
    code = DTYPES.get(gate.dtype)
    if code is None:
        raise ValueError(f"{what}: the gate must be fp16, bf16 or fp32")
    width = shape[-1]
    if gate.dim() == 1 and gate.shape[0] == width:
        gate = gate.contiguous()
        return gate, gate.data_ptr(), code, _CHANNEL, 0
    if gate.shape == shape:
        gate, ld = _rows(gate, width)
        return gate, gate.data_ptr(), code, _ELEMENT, ld
    if gate.shape == (*shape[:-1], 1):
        gate, ld = _rows(gate, 1)
        return gate, gate.data_ptr(), code, _TOKEN, ld
    raise ValueError(f"{what}: a gate must be [{width}], {tuple(shape)} or {(*shape[:-1], 1)}, not {tuple(gate.shape)}")


def _inputs(what, x, residual, weight, post_weight, gate, dtype):
    """The checked inputs of a call: (device, x, residual (rows of one stride), their addresses and row strides, weight,
    post weight and gate with address and type, type codes of x, stream and y, width)."""
    dev = gpu_input(what, x)
    same_gpu(what, dev, residual, weight, post_weight, gate)
    shape = x.shape
    xc = sc = yc = DTYPES.get(x.dtype)
    if xc is None or not shape or not 1 <= shape[-1] <= MAX_WIDTH:
        raise ValueError(f"{what}: x must be [.., W] with W from 1 to {MAX_WIDTH}, fp16, bf16 or fp32")
    width = shape[-1]
    r_at = ldr = 0
    if residual is not None:
        sc = DTYPES.get(residual.dtype)
        if residual.shape != shape or sc not in (xc, 2):
            raise ValueError(f"{what}: the residual must have x's shape, and x's type or fp32")
        residual, ldr = _rows(residual, width)
        r_at = residual.data_ptr()
    if dtype is not None:
        yc = DTYPES.get(dtype)
        if yc not in (xc, 2):
            raise ValueError(f"{what}: y must be of x's type or fp32")
    x, ldx = _rows(x, width)
    return (dev, x, residual, x.data_ptr(), r_at, ldx, ldr, _weight(what, "weight", weight, width),
            _weight(what, "post_weight", post_weight, width), _gate(what, gate, shape), xc, sc, yc, width)


def _like(t, contiguous, dtype):
    """An empty tensor of t's shape with packed rows."""
    return torch.empty_like(t) if contiguous and t.dtype == dtype else t.new_empty(t.shape, dtype=dtype)


def _forward(what, x, residual, weight, post_weight, gate, scale, eps, dtype, keep_h):
    dev, x2, r2, x_at, r_at, ldx, ldr, w, pw, g, xc, sc, yc, width = _inputs(what, x, residual, weight, post_weight, gate,
                                                                           dtype)
    packed = x.is_contiguous()
    h = y = None
    if keep_h:
        h = _like(x, packed, x.dtype if residual is None else residual.dtype)
    if weight is not None:
        y = _like(x, packed, dtype or x.dtype)
    desc = ResidualNorm.PACK.pack(x_at, r_at, 0, 0, 0 if h is None else h.data_ptr(), 0 if y is None else y.data_ptr(), 0, 0, 0,
                                  w[1], pw[1], g[1], 0, 0, ldx, ldr, 0, 0, g[4], x.numel() // width, width, xc, sc, yc,
                                  w[2], pw[2], g[2], g[3], scale, eps, 0)
    call_on(dev, lib().dk_residual_norm_fwd, desc)
    return h, y


def residual_norm_forward(x, residual, weight, post_weight=None, gate=None, residual_scale=1.0, eps=1e-6, dtype=None):
    """(h, y) of x [.., W] and residual (the same shape; None: no stream). h is of the residual's type (x's without
    one), y of `dtype` (x's type, the default, or fp32), None without a weight."""
    return _forward("residual_norm_forward", x, residual, weight, post_weight, gate, residual_scale, eps, dtype, True)


def residual_norm_backward(grad_h, grad_y, x, residual, weight, post_weight=None, gate=None, residual_scale=1.0, eps=1e-6,
                           param_grads=True):
    """(dx, dresidual, dweight, dpost_weight, dgate) of residual_norm_forward from the gradients of h (None: zeros) and
    y (None only without a weight) and the same inputs; None for an input that was None. dweight, dpost_weight and
    the gradient of a channel gate are fp32 [W]; without param_grads these three are None."""
    return _backward("residual_norm_backward", grad_h, grad_y, x, residual, weight, post_weight, gate, residual_scale, eps,
                     (param_grads, param_grads, param_grads), True)


def _backward(what, grad_h, grad_y, x, residual, weight, post_weight, gate, residual_scale, eps, sums_of, gate_grad):
    """residual_norm_backward with the sums over the rows that are asked for (weight, post weight, channel gate) and, where
    asked for, the gradient of another gate."""
    dev, x2, r2, x_at, r_at, ldx, ldr, w, pw, g, xc, sc, yc, width = _inputs(
        what, x, residual, weight, post_weight, gate, None if grad_y is None else grad_y.dtype)
    same_gpu(what, dev, grad_h, grad_y)
    if (grad_y is None) != (weight is None) or (grad_y is not None and grad_y.shape != x.shape):
        raise ValueError(f"{what}: grad_y of x's shape where there is a weight, and only there")
    h_dtype = x.dtype if residual is None else residual.dtype
    gh_at = ldgh = gy_at = ldgy = 0
    if grad_h is not None:
        if grad_h.shape != x.shape or grad_h.dtype != h_dtype:
            raise ValueError(f"{what}: grad_h must have h's shape and type")
        grad_h, ldgh = _rows(grad_h, width)
        gh_at = grad_h.data_ptr()
    if grad_y is not None:
        grad_y, ldgy = _rows(grad_y, width)
        gy_at = grad_y.data_ptr()
    packed, rows, kind = x.is_contiguous(), x.numel() // width, g[3]
    dx = _like(x, packed, x.dtype)
    dres = None if residual is None else _like(x, packed, h_dtype)
    dgate = x.new_empty(gate.shape, dtype=gate.dtype) if kind in (_TOKEN, _ELEMENT) and gate_grad else None
    # the gradients that are sums over the rows: weight, post weight, channel gate
    wanted = [asked and there for asked, there in zip(sums_of, (weight is not None, post_weight is not None, kind == _CHANNEL))]
    count = sum(wanted)
    work, need, dw, dpw = None, 0, None, None
    if count:
        sums = iter(x.new_empty(count, width, dtype=torch.float32).unbind())
        dw, dpw, channel = (next(sums) if want else None for want in wanted)
        dgate = channel if kind == _CHANNEL else dgate
    desc = ResidualNorm.PACK.pack(x_at, r_at, gh_at, gy_at, 0, 0, dx.data_ptr(), 0 if dres is None else dres.data_ptr(),
                                  0 if dgate is None else dgate.data_ptr(), w[1], pw[1], g[1],
                                  0 if dw is None else dw.data_ptr(), 0 if dpw is None else dpw.data_ptr(), ldx, ldr, ldgh,
                                  ldgy, g[4], rows, width, xc, sc, yc, w[2], pw[2], g[2], kind, residual_scale, eps, 0)
    if count:
        need = lib().dk_residual_norm_bwd_workspace(desc)
        # a tensor of its own a call: graphs and streams share none
        work = x.new_empty(need, dtype=torch.uint8) if need > 0 else None
    call_on(dev, lib().dk_residual_norm_bwd, desc, None if work is None else work.data_ptr(), max(need, 0))
    return dx, dres, dw, dpw, dgate


class _ResidualNorm(torch.autograd.Function):
    """apply(x, residual, weight, post_weight, gate, residual_scale, eps, dtype) -> (h, y), or h without a weight."""

    @staticmethod
    def forward(ctx, x, residual, weight, post_weight, gate, scale, eps, dtype):
        h, y = residual_norm_forward(x, residual, weight, post_weight, gate, scale, eps, dtype)
        ctx.save_for_backward(x, residual, weight, post_weight, gate)
        ctx.scale, ctx.eps, ctx.y_dtype = scale, eps, None if y is None else y.dtype
        ctx.set_materialize_grads(False)
        return h if y is None else (h, y)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_h, grad_y=None):
        if grad_h is None and grad_y is None:
            return (None,) * 8
        x, residual, weight, post_weight, gate = ctx.saved_tensors
        if grad_y is None:
            grads_w = None
            if weight is not None:
                # nothing reached y: the norm before the next block drops out
                grads_w, weight = torch.zeros_like(weight), None
        dx, dres, dw, dpw, dgate = _backward("residual_norm", grad_h, grad_y, x, residual, weight, post_weight, gate, ctx.scale,
                                             ctx.eps, ctx.needs_input_grad[2:5], ctx.needs_input_grad[4])
        if grad_y is None:
            dw = grads_w
        elif dw is not None:
            dw = dw.to(weight.dtype)
        if dpw is not None:
            dpw = dpw.to(post_weight.dtype)
        if dgate is not None:
            dgate = dgate.to(gate.dtype)
        return dx, dres, dw, dpw, dgate, None, None, None


def residual_norm(x, residual, weight, post_weight=None, gate=None, residual_scale=1.0, eps=1e-6, dtype=None):
    """residual_norm_forward, differentiable in x, residual, the weights and the gate."""
    out = _ResidualNorm.apply(x, residual, weight, post_weight, gate, residual_scale, eps, dtype)
    return (out, None) if weight is None else out


def rms_norm(x, weight, eps=1e-6, dtype=None):
    """N(x) * weight (of `dtype`: x's type or fp32), differentiable in x and the weight; the stream's start, before the
    first block."""
    return _RmsNorm.apply(x, weight, eps, dtype)


class _RmsNorm(torch.autograd.Function):
    """apply(x, weight, eps, dtype) -> y."""

    @staticmethod
    def forward(ctx, x, weight, eps, dtype):
        if weight is None:
            raise ValueError("rms_norm: needs a weight")
        _, y = _forward("rms_norm", x, None, weight, None, None, 1.0, eps, dtype, False)
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight = ctx.saved_tensors
        dx, _, dw, _, _ = residual_norm_backward(None, grad, x, None, weight, eps=ctx.eps,
                                                 param_grads=ctx.needs_input_grad[1])
        return dx, None if dw is None else dw.to(weight.dtype), None, None
