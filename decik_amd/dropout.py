"""Dropout with masks from a counter-based generator, never stored (dk_dropout_fwd, dk_dropout_bwd).

The packed masks of pack_keep cost a random bool tensor, a pass that packs it and a bit an element that
lives until the backward. Here an element's mask is a function of (seed, offset, row, column): the
forward and the backward form it again, so nothing is kept but the two numbers, and a recomputed
forward drops the same elements. They are read from the device when a kernel runs, so a captured graph
takes a new mask on every replay whose `rng` was advanced before it.

An element's number is one of 65536 values, kept when it is not below rint(65536 p); kept elements are
multiplied by 65536 / (65536 - rint(65536 p)), so the expected value is the input's exactly. Dropped
elements are +0 whatever they held. Branch b of a call at offset o is branch 0 of a call at o + b: a
call with n branches uses up n offsets.
"""

import ctypes

import torch

from ._lib import DTYPES, check, gpu_tensors, lib, on_device, ptr, stream_of

MAX_BRANCHES = 4


def rng_state(seed, offset=0, device="cuda"):
    """int64 tensor (seed, offset) on the GPU, as the calls below take it. In-place changes select
    other masks (rng[1] += n for the next step)."""
    return torch.tensor([_signed(seed), _signed(offset)], dtype=torch.int64, device=device)


def _signed(v):
    v = int(v) % 2 ** 64
    return v - 2 ** 64 if v >= 2 ** 63 else v


def _rows(t):
    """[rows, width] view (a copy only where the rows have no common stride)."""
    t2 = t if t.dim() == 2 else t.reshape(-1, t.shape[-1]) if t.numel() else t.reshape(0, t.shape[-1])
    if t2.stride(-1) == 1 or t2.shape[-1] == 1:
        if t2.stride(0) >= 0:
            return t2
    return t2.contiguous()


def _common(what, t, rng, ps, dtype):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what}: needs GPU tensors")
    if t.dim() < 1:
        raise ValueError(f"{what}: needs a last axis")
    gpu_tensors(what, t.device, rng=rng)
    if rng is None or rng.dtype != torch.int64 or rng.numel() != 2 or not rng.is_contiguous():
        raise ValueError(f"{what}: rng must hold two contiguous int64 values, seed and offset")
    if not 1 <= len(ps) <= MAX_BRANCHES:
        raise ValueError(f"{what}: 1 to {MAX_BRANCHES} branches")
    if t.dtype not in DTYPES or dtype not in DTYPES:
        raise ValueError(f"{what}: fp16, bf16 or fp32 only")
    if dtype != t.dtype and torch.float32 not in (dtype, t.dtype):
        raise ValueError(f"{what}: types must be equal, or one of them fp32")
    return (ctypes.c_double * len(ps))(*(float(p) for p in ps))


def dropout_forward(x, rng, ps, dtype=None):
    """The dropped-out x of each branch: tuple of tensors of x's shape and `dtype` (default x's),
    branch b with drop probability ps[b], from one read of x. x fp16, bf16 or fp32 [.., W]."""
    dtype = x.dtype if dtype is None else dtype
    p = _common("dropout_forward", x, rng, ps, dtype)
    x2 = _rows(x)
    rows, width = x2.shape
    n = len(ps)
    outs = tuple(torch.empty(x.shape, dtype=dtype, device=x.device) for _ in range(n))
    ptrs = (ctypes.c_void_p * n)(*(o.data_ptr() for o in outs))
    lds = (ctypes.c_int64 * n)(*([width] * n))
    with on_device(x.device):
        check(lib().dk_dropout_fwd(ptr(x2), DTYPES[x.dtype], x2.stride(0), ptr(rng), p, n, ptrs, DTYPES[dtype], lds,
                                   rows, width, stream_of(x.device)))
    return outs


def dropout_backward(grads, rng, ps, dtype=None):
    """dx = sum of the branches' gradients through the masks of dropout_forward(x, rng, ps), summed in
    fp32 and rounded once to `dtype` (default the gradients'). A gradient may be None (zeros)."""
    given = [g for g in grads if g is not None]
    if len(grads) != len(ps) or not given:
        raise ValueError("dropout_backward: one gradient a branch, at least one of them not None")
    g0 = given[0]
    dtype = g0.dtype if dtype is None else dtype
    p = _common("dropout_backward", g0, rng, ps, dtype)
    n = len(ps)
    rows2 = []
    for g in grads:
        if g is not None:
            gpu_tensors("dropout_backward", g0.device, grad=g)
            if g.dtype != g0.dtype or g.shape != g0.shape:
                raise ValueError("dropout_backward: gradients must have one shape and type")
        rows2.append(None if g is None else _rows(g))
    rows, width = next(g for g in rows2 if g is not None).shape
    dx = torch.empty(g0.shape, dtype=dtype, device=g0.device)
    ptrs = (ctypes.c_void_p * n)(*(None if g is None else g.data_ptr() for g in rows2))
    lds = (ctypes.c_int64 * n)(*(0 if g is None else g.stride(0) for g in rows2))
    with on_device(g0.device):
        check(lib().dk_dropout_bwd(ptrs, DTYPES[g0.dtype], lds, ptr(rng), p, n, ptr(dx), DTYPES[dtype], width, rows,
                                   width, stream_of(g0.device)))
    return dx


class SeededDropout(torch.autograd.Function):
    """apply(x, rng, ps, dtype) -> the dropped-out x of each branch (a tuple); the backward forms the
    masks again from rng, which must not change in between (autograd raises if it did)."""

    @staticmethod
    def forward(ctx, x, rng, ps, dtype=None):
        ps = tuple(float(p) for p in ps)
        outs = dropout_forward(x, rng, ps, dtype)
        ctx.save_for_backward(rng)
        ctx.ps, ctx.x_dtype = ps, x.dtype
        ctx.set_materialize_grads(False)
        return outs

    @staticmethod
    def backward(ctx, *grads):
        (rng,) = ctx.saved_tensors
        if all(g is None for g in grads):
            return None, None, None, None
        return dropout_backward(grads, rng, ctx.ps, ctx.x_dtype), None, None, None


def seeded_dropout(x, rng, p, dtype=None):
    """Dropout of x with probability p and the mask of (rng, row, column); differentiable in x."""
    return SeededDropout.apply(x, rng, (p,), dtype)[0]
