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

import struct

import torch
from torch.autograd.function import once_differentiable

from ._lib import DTYPES, call_on, gpu_input, lib, same_gpu

MAX_BRANCHES = 4
# arrays of 1 to 4 host values, as the C entries take them
_DOUBLES = [None] + [struct.Struct(f"{n}d").pack for n in range(1, MAX_BRANCHES + 1)]
_POINTERS = [None] + [struct.Struct(f"{n}P").pack for n in range(1, MAX_BRANCHES + 1)]
_LONGS = [None] + [struct.Struct(f"{n}q").pack for n in range(1, MAX_BRANCHES + 1)]


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
    if t2.stride(1) != 1 and t2.shape[1] != 1 or t2.stride(0) < 0:
        t2 = t2.contiguous()
    return t2


def _common(what, t, rng, ps, dtype):
    """(device, packed probabilities, type codes of t and dtype)."""
    dev = gpu_input(what, t)
    same_gpu(what, dev, rng)
    if t.dim() < 1:
        raise ValueError(f"{what}: needs a last axis")
    if rng is None or rng.dtype != torch.int64 or rng.numel() != 2 or not rng.is_contiguous():
        raise ValueError(f"{what}: rng must hold two contiguous int64 values, seed and offset")
    if not 1 <= len(ps) <= MAX_BRANCHES:
        raise ValueError(f"{what}: 1 to {MAX_BRANCHES} branches")
    a, b = DTYPES.get(t.dtype), DTYPES.get(dtype)
    if a is None or b is None:
        raise ValueError(f"{what}: fp16, bf16 or fp32 only")
    if a != b and a != 2 and b != 2:
        raise ValueError(f"{what}: types must be equal, or one of them fp32")
    return dev, _DOUBLES[len(ps)](*ps), a, b


def dropout_forward(x, rng, ps, dtype=None):
    """The dropped-out x of each branch: tuple of tensors of x's shape and `dtype` (default x's),
    branch b with drop probability ps[b], from one read of x. x fp16, bf16 or fp32 [.., W]."""
    dtype = dtype or getattr(x, "dtype", None)
    dev, p, a, b = _common("dropout_forward", x, rng, ps, dtype)
    x2 = _rows(x)
    rows, width = x2.shape
    n = len(ps)
    outs = tuple([torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format) for _ in ps])
    call_on(dev, lib().dk_dropout_fwd, x2.data_ptr(), a, x2.stride(0), rng.data_ptr(), p, n,
            _POINTERS[n](*[o.data_ptr() for o in outs]), b, _LONGS[n](*[width] * n), rows, width)
    return outs


def dropout_backward(grads, rng, ps, dtype=None):
    """dx = sum of the branches' gradients through the masks of dropout_forward(x, rng, ps), summed in
    fp32 and rounded once to `dtype` (default the gradients'). A gradient may be None (zeros)."""
    what = "dropout_backward"
    g0 = next((g for g in grads if g is not None), None)
    if len(grads) != len(ps) or g0 is None:
        raise ValueError(f"{what}: one gradient a branch, at least one of them not None")
    dev, p, a, b = _common(what, g0, rng, ps, dtype or getattr(g0, "dtype", None))
    dtype = dtype or g0.dtype
    rows2, ptrs, lds = [], [], []
    for g in grads:
        if g is None:
            ptrs.append(0)
            lds.append(0)
            continue
        same_gpu(what, dev, g)
        if g.dtype != g0.dtype or g.shape != g0.shape:
            raise ValueError(f"{what}: gradients must have one shape and type")
        g2 = _rows(g)
        rows2.append(g2)
        ptrs.append(g2.data_ptr())
        lds.append(g2.stride(0))
    rows, width = rows2[0].shape
    n = len(ps)
    dx = torch.empty_like(g0, dtype=dtype, memory_format=torch.contiguous_format)
    call_on(dev, lib().dk_dropout_bwd, _POINTERS[n](*ptrs), a, _LONGS[n](*lds), rng.data_ptr(), p, n, dx.data_ptr(), b,
            width, rows, width)
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
    @once_differentiable
    def backward(ctx, *grads):
        (rng,) = ctx.saved_tensors
        if all(g is None for g in grads):
            return None, None, None, None
        return dropout_backward(grads, rng, ctx.ps, ctx.x_dtype), None, None, None


def seeded_dropout(x, rng, p, dtype=None):
    """Dropout of x with probability p and the mask of (rng, row, column); differentiable in x."""
    return SeededDropout.apply(x, rng, (p,), dtype)[0]
