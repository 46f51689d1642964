"""RoPE of the attention inputs: (q_base + q_lora, k) -> rotated fp16 q, k, head-major.

Mirrors FusedQKRope (solution/attn.py:89-126) and its kernels (solution/attn.py:27-86) with one
HIP launch each way (dk_rope_qk_fwd / dk_rope_qk_bwd):
  forward:  q = fp32(q_base) + fp32(q_lora); q * cos + rotate_half(q) * sin in fp32, stored fp16
            as [1, H, T, D] for SDPA; k the same without LoRA
  backward: dq = g * cos + rotate_half^T(g * sin) in fp32, rounded to fp16 once; the projection
            and the LoRA branch both receive it (as in the base)

Next to it, without a counterpart in the reference (dk_qk_rope_fwd / dk_qk_rope_bwd):
  qk_norm_rope_*  RMS norms of every query and key head (weights [D]) with the rotation in one pass
  axes_rope_*     rotary positions with several axes (time, height, width), the angles formed from
                  integer positions and frequencies, with or without the norms
Both take q and k token-major (strided rows of a packed projection output as they are), fp16 or bf16,
and give them head-major [B, H, T, D]; everything is computed in fp32 and rounded once.
"""

import ctypes

import torch

from . import _lib
from ._lib import DTYPES, check, gpu_tensors, lib, on_device, ptr, stream_of


def _rows(t):
    t2 = t.reshape(-1, t.shape[-1])
    return t2 if t2.stride(-1) == 1 else t2.contiguous()


def rope_qk_forward(q_base, q_lora, k, cos, sin, n_heads, n_kv_heads):
    """(q_out [H, T, D], k_out [HK, T, D]) fp16; q_base/q_lora [T, H*D], k [T, HK*D] fp16;
    cos/sin fp32 [T, D]. q_lora may be None (no addition)."""
    qb, kk = _rows(q_base), _rows(k)
    ql = None if q_lora is None else _rows(q_lora)
    n_tok = qb.shape[0]
    d = cos.shape[-1]
    c = cos.reshape(n_tok, d).to(torch.float32).contiguous()
    s = sin.reshape(n_tok, d).to(torch.float32).contiguous()
    q_out = torch.empty((n_heads, n_tok, d), dtype=torch.float16, device=qb.device)
    k_out = torch.empty((n_kv_heads, n_tok, d), dtype=torch.float16, device=qb.device)
    check(lib().dk_rope_qk_fwd(ptr(qb), ptr(ql), qb.stride(0), 0 if ql is None else ql.stride(0), ptr(kk),
                               kk.stride(0), ptr(c), ptr(s), ptr(q_out), ptr(k_out), n_tok, n_heads,
                               n_kv_heads, d, stream_of(qb.device)))
    return q_out, k_out


def rope_qk_backward(grad_q, grad_k, cos, sin):
    """(dq [T, H*D], dk [T, HK*D]) fp16 from head-major fp16 gradients [H, T, D], [HK, T, D]."""
    gq = grad_q.reshape(-1, grad_q.shape[-2], grad_q.shape[-1]).to(torch.float16).contiguous()
    gk = grad_k.reshape(-1, grad_k.shape[-2], grad_k.shape[-1]).to(torch.float16).contiguous()
    n_heads, n_tok, d = gq.shape
    n_kv = gk.shape[0]
    c = cos.reshape(n_tok, d).to(torch.float32).contiguous()
    s = sin.reshape(n_tok, d).to(torch.float32).contiguous()
    dq = torch.empty((n_tok, n_heads * d), dtype=torch.float16, device=gq.device)
    dk = torch.empty((n_tok, n_kv * d), dtype=torch.float16, device=gq.device)
    check(lib().dk_rope_qk_bwd(ptr(gq), ptr(gk), ptr(c), ptr(s), ptr(dq), dq.stride(0), ptr(dk), dk.stride(0),
                               n_tok, n_heads, n_kv, d, stream_of(gq.device)))
    return dq, dk


class FusedQKRope(torch.autograd.Function):
    """(q_base + q_lora, k) -> RoPE'd fp16 q [1, HQ, T, D] and k [1, HK, T, D]
    (solution/attn.py:89-126)."""

    @staticmethod
    def forward(ctx, q_base, q_lora, k, cos, sin, n_heads, n_kv_heads):
        q_out, k_out = rope_qk_forward(q_base, q_lora, k, cos, sin, n_heads, n_kv_heads)
        ctx.save_for_backward(cos, sin)
        return q_out.unsqueeze(0), k_out.unsqueeze(0)

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        cos, sin = ctx.saved_tensors
        dq, dk = rope_qk_backward(grad_q, grad_k, cos, sin)
        # q_lora may be absent (None) when the LoRA term is already in q_base
        return dq, dq.clone() if ctx.needs_input_grad[1] else None, dk, None, None, None, None


def _token_rows(what, name, t, heads, d):
    """(tensor whose [B * T] rows have one stride, that stride, B, T) of a [B, T, H * D] or [T, H * D] tensor."""
    if t.dim() not in (2, 3) or t.shape[-1] != heads * d:
        raise ValueError(f"{what}: {name} must be [B, T, {heads * d}] or [T, {heads * d}], not {tuple(t.shape)}")
    b, n = (1, t.shape[0]) if t.dim() == 2 else t.shape[:2]
    row = t.stride(-2)
    if t.stride(-1) != 1 or (n > 1 and row < heads * d) or (b > 1 and t.stride(0) != n * row):
        t = t.contiguous()
        row = t.stride(-2)
    elif n == 1 and b > 1:
        row = t.stride(0)  # one token a sequence: the rows are the batch entries
        if row < heads * d:
            t = t.contiguous()
            row = heads * d
    return t, row, b, n


def _rotation(what, desc, device, batch, tokens, d, cos=None, sin=None, positions=None, inv_freq=None, sections=None,
              interleaved=False):
    """Fill the rotation fields of `desc`; returns the tensors to keep alive."""
    if cos is not None:
        gpu_tensors(what, device, cos=cos, sin=sin)
        keep = []
        for t in (cos, sin):
            if t.shape != cos.shape or tuple(t.shape) not in ((tokens, d), (1, tokens, d), (batch, tokens, d)):
                raise ValueError(f"{what}: cos and sin must be [T, D] or [B, T, D] of T = {tokens}, D = {d}")
            keep.append(t.to(torch.float32).contiguous())
        desc.cos, desc.sin = keep[0].data_ptr(), keep[1].data_ptr()
        desc.table_batch_stride = tokens * d if cos.dim() == 3 and cos.shape[0] > 1 else 0
        return keep
    gpu_tensors(what, device, positions=positions, inv_freq=inv_freq)
    sections = [int(s) for s in sections]
    n = len(sections)
    if not 1 <= n <= 4:
        raise ValueError(f"{what}: 1 to 4 axes")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: positions must be int32 or int64")
    if tuple(positions.shape) not in ((n, tokens), (n, 1, tokens), (n, batch, tokens)):
        raise ValueError(f"{what}: positions must be [{n}, T] or [{n}, B, T] of T = {tokens}, B = {batch}, not "
                         f"{tuple(positions.shape)}")
    if inv_freq.dim() != 1 or inv_freq.numel() != d // 2:
        raise ValueError(f"{what}: inv_freq must hold {d // 2} frequencies")
    if positions.stride(-1) != 1 and tokens > 1:
        positions = positions.contiguous()
    inv = inv_freq.to(torch.float32).contiguous()
    desc.positions, desc.inv_freq = positions.data_ptr(), inv.data_ptr()
    desc.positions_int64 = int(positions.dtype == torch.int64)
    desc.pos_axis_stride = positions.stride(0)
    desc.pos_batch_stride = positions.stride(1) if positions.dim() == 3 and positions.shape[1] > 1 else 0
    desc.n_axes, desc.interleaved = n, int(bool(interleaved))
    for i, s in enumerate(sections):
        desc.sections[i] = s
    return [positions, inv]


def _norm_weights(what, desc, device, d, q_weight, k_weight):
    if (q_weight is None) != (k_weight is None):
        raise ValueError(f"{what}: norm weights for both q and k, or for neither")
    if q_weight is None:
        return []
    gpu_tensors(what, device, q_weight=q_weight, k_weight=k_weight)
    if tuple(q_weight.shape) != (d,) or tuple(k_weight.shape) != (d,):
        raise ValueError(f"{what}: norm weights must be [{d}]")
    if q_weight.dtype not in DTYPES or k_weight.dtype != q_weight.dtype:
        raise ValueError(f"{what}: norm weights must share one type, fp16, bf16 or fp32")
    keep = [q_weight.contiguous(), k_weight.contiguous()]
    desc.q_weight, desc.k_weight, desc.w_dtype = keep[0].data_ptr(), keep[1].data_ptr(), DTYPES[q_weight.dtype]
    return keep


def _qk_forward(what, q, k, q_weight, k_weight, n_heads, n_kv_heads, eps, d, **rotation):
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise ValueError(f"{what}: needs GPU tensors")
    dev = q.device
    gpu_tensors(what, dev, k=k)
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype:
        raise ValueError(f"{what}: q and k must both be fp16 or both bf16")
    desc = _lib.QkRope()
    q, desc.ld_q, b, t = _token_rows(what, "q", q, n_heads, d)
    k, desc.ld_k, bk, tk = _token_rows(what, "k", k, n_kv_heads, d)
    if (bk, tk) != (b, t):
        raise ValueError(f"{what}: q and k must have the same tokens")
    keep = _norm_weights(what, desc, dev, d, q_weight, k_weight)
    keep += _rotation(what, desc, dev, b, t, d, **rotation)
    q_out = torch.empty((b, n_heads, t, d), dtype=q.dtype, device=dev)
    k_out = torch.empty((b, n_kv_heads, t, d), dtype=q.dtype, device=dev)
    desc.q, desc.k, desc.q_out, desc.k_out = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
    desc.batch, desc.tokens, desc.n_heads, desc.n_kv_heads, desc.head_dim = b, t, n_heads, n_kv_heads, d
    desc.dtype, desc.eps = DTYPES[q.dtype], eps
    with on_device(dev):
        check(lib().dk_qk_rope_fwd(ctypes.byref(desc), stream_of(dev)))
    return q_out, k_out


def _qk_backward(what, grad_q, grad_k, q, k, q_weight, k_weight, eps, weight_grads, **rotation):
    if not isinstance(grad_q, torch.Tensor) or not grad_q.is_cuda:
        raise ValueError(f"{what}: needs GPU tensors")
    dev = grad_q.device
    gpu_tensors(what, dev, grad_k=grad_k, q=q, k=k)
    if grad_q.dim() != 4 or grad_k.dim() != 4 or grad_q.shape[0] != grad_k.shape[0] or \
            grad_q.shape[2:] != grad_k.shape[2:]:
        raise ValueError(f"{what}: gradients must be [B, H, T, D] of the same B, T and D")
    if grad_q.dtype not in (torch.float16, torch.bfloat16) or grad_k.dtype != grad_q.dtype:
        raise ValueError(f"{what}: gradients must both be fp16 or both bf16")
    b, hq, t, d = grad_q.shape
    hk = grad_k.shape[1]
    desc = _lib.QkRope()
    gq, gk = grad_q.contiguous(), grad_k.contiguous()
    keep = _norm_weights(what, desc, dev, d, q_weight, k_weight) + [gq, gk]
    keep += _rotation(what, desc, dev, b, t, d, **rotation)
    dwq = dwk = None
    if q_weight is not None:
        if q is None or k is None or q.dtype != grad_q.dtype or k.dtype != grad_q.dtype:
            raise ValueError(f"{what}: norms need q and k again, of the gradients' type")
        q, desc.ld_q, bq, tq = _token_rows(what, "q", q, hq, d)
        k, desc.ld_k, bk, tk = _token_rows(what, "k", k, hk, d)
        if (bq, tq) != (b, t) or (bk, tk) != (b, t):
            raise ValueError(f"{what}: q, k and their gradients must have the same tokens")
        desc.q, desc.k = q.data_ptr(), k.data_ptr()
        keep += [q, k]
        if weight_grads:
            dwq, dwk = torch.empty((2, d), dtype=torch.float32, device=dev).unbind()
            desc.dw_q, desc.dw_k = dwq.data_ptr(), dwk.data_ptr()
    dq = torch.empty((b, t, hq * d), dtype=gq.dtype, device=dev)
    dk = torch.empty((b, t, hk * d), dtype=gq.dtype, device=dev)
    desc.grad_q, desc.grad_k, desc.q_out, desc.k_out = gq.data_ptr(), gk.data_ptr(), dq.data_ptr(), dk.data_ptr()
    desc.ld_q_out, desc.ld_k_out = hq * d, hk * d
    desc.batch, desc.tokens, desc.n_heads, desc.n_kv_heads, desc.head_dim = b, t, hq, hk, d
    desc.dtype, desc.eps = DTYPES[gq.dtype], eps
    with on_device(dev):
        need = lib().dk_qk_rope_bwd_workspace(ctypes.byref(desc))
        # a tensor of its own a call: graphs and streams share none
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
        check(lib().dk_qk_rope_bwd(ctypes.byref(desc), ptr(ws), max(need, 0), stream_of(dev)))
    return dq, dk, dwq, dwk


def qk_norm_rope_forward(q, k, q_weight, k_weight, cos, sin, n_heads, n_kv_heads, eps=1e-6):
    """(q_out [B, H, T, D], k_out [B, HK, T, D]): each head's RMS norm times its weight, rotated.
    q [B, T, H*D] or [T, H*D], k likewise, fp16 or bf16; q_weight, k_weight [D]; cos, sin [T, D] or
    [B, T, D]."""
    return _qk_forward("qk_norm_rope_forward", q, k, q_weight, k_weight, n_heads, n_kv_heads, eps, cos.shape[-1],
                       cos=cos, sin=sin)


def qk_norm_rope_backward(grad_q, grad_k, q, k, q_weight, k_weight, cos, sin, eps=1e-6, weight_grads=True):
    """(dq [B, T, H*D], dk [B, T, HK*D], dq_weight, dk_weight fp32 [D], None without weight_grads) of
    qk_norm_rope_forward, from head-major gradients of its outputs and the same q and k."""
    return _qk_backward("qk_norm_rope_backward", grad_q, grad_k, q, k, q_weight, k_weight, eps, weight_grads,
                        cos=cos, sin=sin)


def axes_rope_forward(q, k, positions, inv_freq, sections, n_heads, n_kv_heads, interleaved=False, q_weight=None,
                      k_weight=None, eps=1e-6):
    """(q_out, k_out) head-major, rotated by positions with several axes: positions int32 or int64
    [axes, T] or [axes, B, T]; inv_freq [D / 2] (radians a position); sections: how many of the
    frequencies each axis takes, in order of the frequencies, or interleaved (frequency j belongs to
    axis j % axes while that axis has some left, the others to axis 0). With q_weight and k_weight the
    heads are RMS-normalized first. The angles are exact to 2^-24 turns for positions below 2^28."""
    return _qk_forward("axes_rope_forward", q, k, q_weight, k_weight, n_heads, n_kv_heads, eps,
                       2 * inv_freq.shape[-1], positions=positions, inv_freq=inv_freq, sections=sections,
                       interleaved=interleaved)


def axes_rope_backward(grad_q, grad_k, positions, inv_freq, sections, interleaved=False, q=None, k=None, q_weight=None,
                       k_weight=None, eps=1e-6, weight_grads=True):
    """(dq, dk, dq_weight, dk_weight) of axes_rope_forward; q and k again where it had norms (the
    weights' gradients are None where it had none, or without weight_grads)."""
    return _qk_backward("axes_rope_backward", grad_q, grad_k, q, k, q_weight, k_weight, eps, weight_grads,
                        positions=positions, inv_freq=inv_freq, sections=sections, interleaved=interleaved)


def _head_major_grads(ctx, grads, b, t, d):
    """Gradients of q_out and k_out, zeros for one that none reached."""
    return [torch.zeros((b, h, t, d), dtype=ctx.qk_dtype, device=ctx.device) if g is None else g
            for g, h in zip(grads, ctx.heads)]


class _QkRotation(torch.autograd.Function):
    """apply(q, k, q_weight, k_weight, heads, eps, rotation, *rotation tensors); rotation = ("tables",)
    with cos, sin or ("axes", sections, interleaved) with positions, inv_freq."""

    @staticmethod
    def _named(rotation, tensors):
        if rotation[0] == "tables":
            return dict(cos=tensors[0], sin=tensors[1])
        return dict(positions=tensors[0], inv_freq=tensors[1], sections=rotation[1], interleaved=rotation[2])

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, heads, eps, rotation, *tensors):
        d = tensors[0].shape[-1] if rotation[0] == "tables" else 2 * tensors[1].shape[-1]
        outs = _qk_forward("qk rotation", q, k, q_weight, k_weight, *heads, eps, d,
                           **_QkRotation._named(rotation, tensors))
        norm = q_weight is not None
        ctx.save_for_backward(*((q, k, q_weight, k_weight) if norm else ()), *tensors)
        ctx.norm, ctx.eps, ctx.rotation, ctx.heads = norm, eps, rotation, heads
        ctx.shapes, ctx.qk_dtype, ctx.device, ctx.outs = (q.shape, k.shape), q.dtype, q.device, outs[0].shape
        ctx.set_materialize_grads(False)
        return outs

    @staticmethod
    def backward(ctx, *grads):
        if all(g is None for g in grads):
            return (None,) * 9
        saved = ctx.saved_tensors
        q, k, qw, kw = saved[:4] if ctx.norm else (None,) * 4
        tensors = saved[4:] if ctx.norm else saved
        b, _, t, d = ctx.outs
        gq, gk = _head_major_grads(ctx, grads, b, t, d)
        want = ctx.norm and (ctx.needs_input_grad[2] or ctx.needs_input_grad[3])
        dq, dk, dqw, dkw = _qk_backward("qk rotation", gq, gk, q, k, qw, kw, ctx.eps, want,
                                        **_QkRotation._named(ctx.rotation, tensors))
        if want:
            dqw, dkw = dqw.to(qw.dtype), dkw.to(kw.dtype)
        return (dq.reshape(ctx.shapes[0]), dk.reshape(ctx.shapes[1]), dqw, dkw, None, None, None, None, None)


def qk_norm_rope(q, k, q_weight, k_weight, cos, sin, n_heads, n_kv_heads, eps=1e-6):
    """qk_norm_rope_forward, differentiable in q, k and the norm weights."""
    return _QkRotation.apply(q, k, q_weight, k_weight, (n_heads, n_kv_heads), eps, ("tables",), cos, sin)


def axes_rope(q, k, positions, inv_freq, sections, n_heads, n_kv_heads, interleaved=False, q_weight=None, k_weight=None,
              eps=1e-6):
    """axes_rope_forward, differentiable in q, k and the norm weights."""
    return _QkRotation.apply(q, k, q_weight, k_weight, (n_heads, n_kv_heads), eps,
                             ("axes", tuple(int(s) for s in sections), bool(interleaved)), positions, inv_freq)
