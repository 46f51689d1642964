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
  scaled_rope_*   rotary positions of the first part of each head, in halves or in pairs, from positions and
                  frequencies (scaled_frequencies: stretched for long contexts), any strides (dk_scaled_rope_*)
All take q and k token-major (strided rows of a packed projection output as they are), fp16 or bf16,
and give them head-major [B, H, T, D]; everything is computed in fp32 and rounded once.
"""

import math

import torch
from torch.autograd.function import once_differentiable

from ._lib import DTYPES, QkRope, ScaledRope, call_on, check, gpu_input, lib, ptr, same_gpu, stream_of


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


_QK_TYPES = {torch.float16: 0, torch.bfloat16: 1}


def _token_rows(what, t, heads, d):
    """(tensor whose [B * T] rows have one stride, that stride, B, T) of a [B, T, H * D] or [T, H * D] tensor."""
    shape, width = t.shape, heads * d
    if len(shape) not in (2, 3) or shape[-1] != width:
        raise ValueError(f"{what}: q and k must be [B, T, H * D] or [T, H * D], here H * D = {width}, not {tuple(shape)}")
    b, n = (1, shape[0]) if len(shape) == 2 else shape[:2]
    row = t.stride(-2)
    if n == 1 and b > 1:
        row = t.stride(0)  # one token a sequence: the rows are the batch entries
    elif b > 1 and t.stride(0) != n * row:
        row = -1
    if t.stride(-1) != 1 or (b * n > 1 and row < width):
        t, row = t.contiguous(), width
    return t, row, b, n


def _fp32(t):
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.to(torch.float32).contiguous()


def _rotation(what, dev, batch, tokens, d, tables, axes):
    """(cos, sin, positions, inv_freq pointers, strides of tables, axes and batches, axis count, sections,
    interleaved, int64 positions, the tensors behind the pointers) of a descriptor."""
    if tables is not None:
        cos, sin = tables
        same_gpu(what, dev, cos, sin)
        if cos.shape != sin.shape or cos.shape not in ((tokens, d), (batch, tokens, d), (1, tokens, d)):
            raise ValueError(f"{what}: cos and sin must be [T, D] or [B, T, D] of T = {tokens}, D = {d}")
        cos, sin = _fp32(cos), _fp32(sin)
        own = tokens * d if cos.dim() == 3 and cos.shape[0] > 1 else 0
        return cos.data_ptr(), sin.data_ptr(), 0, 0, own, 0, 0, 0, (0, 0, 0, 0), 0, 0, (cos, sin)
    positions, inv_freq, sections, interleaved = axes
    same_gpu(what, dev, positions, inv_freq)
    sections = tuple(int(s) for s in sections)
    n = len(sections)
    if not 1 <= n <= 4:
        raise ValueError(f"{what}: 1 to 4 axes")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: positions must be int32 or int64")
    if positions.shape not in ((n, tokens), (n, batch, tokens), (n, 1, tokens)):
        raise ValueError(f"{what}: positions must be [{n}, T] or [{n}, B, T] of T = {tokens}, B = {batch}, not "
                         f"{tuple(positions.shape)}")
    if inv_freq.shape != (d // 2,):
        raise ValueError(f"{what}: inv_freq must hold {d // 2} frequencies")
    if positions.stride(-1) != 1 and tokens > 1:
        positions = positions.contiguous()
    inv_freq = _fp32(inv_freq)
    per_batch = positions.stride(1) if positions.dim() == 3 and positions.shape[1] > 1 else 0
    return (0, 0, positions.data_ptr(), inv_freq.data_ptr(), 0, positions.stride(0), per_batch, n,
            sections + (0,) * (4 - n), int(bool(interleaved)), int(positions.dtype == torch.int64),
            (positions, inv_freq))


def _norm_weights(what, dev, d, q_weight, k_weight):
    """(weights, their type code), contiguous; (None, None, 0) without norms."""
    if (q_weight is None) != (k_weight is None):
        raise ValueError(f"{what}: norm weights for both q and k, or for neither")
    if q_weight is None:
        return None, None, 0
    same_gpu(what, dev, q_weight, k_weight)
    code = DTYPES.get(q_weight.dtype)
    if q_weight.shape != (d,) or k_weight.shape != (d,) or code is None or k_weight.dtype != q_weight.dtype:
        raise ValueError(f"{what}: norm weights must both be [{d}], of one type, fp16, bf16 or fp32")
    return q_weight.contiguous(), k_weight.contiguous(), code


def _descriptor(at, dw_q, dw_k, weights, rot, lds, b, t, hq, hk, d, code, eps):
    """dk_qk_rope as packed bytes, its fields in order (at: pointers of q, k, their gradients and outputs)."""
    qw, kw, w_code = weights
    cos, sin, pos, inv, table_batch, pos_axis, pos_batch, n_axes, sections, interleaved, pos64, _ = rot
    return QkRope.PACK.pack(*at, 0 if qw is None else qw.data_ptr(), 0 if kw is None else kw.data_ptr(), dw_q, dw_k,
                            cos, sin, pos, inv, *lds, table_batch, pos_axis, pos_batch, b, t, hq, hk, d, code, w_code,
                            n_axes, *sections, interleaved, pos64, eps, 0)


def _qk_forward(what, q, k, q_weight, k_weight, hq, hk, eps, d, tables=None, axes=None):
    dev = gpu_input(what, q)
    same_gpu(what, dev, k)
    code = _QK_TYPES.get(q.dtype)
    if code is None or k.dtype != q.dtype:
        raise ValueError(f"{what}: q and k must both be fp16 or both bf16")
    q, ldq, b, t = _token_rows(what, q, hq, d)
    k, ldk, bk, tk = _token_rows(what, k, hk, d)
    if bk != b or tk != t:
        raise ValueError(f"{what}: q and k must have the same tokens")
    weights = _norm_weights(what, dev, d, q_weight, k_weight)
    rot = _rotation(what, dev, b, t, d, tables, axes)
    q_out, k_out = q.new_empty(b, hq, t, d), q.new_empty(b, hk, t, d)
    at = q.data_ptr(), k.data_ptr(), 0, 0, q_out.data_ptr(), k_out.data_ptr()
    call_on(dev, lib().dk_qk_rope_fwd,
            _descriptor(at, 0, 0, weights, rot, (ldq, ldk, 0, 0), b, t, hq, hk, d, code, eps))
    return q_out, k_out


def _qk_backward(what, grad_q, grad_k, q, k, q_weight, k_weight, eps, weight_grads, tables=None, axes=None):
    dev = gpu_input(what, grad_q)
    same_gpu(what, dev, grad_k, q, k)
    if grad_q.dim() != 4 or grad_k.dim() != 4 or grad_q.shape[0] != grad_k.shape[0] or \
            grad_q.shape[2:] != grad_k.shape[2:]:
        raise ValueError(f"{what}: gradients must be [B, H, T, D] of the same B, T and D")
    code = _QK_TYPES.get(grad_q.dtype)
    if code is None or grad_k.dtype != grad_q.dtype:
        raise ValueError(f"{what}: gradients must both be fp16 or both bf16")
    b, hq, t, d = grad_q.shape
    hk = grad_k.shape[1]
    gq, gk = grad_q.contiguous(), grad_k.contiguous()
    weights = _norm_weights(what, dev, d, q_weight, k_weight)
    rot = _rotation(what, dev, b, t, d, tables, axes)
    ldq = ldk = need = 0
    dws, work = (None, None), None
    if q_weight is None:
        q = k = None
    else:
        if q is None or k is None or q.dtype != gq.dtype or k.dtype != gq.dtype:
            raise ValueError(f"{what}: norms need q and k again, of the gradients' type")
        q, ldq, bq, tq = _token_rows(what, q, hq, d)
        k, ldk, bk, tk = _token_rows(what, k, hk, d)
        if (bq, tq) != (b, t) or (bk, tk) != (b, t):
            raise ValueError(f"{what}: q, k and their gradients must have the same tokens")
        if weight_grads:
            dws = gq.new_empty(2, d, dtype=torch.float32).unbind()
    dq, dk = gq.new_empty(b, t, hq * d), gq.new_empty(b, t, hk * d)
    at = (0 if q is None else q.data_ptr(), 0 if k is None else k.data_ptr(), gq.data_ptr(), gk.data_ptr(),
          dq.data_ptr(), dk.data_ptr())
    dwq, dwk = (0, 0) if dws[0] is None else (dws[0].data_ptr(), dws[1].data_ptr())
    desc = _descriptor(at, dwq, dwk, weights, rot, (ldq, ldk, hq * d, hk * d), b, t, hq, hk, d, code, eps)
    if dwq:
        need = lib().dk_qk_rope_bwd_workspace(desc)
        # a tensor of its own a call: graphs and streams share none
        work = gq.new_empty(need, dtype=torch.uint8) if need > 0 else None
    call_on(dev, lib().dk_qk_rope_bwd, desc, None if work is None else work.data_ptr(), max(need, 0))
    return dq, dk, *dws


def qk_norm_rope_forward(q, k, q_weight, k_weight, cos, sin, n_heads, n_kv_heads, eps=1e-6):
    """(q_out [B, H, T, D], k_out [B, HK, T, D]): each head's RMS norm times its weight, rotated.
    q [B, T, H*D] or [T, H*D], k likewise, fp16 or bf16; q_weight, k_weight [D]; cos, sin [T, D] or
    [B, T, D]."""
    return _qk_forward("qk_norm_rope_forward", q, k, q_weight, k_weight, n_heads, n_kv_heads, eps, cos.shape[-1],
                       tables=(cos, sin))


def qk_norm_rope_backward(grad_q, grad_k, q, k, q_weight, k_weight, cos, sin, eps=1e-6, weight_grads=True):
    """(dq [B, T, H*D], dk [B, T, HK*D], dq_weight, dk_weight fp32 [D], None without weight_grads) of
    qk_norm_rope_forward, from head-major gradients of its outputs and the same q and k."""
    return _qk_backward("qk_norm_rope_backward", grad_q, grad_k, q, k, q_weight, k_weight, eps, weight_grads,
                        tables=(cos, sin))


def axes_rope_forward(q, k, positions, inv_freq, sections, n_heads, n_kv_heads, interleaved=False, q_weight=None,
                      k_weight=None, eps=1e-6):
    """(q_out, k_out) head-major, rotated by positions with several axes: positions int32 or int64
    [axes, T] or [axes, B, T]; inv_freq [D / 2] (radians a position); sections: how many of the
    frequencies each axis takes, in order of the frequencies, or interleaved (frequency j belongs to
    axis j % axes while that axis has some left, the others to axis 0). With q_weight and k_weight the
    heads are RMS-normalized first. The angles are exact to 2^-24 turns for positions below 2^28
    and frequencies up to 2 pi."""
    return _qk_forward("axes_rope_forward", q, k, q_weight, k_weight, n_heads, n_kv_heads, eps,
                       2 * inv_freq.shape[-1], axes=(positions, inv_freq, sections, interleaved))


def axes_rope_backward(grad_q, grad_k, positions, inv_freq, sections, interleaved=False, q=None, k=None, q_weight=None,
                       k_weight=None, eps=1e-6, weight_grads=True):
    """(dq, dk, dq_weight, dk_weight) of axes_rope_forward; q and k again where it had norms (the
    weights' gradients are None where it had none, or without weight_grads)."""
    return _qk_backward("axes_rope_backward", grad_q, grad_k, q, k, q_weight, k_weight, eps, weight_grads,
                        axes=(positions, inv_freq, sections, interleaved))


def _head_major_grads(ctx, grads, b, t, d):
    """Gradients of q_out and k_out, zeros for one that none reached."""
    return [torch.zeros((b, h, t, d), dtype=ctx.qk_dtype, device=ctx.device) if g is None else g
            for g, h in zip(grads, ctx.heads)]


class _QkRotation(torch.autograd.Function):
    """apply(q, k, q_weight, k_weight, heads, eps, rotation, *rotation tensors); rotation = ("tables",)
    with cos, sin or ("axes", sections, interleaved) with positions, inv_freq."""

    @staticmethod
    def _named(rotation, tensors):
        return dict(tables=tensors) if rotation[0] == "tables" else dict(axes=(*tensors, *rotation[1:]))

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, heads, eps, rotation, *tensors):
        if any(ctx.needs_input_grad[7:]):
            raise ValueError("qk rotation: tables and frequencies take no gradient (detach them)")
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
    @once_differentiable
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


LAYOUTS = ("half", "pairs")
# kinds of scaled_frequencies and the keys that each uses
_SCALINGS = {"default": (), "linear": ("factor",), "ntk": ("factor",), "dynamic": ("factor",),
             "yarn": ("factor", "beta_fast", "beta_slow", "attention_factor"),
             "llama3": ("factor", "low_freq_factor", "high_freq_factor"),
             "longrope": ("factor", "short_factor", "long_factor", "attention_factor")}


def scaled_frequencies(rotary_dim, base=10000.0, scaling=None, length=None, device=None):
    """(inv_freq fp32 [rotary_dim / 2] in radians a position, the factor of cos and sin) of a rotation of rotary_dim
    elements, for a context stretched as a model's configuration says. scaling: None or a dict with "rope_type" (or
    "type") and
      default  nothing more
      linear   factor: every frequency over factor
      ntk      factor: base times factor^(R / (R - 2)), which stretches the slowest frequency by factor
      dynamic  factor, original_max_position_embeddings: as ntk for the `length` of the call, where that is longer
      yarn     factor, original_max_position_embeddings; beta_fast 32, beta_slow 1, attention_factor 0.1 ln factor + 1:
               frequencies of more than beta_fast turns in the original length are kept, those of fewer than beta_slow are
               divided by factor, a ramp over their index between
      llama3   factor, low_freq_factor, high_freq_factor, original_max_position_embeddings: the same with a ramp over
               the number of turns
      longrope short_factor, long_factor (a divisor a frequency; the second where `length` is longer than the original),
               original_max_position_embeddings, and factor or attention_factor (sqrt(1 + ln factor / ln original))
    Computed in 64 bits and rounded once. A key that its kind does not use is refused: it would change the result
    elsewhere (original_max_position_embeddings and None values may always be there)."""
    what = "scaled_frequencies"
    r = int(rotary_dim)
    if r < 2 or r % 2:
        raise ValueError(f"{what}: rotary_dim must be even and positive")
    s = dict(scaling or {})
    kind = s.get("rope_type", s.get("type", "default"))
    if kind not in _SCALINGS:
        raise ValueError(f"{what}: unknown kind of scaling {kind!r}")
    unused = sorted(key for key in s if s[key] is not None
                    and key not in ("rope_type", "type", "original_max_position_embeddings") + _SCALINGS[kind])
    if unused:
        raise ValueError(f"{what}: {kind} does not use {', '.join(unused)}")

    def given(name):
        if s.get(name) is None:
            raise ValueError(f"{what}: {kind} needs {name}")
        return s[name]

    i = torch.arange(r // 2, dtype=torch.float64)
    stretch = lambda by: base if r == 2 else base * by ** (r / (r - 2))  # noqa: E731
    inv, attention = float(base) ** (-2.0 * i / r), 1.0
    if kind == "linear":
        inv = inv / given("factor")
    elif kind == "ntk":
        inv = stretch(given("factor")) ** (-2.0 * i / r)
    elif kind == "dynamic":
        factor, original = given("factor"), given("original_max_position_embeddings")
        if length is not None and length > original:
            inv = stretch(factor * length / original - (factor - 1)) ** (-2.0 * i / r)
    elif kind == "yarn":
        factor, original = given("factor"), given("original_max_position_embeddings")
        fast, slow = s.get("beta_fast") or 32.0, s.get("beta_slow") or 1.0
        # the index whose frequency makes n turns in the original length
        index = lambda n: r * math.log(original / (n * 2.0 * math.pi)) / (2.0 * math.log(base))  # noqa: E731
        low, high = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), r - 1)
        slowed = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        inv = inv * (1.0 - slowed) + inv / factor * slowed
        attention = s.get("attention_factor")
        if attention is None:
            attention = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    elif kind == "llama3":
        factor, low, high = given("factor"), given("low_freq_factor"), given("high_freq_factor")
        turns = given("original_max_position_embeddings") * inv / (2.0 * math.pi)
        kept = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        inv = inv * kept + inv / factor * (1.0 - kept)
    elif kind == "longrope":
        original = given("original_max_position_embeddings")
        by = given("long_factor" if length is not None and length > original else "short_factor")
        if len(by) != r // 2:
            raise ValueError(f"{what}: longrope needs {r // 2} divisors")
        inv = inv / torch.tensor(by, dtype=torch.float64)
        attention = s.get("attention_factor")
        if attention is None:
            factor = given("factor")
            attention = math.sqrt(1.0 + math.log(factor) / math.log(original)) if factor > 1.0 else 1.0
    return inv.to(torch.float32).to(device), float(attention)


def _scaled_rope(what, entry, q, k, batch, tokens, heads, d, q_strides, k_strides, positions, inv_freq, layout, factor,
                 shapes):
    dev = q.device
    same_gpu(what, dev, positions, inv_freq)
    code = _QK_TYPES.get(q.dtype)
    if code is None or k.dtype != q.dtype:
        raise ValueError(f"{what}: q and k must both be fp16 or both bf16")
    if layout not in LAYOUTS:
        raise ValueError(f"{what}: layout must be one of {LAYOUTS}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what}: positions must be int32 or int64")
    if positions.shape not in ((tokens,), (batch, tokens), (1, tokens)):
        raise ValueError(f"{what}: positions must be [T] or [B, T] of T = {tokens}, B = {batch}, not {tuple(positions.shape)}")
    if inv_freq.dim() != 1 or 2 * inv_freq.shape[0] > d:
        raise ValueError(f"{what}: inv_freq must hold at most D / 2 = {d // 2} frequencies")
    if tokens > 1 and positions.stride(-1) != 1:
        positions = positions.contiguous()
    inv_freq = _fp32(inv_freq)
    pos_batch = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
    outs = q.new_empty(shapes[0]), q.new_empty(shapes[1])
    call_on(dev, entry, ScaledRope.PACK.pack(q.data_ptr(), k.data_ptr(), outs[0].data_ptr(), outs[1].data_ptr(),
                                             positions.data_ptr(), inv_freq.data_ptr(), *q_strides, *k_strides, pos_batch,
                                             batch, tokens, *heads, d, 2 * inv_freq.shape[0], code, layout == "pairs",
                                             positions.dtype == torch.int64, factor))
    return outs


def _token_major(what, t, heads):
    """(t, B, T, D, strides of batch, token and head) of a [B, T, H * D] or [T, H * D] tensor."""
    shape = t.shape
    if len(shape) not in (2, 3) or heads < 1 or shape[-1] % heads or shape[-1] == 0:
        raise ValueError(f"{what}: q and k must be [B, T, H * D] or [T, H * D], here H = {heads}, not {tuple(shape)}")
    strides = t.stride()
    if strides[-1] != 1 and shape[-1] > 1:
        t = t.contiguous()
        strides = t.stride()
    d = shape[-1] // heads
    if len(shape) == 2:
        return t, 1, shape[0], d, (0, strides[0], d)
    return t, shape[0], shape[1], d, (strides[0], strides[1], d)


def scaled_rope_forward(q, k, positions, inv_freq, n_heads, n_kv_heads, layout="half", factor=1.0):
    """(q_out [B, H, T, D], k_out [B, HK, T, D]): the first 2 len(inv_freq) elements of every head turned by positions
    ([T] or [B, T], int32 or int64) times inv_freq (radians a position), cos and sin times factor; the others as they
    are. layout "half": element j turns with j + len(inv_freq), "pairs": 2 j with 2 j + 1. q [B, T, H*D] or [T, H*D]
    (any strides of the first axes), k likewise, fp16 or bf16. The angles are exact to 2^-24 turns for positions below
    2^28 and frequencies up to 2 pi."""
    what = "scaled_rope_forward"
    gpu_input(what, q)
    same_gpu(what, q.device, k)
    q, b, t, d, q_strides = _token_major(what, q, n_heads)
    k, bk, tk, dk, k_strides = _token_major(what, k, n_kv_heads)
    if (bk, tk, dk) != (b, t, d):
        raise ValueError(f"{what}: q and k must have the same tokens and head size")
    return _scaled_rope(what, lib().dk_scaled_rope_fwd, q, k, b, t, (n_heads, n_kv_heads), d, q_strides, k_strides,
                        positions, inv_freq, layout, factor, ((b, n_heads, t, d), (b, n_kv_heads, t, d)))


def scaled_rope_backward(grad_q, grad_k, positions, inv_freq, layout="half", factor=1.0):
    """(dq [B, T, H*D], dk [B, T, HK*D]) of scaled_rope_forward from gradients [B, H, T, D] of its outputs."""
    what = "scaled_rope_backward"
    gpu_input(what, grad_q)
    same_gpu(what, grad_q.device, grad_k)
    if grad_q.dim() != 4 or grad_k.dim() != 4 or grad_q.shape[0] != grad_k.shape[0] or \
            grad_q.shape[2:] != grad_k.shape[2:]:
        raise ValueError(f"{what}: gradients must be [B, H, T, D] of the same B, T and D")
    b, hq, t, d = grad_q.shape
    hk = grad_k.shape[1]
    grads = [g if d <= 1 or g.stride(3) == 1 else g.contiguous() for g in (grad_q, grad_k)]
    strides = [(g.stride(0), g.stride(2), g.stride(1)) for g in grads]
    return _scaled_rope(what, lib().dk_scaled_rope_bwd, *grads, b, t, (hq, hk), d, *strides, positions, inv_freq, layout,
                        factor, ((b, t, hq * d), (b, t, hk * d)))


class _ScaledRope(torch.autograd.Function):
    """apply(q, k, positions, inv_freq, heads, layout, factor) -> (q_out, k_out)."""

    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, heads, layout, factor):
        if ctx.needs_input_grad[3]:
            raise ValueError("scaled_rope: frequencies take no gradient (detach them)")
        outs = scaled_rope_forward(q, k, positions, inv_freq, *heads, layout, factor)
        ctx.save_for_backward(positions, inv_freq)
        ctx.heads, ctx.layout, ctx.factor, ctx.shapes, ctx.outs = heads, layout, factor, (q.shape, k.shape), outs[0].shape
        ctx.qk_dtype, ctx.device = q.dtype, q.device
        ctx.set_materialize_grads(False)
        return outs

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        if all(g is None for g in grads):
            return (None,) * 7
        b, _, t, d = ctx.outs
        gq, gk = _head_major_grads(ctx, grads, b, t, d)
        dq, dk = scaled_rope_backward(gq, gk, *ctx.saved_tensors, ctx.layout, ctx.factor)
        return dq.reshape(ctx.shapes[0]), dk.reshape(ctx.shapes[1]), None, None, None, None, None


def scaled_rope(q, k, positions, inv_freq, n_heads, n_kv_heads, layout="half", factor=1.0):
    """scaled_rope_forward, differentiable in q and k."""
    return _ScaledRope.apply(q, k, positions, inv_freq, (n_heads, n_kv_heads), layout, factor)
