"""Linear layers in 4-bit integers with a scale and a zero point a group (dk_int4_linear).

A frozen weight [N, K] is held as codes 0 .. 15 with a scale (fp16 or bf16) and, where asked, a zero point for every `group`
columns of a row, about a quarter of fp16's bytes; zero points are 8 where none are given:
  W[n, k] = (code[n, k] - zero[n, k // group]) * scale[n, k // group]
  forward:  y = x . W^T + bias. Up to 32 tokens (64 on weights of up to 2^24) stream the weight to registers: the integers times
            x exactly, each group's sum in fp32 times its scale, rounded once. More go by tiles, with W rounded once to x's
            type (at most half a step of it a weight; fp16 keeps W in steps of 2^-24 at least) and sums in fp32; where W is
            not to be rounded, call it on up to 32 tokens at a time
  backward: dX = dY . W by tiles, W rounded once to dY's type, sums in fp32
quantize_int4 makes such a weight from values, int4_weight from codes, scales and zero points that a checkpoint holds;
both lay the codes out once for the kernels (Int4Weight). Sums are added in an order that depends on the sizes alone.
"""

import ctypes

import torch
from torch.autograd.function import once_differentiable

from ._lib import DTYPES, call_on, check, gpu_input, lib, same_gpu

ROWS, BLOCK = 16, 128  # rows and columns of a tile of packed codes
_TYPES = {torch.float16: 0, torch.bfloat16: 1}


class Int4Weight:
    """A weight [n, k] in groups of `group` columns, as dk_int4_linear takes it: packed uint8 [ceil(n / 16), ceil(k / 128),
    1024] (tiles of 16 rows by 128 columns), meta int32 [ceil(n / 16), ceil(k / group), 16] (scale and zero point),
    scale_dtype. No call changes it."""

    __slots__ = ("packed", "meta", "n", "k", "group", "scale_dtype")

    def __init__(self, packed, meta, n, k, group, scale_dtype):
        self.packed, self.meta, self.n, self.k, self.group, self.scale_dtype = packed, meta, n, k, group, scale_dtype

    @property
    def shape(self):
        return torch.Size((self.n, self.k))

    @property
    def device(self):
        return self.packed.device

    def to(self, device):
        return Int4Weight(self.packed.to(device), self.meta.to(device), self.n, self.k, self.group, self.scale_dtype)

    @property
    def scales(self):
        """[n, groups], of scale_dtype."""
        return (self._by_row() & 0xFFFF).to(torch.int16).view(self.scale_dtype)

    @property
    def zeros(self):
        """uint8 [n, groups]."""
        return (self._by_row() >> 16).to(torch.uint8)

    def _by_row(self):
        tiles, groups, _ = self.meta.shape
        return self.meta.transpose(1, 2).reshape(tiles * ROWS, groups)[:self.n]

    def codes(self):
        """uint8 [n, k], unpacked."""
        tiles, blocks, _ = self.packed.shape
        words = self.packed.view(torch.int32).view(tiles, blocks, 4, ROWS, 4)  # [.., q, row, j]
        cols = torch.stack([(words >> s) & 15 for s in _SHIFTS], -1).to(torch.uint8)
        # [tile, row, block, j, q, column]
        return cols.permute(0, 3, 1, 4, 2, 5).reshape(tiles * ROWS, blocks * BLOCK)[:self.n, :self.k].contiguous()


# bits of columns 0 .. 7 of a word
_SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)


def int4_weight(codes, scales, zeros=None, group=128):
    """Int4Weight of codes [N, K] (uint8, 0 to 15), scales [N, ceil(K / group)] (fp16 or bf16, below 2^117) and zero points of
    the same shape (uint8, 0 to 16; None: 8). group: a multiple of 32. On any device; the layout is made once."""
    what = "int4_weight"
    group = int(group)
    if group < 32 or group % 32 or group > 2 ** 20:
        raise ValueError(f"{what}: group must be a multiple of 32 up to 2^20")
    if codes.dim() != 2 or codes.dtype != torch.uint8 or not 1 <= codes.shape[1] <= 2 ** 20 or codes.shape[0] >= 2 ** 23:
        raise ValueError(f"{what}: codes must be uint8 [N, K], N below 2^23, K from 1 to 2^20")
    n, k = codes.shape
    shape = (n, -(-k // group))
    if tuple(scales.shape) != shape or scales.dtype not in _TYPES:
        raise ValueError(f"{what}: scales must be {list(shape)}, fp16 or bf16")
    if zeros is not None and (tuple(zeros.shape) != shape or zeros.dtype != torch.uint8):
        raise ValueError(f"{what}: zeros must be uint8 {list(shape)}")
    for t in (scales, zeros):
        if t is not None and t.device != codes.device:
            raise ValueError(f"{what}: codes, scales and zeros must be on one device")
    if n and (int(codes.max()) > 15 or (zeros is not None and int(zeros.max()) > 16)):
        raise ValueError(f"{what}: codes must be 0 to 15, zeros 0 to 16")
    if n and not float(scales.detach().abs().max()) < 2.0 ** 117:
        raise ValueError(f"{what}: scales must be numbers below 2^117")
    tiles, blocks = -(-n // ROWS), -(-k // BLOCK)
    cols = torch.zeros((tiles * ROWS, blocks * BLOCK), dtype=torch.uint8, device=codes.device)
    cols[:n, :k] = codes
    cols = cols.view(tiles, ROWS, blocks, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)  # [tile, block, q, row, j, column]
    words = torch.zeros((tiles, blocks, 4, ROWS, 4), dtype=torch.int32, device=codes.device)
    for e, shift in enumerate(_SHIFTS):
        words |= cols[..., e].to(torch.int32) << shift
    meta = torch.zeros((tiles * ROWS, shape[1]), dtype=torch.int32, device=codes.device)
    meta[:n] = scales.contiguous().view(torch.int16).to(torch.int32) & 0xFFFF
    meta[:n] |= 8 << 16 if zeros is None else zeros.to(torch.int32) << 16
    return Int4Weight(words.view(tiles, blocks, 256).view(torch.uint8), meta.view(tiles, ROWS, shape[1]).transpose(1, 2).contiguous(),
                      n, k, group, scales.dtype)


def quantize_int4(w, group=128, symmetric=False, scale_dtype=None):
    """Int4Weight of w [N, K], fp16, bf16 or fp32, rounded to the nearest: with zero points scale = (max - min) / 15 of a
    group's values and 0, zero = rint(-min / scale); symmetric: scale = absmax / 7, zero 8. Scales of scale_dtype
    (default w's type, fp16 for fp32). A group without a finite scale above 0 in that type is all zero points, scale
    0."""
    what = "quantize_int4"
    group = int(group)
    if group < 32 or group % 32:
        raise ValueError(f"{what}: group must be a multiple of 32")
    if not isinstance(w, torch.Tensor) or w.dim() != 2 or w.dtype not in DTYPES or w.shape[1] < 1:
        raise ValueError(f"{what}: w must be [N, K], fp16, bf16 or fp32")
    scale_dtype = scale_dtype or (w.dtype if w.dtype in _TYPES else torch.float16)
    if scale_dtype not in _TYPES:
        raise ValueError(f"{what}: scale_dtype must be fp16 or bf16")
    n, k = w.shape
    groups = -(-k // group)
    width = min(group, k)  # (one group where it is longer than a row)
    v = torch.zeros((n, groups * width), dtype=torch.float32, device=w.device)
    v[:, :k] = w
    v = v.view(n, groups, width)
    if symmetric:
        scales, lo = v.abs().amax(-1) / 7.0, None
    else:
        lo = v.amin(-1).clamp_max(0.0)
        scales = (v.amax(-1).clamp_min(0.0) - lo) / 15.0
    scales = scales.to(scale_dtype)
    ok = scales.isfinite() & (scales > 0)
    scales = torch.where(ok, scales, torch.zeros_like(scales))
    by = torch.where(ok, scales.float(), torch.ones_like(scales, dtype=torch.float32))
    zeros = torch.full_like(by, 8.0) if symmetric else torch.where(ok, torch.round(-lo / by), 8.0).clamp(0, 15)
    codes = torch.round(v / by[..., None]).add_(zeros[..., None]).clamp_(0, 15)
    codes = torch.where(ok[..., None], codes, zeros[..., None]).to(torch.uint8).view(n, groups * width)[:, :k]
    return int4_weight(codes.contiguous(), scales, None if symmetric else zeros.to(torch.uint8), group)


def dequantize_int4(weight, dtype=torch.float32):
    """The values the weight stands for, [N, K] of `dtype`."""
    times = min(weight.group, weight.k)  # (one group where it is longer than a row)
    zeros, scales = (t.float().repeat_interleave(times, 1)[:, :weight.k] for t in (weight.zeros, weight.scales))
    return ((weight.codes().float() - zeros) * scales).to(dtype)


def launch_plan(backward, m, n, k):
    """What a product of these sizes runs as (dk_int4_linear_plan): dict of tile_tokens, waves (of a work-group that streams
    the weight; 0: tiles of 256 rows or columns), shares (waves that share a row's columns) and splits of the sum."""
    out = (ctypes.c_int32 * 4)()
    check(lib().dk_int4_linear_plan(int(backward), m, n, k, out))
    return dict(tile_tokens=out[0], waves=out[1], shares=out[2], splits=out[3])


def _product(what, backward, x, weight, bias, dtype):
    dev = gpu_input(what, x)
    if not isinstance(weight, Int4Weight):
        raise ValueError(f"{what}: the weight must be an Int4Weight")
    same_gpu(what, dev, weight.packed, weight.meta, bias)
    n, k = weight.n, weight.k
    total, cols = (n, k) if backward else (k, n)
    if x.dim() < 1 or x.shape[-1] != total:
        raise ValueError(f"{what}: {'dy [.., N]' if backward else 'x [.., K]'} must end in {total}")
    code = _TYPES.get(x.dtype)
    if code is None:
        raise ValueError(f"{what}: {'dy' if backward else 'x'} must be fp16 or bf16")
    out = code if dtype is None else DTYPES.get(dtype)
    if out not in (code, 2):
        raise ValueError(f"{what}: dtype must be x's type or fp32")
    bias_code = 0
    if bias is not None:
        bias_code = DTYPES.get(bias.dtype)
        if bias.shape != (n,) or bias_code is None:
            raise ValueError(f"{what}: bias must be [{n}], fp16, bf16 or fp32")
        bias = bias.contiguous()
    if total == 0:
        return x.new_zeros(*x.shape[:-1], cols, dtype=dtype)
    x2 = x if x.dim() == 2 else x.reshape(-1, total)
    m = x2.shape[0]
    if x2.stride(1) != 1 and total != 1 or (m > 1 and x2.stride(0) >= 2 ** 22):
        x2 = x2.contiguous()
    ldx = x2.stride(0)
    copy = total % 8 != 0 or x2.data_ptr() % 16 != 0 or (m > 1 and ldx % 8 != 0)
    y = x.new_empty(*x.shape[:-1], cols, dtype=dtype)
    need = lib().dk_int4_linear_workspace(backward, copy, m, n, k)
    # a tensor of its own a call: graphs and streams share none
    work = x.new_empty(need, dtype=torch.uint8) if need > 0 else None
    call_on(dev, lib().dk_int4_linear, backward, x2.data_ptr(), code, ldx, weight.packed.data_ptr(), weight.meta.data_ptr(),
            weight.group, _TYPES[weight.scale_dtype], None if bias is None else bias.data_ptr(),
            bias_code, y.data_ptr(), out, cols, m, n, k, copy, None if work is None else work.data_ptr(), max(need, 0))
    return y


def int4_linear_forward(x, weight, bias=None, dtype=None):
    """y [.., N] (x's type, or dtype = fp32) = x . W^T + bias of x [.., K], fp16 or bf16, and an Int4Weight."""
    return _product("int4_linear_forward", False, x, weight, bias, dtype)


def int4_linear_backward(dy, weight, dtype=None):
    """dX [.., K] (dy's type, or dtype = fp32) = dY . W of dy [.., N], fp16 or bf16."""
    return _product("int4_linear_backward", True, dy, weight, None, dtype)


class Int4Linear(torch.autograd.Function):
    """apply(x, weight, bias) -> y: a linear whose Int4Weight and bias are frozen; gradients reach x."""

    @staticmethod
    def forward(ctx, x, weight, bias=None):
        if any(ctx.needs_input_grad[2:]):  # (two inputs where the call names no bias)
            raise ValueError("Int4Linear: the bias is frozen (detach it)")
        ctx.weight, ctx.named = weight, len(ctx.needs_input_grad)
        return int4_linear_forward(x, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return (int4_linear_backward(grad, ctx.weight), None, None)[:ctx.named]
