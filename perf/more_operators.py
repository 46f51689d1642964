"""Performance cases of operators that join the blocks of a decoder layer, turn its heads and hold its weights in 4 bits.

Three operators, at Qwen2.5-1.5B and 7B sizes and, drawn, at others of the same range:

- norm: the residual stream h = residual_scale * residual + gate * N(x) post_weight (the norm N after a block, its
        gate and its weight each optional) with the RMS norm before the next block, y = N(h) weight, in one
        pass, and the gradients of x, residual, both weights and the gate. N(v) = v / sqrt(mean(v^2) + eps). A gate
        has a value a channel, a token or an element. The stream is held in the blocks' type or in fp32.
- rope: rotary positions of q and k, token-major in, head-major out: the first R = 2 len(inv_freq) elements of a head
        turn by position * inv_freq, in halves (j with j + R / 2) or in pairs (2 j with 2 j + 1), cos and sin
        times a factor; the rest passes through; and the gradients.
- int4: a linear layer whose frozen weight holds 4-bit integers with a scale, and where asked a zero point, for every
        group of columns of a row: W = (code - zero) * scale, zero 8 where there is none; forward for one token to
        many, and the input gradient.

`own` picks between plain torch forms of these and the package's calls.
"""

import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # 16 streams decode a token each through a block with norms on both sides and a channel gate: latency
        dict(name="norm_decode_16", kind="norm", rows=16, width=3584, x="fp16", stream="fp16", post=True, gate="channel",
             scale=1.0, grad=False),
        # a 1.5B fine-tuning step: the plain pre-norm block, fp32 stream, norm weight trained
        dict(name="norm_1p5b_830", kind="norm", rows=830, width=1536, x="fp16", stream="fp32", post=False, gate="none",
             scale=1.0, grad=True),
        # a ragged batch, odd width, a gate of every element
        dict(name="norm_ragged", kind="norm", rows=333, width=1121, x="bf16", stream="bf16", post=True, gate="element",
             scale=0.75, grad=True),
        # a 7B layer at a long packed length, norms on both sides, channel gate
        dict(name="norm_7b_8192", kind="norm", rows=8192, width=3584, x="bf16", stream="bf16", post=True, gate="channel",
             scale=1.0, grad=True),
        # 16 streams decode a token each far into a long context, half of each head turned in pairs: latency
        dict(name="rope_decode_16", kind="rope", batch=16, tokens=1, heads=28, kv_heads=4, head_dim=128, rotary=64, x="fp16",
             layout="pairs", grad=False),
        # a ragged batch, an odd head size, a quarter of the head turned
        dict(name="rope_ragged", kind="rope", batch=3, tokens=683, heads=9, kv_heads=3, head_dim=80, rotary=20, x="bf16",
             layout="half", grad=True),
        # a 7B layer at a long packed length, frequencies scaled for a long context
        dict(name="rope_7b_8192", kind="rope", batch=1, tokens=8192, heads=28, kv_heads=4, head_dim=128, rotary=128, x="bf16",
             layout="half", grad=True),
        # chat on one stream: a single token through the largest 7B projection
        dict(name="int4_decode_1", kind="int4", m=1, n=18944, k=3584, group=128, zeros=True, x="fp16", bias=False, grad=False),
        # 16 streams decode a token each through the 7B down projection
        dict(name="int4_decode_16", kind="int4", m=16, n=3584, k=18944, group=128, zeros=True, x="bf16", bias=False,
             grad=False),
        # odd sizes in every direction, small groups, symmetric, with a bias
        dict(name="int4_ragged", kind="int4", m=37, n=2057, k=1121, group=32, zeros=False, x="fp16", bias=True, grad=True),
        # gate or up of a 1.5B fine-tuning step
        dict(name="int4_1p5b_830", kind="int4", m=830, n=8960, k=1536, group=64, zeros=True, x="fp16", bias=False, grad=True),
        # long prompts through the largest 7B projection: the largest call
        dict(name="int4_7b_4096", kind="int4", m=4096, n=18944, k=3584, group=128, zeros=True, x="bf16", bias=False, grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "rope", "int4", "int4"])
    x = rng.choice(["fp16", "bf16"])
    grad = rng.random() < 0.6
    if kind == "norm":
        width = _log(rng, 64, 8192)
        return dict(kind=kind, rows=_log(rng, 1, min(16384, 8192 * 3584 // width)), width=width, x=x,
                    stream=rng.choice([x, x, "fp32"]), post=rng.random() < 0.6,
                    gate=rng.choice(["none", "channel", "token", "element"]), scale=rng.choice([1.0, 1.0, 0.5, 1.25]),
                    grad=grad)
    if kind == "int4":
        n, k = _log(rng, 128, 18944), _log(rng, 256, 18944)
        m = _log(rng, 1, max(1, min(4096, 4096 * 18944 * 3584 // (n * k))))
        return dict(kind=kind, m=m, n=n, k=k, group=rng.choice([32, 64, 128, 128]), zeros=rng.random() < 0.6, x=x,
                    bias=rng.random() < 0.5, grad=grad)
    head_dim = rng.choice([64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.randint(1, 7)
    batch = rng.choice([1, 1, 2, 3])
    top = 8192 * 32 * 128 // (batch * (heads + kv_heads) * head_dim)
    rotary = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4, 2 * rng.randint(1, head_dim // 2)])
    return dict(kind=kind, batch=batch, tokens=_log(rng, 1, min(8192, top)), heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, rotary=rotary, x=x, layout=rng.choice(["half", "pairs"]), grad=grad)


# ---- inputs --------------------------------------------------------------------------------------

class _Source:
    """Random tensors on the GPU, made from the seed alone."""

    def __init__(self, seed):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.g = torch.Generator(device=self.dev)
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.float16):
        return (torch.randn(shape, generator=self.g, device=self.dev) * std).to(dtype)

    def whole(self, lo, hi, *shape, dtype=torch.int64):
        return torch.randint(lo, hi, shape, generator=self.g, device=self.dev, dtype=dtype)


def _norm_inputs(case, src):
    rows, width, t, s = case["rows"], case["width"], TYPES[case["x"]], TYPES[case["stream"]]
    # the stream of a deep layer: a few channels far above the others
    gain = torch.where(torch.rand(width, generator=src.g, device=src.dev) < 0.01, 10.0, 1.0)
    st = dict(input=src.normal(rows, width, dtype=t),
              residual=(src.normal(rows, width, std=2.0, dtype=torch.float32) * gain).to(s),
              weight=1.0 + src.normal(width, std=0.2, dtype=torch.float32), post_weight=None, gate_values=None)
    if case["post"]:
        st["post_weight"] = 1.0 + src.normal(width, std=0.2, dtype=torch.float32)
    shape = dict(none=None, channel=(width,), token=(rows, 1), element=(rows, width))[case["gate"]]
    if shape is not None:
        # layer scales are trained and kept in fp32, a gate that the model computes comes in its type
        kept = torch.float32 if case["gate"] == "channel" else t
        st["gate_values"] = torch.sigmoid(src.normal(*shape, dtype=torch.float32)).to(kept)
    if case["grad"]:
        st["gh"] = src.normal(rows, width, std=1e-2, dtype=s)
        st["gy"] = src.normal(rows, width, std=1e-2, dtype=t)
    return st


def _frequencies(rotary, dev):
    """inv_freq of base 1000000, stretched fourfold for a long context: the slow frequencies (fewer than one turn in
    32768 positions) divided by 4, the fast ones (over 32 turns) kept, a ramp between; and the factor of cos and sin."""
    half = rotary // 2
    inv = 1.0 / 1000000.0 ** (torch.arange(half, dtype=torch.float64) / half)
    turns = 32768.0 * inv / (2.0 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    return (inv * keep + inv / 4.0 * (1.0 - keep)).float().to(dev), 0.1 * math.log(4.0) + 1.0


def _rope_inputs(case, src):
    t = TYPES[case["x"]]
    b, tok, h, hk, d = (case[s] for s in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
    # q and k as the packed q/k/v projection leaves them: strided rows of one buffer
    qkv = src.normal(b, tok, (h + 2 * hk) * d, dtype=t)
    st = dict(q=qkv[..., :h * d], k=qkv[..., h * d:(h + hk) * d])
    st["positions"] = src.whole(0, 100000, b, 1) + torch.arange(tok, device=src.dev)
    st["inv_freq"], st["factor"] = _frequencies(case["rotary"], src.dev)
    if case["grad"]:
        st["gq"] = src.normal(b, h, tok, d, std=1e-2, dtype=t)
        st["gk"] = src.normal(b, hk, tok, d, std=1e-2, dtype=t)
    return st


def _int4_inputs(case, src):
    """(codes uint8 [n, k], scales [n, groups], zeros uint8 [n, groups] or None, x, bias or None, dy or None)."""
    m, n, k, group, t = case["m"], case["n"], case["k"], case["group"], TYPES[case["x"]]
    groups = -(-k // group)
    w = torch.zeros((n, groups * group), device=src.dev)
    w[:, :k] = src.normal(n, k, std=0.02, dtype=torch.float32)
    w = w.view(n, groups, group)
    if case["zeros"]:
        lo, hi = w.amin(-1).clamp_max(0.0), w.amax(-1).clamp_min(0.0)
        scales = ((hi - lo) / 15.0).to(t)
        zeros = torch.round(-lo / scales.float()).clamp(0, 15)
    else:
        scales = (w.abs().amax(-1) / 7.0).to(t)
        zeros = torch.full_like(scales, 8.0, dtype=torch.float32)
    codes = torch.round(w / scales.float()[..., None]).add_(zeros[..., None]).clamp_(0, 15).to(torch.uint8)
    codes = codes.view(n, -1)[:, :k].contiguous()
    gain = torch.where(torch.rand(k, generator=src.g, device=src.dev) < 0.01, 10.0, 1.0)
    x = (src.normal(m, k, dtype=torch.float32) * gain).to(t)
    bias = src.normal(n, std=0.1, dtype=t) if case["bias"] else None
    dy = src.normal(m, n, std=1e-2, dtype=t) if case["grad"] else None
    return codes, scales, zeros.to(torch.uint8) if case["zeros"] else None, x, bias, dy


def prepare(case, seed):
    src = _Source(seed)
    st = dict(case)
    if case["kind"] == "norm":
        st.update(_norm_inputs(case, src))
    elif case["kind"] == "rope":
        st.update(_rope_inputs(case, src))
    else:
        codes, scales, zeros, st["input"], st["bias_row"], st["dy"] = _int4_inputs(case, src)
        if own:
            from decik_amd import int4

            st["weight"] = int4.int4_weight(codes, scales, zeros, case["group"])
        else:
            st["codes"], st["scales"], st["zero_points"] = codes, scales, zeros
    return st


# ---- the passes ----------------------------------------------------------------------------------

def run(st):
    if own:
        return _own[st["kind"]](st)
    return _plain[st["kind"]](st)


def _own_norm(st):
    from decik_amd import norm

    given = st["input"], st["residual"], st["weight"], st["post_weight"], st["gate_values"], st["scale"], EPS
    outs = norm.residual_norm_forward(*given)
    if not st["grad"]:
        return list(outs)
    return [*outs, *(g for g in norm.residual_norm_backward(st["gh"], st["gy"], *given) if g is not None)]


def _own_rope(st):
    from decik_amd import rope

    outs = rope.scaled_rope_forward(st["q"], st["k"], st["positions"], st["inv_freq"], st["heads"], st["kv_heads"],
                                    st["layout"], st["factor"])
    if not st["grad"]:
        return list(outs)
    return [*outs, *rope.scaled_rope_backward(st["gq"], st["gk"], st["positions"], st["inv_freq"], st["layout"],
                                              st["factor"])]


def _own_int4(st):
    from decik_amd import int4

    y = int4.int4_linear_forward(st["input"], st["weight"], st["bias_row"])
    if not st["grad"]:
        return [y]
    return [y, int4.int4_linear_backward(st["dy"], st["weight"])]


def _plain_norm(st):
    t, s = TYPES[st["x"]], TYPES[st["stream"]]
    x, res, w, pw, gate = st["input"].float(), st["residual"].float(), st["weight"], st["post_weight"], st["gate_values"]
    p, rx = x, None
    if pw is not None:
        rx = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        p = x * rx * pw
    g = None if gate is None else gate.float()
    h = st["scale"] * res + (p if g is None else g * p)
    rh = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    unit = h * rh
    outs = [h.to(s), (unit * w).to(t)]
    if not st["grad"]:
        return outs
    gy = st["gy"].float()
    u = gy * w
    dh = st["gh"].float() + rh * (u - unit * (u * unit).mean(-1, keepdim=True))
    dp = dh if g is None else dh * g
    dx = dp
    if pw is not None:
        v, ux = dp * pw, x * rx
        dx = rx * (v - ux * (v * ux).mean(-1, keepdim=True))
    outs += [dx.to(t), (st["scale"] * dh).to(s), (gy * unit).sum(0)]
    if pw is not None:
        outs.append((dp * x * rx).sum(0))
    if st["gate"] == "channel":
        outs.append((dh * p).sum(0))
    elif st["gate"] == "token":
        outs.append((dh * p).sum(-1, keepdim=True).to(t))
    elif st["gate"] == "element":
        outs.append((dh * p).to(t))
    return outs


def _turn(x, cos, sin, layout):
    """x [b, heads, tokens, d] with its first 2 * cos.shape[-1] elements turned."""
    r = 2 * cos.shape[-1]
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if layout == "half" else (x[..., 0:r:2], x[..., 1:r:2])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([a, b], -1) if layout == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _plain_rope(st):
    t, d, layout = TYPES[st["x"]], st["head_dim"], st["layout"]
    # angles of far positions in 64 bits
    angle = st["positions"].double()[..., None] * st["inv_freq"].double()
    cos, sin = ((f(angle) * st["factor"]).float()[:, None] for f in (torch.cos, torch.sin))
    outs = [_turn(st[s].float().unflatten(-1, (-1, d)).transpose(1, 2), cos, sin, layout).to(t) for s in "qk"]
    if st["grad"]:
        outs += [_turn(st["g" + s].float(), cos, -sin, layout).transpose(1, 2).flatten(2).to(t) for s in "qk"]
    return outs


def _plain_int4(st):
    t, k, group = TYPES[st["x"]], st["k"], st["group"]
    zeros = 8.0 if st["zero_points"] is None else st["zero_points"].float().repeat_interleave(group, 1)[:, :k]
    w = (st["codes"].float() - zeros) * st["scales"].float().repeat_interleave(group, 1)[:, :k]
    y = st["input"].float() @ w.t()
    if st["bias_row"] is not None:
        y = y + st["bias_row"].float()
    if not st["grad"]:
        return [y.to(t)]
    return [y.to(t), (st["dy"].float() @ w).to(t)]


_own = dict(norm=_own_norm, rope=_own_rope, int4=_own_int4)
_plain = dict(norm=_plain_norm, rope=_plain_rope, int4=_plain_int4)


# ---- work and exact values -----------------------------------------------------------------------

def work(case):
    size = {"fp16": 2, "bf16": 2, "fp32": 4}
    es = size[case["x"]]
    if case["kind"] == "int4":
        m, n, k = case["m"], case["n"], case["k"]
        ways = 2 if case["grad"] else 1
        weight = n * (k + 1) // 2 + n * -(-k // case["group"]) * (es + (1 if case["zeros"] else 0))
        # each way reads the weight and one activation and writes the other
        return {"bytes": ways * (weight + es * m * (n + k)) + (es * n if case["bias"] else 0), "flops": ways * 2 * m * n * k}
    if case["kind"] == "norm":
        rows, width, ss = case["rows"], case["width"], size[case["stream"]]
        data, gate = rows * width, case["gate"]
        values = dict(none=0, channel=4 * width, token=es * rows, element=es * data)[gate]
        weights = 4 * width * (2 if case["post"] else 1)
        per = 6 + (4 if case["post"] else 0) + (1 if gate != "none" else 0)
        fwd = {"bytes": 2 * data * (es + ss) + values + weights, "flops": data * per}
        if not case["grad"]:
            return fwd
        # gradients of h and y in, of x and the residual out, the weights' and the gate's
        return {"bytes": fwd["bytes"] + 2 * data * (es + ss) + weights + values, "flops": fwd["flops"] + data * (2 * per + 4)}
    rows = case["batch"] * case["tokens"]
    data = rows * (case["heads"] + case["kv_heads"]) * case["head_dim"]
    ways = 2 if case["grad"] else 1
    turned = rows * (case["heads"] + case["kv_heads"]) * case["rotary"]
    return {"bytes": ways * (2 * data * es + 8 * rows + 2 * case["rotary"]), "flops": ways * 3 * turned}


def _exact_norm(st):
    """The definition in 64 bits, its gradients by automatic differentiation."""
    def leaf(v):
        return None if v is None else v.double().requires_grad_(st["grad"])

    x, res, w, pw, gate = (leaf(st[s]) for s in ("input", "residual", "weight", "post_weight", "gate_values"))

    def unit(v):
        return v * torch.rsqrt(v.square().sum(-1, keepdim=True) / st["width"] + EPS)

    block = x if pw is None else unit(x) * pw
    h = res * st["scale"] + (block if gate is None else block * gate)
    y = unit(h) * w
    if not st["grad"]:
        return [h, y]
    wrt = [v for v in (x, res, w, pw, gate) if v is not None]
    grads = torch.autograd.grad([h, y], wrt, [st["gh"].double(), st["gy"].double()])
    return [h.detach(), y.detach(), *grads]


def _exact_rope(st):
    """Complex numbers turned by the angle."""
    r, d = st["rotary"], st["head_dim"]
    angle = st["positions"].to(torch.float64).unsqueeze(-1) * st["inv_freq"].to(torch.float64)
    turn = torch.polar(torch.full_like(angle, st["factor"]), angle).unsqueeze(1)
    if st["layout"] == "half":
        first, second = torch.arange(r // 2), torch.arange(r // 2) + r // 2
    else:
        first, second = 2 * torch.arange(r // 2), 2 * torch.arange(r // 2) + 1

    def through(x, by):
        z = torch.complex(x[..., first], x[..., second]) * by
        out = x.clone()
        out[..., first], out[..., second] = z.real, z.imag
        return out

    outs = []
    for x, heads in ((st["q"], st["heads"]), (st["k"], st["kv_heads"])):
        outs.append(through(x.double().reshape(*x.shape[:2], heads, d).permute(0, 2, 1, 3).contiguous(), turn))
    if st["grad"]:
        for g in (st["gq"], st["gk"]):
            back = through(g.double(), turn.conj()).permute(0, 2, 1, 3)
            outs.append(back.reshape(*back.shape[:2], -1))
    return outs


def exact(case, seed):
    src = _Source(seed)
    if case["kind"] == "norm":
        return _exact_norm({**case, **_norm_inputs(case, src)})
    if case["kind"] == "rope":
        return _exact_rope({**case, **_rope_inputs(case, src)})
    codes, scales, zeros, x, bias, dy = _int4_inputs(case, src)
    w = torch.empty(codes.shape, dtype=torch.float64, device=codes.device)
    for i in range(scales.shape[1]):
        at = slice(i * case["group"], min(case["k"], (i + 1) * case["group"]))
        zero = 8 if zeros is None else zeros[:, i:i + 1].double()
        w[:, at] = (codes[:, at].double() - zero) * scales[:, i:i + 1].double()
    y = torch.mm(x.double(), w.t().contiguous())
    if bias is not None:
        y += bias.double()
    return [y] if dy is None else [y, torch.mm(dy.double(), w)]
