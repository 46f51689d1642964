"""Performance cases of the operators around the frozen projections of a fine-tuned decoder layer.

Four operators, at Qwen2.5-1.5B and 7B sizes and, drawn, at others of the same range:

- dropout: the inputs of one or more LoRA branches, dropped out with a counter-based generator whose
           mask is not stored, and the gradient back through the same mask. Philox4x32-10, keyed
           with the 64-bit seed; the counter of columns 8 g .. 8 g + 7 of row r is (g, r, low word,
           high word of offset + branch); column 8 g + e compares the 16-bit half e % 2 of output
           word e // 2 with rint(p * 65536) and is kept when it is not below.
- qknorm:  RMS norms of every query and key head with the rotation of rotary positions (given as
           cos / sin tables), token-major in, head-major out, and its gradients.
- axes:    rotary positions with several axes (time, height, width): angles formed from integer
           positions and frequencies, with or without the norms, and the gradients.
- int8:    a linear layer whose frozen weight holds 8-bit integers with a scale per output channel;
           the activations are quantized per token (scale absmax / 127, values
           rint(x * (127 / absmax))), and so is dY * channel scale for the input gradient.

`own` picks between plain torch forms of these and the package's calls.
"""

import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # the q and v adapters of a 1.5B fine-tuning step on its fp32 norm output
        dict(name="dropout_1p5b_830", kind="dropout", rows=830, width=1536, branches=2, p=0.05, x="fp32", out="fp16"),
        # the same two branches of a 7B layer at a long packed length
        dict(name="dropout_7b_8192", kind="dropout", rows=8192, width=3584, branches=2, p=0.1, x="fp16", out="fp16"),
        # one adapter, a width that no vector divides
        dict(name="dropout_ragged", kind="dropout", rows=333, width=1121, branches=1, p=0.25, x="bf16", out="bf16"),
        # 16 streams decode a token each: forward only, where latency counts
        dict(name="qknorm_decode_16", kind="qknorm", batch=16, tokens=1, heads=28, kv_heads=4, head_dim=128, x="fp16",
             grad=False),
        # the attention inputs of a 1.5B fine-tuning step, norm weights trained
        dict(name="qknorm_1p5b_830", kind="qknorm", batch=1, tokens=830, heads=12, kv_heads=2, head_dim=128, x="fp16",
             grad=True),
        # a 7B layer at a long packed length
        dict(name="qknorm_7b_8192", kind="qknorm", batch=1, tokens=8192, heads=28, kv_heads=4, head_dim=128, x="bf16",
             grad=True),
        # two sequences of text and image patches, three axes in consecutive sections
        dict(name="axes_7b_2x2048", kind="axes", batch=2, tokens=2048, heads=28, kv_heads=4, head_dim=128, x="fp16",
             time=16, height=24, width=24, interleaved=False, norm=False, grad=True),
        # a ragged batch of short clips, odd head size, interleaved axes, with the norms
        dict(name="axes_ragged", kind="axes", batch=3, tokens=683, heads=9, kv_heads=3, head_dim=80, x="bf16",
             time=14, height=13, width=13, interleaved=True, norm=True, grad=True),
        # chat on one stream: a single token through the largest 7B projection
        dict(name="int8_decode_1", kind="int8", m=1, n=18944, k=3584, x="fp16", bias=False, grad=False),
        # odd sizes in every direction, with a bias
        dict(name="int8_ragged", kind="int8", m=333, n=2057, k=1121, x="bf16", bias=True, grad=True),
        # gate or up of a 1.5B fine-tuning step
        dict(name="int8_1p5b_830", kind="int8", m=830, n=8960, k=1536, x="fp16", bias=False, grad=True),
        # long-context training: the largest call
        dict(name="int8_7b_8192", kind="int8", m=8192, n=18944, k=3584, x="fp16", bias=False, grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["dropout", "qknorm", "axes", "int8", "int8"])
    if kind == "dropout":
        width = _log(rng, 64, 18944)
        x = rng.choice(["fp16", "bf16", "fp32"])
        return dict(kind=kind, rows=_log(rng, 1, min(8192, 8192 * 3584 // width)), width=width,
                    branches=rng.choice([1, 2, 2]), p=round(rng.uniform(0.01, 0.5), 3), x=x,
                    out=rng.choice(["fp16", "fp32"]) if x == "fp32" else x)
    if kind == "int8":
        n, k = _log(rng, 128, 18944), _log(rng, 256, 18944)
        m = _log(rng, 1, max(1, min(8192, 8192 * 18944 * 3584 // (n * k))))
        return dict(kind=kind, m=m, n=n, k=k, x=rng.choice(["fp16", "bf16"]), bias=rng.random() < 0.5,
                    grad=rng.random() < 0.6)
    head_dim = rng.choice([64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.randint(1, 7)
    batch = rng.choice([1, 1, 2, 3])
    top = 8192 * 32 * 128 // (batch * (heads + kv_heads) * head_dim)
    case = dict(kind=kind, batch=batch, tokens=_log(rng, 1, min(8192, top)), heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, x=rng.choice(["fp16", "bf16"]), grad=rng.random() < 0.7)
    if kind == "axes":
        half, side = head_dim // 2, (head_dim // 2 // 3) - rng.randint(0, 2)
        case.update(time=half - 2 * side, height=side, width=side, interleaved=rng.random() < 0.5, norm=rng.random() < 0.5)
    return case


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


def _axis_positions(src, batch, tokens):
    """[3, batch, tokens]: text (all axes alike) around one block of image or video patches."""
    out = torch.empty((3, batch, tokens), dtype=torch.int64, device=src.dev)
    grid_w, grid_h = 28, 16
    for b in range(batch):
        start = int(torch.randint(0, 60000, (1,), generator=src.g, device=src.dev))
        i = torch.arange(tokens, device=src.dev)
        lead = tokens // 5
        patch = (i >= lead) & (i < tokens - tokens // 5)
        j = i - lead
        frame, row, col = j // (grid_w * grid_h), j // grid_w % grid_h, j % grid_w
        for a, axis in enumerate((frame, row, col)):
            out[a, b] = start + torch.where(patch, lead + axis, i)
    return out


def _inv_freq(head_dim, dev):
    return (1.0 / 1000000.0 ** (torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)).float().to(dev)


def _axis_of(sections, interleaved, dev):
    """The axis that each of the head_dim / 2 frequencies belongs to: consecutive sections, or axis
    j % n while it has frequencies left (axis 0 takes the others)."""
    n, half = len(sections), sum(sections)
    if interleaved:
        axis = [j % n if j < n * sections[j % n] else 0 for j in range(half)]
    else:
        axis = [a for a, s in enumerate(sections) for _ in range(s)]
    return torch.tensor(axis, device=dev)


def _plain_quantize(x32):
    """(integers as fp32, scale) of each row. The quotients divide tensors: a number over a tensor would
    be its rounded reciprocal times the number."""
    top = x32.abs().amax(-1, keepdim=True)
    most = torch.full_like(top, 127.0)
    return torch.round(x32 * torch.where(top > 0, most / top, 0.0)), top / most


def _int8_inputs(case, src):
    m, n, k, t = case["m"], case["n"], case["k"], TYPES[case["x"]]
    w = src.normal(n, k, std=0.02, dtype=torch.float32)
    # a few channels of the activations are ten times the others, as a norm's weights make them
    gain = torch.where(torch.rand(k, generator=src.g, device=src.dev) < 0.01, 10.0, 1.0)
    x = (src.normal(m, k, dtype=torch.float32) * gain).to(t)
    bias = src.normal(n, std=0.1, dtype=t) if case["bias"] else None
    return w, x, bias, src.normal(m, n, std=1e-3, dtype=t) if case["grad"] else None


def prepare(case, seed):
    src = _Source(seed)
    st = dict(case)
    t = TYPES[case["x"]]
    if case["kind"] == "dropout":
        rows, width = case["rows"], case["width"]
        st["input"] = src.normal(rows, width, dtype=t)
        st["rng"] = src.whole(0, 2 ** 62, 2)
        st["grads"] = [src.normal(rows, width, std=1e-2, dtype=TYPES[case["out"]]) for _ in range(case["branches"])]
        return st
    if case["kind"] == "int8":
        w, st["input"], st["bias_row"], st["dy"] = _int8_inputs(case, src)
        if own:
            from decik_amd import int8

            st["wq"], st["ws"] = int8.quantize_int8(w)
        else:
            wq, ws = _plain_quantize(w)
            st["wq"], st["ws"] = wq.to(torch.int8), ws[:, 0].contiguous()
        return st
    b, tok, h, hk, d = (case[s] for s in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
    # q and k as the packed q/k/v projection leaves them: strided rows of one buffer
    qkv = src.normal(b, tok, (h + 2 * hk) * d, dtype=t)
    st["q"], st["k"] = qkv[..., :h * d], qkv[..., h * d:(h + hk) * d]
    if case["kind"] == "qknorm" or case["norm"]:
        st["qw"], st["kw"] = (1.0 + src.normal(d, std=0.2, dtype=torch.float32) for _ in range(2))
    else:
        st["qw"] = st["kw"] = None
    if case["kind"] == "qknorm":
        start = src.whole(0, 30000, b, 1)
        pos = (start + torch.arange(tok, device=src.dev)).double()
        angle = pos[..., None] * _inv_freq(d, src.dev).double()
        angle = torch.cat([angle, angle], -1)
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    else:
        st["sections"] = [case["time"], case["height"], case["width"]]
        st["positions"], st["inv_freq"] = _axis_positions(src, b, tok), _inv_freq(d, src.dev)
    if case["grad"]:
        st["gq"] = src.normal(b, h, tok, d, std=1e-2, dtype=t)
        st["gk"] = src.normal(b, hk, tok, d, std=1e-2, dtype=t)
    return st


# ---- the passes ----------------------------------------------------------------------------------

def run(st):
    if own:
        return _own[st["kind"]](st)
    return _plain[st["kind"]](st)


def _own_dropout(st):
    from decik_amd import dropout

    ps = (st["p"],) * st["branches"]
    outs = dropout.dropout_forward(st["input"], st["rng"], ps, TYPES[st["out"]])
    return [*outs, dropout.dropout_backward(st["grads"], st["rng"], ps, TYPES[st["x"]])]


def _own_qknorm(st):
    from decik_amd import rope

    outs = rope.qk_norm_rope_forward(st["q"], st["k"], st["qw"], st["kw"], st["cos"], st["sin"], st["heads"],
                                     st["kv_heads"], EPS)
    if not st["grad"]:
        return list(outs)
    return [*outs, *rope.qk_norm_rope_backward(st["gq"], st["gk"], st["q"], st["k"], st["qw"], st["kw"], st["cos"],
                                               st["sin"], EPS)]


def _own_axes(st):
    from decik_amd import rope

    outs = rope.axes_rope_forward(st["q"], st["k"], st["positions"], st["inv_freq"], st["sections"], st["heads"],
                                  st["kv_heads"], st["interleaved"], st["qw"], st["kw"], EPS)
    if not st["grad"]:
        return list(outs)
    if not st["norm"]:
        return [*outs, *rope.axes_rope_backward(st["gq"], st["gk"], st["positions"], st["inv_freq"], st["sections"],
                                                st["interleaved"])[:2]]
    return [*outs, *rope.axes_rope_backward(st["gq"], st["gk"], st["positions"], st["inv_freq"], st["sections"],
                                            st["interleaved"], st["q"], st["k"], st["qw"], st["kw"], EPS)]


def _own_int8(st):
    from decik_amd import int8

    y = int8.int8_linear_forward(st["input"], st["wq"], st["ws"], st["bias_row"])
    if not st["grad"]:
        return [y]
    return [y, int8.int8_linear_backward(st["dy"], st["wq"], st["ws"], st["k"])]


def _philox_halves(rng, rows, groups, branch):
    """[rows, groups, 8] 16-bit numbers of one branch, in int64."""
    mask = 0xFFFFFFFF
    dev = rng.device
    k0, k1 = rng[0] & mask, (rng[0] >> 32) & mask
    off = rng[1] + branch
    c = [torch.arange(groups, device=dev).expand(rows, groups), torch.arange(rows, device=dev)[:, None].expand(rows, groups),
         (off & mask).expand(rows, groups), ((off >> 32) & mask).expand(rows, groups)]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & mask) ^ c[1] ^ k0, b & mask, ((a >> 32) & mask) ^ c[3] ^ k1, a & mask]
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    words = torch.stack(c, -1)
    return torch.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, groups, 8)


def _plain_dropout(st):
    rows, width = st["rows"], st["width"]
    thr = round(st["p"] * 65536)
    scale = torch.tensor(65536.0 / (65536 - thr), dtype=torch.float32, device=st["input"].device)
    x = st["input"].float()
    outs, dx = [], torch.zeros_like(x)
    for b in range(st["branches"]):
        keep = (_philox_halves(st["rng"], rows, -(-width // 8), b) >= thr).reshape(rows, -1)[:, :width]
        outs.append(torch.where(keep, x * scale, 0.0).to(TYPES[st["out"]]))
        dx = dx + torch.where(keep, st["grads"][b].float() * scale, 0.0)
    return [*outs, dx.to(TYPES[st["x"]])]


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def _rotate_back(g, cos, sin):
    half = g.shape[-1] // 2
    s = g * sin
    return g * cos + torch.cat([s[..., half:], -s[..., :half]], -1)


def _plain_rotation(st, cos, sin):
    t, d, norm = TYPES[st["x"]], st["head_dim"], st["qw"] is not None
    cos, sin = cos[:, None], sin[:, None]  # [batch, 1, tokens, head_dim]
    outs, grads, weights = [], [], []
    for side, heads, w in (("q", st["heads"], st["qw"]), ("k", st["kv_heads"], st["kw"])):
        x = st[side].float().unflatten(-1, (heads, d)).transpose(1, 2)
        y = x
        if norm:
            r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            y = x * r * w
        outs.append(_rotate(y, cos, sin).to(t))
        if not st["grad"]:
            continue
        g = _rotate_back(st["g" + side].float(), cos, sin)
        if norm:
            weights.append((g * x * r).sum((0, 1, 2)))
            g = g * w
            g = r * (g - x * (r * r) * (g * x).mean(-1, keepdim=True))
        grads.append(g.transpose(1, 2).flatten(2).to(t))
    return [*outs, *grads, *weights]


def _plain_qknorm(st):
    return _plain_rotation(st, st["cos"], st["sin"])


def _plain_axes(st):
    # angles of far positions in 64 bits
    axis = _axis_of(st["sections"], st["interleaved"], st["inv_freq"].device)
    angle = st["positions"][axis].permute(1, 2, 0).double() * st["inv_freq"].double()
    angle = torch.cat([angle, angle], -1)
    return _plain_rotation(st, angle.cos().float(), angle.sin().float())


def _plain_int8(st):
    t, n, k = TYPES[st["x"]], st["n"], st["k"]
    w = st["wq"][:n, :k].float()
    xq, xs = _plain_quantize(st["input"].float())
    y = (xq @ w.t()) * xs * st["ws"]
    if st["bias_row"] is not None:
        y = y + st["bias_row"].float()
    if not st["grad"]:
        return [y.to(t)]
    gq, gs = _plain_quantize(st["dy"].float() * st["ws"])
    return [y.to(t), ((gq @ w) * gs).to(t)]


_own = dict(dropout=_own_dropout, qknorm=_own_qknorm, axes=_own_axes, int8=_own_int8)
_plain = dict(dropout=_plain_dropout, qknorm=_plain_qknorm, axes=_plain_axes, int8=_plain_int8)


# ---- work and exact values -----------------------------------------------------------------------

def work(case):
    size = {"fp16": 2, "bf16": 2, "fp32": 4}
    es = size[case["x"]]
    if case["kind"] == "dropout":
        n, nb = case["rows"] * case["width"], case["branches"]
        return {"bytes": n * 2 * (es + nb * size[case["out"]]), "flops": n * nb * 3}
    if case["kind"] == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        ways = 2 if case["grad"] else 1
        # each way reads the weight, its scales and one activation and writes the other
        return {"bytes": ways * (n * k + 4 * n + es * m * (n + k)) + (es * n if case["bias"] else 0),
                "flops": ways * 2 * m * n * k}
    rows = case["batch"] * case["tokens"]
    d = case["head_dim"]
    data = rows * (case["heads"] + case["kv_heads"]) * d
    norm = case["kind"] == "qknorm" or case["norm"]
    table = rows * 2 * d * 4 if case["kind"] == "qknorm" else rows * 24 + 2 * d
    weights = 8 * d if norm else 0
    fwd = {"bytes": 2 * data * es + table + weights, "flops": data * (8 if norm else 3)}
    if not case["grad"]:
        return fwd
    return {"bytes": fwd["bytes"] + (3 if norm else 2) * data * es + table + 2 * weights,
            "flops": fwd["flops"] + data * (14 if norm else 3)}


def _exact_bits(rng, rows, cols, branch):
    """16-bit numbers [rows, cols], by the generator's definition on 16-bit limbs."""
    dev = rng.device
    col, row = torch.arange(cols, device=dev), torch.arange(rows, device=dev)
    group = (col // 8)[None, :] + 0 * row[:, None]
    seed, off = int(rng[0]), (int(rng[1]) + branch) % 2 ** 64
    c = [group, row[:, None] + 0 * col[None, :], torch.full_like(group, off % 2 ** 32),
         torch.full_like(group, off // 2 ** 32)]

    def product(a, m):
        lo, hi = (a % 65536) * m, (a // 65536) * m
        low = lo + (hi % 65536) * 65536
        return low // 2 ** 32 + hi // 65536, low % 2 ** 32

    for i in range(10):
        k0, k1 = (seed + i * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + i * 0xBB67AE85) % 2 ** 32
        h0, l0 = product(c[0], 0xD2511F53)
        h1, l1 = product(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
    word = torch.stack(c).gather(0, (col % 8 // 2)[None, None, :].expand(1, rows, cols))[0]
    return torch.where(col % 2 == 1, word // 65536, word % 65536)


def _exact_rotation(st, angle, cos, sin):
    """One axis of complex numbers: (x[j], x[j + D / 2]) turned by the angle of frequency j, or with
    given tables by its cos and sin of each half."""
    d, half = st["head_dim"], st["head_dim"] // 2
    if angle is not None:
        cos, sin = torch.cos(angle).repeat(1, 1, 2), torch.sin(angle).repeat(1, 1, 2)
    c = [t[:, None].contiguous() for t in (cos[..., :half], cos[..., half:], sin[..., :half], sin[..., half:])]
    outs, grads, weights = [], [], []
    for x, g, w, heads in ((st["q"], st.get("gq"), st["qw"], st["heads"]), (st["k"], st.get("gk"), st["kw"], st["kv_heads"])):
        x = x.double().reshape(*x.shape[:2], heads, d).permute(0, 2, 1, 3)
        rms = (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() if w is not None else 1.0
        unit = x / rms
        y = unit * w.double() if w is not None else unit
        a, b = y[..., :half], y[..., half:]
        outs.append(torch.cat([a * c[0] - b * c[2], b * c[1] + a * c[3]], -1))
        if not st["grad"]:
            continue
        ga, gb = g.double()[..., :half], g.double()[..., half:]
        gy = torch.cat([ga * c[0] + gb * c[3], gb * c[1] - ga * c[2]], -1)
        if w is not None:
            weights.append((gy * unit).sum(dim=(0, 1, 2)))
            gy = gy * w.double()
            gy = (gy - unit * (gy * unit).sum(-1, keepdim=True) / d) / rms
        grads.append(gy.permute(0, 2, 1, 3).reshape(*gy.shape[:1], gy.shape[2], heads * d))
    return outs + grads + weights


def _exact_levels(x):
    """The integers and scales of each row in 64 bits, rounded to fp32 where the definition is."""
    top = x.abs().max(-1, keepdim=True).values
    factor = (127.0 / top.clamp_min(1e-30)).float().double()
    return (x * factor).float().round().double(), (top / 127.0)


def exact(case, seed):
    if case["kind"] == "int8":
        w, x, bias, dy = _int8_inputs(case, _Source(seed))
        channels, ws = _exact_levels(w.double())
        ws = ws[:, 0].float().double()
        levels, scale = _exact_levels(x.double())
        y = torch.mm(levels, channels.t().contiguous()) * scale * ws
        if bias is not None:
            y = y + bias.double()
        if dy is None:
            return [y]
        levels, scale = _exact_levels((dy.double() * ws).float().double())
        return [y, torch.mm(levels, channels) * scale]
    st = prepare(case, seed)
    if case["kind"] == "dropout":
        thr = int(torch.tensor(case["p"] * 65536, dtype=torch.float64).round())
        kept = [_exact_bits(st["rng"], case["rows"], case["width"], b) >= thr for b in range(case["branches"])]
        factor = 65536.0 / (65536.0 - thr)
        outs = [st["input"].double() * factor * k for k in kept]
        return [*outs, sum(g.double() * factor * k for g, k in zip(st["grads"], kept))]
    if case["kind"] == "qknorm":
        return _exact_rotation(st, None, st["cos"].double(), st["sin"].double())
    s, pos = st["sections"], st["positions"].double()
    ends = [sum(s[:a + 1]) for a in range(len(s))]
    angle = torch.empty((case["batch"], case["tokens"], sum(s)), dtype=torch.float64, device=pos.device)
    for j in range(sum(s)):
        if case["interleaved"]:
            a = j % len(s) if j // len(s) < s[j % len(s)] else 0
        else:
            a = next(i for i in range(len(s)) if j < ends[i])
        angle[..., j] = pos[a] * float(st["inv_freq"][j])
    return _exact_rotation(st, angle, None, None)
