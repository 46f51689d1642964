"""The new operators together, as an attention layer uses them: frozen 8-bit q/k/v projections, the q and
v LoRA branches with seeded dropout, norms and multi-axis rotation of the heads; forward and backward,
eager and captured."""

import numpy as np
import pytest
import torch

from helpers import assert_close, randn16
from test_dropout_gpu import keep_mask
from test_qk_rope_gpu import axis_table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("x_dtype", [torch.float16, torch.float32])
def test_seeded_pair_is_the_packed_pair(x_dtype, device):
    """LoRAPairSeeded against LoRAPair with the same masks packed, bit for bit (p = 1/4: the same
    scale either way)."""
    from decik_amd.dropout import rng_state
    from decik_amd.lora import LoRAPair, LoRAPairSeeded, pack_keep

    t, w, r, seed, offset, p = 333, 1536, 16, 77, 2 ** 33 + 5, 0.25
    keeps = [torch.from_numpy(keep_mask(t, w, seed, offset + b, p)).to(device) for b in range(2)]
    bits = pack_keep(*keeps)
    scale = torch.full((1,), 1.0 / (1.0 - p), device=device)
    adapters = [randn16(s, i, device, 0.05) for i, s in enumerate(((r, w), (1536, r), (r, w), (256, r)))]
    grads = [randn16((t, n), 10 + n, device, 1e-2) for n in (1536, 256)]
    results = []
    for seeded in (False, True):
        x = randn16((t, w), 5, device).to(x_dtype).requires_grad_(True)
        ab = [a.clone().requires_grad_(True) for a in adapters]
        if seeded:
            outs = LoRAPairSeeded.apply(x, rng_state(seed, offset, device), *ab, 2.0, 1.5, p, p)
        else:
            outs = LoRAPair.apply(x, bits[0], scale, bits[1], scale, *ab, 2.0, 1.5, p, p)
        results.append([*outs, *torch.autograd.grad(outs, [x, *ab], grads)])
    for a, b in zip(*results):
        assert a.shape == b.shape and torch.equal(a.to(b.dtype), b)


def layer(device, tokens=97, hidden=256, heads=4, kv_heads=2, d=64):
    from decik_amd.int8 import quantize_int8

    g = torch.Generator().manual_seed(3)
    rnd = lambda *s, std=1.0: (torch.randn(s, generator=g) * std).to(device)  # noqa: E731
    ns = [heads * d, kv_heads * d, kv_heads * d]
    st = dict(ns=ns, heads=heads, kv_heads=kv_heads, d=d, x=rnd(tokens, hidden).half(),
              w=[quantize_int8(rnd(n, hidden, std=0.05)) for n in ns], bias=[rnd(n, std=0.1).half() for n in ns],
              ab=[rnd(16, hidden, std=0.1).half(), rnd(ns[0], 16, std=0.1).half(), rnd(16, hidden, std=0.1).half(),
                  rnd(ns[2], 16, std=0.1).half()],
              qw=1 + rnd(d, std=0.2), kw=1 + rnd(d, std=0.2), sections=[12, 10, 10],
              pos=torch.randint(0, 40000, (3, tokens), generator=g).to(device),
              inv=(1e6 ** (-torch.arange(0, d, 2).double() / d)).float().to(device), p=(0.125, 0.25),
              grads=[rnd(1, heads, tokens, d, std=1e-2).half(), rnd(1, kv_heads, tokens, d, std=1e-2).half(),
                     rnd(tokens, ns[2], std=1e-2).half()])
    return st


def forward(st, x, rng, ab, qw, kw):
    from decik_amd.int8 import Int8Linear
    from decik_amd.lora import LoRAPairSeeded
    from decik_amd.rope import axes_rope

    q, k, v = (Int8Linear.apply(x, *w, b) for w, b in zip(st["w"], st["bias"]))
    lq, lv = LoRAPairSeeded.apply(x, rng, *ab, 2.0, 2.0, *st["p"])
    q, v = q + lq, v + lv
    qr, kr = axes_rope(q, k, st["pos"], st["inv"], st["sections"], st["heads"], st["kv_heads"], True, qw, kw)
    return qr, kr, v


def test_attention_inputs(device):
    """Against the chain in 64 bits with the same fp16 roundings between the operators; the bar is the
    framework's (1e-2 of the largest value, 1e-3 of the sum): fp32 against fp64 flips single fp16
    roundings between operators, which the norms and products spread."""
    from decik_amd.dropout import rng_state

    st = layer(device)
    seed, offset = 11, 6
    leaves = [st["x"].clone(), *[a.clone() for a in st["ab"]], st["qw"].clone(), st["kw"].clone()]
    for t in leaves:
        t.requires_grad_(True)
    outs = forward(st, leaves[0], rng_state(seed, offset, device), leaves[1:5], leaves[5], leaves[6])
    got = torch.autograd.grad(outs, leaves, st["grads"])

    # the reference on the CPU: quantization passes gradients on, fp16 roundings pass them on too
    c = lambda t: t.detach().double().cpu()  # noqa: E731
    ref = [c(t).requires_grad_(True) for t in leaves]
    half = lambda t: t + (t.detach().half().double() - t.detach())  # noqa: E731
    x = ref[0]
    rows = x.detach().float()
    top = rows.abs().amax(1, keepdim=True)
    xq = torch.round(rows * (torch.full_like(top, 127) / top)).double() * (top / torch.full_like(top, 127)).double()
    xhat = x + (xq - x.detach())
    q, k, v = (half(xhat @ (c(w) * c(s)[:, None]).t() + c(b)) for (w, s), b in zip(st["w"], st["bias"]))
    loras = []
    for b, (a_i, b_i, p) in enumerate(((1, 2, st["p"][0]), (3, 4, st["p"][1]))):
        keep = torch.from_numpy(keep_mask(*x.shape, seed, offset + b, p))
        xd = half(x * keep / (1 - p))
        loras.append(half(half(half(xd @ ref[a_i].t()) @ ref[b_i].t()) * 2.0))
    q, v = half(q + loras[0]), half(v + loras[1])
    angle = c(st["pos"])[axis_table(st["sections"], True)].t() * c(st["inv"])
    cos, sin = (f(torch.cat([angle, angle], -1))[None] for f in (torch.cos, torch.sin))
    want = []
    for t, w, h in ((q, ref[5], st["heads"]), (k, ref[6], st["kv_heads"])):
        t = t.reshape(-1, h, st["d"]).transpose(0, 1)
        n = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w
        lo, hi = n.chunk(2, -1)
        want.append((n * cos + torch.cat([-hi, lo], -1) * sin)[None])
    want.append(v)
    expect = torch.autograd.grad(want, ref, [c(g) for g in st["grads"]])
    for o, w in zip(outs, want):
        assert_close(o, w.detach().numpy(), what="out")
    for i, (g, w) in enumerate(zip(got, expect)):
        # the 8-bit gradient of x: each of its three terms is off by at most half a step of its row
        if i == 0:
            assert g.dtype == torch.float16
            err, size = (g.double().cpu() - w).norm(), w.norm()
            assert err <= 0.02 * size
        else:
            assert_close(g, w.numpy(), max_rel=1e-2, mean_rel=2e-3, what=f"grad {i}")


def test_captured_layer_steps(device):
    """The layer's forward and backward captured once; replays with other masks and inputs equal the eager
    step, with eager work between them."""
    from decik_amd.dropout import rng_state

    st = layer(device, tokens=64)

    def make_leaves():
        leaves = [st["x"].clone(), *[a.clone() for a in st["ab"]], st["qw"].clone(), st["kw"].clone()]
        return [t.requires_grad_(True) for t in leaves]

    def step(leaves, rng):
        outs = forward(st, leaves[0], rng, leaves[1:5], leaves[5], leaves[6])
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, st["grads"]))

    rng = rng_state(1, 0, device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = make_leaves()
        step(warm, rng)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    captured = make_leaves()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(captured, rng)
    for i in range(4):
        with torch.no_grad():
            rng[1] += 2
            captured[0] += 0.0625
        graph.replay()
        torch.cuda.synchronize()
        eager = make_leaves()
        with torch.no_grad():
            eager[0].copy_(captured[0])
        want = step(eager, rng)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results, want))
        assert not torch.equal(results[0], results[0] * 0)


def test_second_derivatives_are_refused(device):
    """A gradient taken with create_graph is right, and differentiating it again raises instead of leaving
    the operators' part out."""
    from decik_amd.dropout import rng_state, seeded_dropout
    from decik_amd.int8 import Int8Linear, quantize_int8
    from decik_amd.lora import LoRAPairSeeded
    from decik_amd.rope import axes_rope

    rng = rng_state(1, 0, device)
    ab = [randn16(s, i, device, 0.05) for i, s in enumerate(((16, 64), (64, 16), (16, 64), (64, 16)))]
    w = quantize_int8(randn16((64, 64), 8, device))
    pos, inv = torch.arange(8, device=device)[None], torch.ones(16, device=device)
    calls = {
        "dropout": lambda x: seeded_dropout(x, rng, 0.25),
        "pair": lambda x: LoRAPairSeeded.apply(x, rng, *ab, 2.0, 2.0, 0.25, 0.25)[0],
        "rotation": lambda x: axes_rope(x, x, pos, inv, [16], 2, 2)[0],
        "int8": lambda x: Int8Linear.apply(x, *w),
    }
    for name, call in calls.items():
        x = randn16((8, 64), 9, device).requires_grad_(True)
        y = call(x)
        loss = (y.float() ** 2).sum()
        once = torch.autograd.grad(loss, x, retain_graph=True)[0]
        again = torch.autograd.grad(loss, x, create_graph=True)[0]
        assert torch.equal(once, again.detach()), name
        with pytest.raises(RuntimeError, match="twice"):
            (again.float() ** 2).sum().backward()


def test_seeded_pair_edges(device):
    """No tokens, one token, a middle axis, views; adapters that do not fit are refused."""
    from decik_amd.dropout import rng_state
    from decik_amd.lora import LoRAPairSeeded

    w, r, rng = 64, 16, rng_state(1, 0, device)
    ab = [randn16(s, i, device, 0.05).requires_grad_(True) for i, s in enumerate(((r, w), (48, r), (r, w), (32, r)))]
    for shape in ((0, w), (2, 0, w), (1, w), (2, 3, w)):
        x = randn16(shape, 5, device).requires_grad_(True)
        q, v = LoRAPairSeeded.apply(x, rng, *ab, 2.0, 2.0, 0.5, 0.25)
        assert q.shape == (*shape[:-1], 48) and v.shape == (*shape[:-1], 32)
        grads = torch.autograd.grad(q.float().sum() + v.float().sum(), [x, *ab])
        for g, t in zip(grads, [x, *ab]):
            assert g.shape == t.shape and g.dtype == t.dtype and bool(g.isfinite().all())
            assert x.numel() > 0 or not bool(g.any())
    x = randn16((6, 2 * w), 6, device)
    for view in (x[:, w:], x[::2, :w], x[:, ::2]):
        outs = [LoRAPairSeeded.apply(t, rng, *ab, 2.0, 2.0, 0.5, 0.25) for t in (view, view.contiguous())]
        assert all(torch.equal(a, b) for a, b in zip(*outs))
    x = x[:, :w]
    for bad in ([ab[0][:, :32], *ab[1:]], [ab[0][:8], ab[1][:, :8], ab[2][:8], ab[3][:, :8]], [*ab[:3], ab[3][:, :8]],
                [*ab[:2], torch.cat([ab[2]] * 2), torch.cat([ab[3]] * 2, 1)], [ab[0].cpu(), *ab[1:]]):
        with pytest.raises(ValueError):
            LoRAPairSeeded.apply(x, rng, *bad, 2.0, 2.0, 0.5, 0.25)
    for args in ((x.bfloat16(), rng), (x.cpu(), rng), (x, rng.cpu())):
        with pytest.raises(ValueError):
            LoRAPairSeeded.apply(*args, *ab, 2.0, 2.0, 0.5, 0.25)
