"""The residual stream's norms, the scaled rotation and the 4-bit linears together, as a decoder layer uses them: norm,
q/k/v, rotation, attention, o, join with the norm after the block and the gate, gate/up, SwiGLU, down, join; forward and
backward, a token at a time, eager and captured, on two streams."""

import pytest
import torch

from helpers import assert_close, randn16

pytestmark = pytest.mark.gpu
EPS = 1e-6


def layer(device, tokens=97, hidden=256, heads=4, kv_heads=2, d=64, inter=384):
    from decik_amd.int4 import quantize_int4
    from decik_amd.rope import scaled_frequencies

    g = torch.Generator().manual_seed(5)
    rnd = lambda *s, std=1.0: (torch.randn(s, generator=g) * std).to(device)  # noqa: E731
    shapes = dict(q=(heads * d, hidden), k=(kv_heads * d, hidden), v=(kv_heads * d, hidden), o=(hidden, heads * d),
                  gate=(inter, hidden), up=(inter, hidden), down=(hidden, inter))
    inv, factor = scaled_frequencies(32, 1e6, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096),
                                     device=device)
    return dict(heads=heads, kv_heads=kv_heads, d=d, x=rnd(1, tokens, hidden), inv=inv, factor=factor, start=5000,
                w={n: quantize_int4(rnd(*s, std=s[1] ** -0.5), 64) for n, s in shapes.items()},
                # norms before and after each block and the gates of the joins, all trained
                leaves=[1 + rnd(hidden, std=0.2) for _ in range(5)] + [torch.sigmoid(rnd(hidden)) for _ in range(2)],
                grads=[rnd(1, tokens, hidden, std=1e-2), rnd(1, tokens, hidden, std=1e-2).half()])


def attend(q, k, v):
    """Causal attention of q [1, H, T, D] over the last T of k, v [1, HK, S, D] in fp32 (fp64 where they are)."""
    h, hk, t, s = q.shape[1], k.shape[1], q.shape[2], k.shape[2]
    wide = (lambda z: z) if q.dtype == torch.float64 else (lambda z: z.float())  # noqa: E731
    kk, vv = (wide(z).repeat_interleave(h // hk, 1)[0] for z in (k, v))
    score = torch.bmm(wide(q)[0], kk.transpose(1, 2).contiguous()) * q.shape[-1] ** -0.5
    mask = torch.ones(t, s, dtype=torch.bool, device=q.device).tril(s - t)
    p = torch.softmax(score.masked_fill(~mask, float("-inf")), -1)
    return torch.bmm(p, vv).to(q.dtype)[None]


def run(st, x, leaves, past=None, start=None):
    """(stream, normed stream, keys and values) of tokens x [1, T, W], an fp32 stream."""
    from decik_amd.int4 import Int4Linear
    from decik_amd.norm import residual_norm, rms_norm
    from decik_amd.rope import scaled_rope
    from decik_amd.swiglu import SwiGLU

    w, (n1, post1, n2, post2, n3, g1, g2) = st["w"], leaves
    t, d = x.shape[1], st["d"]
    y = rms_norm(x, n1, EPS).half()
    q, k, v = (Int4Linear.apply(y, w[n]) for n in "qkv")
    pos = torch.arange(t, device=x.device) + (st["start"] if start is None else start)
    q, k = scaled_rope(q, k, pos, st["inv"], st["heads"], st["kv_heads"], "pairs", st["factor"])
    v = v.unflatten(-1, (-1, d)).transpose(1, 2)
    if past is not None:
        k, v = torch.cat([past[0], k], 2), torch.cat([past[1], v], 2)
    a = attend(q, k, v).transpose(1, 2).flatten(2)
    h, y = residual_norm(Int4Linear.apply(a, w["o"]), x, n2, post1, g1, 1.0, EPS)
    m = SwiGLU.apply(Int4Linear.apply(y, w["gate"]), Int4Linear.apply(y, w["up"]))
    h, y = residual_norm(Int4Linear.apply(m, w["down"]), h, n3, post2, g2, 1.0, EPS)
    return h, y, (k, v)


def make_leaves(st):
    return [t.clone().requires_grad_(True) for t in (st["x"], *st["leaves"])]


def step(st, leaves):
    h, y, _ = run(st, leaves[0], leaves[1:])
    return [h.detach(), y.detach(), *torch.autograd.grad([h, y], leaves, st["grads"])]


def test_layer(device):
    """Against the chain in 64 bits with the same fp16 roundings between the operators; the bar is the framework's
    (1e-2 of the largest value, 1e-3 of the sum, gradients 2e-3): fp32 against fp64 flips single fp16 roundings between
    operators, which norms and products spread."""
    from decik_amd.int4 import dequantize_int4

    st = layer(device)
    got = step(st, make_leaves(st))
    c = lambda t: t.detach().double().cpu()  # noqa: E731
    ref = [c(t).requires_grad_(True) for t in (st["x"], *st["leaves"])]
    half = lambda t: t + (t.detach().half().double() - t.detach())  # noqa: E731
    w = {n: c(dequantize_int4(q)) for n, q in st["w"].items()}
    x, n1, post1, n2, post2, n3, g1, g2 = ref
    unit = lambda t: t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)  # noqa: E731
    y = half(unit(x) * n1)
    q, k, v = (half(y @ w[n].t()).unflatten(-1, (-1, st["d"])).transpose(1, 2) for n in "qkv")
    angle = (torch.arange(x.shape[1]) + st["start"]).double()[:, None] * c(st["inv"])
    turn = torch.polar(torch.full_like(angle, st["factor"]), angle)

    def turned(t):
        z = torch.view_as_complex(t[..., :32].unflatten(-1, (-1, 2)).contiguous()) * turn
        return half(torch.cat([torch.view_as_real(z).flatten(-2), t[..., 32:]], -1))

    a = half(attend(turned(q), turned(k), v)).transpose(1, 2).flatten(2)
    h = x + g1 * (unit(half(a @ w["o"].t())) * post1)
    y = half(unit(h) * n2)
    gate, up = (half(y @ w[n].t()) for n in ("gate", "up"))
    h = h + g2 * (unit(half(half(torch.nn.functional.silu(gate) * up) @ w["down"].t())) * post2)
    y = half(unit(h) * n3)
    want = [h, y, *torch.autograd.grad([h, y], ref, [c(t) for t in st["grads"]])]
    for i, (a, b) in enumerate(zip(got, want)):
        assert_close(a, b.detach().numpy(), max_rel=1e-2, mean_rel=1e-3 if i < 2 else 2e-3, what=str(i))


def test_a_token_at_a_time(device):
    """Single tokens with the keys and values of those before give the rows of the whole sequence."""
    st = layer(device, tokens=9)
    with torch.no_grad():
        h, y, _ = run(st, st["x"], st["leaves"])
        past = None
        for t in range(9):
            ht, yt, past = run(st, st["x"][:, t:t + 1], st["leaves"], past, st["start"] + t)
            assert_close(ht[0, 0], h[0, t].float().cpu().numpy(), what=f"stream {t}")
            assert_close(yt[0, 0], y[0, t].float().cpu().numpy(), what=f"output {t}")


@pytest.mark.parametrize("tokens", [1, 8, 70])
def test_captured_steps(tokens, device):
    """Forward and backward captured once; replays on other inputs equal the eager step, with eager work between them."""
    st = layer(device, tokens=tokens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(st, make_leaves(st))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    captured = make_leaves(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(st, captured)
    for _ in range(4):
        with torch.no_grad():
            captured[0] += 0.0625
        graph.replay()
        torch.cuda.synchronize()
        eager = make_leaves(st)
        with torch.no_grad():
            eager[0].copy_(captured[0])
        want = step(st, eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results, want))


def test_two_streams(device):
    """Each call has its own workspace and runs on its caller's stream: every result is that of a call alone, bit for bit."""
    from decik_amd.int4 import int4_linear_backward, int4_linear_forward, quantize_int4
    from decik_amd.norm import residual_norm_backward, residual_norm_forward
    from decik_amd.rope import scaled_rope_backward, scaled_rope_forward

    x, res, g = randn16((830, 1001), 1, device), randn16((830, 1001), 2, device), randn16((830, 1001), 3, device)
    nw = [randn16((1001,), 4 + i, device).float() for i in range(3)]
    w = quantize_int4(randn16((700, 1001), 7, device, 0.02), 32)
    dy = randn16((830, 700), 8, device)
    inv, pos = torch.rand(20, device=device), torch.arange(830, device=device)
    qk = randn16((830, 720), 9, device)

    def call():
        outs = scaled_rope_forward(qk, qk[:, :240], pos, inv, 9, 3)
        return [*residual_norm_forward(x, res, *nw), *residual_norm_backward(res, g, x, res, *nw), *outs,
                *scaled_rope_backward(*outs, pos, inv), int4_linear_forward(x, w), int4_linear_forward(x[:5], w),
                int4_linear_backward(dy, w)]

    want = call()
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(call())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_second_derivatives_are_refused(device):
    """A gradient taken with create_graph is right, and differentiating it again raises."""
    from decik_amd.int4 import Int4Linear, quantize_int4
    from decik_amd.norm import residual_norm, rms_norm
    from decik_amd.rope import scaled_rope

    w, one = quantize_int4(randn16((64, 64), 8, device), 32), torch.ones(64, device=device)
    pos, inv = torch.arange(8, device=device), torch.ones(16, device=device)
    calls = dict(int4=lambda x: Int4Linear.apply(x, w), norm=lambda x: residual_norm(x, x, one, one)[1],
                 alone=lambda x: rms_norm(x, one), rotation=lambda x: scaled_rope(x, x, pos, inv, 2, 2)[0])
    for name, call in calls.items():
        x = randn16((8, 64), 9, device).requires_grad_(True)
        loss = (call(x).float() ** 2).sum()
        once = torch.autograd.grad(loss, x, retain_graph=True)[0]
        again = torch.autograd.grad(loss, x, create_graph=True)[0]
        assert torch.equal(once, again.detach()), name
        with pytest.raises(RuntimeError, match="twice"):
            (again.float() ** 2).sum().backward()


def test_far_offsets(device):
    """Rows 2^31 elements apart, and outputs of more than 2^32 elements, give what few rows close together give."""
    from decik_amd.int4 import int4_linear_backward, int4_linear_forward, quantize_int4
    from decik_amd.norm import residual_norm_backward, residual_norm_forward
    from decik_amd.rope import scaled_rope_backward, scaled_rope_forward
    from test_int4_gpu import check_backward, values

    far = 2 ** 31

    def apart(t):
        view = torch.empty((t.shape[0] - 1) * far + t.shape[1], dtype=t.dtype, device=device).as_strided(t.shape, (far, 1))
        return view.copy_(t)

    x, one = randn16((3, 256), 1, device), torch.ones(256, device=device)
    y = apart(x)
    w = quantize_int4(randn16((256, 256), 2, device), 64)
    inv, pos = torch.rand(24, device=device), torch.arange(3, device=device)
    head = lambda t: t[None].unflatten(-1, (4, 64)).transpose(1, 2)  # noqa: E731
    pairs = [(residual_norm_forward(t, t, one, one, t) + residual_norm_backward(t, t, t, t, one, one, t)
              + scaled_rope_forward(t, t, pos, inv, 4, 4) + scaled_rope_backward(head(t), head(t), pos, inv, "pairs")
              + (int4_linear_forward(t, w), int4_linear_backward(t, w))) for t in (x, y)]
    assert all(torch.equal(a, b) for a, b in zip(*pairs))
    del y, pairs
    t, d = 2 ** 23 + 5, 256
    q = randn16((2 * d,), 1, device).expand(t, 2 * d)
    pos, inv = torch.arange(t, dtype=torch.int32, device=device), torch.rand(100, device=device)
    big = scaled_rope_forward(q, q[:, :d], pos, inv, 2, 1)
    assert big[0].numel() > 2 ** 32
    few = scaled_rope_forward(q[-3:], q[-3:, :d], pos[-3:], inv, 2, 1)
    assert all(torch.equal(a[:, :, -3:], b) for a, b in zip(big, few))
    back = scaled_rope_backward(*big, pos, inv)
    assert all(torch.equal(a[:, -3:], b) for a, b in zip(back, scaled_rope_backward(*few, pos[-3:], inv)))
    del big, back
    m, n, k = 2 ** 18 + 1, 16400, 40
    x, w = randn16((m, k), 1, device), quantize_int4(randn16((n, k), 2, device), 32)
    y = int4_linear_forward(x, w)
    assert y.numel() > 2 ** 32 and torch.equal(y[-300:], int4_linear_forward(x[-300:], w))
    dx = int4_linear_backward(y, w)  # (few rows split its sum, which orders it otherwise)
    check_backward(dx[-300:], y[-300:], values(w.codes(), w.scales, w.zeros, 32))
