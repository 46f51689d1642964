"""Norms of q and k heads with the rotation, and rotary positions with several axes
(decik_amd.rope.qk_norm_rope_*, axes_rope_*) against the formulas in 64 bits: values and gradients,
types, head sizes and counts, strides, batches, far positions, one token and none.

Tolerances. With |y|' = |y_a| + |y_b| of a pair, an output is two products and a sum: every fp32 rounding
before the last is within 2^-24 of |y|', a norm adds fewer than 40 of them (sums of up to 32 + 5 terms a
row, the root, two products), formed angles 2^-21 |y|': in all within 2^-18 |y|', then one rounding to
the output type (half a step, eps / 2). dx = r (n w - f mean(n w f)): the same over twice the operations,
2^-17 of r (|n w|' + |f| mean |n w f|). dw: sums of fewer than 256 terms in any chain, 2^-16 of the sum of
magnitudes."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}


def make(shape, dtype, device, seed, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std + mean).to(dtype).to(device)


def pairs(x):
    """[.., D] -> complex [.., D / 2] with the halves as real and imaginary parts."""
    half = x.shape[-1] // 2
    return x[..., :half], x[..., half:]


def both(t):
    return np.concatenate([t, t], -1)


def reference(x, g, w, cos, sin, heads, eps):
    """x [B, T, H*D], g [B, H, T, D] or None, w [D] or None, cos and sin [B, T, D], float64 numpy.
    Returns dict of (value, magnitude) of out, dx, dw."""
    b, t, _ = x.shape
    d = cos.shape[-1]
    x = x.reshape(b, t, heads, d).transpose(0, 2, 1, 3)
    cos, sin = cos[:, None], sin[:, None]
    (ca, cb), (sa, sb) = pairs(cos), pairs(sin)
    r = 1.0 if w is None else 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    f = x * r
    y = f if w is None else f * w
    ya, yb = pairs(y)
    res = dict(out=(np.concatenate([ya * ca - yb * sa, yb * cb + ya * sb], -1), both(abs(ya) + abs(yb))))
    if g is not None:
        ga, gb = pairs(g)
        n = np.concatenate([ga * ca + gb * sb, gb * cb - ga * sa], -1)
        nmag = both(abs(ga) + abs(gb))
        if w is None:
            dx, mag = n, nmag
        else:
            nw = n * w
            dx = r * (nw - f * (nw * f).mean(-1, keepdims=True))
            mag = r * (nmag * abs(w) + abs(f) * (nmag * abs(w) * abs(f)).mean(-1, keepdims=True))
            res["dw"] = ((n * f).sum((0, 1, 2)), (nmag * abs(f)).sum((0, 1, 2)))
        back = lambda v: v.transpose(0, 2, 1, 3).reshape(b, t, heads * d)  # noqa: E731
        res["dx"] = (back(dx), back(mag))
    return res


def check(got, want, rel, what):
    value, mag = (torch.from_numpy(np.ascontiguousarray(v)) for v in want)
    err = (got.double().cpu() - value).abs()
    bound = value.abs() * (torch.finfo(got.dtype).eps / 2) + mag * rel + TINY[got.dtype]
    assert got.shape == value.shape, what
    assert bool((err <= bound).all()), f"{what}: worst excess {(err - bound).max().item():.3e}"


def f64(t):
    return t.detach().double().cpu().numpy()


def axis_table(sections, interleaved):
    n = len(sections)
    if interleaved:
        return [j % n if j < n * sections[j % n] else 0 for j in range(sum(sections))]
    return [a for a, s in enumerate(sections) for _ in range(s)]


def inputs(b, t, h, hk, d, dtype, device, seed=0):
    qkv = make((b, t, (h + 2 * hk) * d), dtype, device, seed)
    q, k = qkv[..., :h * d], qkv[..., h * d:(h + hk) * d]
    return q, k, make((b, h, t, d), dtype, device, seed + 1, 1e-2), make((b, hk, t, d), dtype, device, seed + 2, 1e-2)


def check_all(outs, grads, q, k, gq, gk, qw, kw, cos, sin, h, hk, eps):
    for side, x, g, w, heads, i in (("q", q, gq, qw, h, 0), ("k", k, gk, kw, hk, 1)):
        ref = reference(f64(x), f64(g), None if w is None else f64(w), cos, sin, heads, eps)
        check(outs[i], ref["out"], 2.0 ** -18, f"{side} out")
        check(grads[i], ref["dx"], 2.0 ** -17, f"d{side}")
        if w is not None:
            check(grads[2 + i], ref["dw"], 2.0 ** -16, f"d{side}_weight")
    if qw is None:
        assert grads[2] is None and grads[3] is None


SHAPES = [(1, 1, 28, 4, 128), (16, 1, 28, 4, 128), (1, 830, 12, 2, 128), (3, 33, 5, 5, 64), (2, 65, 9, 3, 80),
          (1, 70, 3, 1, 96), (1, 9, 2, 1, 16), (2, 31, 4, 2, 256), (1, 40, 3, 2, 512), (1, 25, 7, 1, 48)]


@pytest.mark.parametrize("b,t,h,hk,d", SHAPES)
@pytest.mark.parametrize("dtype,w_dtype", [(torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                           (torch.float16, torch.float16)])
def test_norm_rope(b, t, h, hk, d, dtype, w_dtype, device):
    from decik_amd.rope import qk_norm_rope_backward, qk_norm_rope_forward

    q, k, gq, gk = inputs(b, t, h, hk, d, dtype, device)
    qw, kw = make((d,), w_dtype, device, 5, 0.3, 1.0), make((d,), w_dtype, device, 6, 0.3, 1.0)
    # tables whose halves differ, other angles in each batch entry
    angle = make((b, t, d), torch.float32, device, 7, 3.0)
    cos, sin = angle.cos(), angle.sin()
    outs = qk_norm_rope_forward(q, k, qw, kw, cos, sin, h, hk, 1e-5)
    grads = qk_norm_rope_backward(gq, gk, q, k, qw, kw, cos, sin, 1e-5)
    check_all(outs, grads, q, k, gq, gk, qw, kw, f64(cos), f64(sin), h, hk, 1e-5)


@pytest.mark.parametrize("b,t,h,hk,d", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_axes_rope(b, t, h, hk, d, interleaved, norm, device):
    from decik_amd.rope import axes_rope_backward, axes_rope_forward

    dtype = torch.bfloat16 if interleaved else torch.float16
    q, k, gq, gk = inputs(b, t, h, hk, d, dtype, device)
    qw, kw = (make((d,), torch.float32, device, 5 + i, 0.3, 1.0) for i in range(2)) if norm else (None, None)
    side = d // 2 // 3
    sections = [d // 2 - 2 * side, side, side]
    gen = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 2 ** 20, (3, b, t), generator=gen)
    inv = (1e6 ** (-torch.arange(0, d, 2).double() / d)).float().to(device)
    outs = axes_rope_forward(q, k, pos.to(device), inv, sections, h, hk, interleaved, qw, kw)
    grads = axes_rope_backward(gq, gk, pos.to(device), inv, sections, interleaved, q, k, qw, kw)
    angle = pos.numpy()[axis_table(sections, interleaved)].transpose(1, 2, 0).astype(np.float64) * f64(inv)
    check_all(outs, grads, q, k, gq, gk, qw, kw, both(np.cos(angle)), both(np.sin(angle)), h, hk, 1e-6)


def test_many_tokens_a_wave(device):
    """More tokens than waves, so that a wave walks several, and norm gradients over slabs."""
    from decik_amd.rope import qk_norm_rope_backward, qk_norm_rope_forward

    b, t, h, hk, d = 2, 2900, 6, 2, 64
    q, k, gq, gk = inputs(b, t, h, hk, d, torch.float16, device)
    qw, kw = make((d,), torch.float32, device, 5, 0.3, 1.0), make((d,), torch.float32, device, 6, 0.3, 1.0)
    angle = make((t, d), torch.float32, device, 7, 3.0)
    cos, sin = angle.cos(), angle.sin()
    outs = qk_norm_rope_forward(q, k, qw, kw, cos, sin, h, hk)
    grads = qk_norm_rope_backward(gq, gk, q, k, qw, kw, cos, sin)
    shared = [np.broadcast_to(f64(v), (b, t, d)) for v in (cos, sin)]
    check_all(outs, grads, q, k, gq, gk, qw, kw, *shared, h, hk, 1e-6)
    again = qk_norm_rope_backward(gq, gk, q, k, qw, kw, cos, sin)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


@pytest.mark.parametrize("sections", [[64], [32, 32], [16, 16, 16, 16], [0, 64], [64, 0, 0], [40, 1, 23]])
@pytest.mark.parametrize("interleaved", [False, True])
def test_sections(sections, interleaved, device):
    from decik_amd._lib import DecikError
    from decik_amd.rope import axes_rope_forward

    d, n = 128, len(sections)
    table = axis_table(sections, interleaved)
    q, k, _, _ = inputs(1, 5, 2, 1, d, torch.float16, device)
    pos = torch.arange(5 * n).reshape(n, 5) * 37 - 11  # negative positions too
    inv = torch.rand(d // 2, generator=torch.Generator().manual_seed(1)).to(device)
    call = lambda p: axes_rope_forward(q, k, p.to(device), inv, sections, 2, 1, interleaved)  # noqa: E731
    if [table.count(a) for a in range(n)] != sections:
        with pytest.raises(DecikError, match="more frequencies"):
            call(pos)
        return
    angle = pos.numpy()[table].T[None].astype(np.float64) * f64(inv)
    ref = reference(f64(q), None, None, both(np.cos(angle)), both(np.sin(angle)), 2, 0)
    check(call(pos)[0], ref["out"], 2.0 ** -18, "q")
    assert torch.equal(call(pos)[0], call(pos.to(torch.int32))[0])


def test_far_positions(device):
    """Angles of positions up to 2^31: the fixed-point fraction keeps them where fp32 products could
    not (one step of fp32 at 2^31 radians is 256)."""
    from decik_amd.rope import axes_rope_forward

    d, t = 64, 6
    q, k, _, _ = inputs(1, t, 2, 1, d, torch.float16, device)
    pos = torch.tensor([[0, 1, 2 ** 20 + 1, 2 ** 24 + 1, 2 ** 28 - 1, 2 ** 31 - 1]])
    inv = (1e4 ** (-torch.arange(0, d, 2).double() / d)).float().to(device)
    out = axes_rope_forward(q, k, pos.to(device), inv, [d // 2], 2, 1)[0]
    # positions times 24-bit frequencies need 55 bits: the reference angle in extended precision
    angle = (pos.numpy()[0][:, None].astype(np.longdouble) * f64(inv).astype(np.longdouble))[None]
    cos, sin = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
    ref = reference(f64(q), None, None, both(cos), both(sin), 2, 0)
    # the fraction's error, 2^-55 turns a position at most: 2^-24 turns = 2^-21 radians at 2^31
    check(out, ref["out"], 2.0 ** -18, "q")


@pytest.mark.parametrize("freq", [-1.0, -1e-3, -2.0 ** -40, -1e-30, 1e-30, 0.0])
def test_signs_of_frequencies(freq, device):
    """Negative frequencies turn the other way, tiny ones not at all."""
    from decik_amd.rope import axes_rope_forward

    d, t = 64, 5
    q, k, _, _ = inputs(1, t, 2, 1, d, torch.float16, device)
    pos = torch.tensor([[0, 1, 77, 2 ** 20, 2 ** 28]])
    inv = torch.full((d // 2,), freq, dtype=torch.float32, device=device)
    out = axes_rope_forward(q, k, pos.to(device), inv, [d // 2], 2, 1)[0]
    angle = (pos.numpy()[0][:, None].astype(np.longdouble) * f64(inv).astype(np.longdouble))[None]
    cos, sin = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
    ref = reference(f64(q), None, None, both(cos), both(sin), 2, 0)
    # the fraction's error, 2^-54 turns a position at most: 2^-26 turns = 2^-23 radians at 2^28
    check(out, ref["out"], 2.0 ** -18, "q")


def test_strides(device):
    from decik_amd.rope import axes_rope_forward, qk_norm_rope_backward, qk_norm_rope_forward

    h, hk, d, t = 3, 1, 32, 10
    big = make((2, t, 2 * 5 * d + 3), torch.float16, device, 1)
    qw, kw = make((d,), torch.float32, device, 5, 0.3, 1.0), make((d,), torch.float32, device, 6, 0.3, 1.0)
    angle = make((t, d), torch.float32, device, 7, 3.0)
    cos, sin = angle.cos(), angle.sin()
    views = [(big[..., 1:1 + h * d], big[..., 101:101 + hk * d]),           # odd row stride, odd start
             (big[:, ::2, :h * d][:, :5], big[:, ::2, -hk * d:][:, :5]),    # every other token
             (big[:1, 0, :h * d], big[:1, 0, 100:100 + hk * d]),            # one row
             (big[:, :1, :h * d], big[:, :1, 99:99 + hk * d]),              # one token a sequence, far apart
             (big[0].t()[:h * d].t(), big[1].t()[:hk * d].t()),
             (big[..., :2 * h * d:2], big[..., :2 * hk * d:2]),             # no unit stride
             (big[:1, :, :h * d].expand(2, t, h * d), big[..., :hk * d])]   # a shared q
    for q, k in views:
        n = q.shape[-2]
        want = qk_norm_rope_forward(q.contiguous(), k.contiguous(), qw, kw, cos[:n], sin[:n], h, hk)
        got = qk_norm_rope_forward(q, k, qw, kw, cos[:n], sin[:n], h, hk)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        gq, gk = torch.randn_like(got[0]), torch.randn_like(got[1])
        got = qk_norm_rope_backward(gq.transpose(1, 2).contiguous().transpose(1, 2), gk, q, k, qw, kw, cos[:n], sin[:n])
        want = qk_norm_rope_backward(gq, gk, q.contiguous(), k.contiguous(), qw, kw, cos[:n], sin[:n])
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    pos = torch.randint(0, 999, (2, t, 3), device=device).permute(2, 0, 1)  # tokens not contiguous
    inv = torch.rand(d // 2, device=device)
    q, k = views[0]
    got = axes_rope_forward(q, k, pos, inv, [8, 4, 4], h, hk)
    want = axes_rope_forward(q, k, pos.contiguous(), inv, [8, 4, 4], h, hk)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_special_rows(device):
    """A row of zeros keeps finite values; infinities and NaN stay in their own head rows."""
    from decik_amd.rope import qk_norm_rope_backward, qk_norm_rope_forward

    h, hk, d, t = 4, 2, 64, 5
    q, k, gq, gk = inputs(1, t, h, hk, d, torch.float16, device)
    q, k = q.clone(), k.clone()
    qw, kw = make((d,), torch.float32, device, 5, 0.3, 1.0), make((d,), torch.float32, device, 6, 0.3, 1.0)
    angle = make((t, d), torch.float32, device, 7, 3.0)
    args = (qw, kw, angle.cos(), angle.sin())
    clean = qk_norm_rope_forward(q, k, *args, h, hk)
    dclean = qk_norm_rope_backward(gq, gk, q, k, *args)
    q[0, 1, :d], q[0, 2, d + 3], k[0, 3, 7] = 0, float("nan"), float("inf")
    out = qk_norm_rope_forward(q, k, *args, h, hk)
    dout = qk_norm_rope_backward(gq, gk, q, k, *args)
    assert bool((out[0][0, 0, 1] == 0).all()) and bool(torch.isfinite(dout[0][0, 1, :d]).all())
    assert bool(torch.isnan(out[0][0, 1, 2]).all()) and not bool(torch.isfinite(out[1][0, 0, 3]).all())
    same = torch.ones((h, t), dtype=torch.bool, device=device)
    same[0, 1] = same[1, 2] = False
    assert torch.equal(out[0][0][same], clean[0][0][same])
    assert torch.equal(dout[0].reshape(t, h, d).transpose(0, 1)[same], dclean[0].reshape(t, h, d).transpose(0, 1)[same])


def test_no_tokens(device):
    from decik_amd.rope import axes_rope_forward, qk_norm_rope_backward, qk_norm_rope_forward

    w, e = torch.ones(32, device=device), lambda *s: torch.empty(s, dtype=torch.float16, device=device)  # noqa: E731
    tab = torch.empty((0, 32), device=device)
    q, k = qk_norm_rope_forward(e(1, 0, 64), e(1, 0, 32), w, w, tab, tab, 2, 1)
    assert q.shape == (1, 2, 0, 32) and k.shape == (1, 1, 0, 32)
    g = qk_norm_rope_backward(e(1, 2, 0, 32), e(1, 1, 0, 32), e(1, 0, 64), e(1, 0, 32), w, w, tab, tab)
    assert g[0].shape == (1, 0, 64) and bool((g[2] == 0).all()) and bool((g[3] == 0).all())
    pos = torch.empty((1, 0), dtype=torch.int64, device=device)
    assert axes_rope_forward(e(0, 64), e(0, 32), pos, w[:16], [16], 2, 1)[0].shape == (1, 2, 0, 32)


@pytest.mark.parametrize("kind", ["tables", "axes", "axes_norm"])
def test_autograd(kind, device):
    from decik_amd.rope import (axes_rope, axes_rope_backward, qk_norm_rope, qk_norm_rope_backward)

    b, t, h, hk, d = 2, 7, 4, 2, 32
    q, k, gq, gk = inputs(b, t, h, hk, d, torch.bfloat16, device)
    q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    qw, kw = (make((d,), torch.bfloat16, device, 5 + i, 0.3, 1.0).requires_grad_(True) for i in range(2))
    angle = make((t, d), torch.float32, device, 7, 3.0)
    pos, inv = torch.randint(0, 99, (2, t), device=device), torch.rand(d // 2, device=device)
    if kind == "tables":
        outs = qk_norm_rope(q, k, qw, kw, angle.cos(), angle.sin(), h, hk)
        want = qk_norm_rope_backward(gq, gk, q, k, qw, kw, angle.cos(), angle.sin())
    elif kind == "axes":
        outs = axes_rope(q, k, pos, inv, [10, 6], h, hk)
        want = axes_rope_backward(gq, gk, pos, inv, [10, 6])
    else:
        outs = axes_rope(q, k, pos, inv, [8, 8], h, hk, True, qw, kw)
        want = axes_rope_backward(gq, gk, pos, inv, [8, 8], True, q, k, qw, kw)
    leaves = (q, k, qw, kw) if kind != "axes" else (q, k)
    got = torch.autograd.grad(outs, leaves, (gq, gk), retain_graph=True)
    for x, y, leaf in zip(got, want, leaves):
        assert x.dtype == leaf.dtype and torch.equal(x, y.to(leaf.dtype).reshape(leaf.shape))
    # only one output used: the other's gradients are zero
    (only_k,) = torch.autograd.grad(outs[0], (k,), gq)
    assert bool((only_k == 0).all())


def test_gradients_by_differences(device):
    """<dx, h> and <dw, h> against central differences of the formula in 64 bits, along random
    directions: the differences' own error is of third order in the step (1e-4)."""
    from decik_amd.rope import qk_norm_rope_backward

    h, hk, d, t = 2, 1, 32, 3
    q, k, gq, gk = inputs(1, t, h, hk, d, torch.bfloat16, device)
    qw, kw = make((d,), torch.float32, device, 5, 0.3, 1.0), make((d,), torch.float32, device, 6, 0.3, 1.0)
    angle = make((t, d), torch.float32, device, 7, 3.0)
    grads = qk_norm_rope_backward(gq, gk, q, k, qw, kw, angle.cos(), angle.sin())
    cos, sin, x, g, w = (f64(v) for v in (angle.cos()[None], angle.sin()[None], q, gq, qw))
    loss = lambda xx, ww: (reference(xx, None, ww, cos, sin, h, 1e-6)["out"][0] * g).sum()  # noqa: E731
    rng = np.random.default_rng(1)
    for i, (at, got) in enumerate(((x, grads[0]), (w, grads[2]))):
        step = rng.standard_normal(at.shape)
        e = 1e-4
        moved = [(loss(x + s * e * step, w) if i == 0 else loss(x, w + s * e * step)) for s in (1, -1)]
        diff = (moved[0] - moved[1]) / (2 * e)
        have = (f64(got) * step).sum()
        # dx is rounded to bf16: half a step of each value times its direction
        slack = (abs(f64(got) * step)).sum() * (2.0 ** -8 if i == 0 else 2.0 ** -16) + 1e-6
        assert abs(diff - have) <= slack


def test_captured_step(device):
    """Forward and backward with weight gradients, captured and replayed with eager work between."""
    from decik_amd.rope import qk_norm_rope_backward, qk_norm_rope_forward

    h, hk, d, t = 4, 2, 64, 50
    q, k, gq, gk = inputs(1, t, h, hk, d, torch.float16, device)
    qw, kw = make((d,), torch.float32, device, 5, 0.3, 1.0), make((d,), torch.float32, device, 6, 0.3, 1.0)
    angle = make((t, d), torch.float32, device, 7, 3.0)
    cos, sin = angle.cos(), angle.sin()

    def step():
        return (*qk_norm_rope_forward(q, k, qw, kw, cos, sin, h, hk),
                *qk_norm_rope_backward(gq, gk, q, k, qw, kw, cos, sin))

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs on one capture stream share no workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for i in range(3):
        with torch.no_grad():
            q += 0.125
            gq *= 0.5
        for graph, _ in graphs:
            graph.replay()
        want = step()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(x, y) for x, y in zip(outs, want))


def test_refusals(device):
    from decik_amd._lib import DecikError
    from decik_amd.rope import axes_rope_backward, axes_rope_forward, qk_norm_rope_backward, qk_norm_rope_forward

    h, hk, d, t = 2, 1, 32, 4
    q, k, gq, gk = inputs(1, t, h, hk, d, torch.float16, device)
    w, tab = torch.ones(d, device=device), torch.ones((t, d), device=device)
    pos, inv = torch.zeros((1, t), dtype=torch.int64, device=device), torch.ones(d // 2, device=device)
    bad = [lambda: qk_norm_rope_forward(q.cpu(), k, w, w, tab, tab, h, hk),
           lambda: qk_norm_rope_forward(q, k.cpu(), w, w, tab, tab, h, hk),
           lambda: qk_norm_rope_forward(q, k, w, w, tab.cpu(), tab, h, hk),
           lambda: qk_norm_rope_forward(q.float(), k.float(), w, w, tab, tab, h, hk),
           lambda: qk_norm_rope_forward(q, k.bfloat16(), w, w, tab, tab, h, hk),
           lambda: qk_norm_rope_forward(q, k, w, None, tab, tab, h, hk),
           lambda: qk_norm_rope_forward(q, k, w[:16], w[:16], tab, tab, h, hk),
           lambda: qk_norm_rope_forward(q, k, w, w, tab[:3], tab[:3], h, hk),
           lambda: qk_norm_rope_forward(q, k, w, w, tab, tab[:3], h, hk),
           lambda: qk_norm_rope_forward(q, k, w, w, tab, tab, h + 1, hk),
           lambda: qk_norm_rope_forward(q, k[:, :3], w, w, tab, tab, h, hk),
           lambda: qk_norm_rope_backward(gq, gk, q[:, :3], k, w, w, tab, tab),
           lambda: qk_norm_rope_backward(gq, gk, None, None, w, w, tab, tab),
           lambda: qk_norm_rope_backward(gq[0], gk[0], q, k, w, w, tab, tab),
           lambda: axes_rope_forward(q, k, pos.float(), inv, [16], h, hk),
           lambda: axes_rope_forward(q, k, pos[:, :3], inv, [16], h, hk),
           lambda: axes_rope_forward(q, k, pos, inv, [8, 8], h, hk),
           lambda: axes_rope_forward(q, k, pos, inv, [], h, hk),
           lambda: axes_rope_backward(gq, gk[:, :, :3], pos, inv, [16])]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    from decik_amd.rope import axes_rope, qk_norm_rope
    for call in (lambda: qk_norm_rope(q, k, w, w, tab.clone().requires_grad_(True), tab, h, hk),
                 lambda: axes_rope(q, k, pos, inv.clone().requires_grad_(True), [16], h, hk)):
        with pytest.raises(ValueError, match="no gradient"):
            call()
    for sections in ([15], [-1]):
        with pytest.raises(DecikError, match="sections"):
            axes_rope_forward(q, k, pos, inv, sections, h, hk)
    small = torch.empty((1, t, 8), dtype=torch.float16, device=device)
    with pytest.raises(DecikError, match="head_dim"):
        axes_rope_forward(small, small, pos, inv[:4], [4], 1, 1)


@pytest.mark.parametrize("b,t,h,hk,d", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tables_without_norms(b, t, h, hk, d, dtype, device):
    """No norm weights: the rotation by tables alone, which needs neither q nor k for its backward."""
    from decik_amd.rope import qk_norm_rope, qk_norm_rope_backward, qk_norm_rope_forward

    q, k, gq, gk = inputs(b, t, h, hk, d, dtype, device)
    angle = make((b, t, d), torch.float32, device, 7, 3.0)
    cos, sin = angle.cos(), angle.sin()
    outs = qk_norm_rope_forward(q, k, None, None, cos, sin, h, hk)
    grads = qk_norm_rope_backward(gq, gk, None, None, None, None, cos, sin)
    check_all(outs, grads, q, k, gq, gk, None, None, f64(cos), f64(sin), h, hk, 0.0)
    q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
    got = torch.autograd.grad(qk_norm_rope(q, k, None, None, cos, sin, h, hk), (q, k), (gq, gk))
    assert all(torch.equal(x, y) for x, y in zip(got, grads))
