"""The residual stream with its norms and gate (decik_amd.norm) against the formulas in 64 bits: values and gradients,
types, widths from one element to the largest, gates, strides, streams of fp32, empty batches, rows that hold no number.

Tolerances, with H = |scale residual| + |gate p| an element of h, R = rms(H) / rms(h) >= 1 of its row. A row's sum of squares
has at most 26 roundings in any chain (4 passes, 3 + 6 + 8 partial sums, its mean), halved by the root; with the
products rx, post weight and gate an element of h is within 2^-19 H. rh then is within 2^-19 R of itself, a normalized
element within 2^-18 U, U = rh H + |unit| R. With u = gy w and C = mean(|u| U), dh is within 2^-17 of
D = |gh| + rh (|u| (1 + R) + U C), and what follows from dh (dgate, v, dx) within 2^-16 of the same expression of
magnitudes, as are the sums over rows (fewer than 256 terms in any chain). Last, one rounding to the output type."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -149}
EPS = 1e-5


def make(shape, dtype, device, seed, std=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std + mean).to(dtype).to(device)


def f64(t):
    return None if t is None else t.detach().double().cpu()


def reference(gh, gy, x, residual, weight, post, gate, scale, eps):
    """{name: (value, magnitude)} of h, y, dx, dres, dw, dpw, dgate in float64; gradients where gh or gy is given."""
    gh, gy, x, residual, weight, post, gate = (f64(t) for t in (gh, gy, x, residual, weight, post, gate))
    zero = torch.zeros_like(x)
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    rx = torch.ones_like(mean(x)) if post is None else 1.0 / torch.sqrt(mean(x * x) + eps)
    ux = x * rx
    p = ux if post is None else ux * post
    g = torch.ones_like(x) if gate is None else gate.expand_as(x)
    res = zero if residual is None else residual * scale
    h = res + g * p
    hm = res.abs() + (g * p).abs()
    out = dict(h=(h, hm * 2.0 ** -19))
    dh, dm = (zero, zero) if gh is None else (gh, gh.abs())
    if weight is not None:
        rh = 1.0 / torch.sqrt(mean(h * h) + eps)
        ratio = torch.sqrt(mean(hm * hm) + eps) * rh
        unit, um = h * rh, hm * rh + (h * rh).abs() * ratio
        out["y"] = (unit * weight, um * weight.abs() * 2.0 ** -18)
        if gy is not None:
            u = gy * weight
            out["dw"] = ((gy * unit).reshape(-1, x.shape[-1]).sum(0), (gy.abs() * um).reshape(-1, x.shape[-1]).sum(0) * 2.0 ** -16)
            dh = dh + rh * (u - unit * mean(u * unit))
            dm = dm + rh * (u.abs() * (1 + ratio) + um * mean(u.abs() * um))
    if gh is None and gy is None:
        return out
    if residual is not None:
        out["dres"] = (scale * dh, abs(scale) * dm * 2.0 ** -17)
    if gate is not None:
        dg, gm = dh * p, dm * p.abs() * 2.0 ** -16
        if gate.dim() == 1 and gate.shape[0] == x.shape[-1]:
            dg, gm = dg.reshape(-1, x.shape[-1]).sum(0), gm.reshape(-1, x.shape[-1]).sum(0)
        elif gate.shape != x.shape:
            dg, gm = dg.sum(-1, keepdim=True), gm.sum(-1, keepdim=True)
        out["dgate"] = (dg, gm)
    dp, pm = dh * g, dm * g.abs()
    if post is None:
        out["dx"] = (dp, pm * 2.0 ** -17)
    else:
        out["dpw"] = ((dp * ux).reshape(-1, x.shape[-1]).sum(0), (pm * ux.abs()).reshape(-1, x.shape[-1]).sum(0) * 2.0 ** -16)
        v, vm = dp * post, pm * post.abs()
        out["dx"] = (rx * (v - ux * mean(v * ux)), rx * (vm + ux.abs() * mean(vm * ux.abs())) * 2.0 ** -16)
    return out


def check(got, want, what):
    value, mag = want
    assert got.shape == value.shape, what
    err = (got.double().cpu() - value).abs()
    bound = value.abs() * (torch.finfo(got.dtype).eps / 2) + mag + TINY[got.dtype]
    assert bool((err <= bound).all()), f"{what}: worst excess {(err - bound).max().item():.3e}"


NAMES = ("dx", "dres", "dw", "dpw", "dgate")


def run_and_check(x, residual, weight, post, gate, scale, gh, gy, dtype=None):
    from decik_amd.norm import residual_norm_backward, residual_norm_forward

    ref = reference(gh, gy, x, residual, weight, post, gate, scale, EPS)
    h, y = residual_norm_forward(x, residual, weight, post, gate, scale, EPS, dtype)
    check(h, ref["h"], "h")
    assert (y is None) == (weight is None)
    if y is not None:
        check(y, ref["y"], "y")
    grads = residual_norm_backward(gh, gy, x, residual, weight, post, gate, scale, EPS)
    for name, g in zip(NAMES, grads):
        assert (g is None) == (name not in ref), name
        if g is not None:
            check(g, ref[name], name)
    return h, y, grads


def gate_of(kind, shape, dtype, device):
    if kind == "none":
        return None
    full = dict(channel=(shape[-1],), token=(*shape[:-1], 1), element=shape)[kind]
    return torch.sigmoid(make(full, F32, device, 77)).to(dtype)


# one element, odd and ragged rows, where passes of 512 threads begin and end, the largest; many short rows
SIZES = [(1, 1), (1, 8), (3, 7), (16, 3584), (33, 1121), (830, 1536), (5, 4096), (4, 4097), (3, 8192), (2, 8193), (2, 16384),
         (9, 16381), (700, 65), (2000, 512), (5000, 24)]


@pytest.mark.parametrize("rows,width", SIZES)
@pytest.mark.parametrize("post,gate", [(True, "channel"), (False, "none"), (True, "element"), (True, "token")])
def test_sizes(rows, width, post, gate, device):
    if width == 1 and gate == "token":
        pytest.skip("a gate [rows, 1] is one value an element here")
    x, res = make((rows, width), BF16, device, 1), make((rows, width), BF16, device, 2, 2.0)
    w, pw = make((width,), F32, device, 3, 0.2, 1.0), make((width,), F32, device, 4, 0.2, 1.0) if post else None
    g = gate_of(gate, (rows, width), F32 if gate == "channel" else BF16, device)
    gh, gy = make((rows, width), BF16, device, 5, 1e-2), make((rows, width), BF16, device, 6, 1e-2)
    run_and_check(x, res, w, pw, g, 0.75, gh, gy)


@pytest.mark.parametrize("x_type,stream,y_type", [(F16, F16, F16), (F16, F16, F32), (F16, F32, F16), (F16, F32, F32),
                                                  (BF16, BF16, F32), (BF16, F32, BF16), (BF16, F32, F32), (F32, F32, F32)])
@pytest.mark.parametrize("width", [1536, 1121, 5000, 9000])
def test_types(x_type, stream, y_type, width, device):
    rows = 21
    x, res = make((rows, width), x_type, device, 1), make((rows, width), stream, device, 2, 2.0)
    for w_type, gate in ((F32, "channel"), (x_type, "element"), (F16, "token"), (BF16, "none")):
        w, pw = make((width,), w_type, device, 3, 0.2, 1.0), make((width,), w_type, device, 4, 0.2, 1.0)
        g = gate_of(gate, (rows, width), w_type, device)
        gh, gy = make((rows, width), stream, device, 5, 1e-2), make((rows, width), y_type, device, 6, 1e-2)
        run_and_check(x, res, w, pw, g, 1.0, gh, gy, y_type)


@pytest.mark.parametrize("width", [640, 333])
def test_parts_that_are_absent(width, device):
    from decik_amd.norm import residual_norm_backward

    rows = 13
    x, res = make((rows, width), F16, device, 1), make((rows, width), F16, device, 2)
    w, pw = make((width,), F16, device, 3, 0.2, 1.0), make((width,), F16, device, 4, 0.2, 1.0)
    g = gate_of("channel", (rows, width), F16, device)
    gh, gy = make((rows, width), F16, device, 5), make((rows, width), F16, device, 6)
    run_and_check(x, None, w, None, None, 1.0, None, gy)      # a norm alone
    run_and_check(x, None, w, pw, g, 3.0, gh, gy)             # no stream: its scale means nothing
    run_and_check(x, res, None, pw, g, 0.5, gh, None)         # the last join: no norm after it
    run_and_check(x, res, None, None, None, -1.0, gh, None)   # a sum
    run_and_check(x, res, w, pw, g, 0.0, None, gy)            # the stream's gradient is zero
    full = residual_norm_backward(gh, gy, x, res, w, pw, g)
    bare = residual_norm_backward(gh, gy, x, res, w, pw, g, param_grads=False)
    assert bare[2:] == (None, None, None) and all(torch.equal(a, b) for a, b in zip(full[:2], bare[:2]))


def test_strides_and_leading_axes(device):
    """Views of wider buffers, a residual row shared by all tokens, transposed and three-axis tensors: the values of
    contiguous copies."""
    from decik_amd.norm import residual_norm_backward, residual_norm_forward

    b, t, width = 3, 5, 203
    wide = make((b * t, 2 * width + 3), F16, device, 1)
    x = wide[:, 3:3 + width].unflatten(0, (b, t))
    res = make((1, 1, width), F16, device, 2).expand(b, t, width)
    gate = make((b, t, 2 * width), F16, device, 3)[..., ::2]
    token = make((b, t, 4), F16, device, 8)[..., 1:2]
    gh = make((t, b, width), F16, device, 4).transpose(0, 1)
    gy = make((b, t, width), F16, device, 5)
    w, pw = make((2 * width,), F32, device, 6)[::2], make((width,), F32, device, 7)
    for g in (gate, token):
        got = residual_norm_forward(x, res, w, pw, g, 0.5, EPS)
        want = residual_norm_forward(x.contiguous(), res.contiguous(), w.contiguous(), pw, g.contiguous(), 0.5, EPS)
        assert all(torch.equal(a, c) for a, c in zip(got, want)) and got[0].shape == (b, t, width)
        got = residual_norm_backward(gh, gy, x, res, w, pw, g, 0.5, EPS)
        want = residual_norm_backward(gh.contiguous(), gy, x.contiguous(), res.contiguous(), w.contiguous(), pw,
                                      g.contiguous(), 0.5, EPS)
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    one = residual_norm_forward(x[0, 0], res[0, 0], w, pw, gate[0, 0])[0]
    assert one.shape == (width,)


def test_nothing_to_do(device):
    from decik_amd.norm import residual_norm_backward, residual_norm_forward

    x = torch.empty((0, 96), dtype=F16, device=device)
    w = torch.ones(96, device=device)
    h, y = residual_norm_forward(x, x, w, w, w)
    assert h.shape == y.shape == (0, 96)
    dx, dres, dw, dpw, dgate = residual_norm_backward(x, x, x, x, w, w, w)
    assert dx.shape == dres.shape == (0, 96)
    assert all(torch.equal(t, torch.zeros(96, device=device)) for t in (dw, dpw, dgate))


def test_rows_without_numbers_stay_alone(device):
    """An infinity, a NaN, a row of zeros: only their own rows show it, and zeros give zeros."""
    from decik_amd.norm import residual_norm_backward, residual_norm_forward

    rows, width = 9, 1121
    x, res = make((rows, width), F16, device, 1), make((rows, width), F16, device, 2)
    w, pw = make((width,), F32, device, 3), make((width,), F32, device, 4)
    gh, gy = make((rows, width), F16, device, 5), make((rows, width), F16, device, 6)
    clean = residual_norm_forward(x, res, w, pw) + residual_norm_backward(gh, gy, x, res, w, pw)[:2]
    x2, res2 = x.clone(), res.clone()
    x2[2, 1120], res2[4, 0] = float("inf"), float("nan")
    x2[6] = res2[6] = 0.0
    got = residual_norm_forward(x2, res2, w, pw) + residual_norm_backward(gh, gy, x2, res2, w, pw)[:2]
    keep = [0, 1, 3, 5, 7, 8]
    for a, b in zip(got, clean):
        assert torch.equal(a[keep], b[keep])
        assert not bool(torch.isfinite(a[2].sum())) and not bool(torch.isfinite(a[4].sum()))
    assert not got[0][6].any() and not got[1][6].any()


def test_values_past_the_output_type(device):
    """h and y beyond fp16: infinities as the type's rounding gives them, and an fp32 stream keeps them."""
    from decik_amd.norm import residual_norm_forward

    x = torch.full((2, 64), 60000.0, dtype=F16, device=device)
    w = torch.ones(64, device=device)
    h, y = residual_norm_forward(x, x, w)
    assert bool(torch.isinf(h).all()) and torch.allclose(y.float(), torch.ones_like(y, dtype=F32), atol=2.0 ** -11)
    h, _ = residual_norm_forward(x, x.float(), w)
    assert torch.equal(h, torch.full_like(h, float(x[0, 0]) * 2))


def test_same_bits_every_run(device):
    from decik_amd.norm import residual_norm_backward

    rows, width = 1300, 1121
    x, res = make((rows, width), BF16, device, 1), make((rows, width), F32, device, 2)
    w, pw, g = (make((width,), F32, device, s) for s in (3, 4, 5))
    gh, gy = make((rows, width), F32, device, 6), make((rows, width), BF16, device, 7)
    first = residual_norm_backward(gh, gy, x, res, w, pw, g)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, residual_norm_backward(gh, gy, x, res, w, pw, g)))


@pytest.mark.parametrize("gate", ["none", "channel", "token", "element"])
def test_autograd(gate, device):
    """The autograd form gives the functions' values, in the inputs' types."""
    from decik_amd.norm import residual_norm, residual_norm_backward, residual_norm_forward

    b, t, width = 2, 7, 320
    x, res = make((b, t, width), F16, device, 1), make((b, t, width), F32, device, 2)
    w, pw = make((width,), F16, device, 3), make((width,), F32, device, 4)
    g = gate_of(gate, (b, t, width), F16, device)
    leaves = [None if v is None else v.clone().requires_grad_() for v in (x, res, w, pw, g)]
    h, y = residual_norm(*leaves, 0.5, EPS)
    gh, gy = make(h.shape, F32, device, 5), make(y.shape, F16, device, 6)
    assert all(torch.equal(a, c) for a, c in zip((h, y), residual_norm_forward(x, res, w, pw, g, 0.5, EPS)))
    torch.autograd.backward([h, y], [gh, gy])
    want = residual_norm_backward(gh, gy, x, res, w, pw, g, 0.5, EPS)
    for leaf, value in zip(leaves, want):
        if leaf is not None:
            assert leaf.grad.dtype == leaf.dtype and torch.equal(leaf.grad, value.to(leaf.dtype))


def test_autograd_where_one_output_is_used(device):
    from decik_amd.norm import residual_norm, residual_norm_backward, rms_norm

    x, res = make((11, 96), F32, device, 1), make((11, 96), F32, device, 2)
    w, pw = make((96,), F32, device, 3), make((96,), F32, device, 4)
    gr = make((11, 96), F32, device, 5)

    def leaves():
        return [v.clone().requires_grad_() for v in (x, res, w, pw)]

    a = leaves()
    residual_norm(*a, eps=EPS)[1].backward(gr)
    want = residual_norm_backward(None, gr, x, res, w, pw, eps=EPS)
    assert all(torch.equal(v.grad, g) for v, g in zip(a, want))
    a = leaves()
    residual_norm(*a, eps=EPS)[0].backward(gr)
    want = residual_norm_backward(gr, None, x, res, None, pw, eps=EPS)
    assert torch.equal(a[0].grad, want[0]) and torch.equal(a[1].grad, want[1]) and torch.equal(a[3].grad, want[3])
    assert not a[2].grad.any()
    a = leaves()
    rms_norm(a[0], a[2], EPS).backward(gr)
    want = residual_norm_backward(None, gr, x, None, w, eps=EPS)
    assert torch.equal(a[0].grad, want[0]) and torch.equal(a[2].grad, want[2])
    a = leaves()
    h, none = residual_norm(a[0], a[1], None, a[3], eps=EPS)
    assert none is None
    h.backward(gr)
    assert torch.equal(a[0].grad, residual_norm_backward(gr, None, x, res, None, pw, eps=EPS)[0])


def test_gradients_against_differences(device):
    """Central differences of the 64-bit formula along random directions (step 1e-5: truncation and rounding far below
    the bound) against the kernels' gradients."""
    from decik_amd.norm import residual_norm_backward

    rows, width = 6, 50
    given = [make((rows, width), F32, device, 1), make((rows, width), F32, device, 2), make((width,), F32, device, 3),
             make((width,), F32, device, 4), make((width,), F32, device, 5)]
    gh, gy = make((rows, width), F32, device, 6), make((rows, width), F32, device, 7)
    grads = residual_norm_backward(gh, gy, *given, 0.8, EPS)
    ref = reference(gh, gy, *given, 0.8, EPS)

    def loss(values):
        out = reference(None, None, *values, 0.8, EPS)
        return float((out["h"][0] * f64(gh)).sum() + (out["y"][0] * f64(gy)).sum())

    for i, (name, v) in enumerate(zip(("dx", "dres", "dw", "dpw", "dgate"), given)):
        d = torch.from_numpy(np.random.default_rng(i).standard_normal(tuple(v.shape)))
        step = 1e-5
        moved = [[f64(t) + (s * step * d if j == i else 0) for j, t in enumerate(given)] for s in (1, -1)]
        slope = (loss(moved[0]) - loss(moved[1])) / (2 * step)
        got = float((f64(grads[i]) * d).sum())
        bound = float(((ref[name][1] + ref[name][0].abs() * 2.0 ** -24) * d.abs()).sum()) + 1e-6 * float(ref[name][0].norm() * d.norm())
        assert abs(got - slope) <= bound, name


def test_far_rows(device):
    """Element offsets past 2^31."""
    from decik_amd.norm import residual_norm_backward, residual_norm_forward

    rows, width = 140000, 16384
    x = torch.zeros((rows, width), dtype=F16, device=device)
    x[-3:] = make((3, width), F16, device, 1)
    w = make((width,), F32, device, 2)
    h, y = residual_norm_forward(x, x, w)
    hs, ys = residual_norm_forward(x[-3:], x[-3:], w)
    assert torch.equal(h[-3:], hs) and torch.equal(y[-3:], ys) and not y[:5].any()
    del h, y
    dx, _, dw, _, _ = residual_norm_backward(x, x, x, None, w)
    dxs, _, dws, _, _ = residual_norm_backward(x[-3:], x[-3:], x[-3:], None, w)
    assert torch.equal(dx[-3:], dxs)
    assert torch.allclose(dw, dws, rtol=2.0 ** -20, atol=0)  # three terms, added in another order


def test_refusals(device):
    from decik_amd.norm import residual_norm, residual_norm_backward, residual_norm_forward, rms_norm

    x, w = make((4, 64), F16, device, 1), torch.ones(64, device=device)
    bad = [
        ((x, x[:, :32], w), {}, "residual"), ((x, x.bfloat16(), w), {}, "residual"), ((x, x[:2], w), {}, "residual"),
        ((x, x, w[:32]), {}, "weight"), ((x, x, w.double()), {}, "weight"), ((x, x, w, w[:1]), {}, "post_weight"),
        ((x, x, w, None, x[:, :2]), {}, "gate"), ((x, x, w, None, w.double()), {}, "gate"), ((x, x, w, None, x[:1]), {}, "gate"),
        ((x.double(), None, w), {}, "fp16"), ((x, x, w), dict(dtype=BF16), "y must"), ((x.cpu(), None, w), {}, "GPU"),
        ((x, x.cpu(), w), {}, "GPU"), ((x, None, w.cpu()), {}, "GPU"),
        ((make((2, 16385), F16, device, 1), None, None), {}, "16384"), ((torch.empty((3, 0), dtype=F16, device=device), None, None), {}, "W from 1")]
    for args, kw, msg in bad:
        with pytest.raises(ValueError, match=msg):
            residual_norm_forward(*args, **kw)
    for gh, gy, weight, msg in ((x, None, w, "grad_y"), (x, x, None, "grad_y"), (x[:2], x, w, "grad_h"), (x.float(), x, w, "grad_h"),
                                (x, x[:2], w, "grad_y"), (x, x.bfloat16(), w, "y must")):
        with pytest.raises(ValueError, match=msg):
            residual_norm_backward(gh, gy, x, x, weight)
    with pytest.raises(ValueError, match="weight"):
        rms_norm(x, None)
    leaf = x.float().requires_grad_()
    h, y = residual_norm(leaf, None, w)
    (g,) = torch.autograd.grad(y.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
