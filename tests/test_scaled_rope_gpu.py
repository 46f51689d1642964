"""Rotary positions of part of each head, in halves and in pairs (decik_amd.rope.scaled_rope_*) against complex numbers
in 64 bits: layouts, head and rotary sizes that fall to each form of the kernel, strides, far positions, one token, none.

Tolerance: a cosine and sine are within 2^-21 (the angle 2^-24 turns, its half turn rounded to 24 bits, the function 2 units),
times the factor; an output is two products and a sum: within 2^-20 factor (|a| + |b|) before its one rounding (half a
step). Elements past the rotary ones are copies."""

import pytest
import torch

F16, BF16 = torch.float16, torch.bfloat16
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134}


def make(shape, dtype, device, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).to(device)


def frequencies(r, device, base=1e6):
    return (base ** (-torch.arange(0, r, 2, dtype=torch.float64) / max(r, 1))).float().to(device)


def split(r, layout):
    i = torch.arange(r // 2)
    return (i, i + r // 2) if layout == "half" else (2 * i, 2 * i + 1)


def turned(x, positions, inv_freq, layout, factor, sign):
    """(value, magnitude) of x [B, H, T, D] in float64 on the CPU."""
    x, inv = x.double().cpu(), inv_freq.double().cpu()
    angle = positions.cpu().to(torch.float64).expand(x.shape[0], x.shape[2])[..., None] * inv
    by = torch.polar(torch.full_like(angle, factor), sign * angle)[:, None]
    a, b = split(2 * inv.numel(), layout)
    z = torch.complex(x[..., a], x[..., b]) * by
    out, mag = x.clone(), torch.zeros_like(x)
    out[..., a], out[..., b] = z.real, z.imag
    mag[..., a] = mag[..., b] = (x[..., a].abs() + x[..., b].abs()) * abs(factor) * 2.0 ** -20
    return out, mag


def check(got, want, what):
    value, mag = want
    assert got.shape == value.shape, what
    err = (got.double().cpu() - value).abs()
    bound = value.abs() * (torch.finfo(got.dtype).eps / 2) + mag + TINY[got.dtype] * (mag > 0)
    bound = torch.where(mag > 0, bound, torch.zeros_like(bound))  # a copy, or a turned zero
    assert bool((err <= bound).all()), f"{what}: worst excess {(err - bound).max().item():.3e}"


def token_major(x):
    return x.transpose(1, 2).flatten(2)


# head sizes and rotary parts: whole halves (16 by 16), halves of any size, pairs, sizes that no vector divides
SIZES = [(128, 128), (128, 64), (128, 32), (64, 64), (80, 20), (80, 80), (96, 24), (256, 256), (128, 2), (128, 0), (40, 40), (64, 34),
         (72, 70), (8, 6), (12, 8), (7, 6), (1, 0), (100, 50), (512, 256), (1024, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("d,r", SIZES)
@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_sizes(d, r, layout, dtype, device):
    from decik_amd.rope import scaled_rope_backward, scaled_rope_forward

    for b, t, h, hk in ((1, 1, 5, 1), (2, 37, 3, 2)):
        qkv = make((b, t, (h + 2 * hk) * d), dtype, device, 1)
        q, k = qkv[..., :h * d], qkv[..., h * d:(h + hk) * d]
        pos = torch.randint(0, 100000, (b, t), generator=torch.Generator().manual_seed(2)).to(device)
        inv = frequencies(r, device)
        outs = scaled_rope_forward(q, k, pos, inv, h, hk, layout, 1.25)
        for name, x, o, heads in (("q", q, outs[0], h), ("k", k, outs[1], hk)):
            check(o, turned(x.unflatten(-1, (heads, d)).transpose(1, 2), pos, inv, layout, 1.25, 1), name)
        gq, gk = make((b, h, t, d), dtype, device, 3), make((b, hk, t, d), dtype, device, 4)
        grads = scaled_rope_backward(gq, gk, pos, inv, layout, 1.25)
        for name, g, o in (("dq", gq, grads[0]), ("dk", gk, grads[1])):
            value, mag = turned(g, pos, inv, layout, 1.25, -1)
            check(o, (token_major(value), token_major(mag)), name)


# tokens that spread one to a work-group, several, a last work-group that is not full; many heads and one
@pytest.mark.gpu
@pytest.mark.parametrize("b,t,h,hk,d,r", [(1, 8195, 3, 1, 64, 64), (3, 683, 9, 3, 80, 20), (1, 5000, 28, 4, 128, 128), (16, 1, 28, 4, 128, 64),
                                          (1, 2, 300, 8, 128, 96), (1, 9000, 1, 1, 16, 16), (2, 1025, 2, 1, 24, 24)])
@pytest.mark.parametrize("layout", ["half", "pairs"])
def test_counts(b, t, h, hk, d, r, layout, device):
    from decik_amd.rope import scaled_rope_backward, scaled_rope_forward

    q, k = make((b, t, h * d), BF16, device, 1), make((b, t, hk * d), BF16, device, 2)
    pos, inv = torch.arange(t, device=device), frequencies(r, device)
    outs = scaled_rope_forward(q, k, pos, inv, h, hk, layout)
    check(outs[0], turned(q.unflatten(-1, (h, d)).transpose(1, 2), pos, inv, layout, 1.0, 1), "q")
    check(outs[1], turned(k.unflatten(-1, (hk, d)).transpose(1, 2), pos, inv, layout, 1.0, 1), "k")
    back = scaled_rope_backward(*outs, pos, inv, layout)
    for x, o in ((outs[0], back[0]), (outs[1], back[1])):
        value, mag = turned(x, pos, inv, layout, 1.0, -1)
        check(o, (token_major(value), token_major(mag)), "back")


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "pairs"])
def test_strides_and_positions(layout, device):
    """Views of other orders and batches, shared and strided positions of both types, two axes: what copies give."""
    from decik_amd.rope import scaled_rope_backward, scaled_rope_forward

    b, t, h, hk, d, r = 3, 11, 4, 2, 32, 16
    q = make((t, b, h * d), F16, device, 1).transpose(0, 1)
    k = make((b, 2 * t, 3 * hk * d + 1), F16, device, 2)[:, ::2, 1:1 + hk * d]
    gq = make((b, t, h, d), F16, device, 3).transpose(1, 2)
    gk = make((b, hk, d, t), F16, device, 4).transpose(2, 3)
    inv = frequencies(r, device)
    for pos in (torch.arange(t, device=device), torch.arange(t, device=device, dtype=torch.int32)[None],
                torch.arange(2 * b * t, device=device).reshape(b, 2 * t)[:, ::2], torch.arange(t, device=device).expand(b, t)):
        full = pos.expand(b, t).contiguous().long()
        got = scaled_rope_forward(q, k, pos, inv, h, hk, layout, 0.5)
        want = scaled_rope_forward(q.contiguous(), k.contiguous(), full, inv, h, hk, layout, 0.5)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        got = scaled_rope_backward(gq, gk, pos, inv, layout, 0.5)
        want = scaled_rope_backward(gq.contiguous(), gk.contiguous(), full, inv, layout, 0.5)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    one = scaled_rope_forward(q[0], k[0], full[0], inv, h, hk, layout, 0.5)
    assert one[0].shape == (1, h, t, d)
    assert torch.equal(one[0], scaled_rope_forward(q[:1], k[:1], full[:1], inv, h, hk, layout, 0.5)[0])
    none = scaled_rope_forward(q[:, :0], k[:, :0], full[:, :0], inv, h, hk, layout)
    assert none[0].shape == (b, h, 0, d) and none[1].shape == (b, hk, 0, d)


@pytest.mark.gpu
def test_far_and_negative_positions(device):
    from decik_amd.rope import scaled_rope_forward

    pos = torch.tensor([0, 1, 2 ** 20 + 1, 2 ** 28 - 1, -1, -12345, 2 ** 24 + 3], device=device)
    x = make((len(pos), 2 * 64), F16, device, 1)
    inv = torch.cat([torch.tensor([6.28, 1.0, -0.7, 0.0]), torch.rand(28, generator=torch.Generator().manual_seed(1))]).to(device)
    for layout in ("half", "pairs"):
        q, k = scaled_rope_forward(x, x, pos, inv, 2, 2, layout)
        check(q, turned(x.unflatten(-1, (2, 64)).transpose(0, 1)[None], pos, inv, layout, 1.0, 1), layout)
        assert torch.equal(q, k)


@pytest.mark.gpu
def test_values_without_numbers_stay_in_their_pair(device):
    from decik_amd.rope import scaled_rope_forward

    for layout in ("half", "pairs"):
        for d, r in ((64, 32), (40, 20)):
            a, b = split(r, layout)
            x = make((3, d), F16, device, 1)
            bad = x.clone()
            bad[1, a[3]] = float("nan")
            bad[2, d - 1] = float("inf")
            inv, pos = frequencies(r, device), torch.arange(3, device=device)
            clean, got = scaled_rope_forward(x, x, pos, inv, 1, 1, layout)[0][0, 0], scaled_rope_forward(bad, bad, pos, inv, 1, 1, layout)[0][0, 0]
            differ = (clean != got) | got.isnan()
            want = torch.zeros_like(differ)
            want[1, a[3]] = want[1, b[3]] = want[2, d - 1] = True
            assert torch.equal(differ, want)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "pairs"])
def test_autograd_and_differences(layout, device):
    """Gradients through autograd equal the backward's; along a direction they equal differences of the 64-bit form,
    which is linear in x, so that a difference of step 1 is exact."""
    from decik_amd.rope import scaled_rope, scaled_rope_backward

    b, t, h, hk, d, r = 2, 5, 3, 1, 48, 32
    q, k = make((b, t, h * d), F16, device, 1).requires_grad_(), make((b, t, hk * d), F16, device, 2).requires_grad_()
    pos, inv = torch.arange(40, 40 + t, device=device), frequencies(r, device)
    outs = scaled_rope(q, k, pos, inv, h, hk, layout, 1.1)
    gq, gk = make(outs[0].shape, F16, device, 3), make(outs[1].shape, F16, device, 4)
    torch.autograd.backward(outs, [gq, gk])
    want = scaled_rope_backward(gq, gk, pos, inv, layout, 1.1)
    assert torch.equal(q.grad, want[0]) and torch.equal(k.grad, want[1])
    step = make((b, t, h * d), F16, device, 5)
    slope = (turned(step.unflatten(-1, (h, d)).transpose(1, 2), pos, inv, layout, 1.1, 1)[0] * gq.double().cpu()).sum()
    value, mag = turned(gq, pos, inv, layout, 1.1, -1)
    room = ((token_major(value).abs() * 2.0 ** -11 + token_major(mag) + TINY[F16]) * step.double().cpu().abs()).sum()
    assert abs(float((q.grad.double().cpu() * step.double().cpu()).sum() - slope)) <= float(room)
    q.grad = k.grad = None
    scaled_rope(q, k, pos, inv, h, hk, layout, 1.1)[0].backward(gq)
    assert torch.equal(q.grad, want[0]) and not k.grad.any()
    flat = scaled_rope(q[0], k[0], pos, inv, h, hk, layout, 1.1)[1].sum()
    (g,) = torch.autograd.grad(flat, k, create_graph=False)
    assert g.shape == k.shape


@pytest.mark.gpu
def test_refusals(device):
    from decik_amd.rope import scaled_rope, scaled_rope_backward, scaled_rope_forward

    q, k = make((2, 5, 4 * 16), F16, device, 1), make((2, 5, 2 * 16), F16, device, 2)
    pos, inv = torch.arange(5, device=device), frequencies(16, device)
    bad = [
        ((q, k, pos, inv, 3, 2), {}, "H = 3"), ((q, k, pos, inv, 4, 4), {}, "head size"), ((q, k[:, :4], pos, inv, 4, 2), {}, "tokens"),
        ((q, k.bfloat16(), pos, inv, 4, 2), {}, "both"), ((q.float(), k.float(), pos, inv, 4, 2), {}, "fp16"),
        ((q, k, pos[:4], inv, 4, 2), {}, "positions"), ((q, k, pos.float(), inv, 4, 2), {}, "int32"),
        ((q, k, pos, frequencies(18, device), 4, 2), {}, "frequencies"), ((q, k, pos, inv[None], 4, 2), {}, "frequencies"),
        ((q, k, pos, inv, 4, 2, "interleaved"), {}, "layout"), ((q.cpu(), k, pos, inv, 4, 2), {}, "GPU"),
        ((q, k, pos.cpu(), inv, 4, 2), {}, "GPU"), ((q[0, 0], k, pos, inv, 4, 2), {}, "must be"), ((q, k, pos, inv, 0, 2), {}, "must be")]
    for args, kw, msg in bad:
        with pytest.raises(ValueError, match=msg):
            scaled_rope_forward(*args, **kw)
    g = make((2, 4, 5, 16), F16, device, 1)
    for args, msg in (((g, g[:1], pos, inv), "same B"), ((g[0], g[0], pos, inv), "gradients"), ((g, g.float(), pos, inv), "both"),
                      ((g, g, pos, frequencies(32, device)), "frequencies")):
        with pytest.raises(ValueError, match=msg):
            scaled_rope_backward(*args)
    with pytest.raises(ValueError, match="detach"):
        scaled_rope(q, k, pos, inv.clone().requires_grad_(), 4, 2)


# ---- frequencies ---------------------------------------------------------------------------------

def plain(r, base):
    return base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)


def test_frequency_formulas():
    from decik_amd.rope import scaled_frequencies

    r, base, half = 128, 1e6, 64
    inv, one = scaled_frequencies(r, base)
    assert inv.dtype == torch.float32 and one == 1.0 and torch.equal(inv, plain(r, base).float())
    assert torch.equal(scaled_frequencies(r, base, dict(type="linear", factor=8.0))[0], (plain(r, base) / 8).float())
    # ntk: the first frequency stays, the last is divided by the factor
    inv = scaled_frequencies(r, base, dict(rope_type="ntk", factor=8.0))[0].double()
    assert inv[0] == 1.0 and abs(float(inv[-1] * 8 / plain(r, base)[-1]) - 1) < 1e-6
    dyn = dict(rope_type="dynamic", factor=4.0, original_max_position_embeddings=1024)
    assert torch.equal(scaled_frequencies(r, base, dyn, length=1024)[0], plain(r, base).float())
    assert torch.equal(scaled_frequencies(r, base, dyn, length=2048)[0],
                       scaled_frequencies(r, base, dict(rope_type="ntk", factor=5.0))[0])
    # yarn: fast ones kept, slow ones divided, a monotone share between, 0.1 ln s + 1
    inv, factor = scaled_frequencies(r, base, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768))
    ratio = plain(r, base) / inv.double()
    turns = 32768 * plain(r, base) / (2 * torch.pi)
    assert torch.allclose(ratio[turns > 40], torch.ones(1, dtype=torch.float64), atol=1e-6)
    assert torch.allclose(ratio[turns < 0.8], torch.full((1,), 4.0, dtype=torch.float64), atol=1e-6)
    assert bool((ratio.diff() > -1e-6).all()) and abs(factor - (0.1 * torch.log(torch.tensor(4.0)).item() + 1)) < 1e-6
    assert scaled_frequencies(r, base, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768, attention_factor=2.0))[1] == 2.0
    inv, factor = scaled_frequencies(r, 5e5, dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                                  original_max_position_embeddings=8192))
    ratio, turns = plain(r, 5e5) / inv.double(), 8192 * plain(r, 5e5) / (2 * torch.pi)
    assert factor == 1.0 and torch.allclose(ratio[turns > 4], torch.ones(1, dtype=torch.float64), atol=1e-6)
    assert torch.allclose(ratio[turns < 1], torch.full((1,), 8.0, dtype=torch.float64), atol=1e-6)
    mid = (turns > 1) & (turns < 4)
    share = (turns[mid] - 1) / 3
    assert torch.allclose(1 / ratio[mid], share + (1 - share) / 8, atol=1e-6)
    long = dict(rope_type="longrope", short_factor=[1.0] * half, long_factor=[2.0] * half, factor=16.0,
                original_max_position_embeddings=4096)
    inv, factor = scaled_frequencies(r, base, long, length=4096)
    assert torch.equal(inv, plain(r, base).float()) and abs(factor - (1 + 4 / 12) ** 0.5) < 1e-6
    assert torch.equal(scaled_frequencies(r, base, long, length=4097)[0], (plain(r, base) / 2).float())
    assert scaled_frequencies(2, base, dict(rope_type="ntk", factor=8.0))[0].tolist() == [1.0]


def test_frequency_refusals():
    from decik_amd.rope import scaled_frequencies

    for args, msg in (((7,), "even"), ((0,), "even"), ((8, 1e4, dict(rope_type="other")), "unknown"), ((8, 1e4, dict(rope_type="linear")), "factor"),
                      ((8, 1e4, dict(rope_type="yarn", factor=2.0)), "original"),
                      ((8, 1e4, dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=8, mscale=0.7)), "mscale"),
                      ((8, 1e4, dict(factor=2.0)), "factor"),
                      ((8, 1e4, dict(rope_type="longrope", short_factor=[1.0], original_max_position_embeddings=8, factor=2.0)), "divisors")):
        with pytest.raises(ValueError, match=msg):
            scaled_frequencies(*args)
