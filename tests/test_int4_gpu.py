"""Linear layers in 4-bit integers (decik_amd.int4) against the formulas in 64 bits: every form (few tokens by 4, 8
and 16 waves; tiles whole and split), groups, zero points, types, odd sizes, strides, and the
packing, on the CPU.

Tolerances, with S = sum over k of |x| scale |code - zero|. Few tokens: operands are exact, a chain of fp32 sums has at most
32 + K / 32 terms (32 in an MFMA, then MFMAs, groups, waves or splits), so the sum is within (64 + K / 32) 2^-24 of S;
then one rounding, half a step. Many tokens and the backward: a weight is rounded once, half a step of its type (fp16: at
least 2^-25; the scale's 11 bits times the code's 11 are exact before that); the sums as before."""

import pytest
import torch

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134, F32: 2.0 ** -149}


def make(shape, dtype, device, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).to(device)


def random_parts(n, k, group, dtype, seed, zeros=True):
    g = torch.Generator().manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    scales = (torch.rand((n, groups), generator=g) * 0.02 + 1e-3).to(dtype)
    zs = torch.randint(0, 17, (n, groups), generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales, zs


def values(codes, scales, zeros, group):
    """W in float64."""
    k = codes.shape[1]
    times = min(group, k)  # (one group where it is longer than a row)
    s = scales.double().repeat_interleave(times, 1)[:, :k]
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(times, 1)[:, :k]
    return (codes.double() - z) * s


def check(got, value, mag, what):
    assert got.shape == value.shape, what
    err = (got.double() - value).abs()
    bound = value.abs() * (torch.finfo(got.dtype).eps / 2) + mag + TINY[got.dtype]
    assert bool((err <= bound).all()), f"{what}: worst excess {(err - bound).max().item():.3e}"


def rounded_once(w, dtype, terms):
    """What a weight of the tiles and a sum of `terms` of its products may be off by."""
    off = w.abs() * (torch.finfo(dtype).eps / 2 * 1.01 + (64 + terms / 32) * 2.0 ** -24)
    return off + (2.0 ** -25 if dtype == F16 else 0.0)


def check_forward(y, x, w, bias, what="y"):
    from decik_amd.int4 import launch_plan

    k = x.shape[1]
    xd, w = x.double(), w.to(x.device)
    value = xd @ w.t().contiguous()
    if launch_plan(False, x.shape[0], w.shape[0], k)["waves"] == 0:
        off = rounded_once(w, x.dtype, k)
    else:
        off = w.abs() * (64 + k / 32) * 2.0 ** -24
    mag = xd.abs() @ off.t().contiguous()
    if bias is not None:
        value = value + bias.double()
        mag = mag + (value.abs() + bias.double().abs()) * 2.0 ** -24
    check(y, value, mag, what)


def check_backward(dx, dy, w, what="dx"):
    dd, w = dy.double(), w.to(dy.device)
    check(dx, dd @ w, dd.abs() @ rounded_once(w, dy.dtype, dy.shape[1]), what)


# ---- packing, on the CPU -------------------------------------------------------------------------

@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (3, 127, 32), (5, 128, 128), (7, 129, 64), (2, 300, 96), (4, 1000, 4096), (0, 8, 32)])
def test_packing_round_trip(n, k, group):
    from decik_amd.int4 import dequantize_int4, int4_weight

    codes, scales, zeros = random_parts(n, k, group, BF16, 1)
    w = int4_weight(codes, scales, zeros, group)
    assert w.packed.shape == (-(-n // 16), -(-k // 128), 1024) and w.shape == (n, k)
    assert torch.equal(w.codes(), codes) and torch.equal(w.scales, scales) and torch.equal(w.zeros, zeros)
    assert torch.equal(dequantize_int4(w).double(), values(codes, scales, zeros, group).float().double())
    assert torch.equal(int4_weight(codes, scales, None, group).zeros, torch.full_like(zeros, 8))


def test_one_group_a_row():
    """Groups far longer than a row cost no memory of their length."""
    from decik_amd.int4 import dequantize_int4, quantize_int4

    w = make((5, 70), F32, "cpu", 1, 0.02)
    for symmetric in (False, True):
        one, exact = (quantize_int4(w, g, symmetric) for g in (2 ** 20, 96))
        assert one.meta.shape == (1, 1, 16) and torch.equal(dequantize_int4(one), dequantize_int4(exact))


def test_packed_layout():
    """Bytes 16 (16 q + r) of a tile hold row r; their word j columns 32 j + 8 q + e, column e in bits 4 (e // 2) + 16 (e % 2)."""
    from decik_amd.int4 import int4_weight

    codes, scales, zeros = random_parts(35, 256, 128, F16, 3)
    weight = int4_weight(codes, scales, zeros, 128)
    words = weight.packed.view(torch.int32).long() & 0xFFFFFFFF
    for n, b, q, j, e in ((0, 0, 0, 0, 0), (17, 1, 3, 2, 7), (34, 1, 2, 3, 4), (15, 0, 1, 0, 1)):
        word = int(words[n // 16, b, 4 * (16 * q + n % 16) + j])
        assert word >> (4 * (e // 2) + 16 * (e % 2)) & 15 == int(codes[n, 128 * b + 32 * j + 8 * q + e])
        meta = int(weight.meta[n // 16, b, n % 16])
        assert meta & 0xFFFF == int(scales[n, b].view(torch.int16)) and meta >> 16 == int(zeros[n, b])
    assert not weight.meta[2, :, 3:].any() and not words[2, :].view(2, 4, 16, 4)[:, :, 3:].any()


def test_quantize():
    """Values off by at most half a scale and the scale's own rounding; extremes, zeros and numbers that are none."""
    from decik_amd.int4 import dequantize_int4, quantize_int4

    w = make((9, 300), F32, "cpu", 1, 0.02)
    w[0, :32] = 0.0
    w[1, :32] = w[1, :32].abs() + 0.01
    w[2, 5] = float("inf")
    w[3, 5] = float("nan")
    for symmetric in (False, True):
        for dtype in (F16, BF16):
            q = quantize_int4(w, 32, symmetric, dtype)
            d = dequantize_int4(q)
            assert q.scale_dtype == dtype and not d[0, :32].any() and not d[2, :32].any() and not d[3, :32].any()
            s = q.scales.float().repeat_interleave(32, 1)[:, :300]
            keep = torch.ones_like(w, dtype=torch.bool)
            keep[2:4, :32] = False
            # (a scale rounded down leaves the extremes up to 15 half steps of the scale outside)
            assert bool(((d - w).abs() <= s * (0.5 + 16 * torch.finfo(dtype).eps))[keep].all())


def test_refusals_of_weights():
    from decik_amd.int4 import int4_weight, quantize_int4

    codes, scales, zeros = random_parts(4, 64, 32, F16, 1)
    for args, msg in (((codes.int(), scales, zeros, 32), "uint8"), ((codes[0], scales, zeros, 32), "uint8"), ((codes, scales, zeros, 48), "32"),
                      ((codes, scales, zeros, 64), "scales"), ((codes, scales.float(), zeros, 32), "scales"), ((codes, scales, zeros[:2], 32), "zeros"),
                      ((codes + 1, scales, zeros, 32), "0 to 15"), ((codes, scales, zeros + 17, 32), "0 to 16"), ((codes[:, :0], scales[:, :0], None, 32), "K")):
        with pytest.raises(ValueError, match=msg):
            int4_weight(*args)
    for args, msg in (((codes,), "fp16"), ((scales, 40), "32"), ((scales, 32, False, F32), "scale_dtype"), ((scales[0],), "N, K")):
        with pytest.raises(ValueError, match=msg):
            quantize_int4(*args)


# ---- products ------------------------------------------------------------------------------------

# tokens, rows, columns: each form and what lies around its edges
FORWARD = [(1, 1, 1), (1, 17, 128), (2, 100, 129), (15, 333, 1121), (16, 48, 4096), (16, 48, 8961), (1, 8200, 2100), (3, 16500, 640), (1, 8200, 30),
           (16, 4200, 1100), (9, 8209, 2100), (16, 18944, 1121), (16, 70000, 1030), (16, 40, 18944), (13, 3600, 9728), (7, 257, 70000),
           (17, 40, 640), (31, 257, 5000), (32, 3000, 2049), (29, 4200, 9000), (33, 70, 512), (64, 300, 4100), (40, 3000, 4100), (65, 256, 128), (65, 3, 130), (128, 255, 1000),
           (129, 257, 4096), (300, 700, 1121), (830, 1536, 1536), (257, 1000, 31), (2000, 3000, 1121), (600, 20000, 300),
           (48, 4100, 3000), (33, 5000, 3301), (64, 8190, 1540), (64, 1500, 9000), (64, 4200, 4100)]
BACKWARD = [(1, 1, 1), (1, 128, 17), (2, 129, 300), (16, 1121, 333), (32, 640, 256), (33, 1000, 257), (64, 4096, 128), (65, 31, 600), (128, 2057, 1121),
            (129, 300, 513), (300, 1121, 700), (830, 1536, 1536), (37, 2057, 1121), (50, 200, 600)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", FORWARD)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_forward(m, n, k, dtype, device):
    from decik_amd.int4 import int4_linear_forward, int4_weight

    x, bias = make((m, k), dtype, device, 2), make((n,), dtype, device, 3)
    for group, zeros, scale_dtype in ((32, True, dtype), (64, False, F16), (128, True, BF16), (96, True, dtype), (2 ** 20, True, dtype)):
        parts = random_parts(n, k, group, scale_dtype, group, zeros)
        weight = int4_weight(*(None if p is None else p.to(device) for p in parts), group)
        w = values(*(None if p is None else p.to(device) for p in parts), group)
        check_forward(int4_linear_forward(x, weight, bias), x, w, bias, f"group {group}")
        check_forward(int4_linear_forward(x, weight, None, F32), x, w, None, f"group {group} fp32")


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", BACKWARD)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_backward(m, n, k, dtype, device):
    from decik_amd.int4 import int4_linear_backward, int4_weight

    dy = make((m, n), dtype, device, 2)
    for group, zeros, scale_dtype in ((32, True, dtype), (64, False, F16), (128, True, BF16), (96, True, dtype), (2 ** 20, True, dtype)):
        parts = random_parts(n, k, group, scale_dtype, group, zeros)
        weight = int4_weight(*(None if p is None else p.to(device) for p in parts), group)
        w = values(*(None if p is None else p.to(device) for p in parts), group)
        check_backward(int4_linear_backward(dy, weight), dy, w, f"group {group}")
        check_backward(int4_linear_backward(dy, weight, F32), dy, w, f"group {group} fp32")


def test_every_form_for_few_tokens_is_tested():
    """The sizes above reach every number of waves, one tile of rows a work-group and several, one split of the columns and several; the
    tiles for more tokens are tested one by one below."""
    from decik_amd.int4 import launch_plan

    plans = [launch_plan(False, *s) for s in FORWARD]
    few = {(p["waves"], p["shares"]) for p in plans if p["waves"]}
    assert few >= {(4, 4), (8, 8), (16, 8), (16, 5), (16, 3), (16, 1)}
    assert {p["splits"] > 1 for p in plans if p["waves"] == 8} == {p["splits"] > 1 for p in plans if p["waves"] == 16} == {True, False}
    assert {p["tile_tokens"] for p in plans if not p["waves"]} == {64, 128, 256}
    # more than 16 tokens: on any weight up to 32, on small ones up to 64
    assert any(p["waves"] and m > 32 for (m, _, _), p in zip(FORWARD, plans)) and not launch_plan(False, 33, 8192, 4096)["waves"]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [64, 128, 256])
@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_every_tile(tokens, splits, dtype, device, monkeypatch):
    """Each tile, whole and split, both ways, at sizes with edges in every direction and at whole ones."""
    from decik_amd.int4 import int4_linear_backward, int4_linear_forward, int4_weight, launch_plan

    monkeypatch.setenv("DECIK_INT4_PLAN", f"{tokens},{splits}")
    for m, n, k in ((300, 700, 1121), (tokens, 768, 768), (70, 1300, 650)):
        assert launch_plan(False, m, n, k)["tile_tokens"] == launch_plan(True, m, n, k)["tile_tokens"] == tokens
        assert (launch_plan(False, m, n, k)["splits"] > 1) == (launch_plan(True, m, n, k)["splits"] > 1) == (splits > 1)
        x, dy, bias = make((m, k), dtype, device, 2), make((m, n), dtype, device, 3), make((n,), F32, device, 4)
        for group in (32, 64, 128):
            parts = [p.to(device) for p in random_parts(n, k, group, dtype, group)]
            weight = int4_weight(*parts, group)
            w = values(*parts, group)
            for out in (None, F32):
                check_forward(int4_linear_forward(x, weight, bias, out), x, w, bias, f"forward {m} {group}")
                check_backward(int4_linear_backward(dy, weight, out), dy, w, f"backward {m} {group}")


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_strides_and_batches(m, device):
    """Rows that start anywhere, shared rows, transposed activations, three axes: the values of contiguous copies."""
    from decik_amd.int4 import int4_linear_backward, int4_linear_forward, int4_weight

    n, k = 72, 264
    weight = int4_weight(*(p.to(device) for p in random_parts(n, k, 64, F16, 1)), 64)
    for fn, cols, out in ((int4_linear_forward, k, n), (int4_linear_backward, n, k)):
        wide = make((m, 3 * cols + 8), F16, device, 2)
        for x in (wide[:, 8:8 + cols], wide[:, 3:3 + cols], make((cols, m), F16, device, 3).t(), wide[:1, :cols].expand(m, cols),
                  make((m, 2 * cols), F16, device, 4)[:, ::2]):
            y = fn(x, weight)
            assert y.shape == (m, out) and torch.equal(y, fn(x.contiguous(), weight))
        x3 = make((2, m, cols), F16, device, 5)
        assert torch.equal(fn(x3, weight), fn(x3.reshape(-1, cols), weight).view(2, m, out))
        assert torch.equal(fn(x3[0, 0], weight), fn(x3[0, :1], weight)[0])
        assert fn(x3[:, :0], weight).shape == (2, 0, out)


@pytest.mark.gpu
def test_no_rows_in_the_weight(device):
    from decik_amd.int4 import int4_linear_backward, int4_linear_forward, int4_weight

    weight = int4_weight(*(p.to(device) for p in random_parts(0, 64, 32, F16, 1)), 32)
    assert int4_linear_forward(make((3, 64), F16, device, 1), weight).shape == (3, 0)
    assert torch.equal(int4_linear_backward(make((3, 0), F16, device, 1), weight), torch.zeros((3, 64), dtype=F16, device=device))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 20, 200])
def test_rows_without_numbers_stay_alone(m, device):
    """An infinity or NaN of a token shows in that token alone; what lies behind a row is not read into it."""
    from decik_amd.int4 import int4_linear_backward, int4_linear_forward, int4_weight

    n, k = 200, 328
    weight = int4_weight(*(p.to(device) for p in random_parts(n, k, 32, BF16, 1)), 32)
    for fn, cols in ((int4_linear_forward, k), (int4_linear_backward, n)):
        for dtype in (F16, BF16):
            wide = torch.full((m, cols + 8), float("nan"), dtype=dtype, device=device)
            wide[:, :cols] = make((m, cols), dtype, device, 2)
            x = wide[:, :cols]
            clean = fn(x.contiguous(), weight)
            assert torch.equal(fn(x, weight), clean) and bool(clean.isfinite().all())
            x = x.contiguous()
            x[1, cols - 1], x[2, 0] = float("inf"), float("nan")
            got = fn(x, weight)
            # (an infinity times a code that is the zero point is no number; the others' sign is the weight's)
            w = values(weight.codes(), weight.scales, weight.zeros, 32)
            at = w[:, cols - 1] if fn is int4_linear_forward else w[cols - 1]
            assert torch.equal(got[1].isnan(), at == 0) and torch.equal(got[1] > 0, at > 0)
            keep = [i for i in range(m) if i not in (1, 2)]
            assert torch.equal(got[keep], clean[keep]) and not bool(got[2].isfinite().any())


@pytest.mark.gpu
def test_outputs_take_any_row_length(device):
    """Rows behind the last token and columns behind the last row are left as they were (allocations of the outputs' sizes
    inside larger buffers are written by the C entry)."""
    from decik_amd import _lib
    from decik_amd.int4 import int4_linear_forward, int4_linear_backward, int4_weight

    for m, n, k in ((3, 45, 96), (200, 300, 136), (70, 31, 264)):
        weight = int4_weight(*(p.to(device) for p in random_parts(n, k, 32, F16, 1)), 32)
        for back, cols, total in ((0, n, k), (1, k, n)):
            x = make((m, total), F16, device, 2)
            want = (int4_linear_backward if back else int4_linear_forward)(x, weight)
            out = torch.full((m + 2, cols + 3), 7.0, dtype=F16, device=device)
            copy = int(total % 8 != 0)
            need = _lib.lib().dk_int4_linear_workspace(back, copy, m, n, k)
            work = torch.empty(max(need, 1), dtype=torch.uint8, device=device)
            _lib.call_on(device, _lib.lib().dk_int4_linear, back, x.data_ptr(), 0, total, weight.packed.data_ptr(), weight.meta.data_ptr(), 32, 0, None, 0, out.data_ptr(), 0, cols + 3, m, n, k, copy,
                         work.data_ptr(), need)
            assert torch.equal(out[:m, :cols], want)
            assert bool((out[m:] == 7).all()) and bool((out[:, cols:] == 7).all())


@pytest.mark.gpu
def test_autograd_and_differences(device):
    """Gradients through autograd equal the backward's; along a direction they equal the 64-bit form's, which is linear
    in x, so that a difference of step 1 is exact."""
    from decik_amd.int4 import Int4Linear, int4_linear_backward, int4_weight

    m, n, k, group = 37, 100, 200, 32
    parts = random_parts(n, k, group, F16, 1)
    weight = int4_weight(*(p.to(device) for p in parts), group)
    w = values(*parts, group)
    x, bias, dy = make((m, k), F16, device, 2).requires_grad_(), make((n,), F16, device, 3), make((m, n), F16, device, 4)
    Int4Linear.apply(x, weight, bias).backward(dy)
    assert torch.equal(x.grad, int4_linear_backward(dy, weight))
    step = make((m, k), F16, "cpu", 5).double()
    slope = ((step @ w.t()) * dy.double().cpu()).sum()
    room = ((x.grad.double().cpu().abs() * 2.0 ** -11 + dy.double().cpu().abs() @ (w.abs() * 2.0 ** -10 + 2.0 ** -25)) * step.abs()).sum()
    assert abs(float((x.grad.double().cpu() * step).sum() - slope)) <= float(room)
    x.grad = None
    Int4Linear.apply(x, weight).backward(dy)
    assert torch.equal(x.grad, int4_linear_backward(dy, weight))
    with pytest.raises(ValueError, match="frozen"):
        Int4Linear.apply(x, weight, bias.clone().requires_grad_())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 17, 1121), (16, 513, 18944), (40, 513, 4100), (200, 300, 4096)])
def test_same_bits_every_run(m, n, k, device):
    from decik_amd.int4 import int4_linear_backward, int4_linear_forward, int4_weight

    weight = int4_weight(*(p.to(device) for p in random_parts(n, k, 32, F16, 1)), 32)
    x, dy = make((m, k), F16, device, 2), make((m, n), F16, device, 3)
    y, dx = int4_linear_forward(x, weight), int4_linear_backward(dy, weight)
    for _ in range(3):
        assert torch.equal(y, int4_linear_forward(x, weight)) and torch.equal(dx, int4_linear_backward(dy, weight))


@pytest.mark.gpu
def test_refusals(device):
    from decik_amd.int4 import int4_linear_backward, int4_linear_forward, int4_weight

    weight = int4_weight(*(p.to(device) for p in random_parts(8, 64, 32, F16, 1)), 32)
    x, dy = make((4, 64), F16, device, 1), make((4, 8), F16, device, 2)
    for args, kw, msg in (((x[:, :32], weight), {}, "64"), ((x.float(), weight), {}, "fp16"), ((x, weight), dict(dtype=BF16), "dtype"),
                          ((x.cpu(), weight), {}, "GPU"), ((x, weight.to("cpu")), {}, "GPU"), ((x, weight, dy[0, :4]), {}, "bias"),
                          ((x, weight, dy[0].double()), {}, "bias"), ((x, weight.packed), {}, "Int4Weight"), ((x, weight, dy[0].cpu()), {}, "GPU")):
        with pytest.raises(ValueError, match=msg):
            int4_linear_forward(*args, **kw)
    for args, msg in (((x, weight), "8"), ((dy.float(), weight), "fp16"), ((dy, x), "Int4Weight")):
        with pytest.raises(ValueError, match=msg):
            int4_linear_backward(*args)
