"""Linears in 8-bit integers (decik_amd.int8): the quantizer bit for bit, products against exact integer
sums in 64 bits, both ways, over sizes around every tile and split, strides, special rows, graphs.

Tolerances. The quantizer's definition is in fp32, so integers and scales must be equal. A product is
fp32(sum) * x_scale * w_scale + bias: at most four fp32 roundings (2^-24 each) of the product's magnitude
and the bias', covered by 2^-21 of them, then one rounding to the output type (half a step, eps / 2)."""

import numpy as np
import pytest
import torch

from helpers import randn16

pytestmark = pytest.mark.gpu

TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -149}


def make(shape, dtype, device, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).to(device)


def quantized(x, col_scale=None):
    """(integers, fp32 scales) by the definition, in numpy's fp32."""
    x = x.float().cpu().numpy()
    if col_scale is not None:
        x = x * col_scale.cpu().numpy()
    top = np.abs(x).max(1).astype(np.float32)
    with np.errstate(all="ignore"):
        inv = np.where(top < np.float32(2.0 ** -120), np.float32(0), np.float32(127) / top)
        q = np.rint((x * inv[:, None]).astype(np.float32))
        scale = np.where(top < np.float32(2.0 ** -120), np.float32(0), top / np.float32(127))
    bad = ~np.isfinite(top)
    q[bad], scale[bad] = 0, np.nan
    return q.astype(np.int64), scale.astype(np.float32)


def check(y, acc, xs, ws=None, bias=None):
    value = acc.astype(np.float64) * xs.astype(np.float64)[:, None]
    if ws is not None:
        value = value * ws.astype(np.float64)
    mag = np.abs(value)
    if bias is not None:
        b = bias.double().cpu().numpy()
        value, mag = value + b, mag + np.abs(b)
    value, mag = torch.from_numpy(value), torch.from_numpy(mag)
    assert y.shape == value.shape
    err = (y.double().cpu() - value).abs()
    bound = value.abs() * (torch.finfo(y.dtype).eps / 2) + mag * 2.0 ** -21 + TINY[y.dtype]
    assert bool((err <= bound).all()), f"{int((err > bound).sum())} wrong, worst excess {(err - bound).max():.3e}"


def dot(a, b):
    return (a.astype(np.float64) @ b.astype(np.float64)).astype(np.int64)


def ints(t):
    return t.cpu().numpy().astype(np.int64)


@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 16), (2, 17), (37, 1121), (4, 2048), (6, 2056), (3, 4100),
                                    (3, 8200), (2, 18944), (2, 20488), (1, 131071)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("col", [False, True])
def test_quantizer(rows, k, dtype, col, device):
    from decik_amd.int8 import dequantize_int8, quantize_int8

    x = make((rows, k), dtype, device, 1)
    cs = make((k,), torch.float32, device, 2).abs() if col else None
    q, s = quantize_int8(x, cs)
    wq, ws = quantized(x, cs)
    assert np.array_equal(ints(q), wq) and np.array_equal(s.cpu().numpy(), ws)
    # the padding up to a multiple of 16 holds zeros
    pad = torch.as_strided(q, (rows, (k + 15) // 16 * 16), q.stride())
    assert bool((pad[:, k:] == 0).all())
    assert torch.equal(dequantize_int8(q, s), q.float() * s[:, None])


def test_quantizer_special_rows(device):
    from decik_amd.int8 import quantize_int8

    x = make((8, 100), torch.float32, device, 1)
    x[0] = 0
    x[1, 5], x[2, 99], x[3, 0] = float("inf"), float("nan"), -float("inf")
    x[4] *= 1e-38   # below 2^-120
    x[5] *= 1e-30
    x[6] *= 1e30
    q, s = quantize_int8(x)
    wq, ws = quantized(x)
    assert np.array_equal(ints(q), wq) and np.array_equal(s.cpu().numpy(), ws, equal_nan=True)
    assert bool(torch.isnan(s[1:4]).all()) and s[0] == 0 and s[4] == 0 and s[5] > 0
    assert int(q[5].abs().max()) == 127


@pytest.mark.parametrize("rows", [1, 2, 5])
def test_quantizer_views(rows, device):
    from decik_amd.int8 import quantize_int8

    base = make((16, 301), torch.bfloat16, device, 3)
    for view in (base[:rows, 1:200], base[::3, 5:][:rows], base[:rows, ::2], base.t()[:rows], base[:1].expand(rows, 301),
                 base[:rows, :300].unflatten(1, (2, 150)), base[0, :77]):
        q, s = quantize_int8(view)
        want, wants = quantize_int8(view.contiguous().reshape(-1, view.shape[-1]))
        assert torch.equal(q, want) and torch.equal(s, wants)


def int_matrix(shape, device, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int8).to(device)


# tokens around the few-row kernel's blocks and the tiles, channels around 16 and 256, k around the steps
SIZES = [(1, 1, 1), (1, 16, 64), (1, 257, 1121), (2, 40, 100), (15, 33, 128), (16, 512, 4096), (17, 48, 130),
         (20, 8208, 2100), (31, 300, 257), (32, 8208, 320), (33, 256, 128), (64, 255, 1536), (65, 257, 129), (127, 512, 384),
         (128, 100, 16), (129, 513, 2000), (255, 256, 1024), (256, 256, 256), (257, 700, 640), (300, 2057, 1121),
         (830, 256, 1536), (1000, 1000, 77), (1100, 4200, 512)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_forward_sums(m, n, k, device):
    from decik_amd.int8 import int8_matmul

    xq, wq = int_matrix((m, k), device, 1), int_matrix((n, k), device, 2)
    xs, ws = make((m,), torch.float32, device, 3).abs() * 1e-3, make((n,), torch.float32, device, 4).abs() * 1e-2
    bias = make((n,), torch.bfloat16, device, 5)
    acc = dot(ints(xq), ints(wq).T)
    for dtype, b in ((torch.float16, None), (torch.bfloat16, bias), (torch.float32, bias.float()),
                     (torch.float32, bias.half())):
        y = int8_matmul(xq, xs, wq, ws, b, dtype)
        assert y.dtype == dtype
        check(y, acc, xs.cpu().numpy(), ws.cpu().numpy(), b)


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_linear_both_ways(m, n, k, dtype, device):
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, quantize_int8

    wq, ws = quantize_int8(make((n, k), torch.float32, device, 1, 0.02))
    x, dy = make((m, k), dtype, device, 2), make((m, n), dtype, device, 3, 1e-2)
    xi, xs = quantized(x)
    check(int8_linear_forward(x, wq, ws), dot(xi, ints(wq).T), xs, ws.cpu().numpy())
    gi, gs = quantized(dy, ws)
    check(int8_linear_backward(dy, wq, ws), dot(gi, ints(wq)), gs)


def test_largest_sums(device):
    """The largest magnitudes at the largest k: sums next to 2^31."""
    from decik_amd.int8 import int8_matmul

    k = 131071
    for m in (1, 40):
        xq, wq = (torch.full((r, k), -128, dtype=torch.int8, device=device) for r in (m, 3))
        one = torch.ones(max(m, 3), device=device)
        y = int8_matmul(xq, one[:m], wq, one[:3], None, torch.float32)
        assert bool((y == float(np.float32(128 * 128 * k))).all())


def test_every_split(device):
    """Long k with few tiles: splits of k, both ways, the same integers as one pass."""
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, launch_plan, quantize_int8

    seen = set()
    for m, n, k in ((64, 256, 8960), (64, 8960, 256), (300, 600, 4000), (300, 4000, 600), (830, 1536, 8960)):
        seen |= {(0, launch_plan(False, m, n, k)["splits"] > 1), (1, launch_plan(True, m, k, n)["splits"] > 1)}
        wq, ws = quantize_int8(make((n, k), torch.float32, device, 1, 0.02))
        x, dy = make((m, k), torch.float16, device, 2), make((m, n), torch.float16, device, 3, 1e-2)
        xi, xs = quantized(x)
        bias = make((n,), torch.float16, device, 5)
        check(int8_linear_forward(x, wq, ws, bias), dot(xi, ints(wq).T), xs, ws.cpu().numpy(), bias)
        gi, gs = quantized(dy, ws)
        check(int8_linear_backward(dy, wq, ws), dot(gi, ints(wq)), gs)
    assert {(0, True), (1, True)} <= seen


# (tokens, channels, split) of a tile and sizes that run on it, odd in every direction
TILES = {(64, 64, False): (333, 2057, 1121), (64, 64, True): (301, 131, 9001), (64, 256, False): (2051, 1537, 257),
         (64, 256, True): (831, 1535, 8959), (128, 256, False): (701, 9001, 131), (128, 256, True): (513, 3585, 18945),
         (256, 256, False): (1031, 9001, 257)}


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("transposed", [False, True])
def test_every_tile(tile, transposed, device):
    """Each tile with ragged last tiles and steps, against exact sums (64-bit floats hold them)."""
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, launch_plan, quantize_int8

    m, n, k = TILES[tile]
    p = launch_plan(transposed, m, n, k)
    assert (p["tile_tokens"], p["tile_channels"], p["splits"] > 1) == tile
    if transposed:  # sums over k: the layer's output channels
        wq, ws = quantize_int8(make((k, n), torch.float32, device, 1, 0.02))
        dy = make((m, k), torch.bfloat16, device, 2)
        gq, gs = quantize_int8(dy, ws)
        check(int8_linear_backward(dy, wq, ws), (gq.double() @ wq.double()).cpu().numpy(), gs.cpu().numpy())
    else:
        wq, ws = quantize_int8(make((n, k), torch.float32, device, 1, 0.02))
        x, bias = make((m, k), torch.bfloat16, device, 2), make((n,), torch.float16, device, 3)
        xq, xs = quantize_int8(x)
        acc = (xq.double() @ wq.double().t().contiguous()).cpu().numpy()
        for dtype in (torch.bfloat16, torch.float32):
            check(int8_linear_forward(x, wq, ws, bias, dtype), acc, xs.cpu().numpy(), ws.cpu().numpy(), bias)


def test_rows_do_not_depend_on_the_batch(device):
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, quantize_int8

    wq, ws = quantize_int8(make((500, 1121), torch.float32, device, 1, 0.02))
    x, dy = make((700, 1121), torch.float16, device, 2), make((700, 500), torch.float16, device, 3)
    y, dx = int8_linear_forward(x, wq, ws), int8_linear_backward(dy, wq, ws)
    for m in (1, 16, 20, 33, 64, 100, 256, 500):
        assert torch.equal(int8_linear_forward(x[:m], wq, ws), y[:m])
        assert torch.equal(int8_linear_backward(dy[:m], wq, ws), dx[:m])


def test_foreign_layouts(device):
    """Weights and activations that quantize_int8 did not lay out: odd strides and starts, storage that
    ends inside the last 16 bytes."""
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, int8_matmul, quantize_int8

    big = int_matrix((300, 401), device, 1)
    ws = make((300,), torch.float32, device, 2).abs()
    for view, scale in ((big[:, :130], ws), (big[::2, 3:200], ws[::2]), (big.t()[:300, :299], ws),
                        (big[:, :16], ws), (big.reshape(-1)[:37 * 48].reshape(37, 48), ws[:37]),
                        (big.reshape(-1)[-5 * 33:].reshape(5, 33), ws[:5]), (big[:1, 16:40], ws[:1])):
        n, k = view.shape
        x, dy = make((40, k), torch.float16, device, 3), make((40, n), torch.float16, device, 4)
        xi, xs = quantized(x)
        acc = dot(xi, ints(view).T)
        check(int8_linear_forward(x, view, scale), acc, xs, scale.cpu().numpy())
        check(int8_linear_forward(x[:3], view, scale), acc[:3], xs[:3], scale.cpu().numpy())
        gi, gs = quantized(dy, scale)
        check(int8_linear_backward(dy, view, scale), dot(gi, ints(view)), gs)
        xq, xsc = quantize_int8(x)
        assert torch.equal(int8_matmul(xq, xsc, view, scale), int8_linear_forward(x, view, scale))
        assert torch.equal(int8_matmul(xq.clone(), xsc, view, scale), int8_linear_forward(x, view, scale))


def test_special_rows_stay_in_their_rows(device):
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, quantize_int8

    wq, ws = quantize_int8(make((300, 200), torch.float32, device, 1, 0.02))
    for m in (8, 100):
        x, dy = make((m, 200), torch.float16, device, 2), make((m, 300), torch.float16, device, 3)
        y, dx = int8_linear_forward(x, wq, ws), int8_linear_backward(dy, wq, ws)
        x[0], x[1, 3], x[2, 199], dy[3, 7], dy[4] = 0, float("inf"), float("nan"), float("nan"), 0
        y2, dx2 = int8_linear_forward(x, wq, ws), int8_linear_backward(dy, wq, ws)
        assert bool((y2[0] == 0).all()) and bool(torch.isnan(y2[1:3]).all()) and torch.equal(y2[3:], y[3:])
        assert bool(torch.isnan(dx2[3]).all()) and bool((dx2[4] == 0).all()) and torch.equal(dx2[5:], dx[5:])


def test_empty_and_shapes(device):
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, quantize_int8

    wq, ws = quantize_int8(make((40, 64), torch.float32, device, 1))
    assert int8_linear_forward(torch.empty((0, 64), dtype=torch.float16, device=device), wq, ws).shape == (0, 40)
    assert int8_linear_backward(torch.empty((2, 0, 40), device=device), wq, ws).shape == (2, 0, 64)
    x = make((2, 3, 64), torch.bfloat16, device, 2)
    y = int8_linear_forward(x, wq, ws)
    assert y.shape == (2, 3, 40) and torch.equal(y.reshape(6, 40), int8_linear_forward(x.reshape(6, 64), wq, ws))
    assert int8_linear_forward(x[0, 0], wq, ws).shape == (40,)
    assert int8_linear_forward(x, wq, ws, dtype=torch.float32).dtype == torch.float32


def test_autograd(device):
    """Gradients against the dequantized linear: each term of a row is off by at most half a step of the
    row's gradient scale, g_scale / 2 * |wq|; then fp32 and output roundings."""
    from decik_amd.int8 import Int8Linear, dequantize_int8, quantize_int8

    wq, ws = quantize_int8(make((130, 96), torch.float32, device, 1, 0.02))
    x = make((2, 33, 96), torch.float16, device, 2).requires_grad_(True)
    bias = make((130,), torch.float16, device, 3)
    with pytest.raises(ValueError, match="frozen"):
        Int8Linear.apply(x, wq, ws, bias.clone().requires_grad_(True))
    y = Int8Linear.apply(x, wq, ws, bias)
    dy = make(y.shape, torch.float16, device, 4)
    y.backward(dy)
    w = dequantize_int8(wq, ws).double()
    want = (dy.double() @ w).reshape(66, 96)
    _, gs = quantize_int8(dy, ws)
    slack = gs.double()[:, None] * 0.5 * wq.double().abs().sum(0)
    got = x.grad.double().reshape(66, 96)
    bound = slack * 1.001 + want.abs() * 2.0 ** -11 + slack * 2.0 ** -10 + 2.0 ** -25
    assert bool(((got - want).abs() <= bound).all())
    assert x.grad.dtype == torch.float16
    # the forward along a direction: quantized twice, half a step a term each
    xi, xs = quantized(x.detach().reshape(66, 96))
    lin = torch.from_numpy(xi * xs.astype(np.float64)[:, None]).to(device) @ w.T + bias.double()
    assert bool(((y.reshape(66, 130).double() - lin).abs() <= lin.abs() * 2.0 ** -11 + 2.0 ** -16).all())


def test_without_bias(device):
    """The bias left out of the call, or given as None: the same values and gradients."""
    from decik_amd.int8 import Int8Linear, quantize_int8

    w = quantize_int8(randn16((48, 80), 3, device))
    results = []
    for args in (w, (*w, None)):
        x = randn16((5, 80), 4, device).requires_grad_(True)
        y = Int8Linear.apply(x, *args)
        results.append((y, torch.autograd.grad(y, x, torch.ones_like(y))[0]))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_captured_graphs(device):
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, quantize_int8

    wq, ws = quantize_int8(make((512, 4096), torch.float32, device, 1, 0.02))
    xs = [make((m, 4096), torch.float16, device, m) for m in (1, 64)]
    dy = make((64, 512), torch.float16, device, 9)
    step = lambda: [int8_linear_forward(x, wq, ws) for x in xs] + [int8_linear_backward(dy, wq, ws)]  # noqa: E731
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for i in range(3):
        for x in xs:
            x += 0.25
        dy *= -1.5
        for graph, _ in graphs:
            graph.replay()
        want = step()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_other_stream(device):
    from decik_amd.int8 import int8_linear_forward, quantize_int8

    wq, ws = quantize_int8(make((256, 8960), torch.float32, device, 1, 0.02))
    x = make((64, 8960), torch.float16, device, 2)
    want = int8_linear_forward(x, wq, ws)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(int8_linear_forward(x, wq, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_refusals(device):
    from decik_amd._lib import DecikError
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, int8_matmul, quantize_int8

    wq, ws = quantize_int8(make((40, 64), torch.float32, device, 1))
    x = make((4, 64), torch.float16, device, 2)
    xq, xs = quantize_int8(x)
    bad = [lambda: quantize_int8(x.cpu()), lambda: quantize_int8(x.double()), lambda: quantize_int8(x, ws),
           lambda: quantize_int8(x, ws[:1].half().expand(64)), lambda: int8_linear_forward(x[:, :60], wq, ws),
           lambda: int8_linear_forward(x, wq.cpu(), ws), lambda: int8_linear_forward(x, wq.float(), ws),
           lambda: int8_linear_forward(x, wq, ws[:10]), lambda: int8_linear_forward(x, wq, ws, x[0]),
           lambda: int8_linear_forward(x, wq, ws, dtype=torch.float64), lambda: int8_linear_backward(x, wq, ws),
           lambda: int8_linear_backward(make((4, 40), torch.float16, device, 1), wq, ws, 60),
           lambda: int8_matmul(xq, xs[:2], wq, ws), lambda: int8_matmul(xq[:, :32], xs, wq, ws),
           lambda: int8_matmul(xq, xs, wq, ws.half())]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(DecikError, match="131071"):
        quantize_int8(torch.zeros((1, 131072), device=device))


# the largest tile with k split, ragged in every direction: seven splits of one narrow tile column, three uneven ones
# of three columns
SPLIT_TILES = {(4121, 257, 18945): 7, (6229, 725, 15023): 3}


@pytest.mark.parametrize("size", SPLIT_TILES)
@pytest.mark.parametrize("transposed", [False, True])
def test_largest_tile_with_splits(size, transposed, device):
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, launch_plan, quantize_int8

    m, n, k = size
    assert launch_plan(transposed, m, n, k) == dict(tile_tokens=256, tile_channels=256, splits=SPLIT_TILES[size],
                                                    fused=False)
    if transposed:  # sums over k: the layer's output channels
        wq, ws = quantize_int8(make((k, n), torch.float32, device, 1, 0.02))
        dy = make((m, k), torch.float16, device, 2)
        gq, gs = quantize_int8(dy, ws)
        acc = (gq.double() @ wq.double()).cpu().numpy()
        for dtype in (torch.float16, torch.float32):
            check(int8_linear_backward(dy, wq, ws, dtype=dtype), acc, gs.cpu().numpy())
    else:
        wq, ws = quantize_int8(make((n, k), torch.float32, device, 1, 0.02))
        x, bias = make((m, k), torch.float16, device, 2), make((n,), torch.float32, device, 3)
        xq, xs = quantize_int8(x)
        acc = (xq.double() @ wq.double().t().contiguous()).cpu().numpy()
        for dtype in (torch.float16, torch.float32):
            check(int8_linear_forward(x, wq, ws, bias, dtype), acc, xs.cpu().numpy(), ws.cpu().numpy(), bias)
