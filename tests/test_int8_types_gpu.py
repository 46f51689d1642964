"""Types of the 8-bit linear (decik_amd.int8): fp32 activations and gradients, outputs unlike the inputs, both ways on
every tile. Tolerances: test_int8_gpu."""

import pytest
import torch

from test_int8_gpu import SIZES, TILES, check, dot, ints, make, quantized

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_fp32_both_ways(m, n, k, device):
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, quantize_int8

    wq, ws = quantize_int8(make((n, k), torch.float32, device, 1, 0.02))
    x, dy = make((m, k), torch.float32, device, 2), make((m, n), torch.float32, device, 3, 1e-2)
    xi, xs = quantized(x)
    y = int8_linear_forward(x, wq, ws)
    assert y.dtype == torch.float32
    check(y, dot(xi, ints(wq).T), xs, ws.cpu().numpy())
    gi, gs = quantized(dy, ws)
    dx = int8_linear_backward(dy, wq, ws)
    assert dx.dtype == torch.float32
    check(dx, dot(gi, ints(wq)), gs)


@pytest.mark.parametrize("m", [1, 2, 5, 40])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out", TYPES)
def test_outputs_unlike_inputs(m, dtype, out, device):
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, quantize_int8

    n, k = 131, 301
    wq, ws = quantize_int8(make((n, k), torch.float32, device, 1, 0.02))
    x, dy, bias = make((m, k), dtype, device, 2), make((m, n), dtype, device, 3, 1e-2), make((n,), dtype, device, 4)
    xi, xs = quantized(x)
    y = int8_linear_forward(x, wq, ws, bias, out)
    assert y.dtype == out
    check(y, dot(xi, ints(wq).T), xs, ws.cpu().numpy(), bias)
    gi, gs = quantized(dy, ws)
    dx = int8_linear_backward(dy, wq, ws, dtype=out)
    assert dx.dtype == out
    check(dx, dot(gi, ints(wq)), gs)


@pytest.mark.parametrize("tile", TILES)
def test_every_tile_in_every_type(tile, device):
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, quantize_int8

    m, n, k = TILES[tile]
    w = quantize_int8(make((n, k), torch.float32, device, 1, 0.02))
    x = make((m, k), torch.float32, device, 2)
    xq, xs = quantize_int8(x)
    acc = (xq.double() @ w[0].double().t().contiguous()).cpu().numpy()
    for out in TYPES:
        check(int8_linear_forward(x, *w, dtype=out), acc, xs.cpu().numpy(), w[1].cpu().numpy())
    w = quantize_int8(make((k, n), torch.float32, device, 3, 0.02))
    gq, gs = quantize_int8(x, w[1])
    acc = (gq.double() @ w[0].double()).cpu().numpy()
    for out in TYPES:
        check(int8_linear_backward(x, *w, dtype=out), acc, gs.cpu().numpy())
