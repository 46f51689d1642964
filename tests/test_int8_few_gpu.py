"""The forms of the 8-bit linear for a few tokens (decik_amd.int8): the weight streamed to registers, x quantized before
(one or two blocks of 16 tokens, 4 or 16 waves a work-group) or inside the product (one or two tokens, 4 or 16 waves),
around the sizes where one gives way to another. Tolerances: test_int8_gpu."""

import pytest
import torch

from test_int8_gpu import check, dot, int_matrix, ints, make, quantized

# streamed to registers: blocks of tokens x waves. 16 waves below 8177 channels from k = 8192 on.
STREAMED = [(3, 40, 1000), (9, 2057, 1121), (16, 777, 4099), (13, 513, 8961), (16, 1121, 8192), (5, 100, 8191),
            (17, 300, 1121), (31, 100, 640), (32, 131, 4100), (17, 257, 8961), (29, 257, 9001), (32, 500, 8192)]
TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("size", STREAMED)
def test_sizes_are_streamed(size):
    from decik_amd.int8 import launch_plan

    assert launch_plan(False, *size) == dict(tile_tokens=0, tile_channels=16, splits=1, fused=False)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", STREAMED)
def test_streamed(m, n, k, device):
    from decik_amd.int8 import int8_linear_forward, int8_matmul, quantize_int8

    wq, ws = int_matrix((n, k), device, 1), make((n,), torch.float32, device, 2).abs() * 1e-2
    for dtype in TYPES:
        x, bias = make((m, k), dtype, device, 3), make((n,), dtype, device, 4)
        xi, xs = quantized(x)
        acc = dot(xi, ints(wq).T)
        for out in TYPES:
            y = int8_linear_forward(x, wq, ws, bias, out)
            check(y, acc, xs, ws.cpu().numpy(), bias)
            assert torch.equal(int8_matmul(*quantize_int8(x), wq, ws, bias, out), y)


# 16 waves below 8177 channels; x quantized inside as long as its integers (k to the next 64) take 32 KB
@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 8176, 200), (1, 8177, 1121), (2, 8209, 640), (2, 18944, 129), (1, 33, 32768),
                                   (1, 33, 32769), (2, 33, 16384), (2, 33, 16385), (1, 8193, 16385), (2, 1, 1)])
def test_quantized_inside(m, n, k, device):
    from decik_amd.int8 import int8_linear_forward, int8_matmul, launch_plan, quantize_int8

    assert launch_plan(False, m, n, k)["fused"] == (m * ((k + 63) // 64 * 64) <= 32768)
    wq, ws = int_matrix((n, k), device, 1), make((n,), torch.float32, device, 2).abs() * 1e-2
    for dtype in TYPES:
        x, bias = make((m, k), dtype, device, 3), make((n,), dtype, device, 4)
        xi, xs = quantized(x)
        acc = dot(xi, ints(wq).T)
        for out, b in zip(TYPES, (bias, None, bias)):
            y = int8_linear_forward(x, wq, ws, b, out)
            check(y, acc, xs, ws.cpu().numpy(), b)
            # quantized before the product: the same bits
            assert torch.equal(int8_matmul(*quantize_int8(x), wq, ws, b, out), y)
