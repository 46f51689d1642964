"""The largest scales of a 4-bit weight. bf16 operands are formed as (1024 + code) scale - (1024 + zero) scale, whose products are
numbers in fp32 for scales below 2^117; others are refused, as are scales that are no numbers."""

import pytest
import torch

from test_int4_gpu import BF16, F16, F32, random_parts
from test_int4_scales_gpu import ones_at, spread, weight_of


@pytest.mark.parametrize("scale", [float("inf"), -float("inf"), float("nan"), 2.0 ** 117, -(2.0 ** 117), 3e38])
def test_refusals(scale):
    from decik_amd.int4 import int4_weight

    codes, scales, zeros = random_parts(4, 64, 32, BF16, 1)
    scales[2, 1] = scale
    with pytest.raises(ValueError, match="2\\^117"):
        int4_weight(codes, scales, zeros, 32)
    if scale * 0 != 0:
        with pytest.raises(ValueError, match="2\\^117"):
            int4_weight(codes, scales.to(F16), zeros, 32)
    scales[2, 1] = -1.9921875 * 2.0 ** 116
    assert int4_weight(codes, scales, zeros, 32).scales[2, 1] == scales[2, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("plan", ["64,1", "128,2", "256,1"])
def test_the_largest_come_out(plan, device, monkeypatch):
    from decik_amd.int4 import int4_linear_backward, int4_linear_forward

    monkeypatch.setenv("DECIK_INT4_PLAN", plan)
    m, n, k, group = 270, 523, 650, 32
    weight, w = weight_of(n, k, group, spread(n, k, group, BF16, 100, 116.9, 1), 1, device)
    w = w.float().to(BF16).float()
    cols, rows = torch.arange(m) * 2 % k, torch.arange(m) * 5 % n
    assert torch.equal(int4_linear_forward(ones_at(cols, k, BF16, device), weight, None, F32), w[:, cols].t())
    assert torch.equal(int4_linear_backward(ones_at(rows, n, BF16, device), weight, F32), w[rows])
