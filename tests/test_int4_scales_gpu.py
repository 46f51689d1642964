"""The weights that the 4-bit products stand for, seen one by one: tokens with a single 1 read columns (backward: rows) of W,
so that an fp32 output is W as the matrix cores take it. Few tokens: W itself, exactly. Tiles and the backward: W rounded once
to the activations' type, whatever the scales' type -- bf16 scales reach far below and above fp16's."""

import pytest
import torch

from test_int4_gpu import BF16, F16, F32, check_backward, check_forward, make, random_parts, values


def weight_of(n, k, group, scales, seed, device):
    """(Int4Weight, W in float64) of random codes and zero points."""
    from decik_amd.int4 import int4_weight

    codes, _, zeros = random_parts(n, k, group, F16, seed)
    parts = [t.to(device) for t in (codes, scales, zeros)]
    return int4_weight(*parts, group), values(*parts, group)


def spread(n, k, group, dtype, low, high, seed):
    """Scales of all significant bits between 2^low and 2^high, either sign."""
    g = torch.Generator().manual_seed(seed)
    shape = (n, -(-k // group))
    size = torch.exp2(torch.rand(shape, generator=g, dtype=torch.float64) * (high - low) + low)
    return (size * (1 - 2 * torch.randint(0, 2, shape, generator=g))).to(dtype)


def ones_at(cols, total, dtype, device):
    x = torch.zeros((len(cols), total), dtype=dtype, device=device)
    x[torch.arange(len(cols)), cols] = 1.0
    return x


# fp16 holds a scale of eight bits from 2^-17 on, and its smallest values are steps of 2^-24; sixteen of the largest stay below
# 65504 (an infinite weight would show in every token)
RANGES = {F16: (-24, 11.9), BF16: (-28, 11.9)}


@pytest.mark.gpu
@pytest.mark.parametrize("plan", ["64,1", "64,3", "128,1", "128,2", "256,1", "256,2"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scale_dtype", [F16, BF16])
def test_weights_are_rounded_once(plan, dtype, scale_dtype, device, monkeypatch):
    from decik_amd.int4 import int4_linear_backward, int4_linear_forward

    monkeypatch.setenv("DECIK_INT4_PLAN", plan)
    m, n, k = 270, 523, 650
    for group in (32, 64, 128):
        weight, w = weight_of(n, k, group, spread(n, k, group, scale_dtype, *RANGES[scale_dtype], group), group, device)
        # (at most 13 bits for bf16 scales, 16 for fp16's: exact in fp32, from which each type rounds)
        w = w.float().to(dtype).float()
        cols, rows = torch.arange(m) * 2 % k, torch.arange(m) * 5 % n
        assert torch.equal(int4_linear_forward(ones_at(cols, k, dtype, device), weight, None, F32), w[:, cols].t())
        assert torch.equal(int4_linear_backward(ones_at(rows, n, dtype, device), weight, F32), w[rows])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 16, 29])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scale_dtype", [F16, BF16])
def test_few_tokens_round_no_weight(m, dtype, scale_dtype, device):
    from decik_amd.int4 import int4_linear_forward

    n, k = 523, 650
    for group in (32, 64, 128):
        weight, w = weight_of(n, k, group, spread(n, k, group, scale_dtype, *RANGES[scale_dtype], group), group, device)
        cols = torch.arange(m) * 23 % k
        assert torch.equal(int4_linear_forward(ones_at(cols, k, dtype, device), weight, None, F32), w[:, cols].t().float())


@pytest.mark.gpu
def test_pieces_of_few_tokens_round_no_weight(device):
    """What a caller does with more tokens where W is not to be rounded."""
    from decik_amd.int4 import int4_linear_forward, launch_plan

    n, k, m = 4200, 4100, 100
    weight, w = weight_of(n, k, 128, spread(n, k, 128, F16, -24, 11.9, 1), 1, device)
    cols = torch.arange(m) * 41 % k
    x = ones_at(cols, k, F16, device)
    assert launch_plan(False, 32, n, k)["waves"] and not launch_plan(False, m, n, k)["waves"]
    exact = w[:, cols].t().float()
    assert torch.equal(torch.cat([int4_linear_forward(p, weight, None, F32) for p in x.split(32)]), exact)
    assert torch.equal(int4_linear_forward(x, weight, None, F32), w[:, cols].t().half().float())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [40, 300])
def test_zero_weights_under_scales_past_fp16(m, device):
    """Codes that are their zero points stand for 0 under any scale: what a scale of 1 gives."""
    from decik_amd.int4 import int4_linear_backward, int4_linear_forward, int4_weight

    n, k, group = 3000, 6000, 32  # (40 tokens of so many weights go by tiles)
    codes, scales, zeros = (t.to(device) for t in random_parts(n, k, group, BF16, 1))
    zeros[::3, 2] = zeros[::3, 2].clamp(max=15)
    codes[::3, 64:96] = zeros[::3, 2:3]
    one, large = scales.clone(), scales.clone()
    one[::3, 2], large[::3, 2] = 1.0, 70144.0
    x, dy = make((m, k), F16, device, 2), make((m, n), F16, device, 3)
    for fn, by in ((int4_linear_forward, x), (int4_linear_backward, dy)):
        want, got = (fn(by, int4_weight(codes, s, zeros, group)) for s in (one, large))
        assert bool(want.isfinite().all()) and torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(70, 1300, 650), (830, 1536, 1121)])
def test_products_of_small_bf16_scales(m, n, k, device):
    from decik_amd.int4 import int4_linear_backward, int4_linear_forward

    for group in (32, 128):
        weight, w = weight_of(n, k, group, spread(n, k, group, BF16, -20, -15, group), group, device)
        x, dy = make((m, k), F16, device, 2), make((m, n), F16, device, 3)
        for out in (None, F32):
            check_forward(int4_linear_forward(x, weight, None, out), x, w, None, f"forward {group}")
            check_backward(int4_linear_backward(dy, weight, out), dy, w, f"backward {group}")
