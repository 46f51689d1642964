"""4-bit linears whose gradient rows are 2^22 elements and more: the plans and strides that keep a tile's rows inside a buffer
of 2^31 bytes (on the CPU), and the products."""

import ctypes

import pytest
import torch

from test_int4_gpu import F16, check_backward, make, random_parts, values
from test_more_ops_abi import error, lin

LONG = 1 << 22


def span(tokens, m, ld):
    """Bytes from the first to behind the last row of a tile."""
    return min(tokens, m) * ld * 2


@pytest.mark.parametrize("forced", [None, "256,1", "128,2"])
def test_rows_of_a_tile_lie_in_a_buffer(forced, monkeypatch):
    from decik_amd.int4 import launch_plan

    if forced:
        monkeypatch.setenv("DECIK_INT4_PLAN", forced)
    for n in (LONG - 8, LONG - 1, LONG, LONG + 3, LONG + 8, 2 * LONG - 1):
        for m in (2, 64, 65, 200, 256, 4000):
            for k in (1, 40, 4096):
                padded = (n + 7) // 8 * 8
                assert span(launch_plan(True, m, n, k)["tile_tokens"], m, padded) <= 2 ** 31
    assert launch_plan(True, 256, LONG - 8, 4096)["tile_tokens"] > 64


def test_strides():
    """Refused before a launch, or taken as far as the workspace's check."""
    need = dict(m=2, k=64, ldy=64)
    assert "workspace" in error(lin(1, n=LONG + 8, ldx=LONG + 8, **need))
    assert "workspace" in error(lin(1, n=2 * LONG - 8, ldx=2 * LONG - 8, **need))
    assert "workspace" in error(lin(1, n=LONG + 3, ldx=0, copy=1, **need))
    assert "stride" in error(lin(1, n=LONG + 8, ldx=2 * LONG, **need))
    assert "stride" in error(lin(1, n=LONG - 8, ldx=LONG, **need))
    assert "stride" in error(lin(0, n=LONG + 8, ldx=LONG, m=100, k=64, ldy=LONG + 8))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [LONG + 8, LONG + 3])
def test_gradients_of_long_rows(n, device):
    """Packed rows, rows of a wider buffer, one row shared by all tokens; 65 tokens are two tiles."""
    from decik_amd.int4 import int4_linear_backward, int4_weight

    k, group = 40, 32
    parts = [t.to(device) for t in random_parts(n, k, group, F16, 1)]
    weight, w = int4_weight(*parts, group), values(*parts, group)
    dy = torch.randn((65, n), generator=torch.Generator(device).manual_seed(2), device=device).to(F16)
    full = int4_linear_backward(dy, weight)
    check_backward(full, dy, w)
    check_backward(int4_linear_backward(dy[:2], weight), dy[:2], w)
    wide = torch.zeros((3, n + 24), dtype=F16, device=device)[:, 8:8 + n].copy_(dy[:3])
    assert torch.equal(int4_linear_backward(wide, weight), int4_linear_backward(dy[:3], weight))
    shared = dy[:1].expand(65, n)
    assert torch.equal(int4_linear_backward(shared, weight), int4_linear_backward(shared.contiguous(), weight))


@pytest.mark.gpu
def test_a_step_with_long_rows(device):
    from decik_amd.int4 import Int4Linear, int4_linear_backward, int4_weight

    n, k = LONG + 8, 40
    weight = int4_weight(*(t.to(device) for t in random_parts(n, k, 32, F16, 1)), 32)
    x = make((2, k), F16, device, 2).requires_grad_()
    dy = make((2, n), F16, device, 3)
    Int4Linear.apply(x, weight).backward(dy)
    assert torch.equal(x.grad, int4_linear_backward(dy, weight))
