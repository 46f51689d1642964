"""Element offsets past 32 bits: the dropout, rotation and 8-bit entries on rows that lie far apart and on
outputs of more than 2^32 elements give, bit for bit, what they give on few rows close together."""

import numpy as np
import pytest
import torch

from helpers import randn16
from test_dropout_gpu import M32, philox

pytestmark = pytest.mark.gpu

FAR = 2 ** 31


def far(t):
    """A copy of t [rows, width] whose rows lie 2^31 elements apart."""
    rows, width = t.shape
    base = torch.empty((rows - 1) * FAR + width, dtype=t.dtype, device=t.device)
    view = base.as_strided((rows, width), (FAR, 1))
    view.copy_(t)
    return view


def test_far_rows(device):
    from decik_amd.dropout import dropout_backward, dropout_forward, rng_state
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, quantize_int8
    from decik_amd.rope import qk_norm_rope_backward, qk_norm_rope_forward

    x = randn16((3, 256), 1, device)
    y = far(x)
    rng = rng_state(3, 4, device)
    assert torch.equal(dropout_forward(y, rng, (0.3,))[0], dropout_forward(x, rng, (0.3,))[0])
    assert torch.equal(dropout_backward([y, x], rng, (0.3, 0.2)), dropout_backward([x, x], rng, (0.3, 0.2)))
    for a, b in zip(quantize_int8(y), quantize_int8(x)):
        assert torch.equal(a, b)
    w = quantize_int8(randn16((256, 256), 2, device))
    for m in (2, 3):  # quantized inside the product, and before it
        assert torch.equal(int8_linear_forward(y[:m], *w), int8_linear_forward(x[:m], *w))
        assert torch.equal(int8_linear_backward(y[:m], *w), int8_linear_backward(x[:m], *w))
    nw, tab = randn16((64,), 3, device), torch.rand((3, 64), device=device)
    for a, b in zip(*(qk_norm_rope_forward(t, t, nw, nw, tab, tab, 4, 4) for t in (y, x))):
        assert torch.equal(a, b)
    g = randn16((1, 4, 3, 64), 4, device)
    for a, b in zip(*(qk_norm_rope_backward(g, g, t, t, nw, nw, tab, tab) for t in (y, x))):
        assert torch.equal(a, b)


def test_far_weights(device):
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, quantize_int8

    n, k, ld = 1100, 64, 2 ** 22
    wq, ws = quantize_int8(randn16((n, k), 1, device))
    base = torch.zeros((n - 1) * ld + k, dtype=torch.int8, device=device)
    wide = base.as_strided((n, k), (ld, 1))
    wide.copy_(wq)
    for m in (1, 5, 70, 400):
        x, dy = randn16((m, k), 2, device), randn16((m, n), 3, device)
        assert torch.equal(int8_linear_forward(x, wide, ws), int8_linear_forward(x, wq, ws))
        assert torch.equal(int8_linear_backward(dy, wide, ws), int8_linear_backward(dy, wq, ws))


def test_large_dropout(device):
    from decik_amd.dropout import dropout_backward, dropout_forward, rng_state

    rows, width, seed, offset, p = 2 ** 20 + 3, 4096, 9, 5, 0.25
    x = randn16((1, width), 1, device)
    rng = rng_state(seed, offset, device)
    (out,) = dropout_forward(x.expand(rows, width), rng, (p,))
    assert out.numel() > 2 ** 32
    g = np.arange(width // 8)
    for row in (0, rows // 2, rows - 1):
        words = philox([g, np.full_like(g, row), np.full_like(g, offset), np.zeros_like(g)], (seed & M32, seed >> 32))
        bits = np.stack([(words[e // 2] >> np.uint64(16 * (e % 2))) & np.uint64(0xFFFF) for e in range(8)], 1)
        keep = torch.from_numpy(bits.reshape(-1) >= np.uint64(round(p * 65536))).to(device)
        want = torch.where(keep, (x[0].float() * (1 / (1 - p))).half(), torch.zeros_like(x[0]))
        assert torch.equal(out[row], want), row
    # the masks once more: zeros stay, and the kept are scaled again
    assert torch.equal(dropout_backward([out], rng, (p,))[-1], (out[-1].float() * (1 / (1 - p))).half())


def test_large_rotation(device):
    from decik_amd.rope import axes_rope_backward, axes_rope_forward

    t, d = 2 ** 23 + 5, 256
    row = randn16((2 * d,), 1, device)
    q, k = row.expand(t, 2 * d), row[:d].expand(t, d)
    pos = torch.arange(t, dtype=torch.int32, device=device)[None]
    inv = (1e4 ** (-torch.arange(0, d, 2).double() / d)).float().to(device)
    big = axes_rope_forward(q, k, pos, inv, [d // 2], 2, 1)
    assert big[0].numel() > 2 ** 32
    few = axes_rope_forward(q[-3:], k[-3:], pos[:, -3:], inv, [d // 2], 2, 1)
    for a, b in zip(big, few):
        assert torch.equal(a[:, :, -3:], b)
    back = axes_rope_backward(*big, pos, inv, [d // 2])
    want = axes_rope_backward(*few, pos[:, -3:], inv, [d // 2])
    for a, b in zip(back[:2], want[:2]):
        assert torch.equal(a[:, -3:], b)


def test_large_products(device):
    from decik_amd.int8 import int8_linear_backward, int8_linear_forward, quantize_int8

    m, n, k = 2 ** 18 + 1, 16400, 16
    x = randn16((m, k), 1, device)
    y = int8_linear_forward(x, *quantize_int8(randn16((n, k), 2, device)))
    assert y.numel() > 2 ** 32
    assert torch.equal(y[-300:], int8_linear_forward(x[-300:], *quantize_int8(randn16((n, k), 2, device))))
    del y
    w = quantize_int8(randn16((k, n), 3, device))
    dx = int8_linear_backward(x, *w)
    assert torch.equal(dx[-300:], int8_linear_backward(x[-300:], *w))
