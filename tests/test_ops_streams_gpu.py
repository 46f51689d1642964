"""Seeded dropout, the rotations and the seeded LoRA pair on two streams at once: each call has its own workspace and
runs on its caller's stream, so every result is that of a call alone, bit for bit."""

import pytest
import torch

from helpers import randn16

pytestmark = pytest.mark.gpu


def on_two_streams(call):
    want = call()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(call())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_dropout(device):
    from decik_amd.dropout import dropout_backward, dropout_forward, rng_state

    x, g, rng = randn16((830, 1536), 1, device), randn16((830, 1536), 2, device), rng_state(3, 4, device)
    on_two_streams(lambda: (*dropout_forward(x, rng, (0.1, 0.4)), dropout_backward([g, x], rng, (0.1, 0.4))))


@pytest.mark.parametrize("norm", [False, True])
def test_rotations(norm, device):
    from decik_amd.rope import (axes_rope_backward, axes_rope_forward, qk_norm_rope_backward,
                                qk_norm_rope_forward)

    t, h, hk, d = 830, 12, 2, 128
    q, k = randn16((t, h * d), 1, device), randn16((t, hk * d), 2, device)
    gq, gk = randn16((1, h, t, d), 3, device, 1e-2), randn16((1, hk, t, d), 4, device, 1e-2)
    w = (randn16((d,), 5, device), randn16((d,), 6, device)) if norm else (None, None)
    cos, sin = (randn16((t, d), 7 + i, device).float() for i in range(2))
    pos = torch.arange(3 * t, device=device).reshape(3, t)
    inv = (1e6 ** (-torch.arange(0, d, 2).double() / d)).float().to(device)
    sections = [16, 24, 24]

    def call():
        outs = (*qk_norm_rope_forward(q, k, *w, cos, sin, h, hk),
                *qk_norm_rope_backward(gq, gk, q, k, *w, cos, sin),
                *axes_rope_forward(q, k, pos, inv, sections, h, hk, False, *w),
                *axes_rope_backward(gq, gk, pos, inv, sections, False, q, k, *w))
        return [o for o in outs if o is not None]

    on_two_streams(call)


@pytest.mark.parametrize("rank", [16, 32])
def test_seeded_pair(rank, device):
    from decik_amd.dropout import rng_state
    from decik_amd.lora import LoRAPairSeeded

    w, rng = 512, rng_state(5, 6, device)
    shapes = ((rank, w), (384, rank), (rank, w), (128, rank))
    x = randn16((300, w), 1, device).requires_grad_(True)
    ab = [randn16(s, 2 + i, device, 0.05).requires_grad_(True) for i, s in enumerate(shapes)]
    grads = [randn16((300, n), 10 + n, device, 1e-2) for n in (384, 128)]

    def call():
        outs = LoRAPairSeeded.apply(x, rng, *ab, 2.0, 1.5, 0.1, 0.25)
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, [x, *ab], grads)]

    on_two_streams(call)
