"""The autograd form of the residual stream forms the gradients that are asked for: sums over the rows only for the weights
and the channel gate that want one, a gate's gradient only where it does. What is formed is what the whole backward gives."""

import pytest
import torch

from test_norm_gpu import EPS, F16, F32, gate_of, make

pytestmark = pytest.mark.gpu


ASKED = [(0,), (1,), (2,), (3,), (4,), (0, 1), (2, 4), (0, 3), (0, 1, 2, 3, 4)]


@pytest.mark.parametrize("asked,gate", [(a, g) for a in ASKED for g in ("none", "channel", "token", "element") if (a, g) != ((4,), "none")])
def test_only_what_is_asked_for(asked, gate, device, monkeypatch):
    from decik_amd import _lib, norm

    b, t, width = 2, 19, 320
    inputs = [make((b, t, width), F16, device, 1), make((b, t, width), F32, device, 2), make((width,), F32, device, 3),
              make((width,), F32, device, 4), gate_of(gate, (b, t, width), F32, device)]
    leaves = [v.clone().requires_grad_() if i in asked and v is not None else v for i, v in enumerate(inputs)]
    h, y = norm.residual_norm(*leaves, 0.5, EPS)
    gh, gy = make(h.shape, F32, device, 5), make(y.shape, F16, device, 6)
    want = norm.residual_norm_backward(gh, gy, *inputs, 0.5, EPS)
    calls, call_on = [], norm.call_on

    def spy(dev, fn, desc, *args):
        calls.append(_lib.ResidualNorm.from_buffer_copy(desc))
        return call_on(dev, fn, desc, *args)

    monkeypatch.setattr(norm, "call_on", spy)
    torch.autograd.backward([h, y], [gh, gy])
    for i, leaf in enumerate(leaves):
        if leaf is not None and leaf.requires_grad:
            assert torch.equal(leaf.grad, want[i].to(leaf.dtype))
    (d,) = calls
    assert (d.dweight is not None, d.dpost_weight is not None) == (2 in asked, 3 in asked)
    assert (d.dgate is not None) == (4 in asked and gate != "none")
