"""Seeded dropout (decik_amd.dropout) against its definition in 64 bits: masks of the published
generator bit for bit, values within their roundings, forward and backward, types, widths that no
vector divides, strides, infinities and NaN in dropped places, replays of a captured graph.

Tolerance: a kept value is fp32(x * scale), scale itself rounded to fp32 (2^-24 each), rounded once to
the output type (half a step, eps / 2): |out - exact| <= |exact| (eps / 2 + 2^-22) + the type's
smallest half step. A sum of nb branches adds nb - 1 roundings of partial sums, each within 2^-24 of the
sum of magnitudes: 2^-21 of it covers four branches."""

import numpy as np
import pytest
import torch

M32 = 0xFFFFFFFF


def philox(c, key):
    """Philox4x32-10 on uint64 arrays c[0..3] (values below 2^32), key two Python ints."""
    c = [np.asarray(v, np.uint64) for v in c]
    k0, k1 = key
    for _ in range(10):
        a = c[0] * np.uint64(0xD2511F53)
        b = c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & np.uint64(M32),
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & np.uint64(M32)]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return c


def keep_mask(rows, width, seed, offset, p):
    groups = -(-width // 8)
    g, r = np.meshgrid(np.arange(groups), np.arange(rows))
    offset %= 2 ** 64
    words = philox([g, r, np.full_like(g, offset & M32), np.full_like(g, 0) + np.uint64(offset >> 32)],
                   (seed & M32, (seed >> 32) & M32))
    halves = np.empty((rows, groups, 8), np.uint64)
    for e in range(8):
        halves[:, :, e] = (words[e // 2] >> np.uint64(16 * (e % 2))) & np.uint64(0xFFFF)
    return halves.reshape(rows, -1)[:, :width] >= np.uint64(round(p * 65536))


def scale_of(p):
    thr = round(p * 65536)
    return 65536.0 / (65536 - thr) if thr < 65536 else 0.0


TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def check(out, exact, mags=None):
    exact = torch.from_numpy(exact)
    mags = exact.abs() if mags is None else torch.from_numpy(mags)
    err = (out.double().cpu() - exact).abs()
    bound = exact.abs() * (torch.finfo(out.dtype).eps / 2 + 2.0 ** -22) + mags * 2.0 ** -21 + TINY[out.dtype]
    assert bool((err <= bound).all()), f"worst excess {(err - bound).max().item():.3e}"


def test_generator_known_answers():
    """The generator's published test vectors."""
    cases = [((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
             ((M32,) * 4, (M32, M32), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
             ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
              (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))]
    for c, k, want in cases:
        assert tuple(int(v) for v in philox(c, k)) == want


gpu = pytest.mark.gpu
SEED = 0x1234567890ABCDEF


def make(shape, dtype, device, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).to(device)


@gpu
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 8), (3, 7), (5, 9), (64, 64), (333, 1121), (830, 1536), (2, 18944)])
@pytest.mark.parametrize("x_dtype,dtype", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                           (torch.float32, torch.float16), (torch.float32, torch.float32)])
def test_forward_backward(rows, width, x_dtype, dtype, device):
    from decik_amd.dropout import dropout_backward, dropout_forward, rng_state

    ps, offset = (0.05, 0.3), 2 ** 32 - 1  # branch 1's offset has a high word
    x = make((rows, width), x_dtype, device, 1)
    rng = rng_state(SEED, offset, device)
    outs = dropout_forward(x, rng, ps, dtype)
    xd = x.double().cpu().numpy()
    masks = [keep_mask(rows, width, SEED, offset + b, p) for b, p in enumerate(ps)]
    for o, m, p in zip(outs, masks, ps):
        assert o.dtype == dtype and o.shape == x.shape
        assert np.array_equal((o != 0).cpu().numpy() | (xd == 0), m | (xd == 0))
        check(o, np.where(m, xd * scale_of(p), 0.0))
    grads = [make((rows, width), dtype, device, 2 + b, 1e-2) for b in range(2)]
    terms = [np.where(m, g.double().cpu().numpy() * scale_of(p), 0.0) for g, m, p in zip(grads, masks, ps)]
    dx = dropout_backward(grads, rng, ps, x_dtype)
    assert dx.dtype == x_dtype
    check(dx, sum(terms), sum(abs(t) for t in terms))


@gpu
@pytest.mark.parametrize("nb", [1, 2, 3, 4])
def test_branches_are_offsets(nb, device):
    from decik_amd.dropout import dropout_backward, dropout_forward, rng_state

    x = make((37, 100), torch.float16, device, 3)
    ps = (0.5, 0.1, 0.25, 0.75)[:nb]
    outs = dropout_forward(x, rng_state(9, 100, device), ps)
    for b in range(nb):
        (alone,) = dropout_forward(x, rng_state(9, 100 + b, device), ps[b:b + 1])
        assert torch.equal(outs[b], alone)
    # a missing gradient counts as zeros, wherever it stands
    grads = [make((37, 100), torch.float16, device, 10 + b) for b in range(nb)]
    for gone in range(nb if nb > 1 else 0):
        some = [None if b == gone else g for b, g in enumerate(grads)]
        zero = [torch.zeros_like(g) if b == gone else g for b, g in enumerate(grads)]
        rng = rng_state(9, 100, device)
        assert torch.equal(dropout_backward(some, rng, ps), dropout_backward(zero, rng, ps))


@gpu
@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 0.5, 1 - 2.0 ** -16, 1 - 2.0 ** -18, 1.0])
def test_extreme_probabilities(p, device):
    from decik_amd.dropout import dropout_forward, rng_state

    x = make((64, 512), torch.float32, device, 4)
    (o,) = dropout_forward(x, rng_state(5, 6, device), (p,))
    check(o, np.where(keep_mask(64, 512, 5, 6, p), x.double().cpu().numpy() * scale_of(p), 0.0))
    if round(p * 65536) == 0:
        assert torch.equal(o, x)


@gpu
def test_dropped_places_are_zero_whatever_they_held(device):
    from decik_amd.dropout import dropout_backward, dropout_forward, rng_state

    x = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0, -1.0, 1.0, 65504.0, 2.0], device=device)
    x = x.to(torch.float16).repeat(16, 9)
    m = torch.from_numpy(keep_mask(16, 72, 7, 8, 0.5)).to(device)
    (o,) = dropout_forward(x, rng_state(7, 8, device), (0.5,))
    want = torch.where(m, (x.float() * 2).half(), torch.zeros_like(x))
    assert torch.equal(o.view(torch.int16)[~m], torch.zeros_like(o.view(torch.int16))[~m])
    assert torch.equal(torch.nan_to_num(o.float(), 9e9), torch.nan_to_num(want.float(), 9e9))
    dx = dropout_backward([x], rng_state(7, 8, device), (0.5,))
    assert torch.equal(dx.view(torch.int16), o.view(torch.int16))


@gpu
def test_strides_shapes_and_empty(device):
    from decik_amd.dropout import dropout_backward, dropout_forward, rng_state

    rng = rng_state(11, 0, device)
    base = make((40, 301), torch.bfloat16, device, 5)
    for view in (base[:, 3:204], base[::2, 1:], base[:, ::3], base.t(), base[:1].expand(40, 301),
                 base[:, :300].unflatten(1, (3, 100)), base[0]):
        (o,) = dropout_forward(view, rng, (0.2,))
        (want,) = dropout_forward(view.contiguous(), rng, (0.2,))
        assert o.shape == view.shape and torch.equal(o, want)
        assert torch.equal(dropout_backward([view], rng, (0.2,)), want)
    for shape in ((0, 16), (16, 0), (2, 0, 8)):
        (o,) = dropout_forward(torch.empty(shape, device=device), rng, (0.2,))
        assert o.shape == shape


@gpu
def test_writes_stay_in_their_rows(device):
    """Rows of odd width, one after the other: each group's tail ends where its row ends."""
    from decik_amd._lib import DTYPES, check as ok, lib, ptr, stream_of
    from decik_amd.dropout import rng_state
    import ctypes

    x = make((9, 21), torch.float16, device, 6)
    out = torch.full((9, 32), 77.0, dtype=torch.float16, device=device)
    ok(lib().dk_dropout_fwd(ptr(x), DTYPES[x.dtype], 21, ptr(rng_state(1, 2, device)), (ctypes.c_double * 1)(0.5), 1,
                            (ctypes.c_void_p * 1)(out.data_ptr()), DTYPES[x.dtype], (ctypes.c_int64 * 1)(32), 9, 21,
                            stream_of(device)))
    assert bool((out[:, 21:] == 77.0).all())


@gpu
def test_autograd_and_gradient_by_differences(device):
    from decik_amd.dropout import SeededDropout, rng_state, seeded_dropout

    rng = rng_state(3, 4, device)
    x = make((6, 21), torch.float32, device, 7).requires_grad_(True)
    outs = SeededDropout.apply(x, rng, (0.3, 0.6))
    w = [make((6, 21), torch.float32, device, 8 + b) for b in range(2)]
    sum((o * v).sum() for o, v in zip(outs, w)).backward()
    # the outputs are linear in x: a difference of any size is the gradient, up to fp32 rounding
    with torch.no_grad():
        h = make((6, 21), torch.float32, device, 20)
        moved = SeededDropout.apply(x + h, rng, (0.3, 0.6))
        diff = sum(((m.double() - o.double()) * v.double()).sum() for m, o, v in zip(moved, outs, w))
        mags = sum(((m.double().abs() + o.double().abs()) * v.double().abs()).sum() for m, o, v in zip(moved, outs, w))
        assert abs(diff - (x.grad.double() * h.double()).sum()) <= mags * 2.0 ** -20
    # one output unused
    y = seeded_dropout(x, rng, 0.3)
    (g,) = torch.autograd.grad(SeededDropout.apply(x, rng, (0.3, 0.6))[0].sum(), x)
    (g1,) = torch.autograd.grad(y.sum(), x)
    assert torch.equal(g, g1)
    # a changed rng between forward and backward is an error
    y = seeded_dropout(x, rng, 0.3)
    rng[1] += 1
    with pytest.raises(RuntimeError):
        y.sum().backward()


@gpu
def test_captured_graph_takes_new_masks(device):
    from decik_amd.dropout import dropout_backward, dropout_forward, rng_state

    x, g = make((100, 77), torch.float16, device, 9), make((100, 77), torch.float16, device, 10)
    rng = rng_state(21, 0, device)
    dropout_forward(x, rng, (0.4,))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (o,) = dropout_forward(x, rng, (0.4,))
        dx = dropout_backward([g], rng, (0.4,))
    for step in range(4):
        rng[1] += 1
        graph.replay()
        (want,) = dropout_forward(x, rng, (0.4,))
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(dx, dropout_backward([g], rng, (0.4,)))


@gpu
def test_refusals(device):
    from decik_amd._lib import DecikError
    from decik_amd.dropout import dropout_backward, dropout_forward, rng_state

    x, rng = make((4, 16), torch.float16, device, 1), rng_state(0, 0, device)
    for bad in (-0.1, 1.1, float("nan")):
        with pytest.raises(DecikError, match="p must be"):
            dropout_forward(x, rng, (bad,))
    for call in (lambda: dropout_forward(x.cpu(), rng, (0.1,)), lambda: dropout_forward(x, rng.cpu(), (0.1,)),
                 lambda: dropout_forward(x, rng.to(torch.int32), (0.1,)), lambda: dropout_forward(x, rng[:1], (0.1,)),
                 lambda: dropout_forward(x, rng, ()), lambda: dropout_forward(x, rng, (0.1,) * 5),
                 lambda: dropout_forward(x, rng, (0.1,), torch.bfloat16),
                 lambda: dropout_forward(x.to(torch.float64), rng, (0.1,)),
                 lambda: dropout_backward([None], rng, (0.1,)), lambda: dropout_backward([x], rng, (0.1, 0.2)),
                 lambda: dropout_backward([x, x[:2]], rng, (0.1, 0.2))):
        with pytest.raises(ValueError):
            call()


@gpu
@pytest.mark.parametrize("nb", [1, 2, 3])
@pytest.mark.parametrize("x_dtype,dtype", [(torch.float32, torch.bfloat16), (torch.float16, torch.float32),
                                           (torch.bfloat16, torch.float32)])
def test_pairs_of_types(nb, x_dtype, dtype, device):
    """The pairs with fp32 on one side that the branches above leave out, forward and backward."""
    from decik_amd.dropout import dropout_backward, dropout_forward, rng_state

    rows, width, offset, ps = 37, 1121, 12, (0.05, 0.3, 0.6)[:nb]
    x = make((rows, width), x_dtype, device, 1)
    rng = rng_state(SEED, offset, device)
    outs = dropout_forward(x, rng, ps, dtype)
    xd = x.double().cpu().numpy()
    masks = [keep_mask(rows, width, SEED, offset + b, p) for b, p in enumerate(ps)]
    for o, m, p in zip(outs, masks, ps):
        assert o.dtype == dtype and o.shape == x.shape
        check(o, np.where(m, xd * scale_of(p), 0.0))
    grads = [make((rows, width), dtype, device, 2 + b, 1e-2) for b in range(nb)]
    terms = [np.where(m, g.double().cpu().numpy() * scale_of(p), 0.0) for g, m, p in zip(grads, masks, ps)]
    dx = dropout_backward(grads, rng, ps, x_dtype)
    assert dx.dtype == x_dtype
    check(dx, sum(terms), sum(abs(t) for t in terms))
