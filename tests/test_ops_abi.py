"""The C entries of seeded dropout, q/k norms and rotation, and 8-bit linears without a GPU: descriptor
layout, refusals (argument checks run before any GPU call; the pointers are never followed), workspace
sizes, empty calls."""

import ctypes
import os
import struct
import subprocess

import pytest

from decik_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an aligned fake pointer


def error(rc):
    assert rc != 0
    return _lib.lib().dk_last_error().decode()


def test_descriptor_layout(tmp_path):
    names = [f[0] for f in _lib.QkRope._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "decik_nf4.h"\nint main(void){'
                   'printf("%zu\\n", sizeof(dk_qk_rope));' +
                   "".join(f'printf("%zu\\n", offsetof(dk_qk_rope, {n}));' for n in names) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.QkRope)] + [getattr(_lib.QkRope, n).offset for n in names]
    assert _lib.QkRope.PACK.size == ctypes.sizeof(_lib.QkRope)


# ---- dropout -------------------------------------------------------------------------------------

def drop_fwd(x=P, dt=0, ldx=64, rng=P, ps=(0.5,), outs=None, odt=0, ldo=None, rows=4, width=64):
    n = len(ps)
    return _lib.lib().dk_dropout_fwd(x, dt, ldx, rng, struct.pack(f"{n}d", *ps) if n else struct.pack("d", 0), n,
                                     struct.pack(f"{max(n, 1)}P", *(outs or [P] * max(n, 1))), odt,
                                     struct.pack(f"{max(n, 1)}q", *(ldo or [width] * max(n, 1))), rows, width, None)


def drop_bwd(grads=(P,), dt=0, ldg=(64,), rng=P, ps=(0.5,), dx=P, odt=0, ld=64, rows=4, width=64):
    n = len(ps)
    return _lib.lib().dk_dropout_bwd(struct.pack(f"{n}P", *grads), dt, struct.pack(f"{n}q", *ldg), rng,
                                     struct.pack(f"{n}d", *ps), n, dx, odt, ld, rows, width, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(ps=()), "branches"), (dict(ps=(0.1,) * 5), "branches"), (dict(ps=(-0.1,)), "p must"), (dict(ps=(1.5,)), "p must"),
    (dict(ps=(float("nan"),)), "p must"), (dict(dt=3), "types"), (dict(dt=0, odt=1), "types"), (dict(rows=-1), "negative"),
    (dict(width=-8), "negative"), (dict(rows=1 << 31, width=8), "2^31"), (dict(rows=3, width=1 << 33), "2^32"),
    (dict(rng=None), "rng"), (dict(rng=P + 4), "rng"), (dict(x=None), "null"), (dict(outs=[0]), "null"),
    (dict(ldo=[63]), "overlap"), (dict(ldx=-64), "negative row")])
def test_dropout_forward_refusals(kw, msg):
    assert msg in error(drop_fwd(**kw))


@pytest.mark.parametrize("kw,msg", [
    (dict(dx=None), "null"), (dict(ld=60), "overlap"), (dict(ldg=(-1,)), "negative row"), (dict(odt=1), "types"),
    (dict(ps=(2.0,)), "p must")])
def test_dropout_backward_refusals(kw, msg):
    assert msg in error(drop_bwd(**kw))


def test_empty_dropout():
    assert drop_fwd(x=None, rng=None, rows=0) == 0 and drop_fwd(x=None, rng=None, rows=5, width=0) == 0
    assert drop_bwd(grads=(0,), dx=None, rng=None, rows=0) == 0


# ---- norms and rotation --------------------------------------------------------------------------

def qk(**kw):
    d = _lib.QkRope()
    for f in ("q", "k", "q_out", "k_out", "cos", "sin", "grad_q", "grad_k"):
        setattr(d, f, P)
    d.batch, d.tokens, d.n_heads, d.n_kv_heads, d.head_dim = 2, 5, 4, 2, 64
    d.ld_q = d.ld_q_out = 4 * 64
    d.ld_k = d.ld_k_out = 2 * 64
    axes = kw.pop("axes", None)
    if axes is not None:
        d.cos = d.sin = None
        d.positions = d.inv_freq = P
        d.n_axes = len(axes)
        for i, s in enumerate(axes):
            d.sections[i] = s
    for f, v in kw.items():
        setattr(d, f, v)
    return bytes(d)


COMMON = [(dict(dtype=2), "fp16 or bf16"), (dict(head_dim=8), "head_dim"), (dict(head_dim=72), "head_dim"),
          (dict(head_dim=528), "head_dim"), (dict(n_heads=0), "heads"), (dict(n_kv_heads=0), "heads"),
          (dict(tokens=-1), "tokens"), (dict(batch=1 << 20, tokens=1 << 12), "tokens"), (dict(q_weight=P), "both q and k"),
          (dict(q_weight=P, k_weight=P, w_dtype=7), "weight type"), (dict(cos=None), "cos and sin"),
          (dict(sin=None), "cos and sin"), (dict(cos=P + 2), "cos and sin"), (dict(axes=[32], positions=None), "positions"),
          (dict(axes=[32], inv_freq=None), "positions"), (dict(n_axes=5), "axes"), (dict(n_axes=-1), "axes"),
          (dict(axes=[16, 15]), "sections"), (dict(axes=[-2, 34]), "sections"), (dict(axes=[0, 32], interleaved=1), "interleaved"),
          (dict(q_out=None), "null")]


@pytest.mark.parametrize("kw,msg", COMMON + [(dict(q=None), "null"), (dict(ld_q=255), "strides"), (dict(ld_k=0), "strides")])
def test_qk_forward_refusals(kw, msg):
    assert msg in error(_lib.lib().dk_qk_rope_fwd(qk(**kw), None))


NORM = dict(q_weight=P, k_weight=P, w_dtype=2)


@pytest.mark.parametrize("kw,msg", COMMON + [
    (dict(grad_q=None), "null"), (dict(ld_q_out=255), "strides"), (dict(NORM, q=None), "again"), (dict(NORM, ld_q=10), "strides"),
    (dict(dw_q=P, dw_k=P), "no norm weights"), (dict(NORM, dw_q=P), "both"), (dict(NORM, dw_q=P, dw_k=P), "workspace")])
def test_qk_backward_refusals(kw, msg):
    assert msg in error(_lib.lib().dk_qk_rope_bwd(qk(**kw), None, 0, None))


def test_qk_workspace_and_empty():
    L = _lib.lib()
    assert L.dk_qk_rope_bwd_workspace(qk()) == 0 and L.dk_qk_rope_bwd_workspace(qk(**NORM)) == 0
    need = L.dk_qk_rope_bwd_workspace(qk(**NORM, dw_q=P, dw_k=P))
    assert need > 0 and need % (2 * 64 * 4) == 0
    assert "workspace" in error(L.dk_qk_rope_bwd(qk(**NORM, dw_q=P, dw_k=P), P, need - 1, None))
    assert "workspace" in error(L.dk_qk_rope_bwd(qk(**NORM, dw_q=P, dw_k=P), P + 4, need, None))
    assert L.dk_qk_rope_bwd_workspace(qk(head_dim=8)) == -1
    assert "null" in error(L.dk_qk_rope_fwd(None, None))
    empty = qk(tokens=0, q=None, k=None, cos=None, sin=None, q_out=None, k_out=None, grad_q=None, grad_k=None)
    assert L.dk_qk_rope_fwd(empty, None) == 0 and L.dk_qk_rope_bwd(empty, None, 0, None) == 0


# ---- 8-bit linears -------------------------------------------------------------------------------

def quant(x=P, dt=0, ldx=64, col=None, q=P, ldq=64, scale=P, rows=4, k=64):
    return _lib.lib().dk_int8_quantize(x, dt, ldx, col, q, ldq, scale, rows, k, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dt=5), "type"), (dict(rows=-1), "rows"), (dict(rows=1 << 23), "rows"), (dict(k=0), "131071"), (dict(k=131072), "131071"),
    (dict(x=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"), (dict(ldx=-1), "stride"), (dict(ldq=72), "aligned"),
    (dict(q=P + 8), "aligned"), (dict(k=65, ldq=64), "aligned"), (dict(ldq=1 << 23), "aligned")])
def test_quantize_refusals(kw, msg):
    assert msg in error(quant(**kw))


def lin(tr=0, xq=P, ldx=64, xs=P, wq=P, ldw=64, ws=P, bias=None, bdt=0, y=P, ydt=0, ldy=32, m=40, n=32, k=64, work=None, wb=0):
    return _lib.lib().dk_int8_linear(tr, xq, ldx, xs, wq, ldw, ws, bias, bdt, y, ydt, ldy, m, n, k, work, wb, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(m=-1), "2^23"), (dict(n=1 << 23), "2^23"), (dict(m=1 << 20, n=1 << 18), "2^38"), (dict(k=131072), "131071"),
    (dict(ydt=3), "type"), (dict(bias=P, bdt=9), "type"),
    (dict(tr=1), "transposed"), (dict(tr=1, ws=None, bias=P), "transposed"), (dict(xq=None), "null"), (dict(ws=None), "null"),
    (dict(y=None), "null"), (dict(ldx=56), "aligned"), (dict(xq=P + 4), "aligned"), (dict(ldw=60), "aligned"),
    (dict(tr=1, ws=None, ldw=16), "aligned"), (dict(ldy=31), "overlap"), (dict(m=300, k=131071, ldx=131072, ldw=131072), "workspace")])
def test_linear_refusals(kw, msg):
    assert msg in error(lin(**kw))


def x_fwd(x=P, dt=0, ldx=64, wq=P, ldw=64, ws=P, bias=None, bdt=0, y=P, ydt=0, ldy=32, m=40, n=32, k=64, work=None, wb=0):
    return _lib.lib().dk_int8_linear_fwd(x, dt, ldx, wq, ldw, ws, bias, bdt, y, ydt, ldy, m, n, k, work, wb, None)


def x_bwd(dy=P, dt=0, lddy=32, wq=P, ldw=64, ws=P, dx=P, xdt=0, lddx=64, m=40, n=32, k=64, work=None, wb=0):
    return _lib.lib().dk_int8_linear_bwd(dy, dt, lddy, wq, ldw, ws, dx, xdt, lddx, m, n, k, work, wb, None)


@pytest.mark.parametrize("m", [1, 40])
@pytest.mark.parametrize("kw,msg", [
    (dict(k=0), "131071"), (dict(n=-1), "2^23"), (dict(x=None), "null"), (dict(ws=None), "null"), (dict(wq=None), "null"),
    (dict(y=None), "null"), (dict(dt=4), "type"), (dict(ydt=4), "type"), (dict(bias=P, bdt=4), "type")])
def test_linear_x_forward_refusals(m, kw, msg):
    assert msg in error(x_fwd(m=m, **kw))


def test_linear_x_workspace():
    L = _lib.lib()
    assert "workspace" in error(x_fwd()) and "workspace" in error(x_bwd())
    need = L.dk_int8_linear_x_workspace(0, 40, 32, 64)
    assert need >= 40 * 128 + 160
    assert "workspace" in error(x_fwd(work=P, wb=100)) and "workspace" in error(x_fwd(work=P + 8, wb=need))
    assert "aligned" in error(x_fwd(m=1, ldw=40)) and "aligned" in error(x_fwd(m=1, wq=P + 1))
    assert L.dk_int8_linear_x_workspace(0, 1, 32, 64) == 0  # quantized inside the product
    assert L.dk_int8_linear_x_workspace(1, 1, 32, 64) > 0
    assert L.dk_int8_linear_x_workspace(0, -1, 32, 64) == -1 and L.dk_int8_linear_x_workspace(1, 1, 131072, 64) == -1
    assert "overlap" in error(lin(ldy=1)) and "strides" in error(x_fwd(ldy=31)) and "strides" in error(x_bwd(lddx=63))


def test_empty_linears():
    assert quant(x=None, q=None, scale=None, rows=0) == 0
    assert lin(m=0, xq=None, y=None) == 0 and lin(n=0, wq=None, y=None) == 0
    assert x_fwd(m=0, x=None, y=None) == 0 and x_bwd(m=0, dy=None, dx=None) == 0


def test_linear_plans_cover_their_tiles():
    """Whatever the sizes, the workspace is what the planned splits take: whole slabs of m rows."""
    L = _lib.lib()
    for m in (1, 9, 33, 64, 65, 257, 830, 8192):
        for n in (1, 255, 1536, 18944):
            for k in (1, 128, 1121, 8960, 131071):
                for tr in (0, 1):
                    need = L.dk_int8_linear_workspace(tr, m, n, k)
                    slab = 4 * m * ((n + 3) // 4 * 4)
                    assert need == 0 or (need % slab == 0 and 2 <= need // slab <= 32)


def test_linear_plan_query():
    from decik_amd.int8 import launch_plan

    assert launch_plan(False, 1, 18944, 3584) == dict(tile_tokens=0, tile_channels=16, splits=1, fused=True)
    assert not launch_plan(True, 1, 64, 64)["fused"] and launch_plan(True, 1, 64, 64)["tile_tokens"] == 64
    for bad in ((-1, 1, 1), (1, 1 << 23, 1), (1, 1, 0), (1, 1, 131072)):
        with pytest.raises(_lib.DecikError):
            launch_plan(False, *bad)
    assert _lib.lib().dk_int8_linear_plan(0, 1, 1, 1, None) != 0


def test_every_form_that_the_planner_chooses_is_run():
    """Tiles with and without splits over a sweep of sizes: the GPU tests name a size for each of them, and the sizes
    they name are planned so."""
    from decik_amd.int8 import launch_plan
    from test_int8_gpu import SPLIT_TILES, TILES

    def form(transposed, m, n, k):
        p = launch_plan(transposed, m, n, k)
        return p["tile_tokens"], p["tile_channels"], p["splits"] > 1

    tested = {(0, 16, False): (16, 512, 4096), **TILES, (256, 256, True): next(iter(SPLIT_TILES))}
    for transposed in (False, True):
        for f, size in tested.items():
            if f[0] > 0 or not transposed:
                assert form(transposed, *size) == f
        seen = {form(transposed, m, n, k)
                for m in (1, 2, 8, 16, 32, 33, 64, 100, 257, 512, 830, 2051, 6229, 8192, 65536, (1 << 23) - 1)
                for n in (1, 16, 64, 255, 384, 724, 1536, 2057, 3584, 8960, 18944, 151936, (1 << 23) - 1)
                for k in (1, 64, 129, 256, 512, 1121, 2048, 3584, 8960, 15022, 18944, 40000, 131071) if m * n < 1 << 38}
        assert seen <= set(tested) and len(seen) == (8 if transposed else 9)
