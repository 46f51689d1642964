"""The C entries of the residual stream, the scaled rotation and the 4-bit linears without a GPU: descriptor layouts,
refusals (argument checks run before any GPU call; the pointers are never followed), workspace sizes, empty calls."""

import ctypes
import os
import subprocess

import pytest

from decik_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an aligned fake pointer


def error(rc):
    assert rc != 0
    return _lib.lib().dk_last_error().decode()


@pytest.mark.parametrize("struct,name", [(_lib.ResidualNorm, "dk_residual_norm"), (_lib.ScaledRope, "dk_scaled_rope")])
def test_descriptor_layout(struct, name, tmp_path):
    names = [f[0] for f in struct._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "decik_nf4.h"\nint main(void){'
                   f'printf("%zu\\n", sizeof({name}));' +
                   "".join(f'printf("%zu\\n", offsetof({name}, {n}));' for n in names) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(struct)] + [getattr(struct, n).offset for n in names]
    assert struct.PACK.size == ctypes.sizeof(struct)


# ---- the residual stream -------------------------------------------------------------------------

def norm(**kw):
    d = _lib.ResidualNorm()
    for f in ("x", "residual", "h", "y", "dx", "grad_y", "weight"):
        setattr(d, f, P)
    d.rows, d.width, d.weight_dtype = 5, 64, 2
    d.ld_x = d.ld_residual = d.ld_grad_y = 64
    for f, v in kw.items():
        setattr(d, f, v)
    return bytes(d)


COMMON = [(dict(x_dtype=3), "x must"), (dict(stream_dtype=1), "x must"), (dict(x_dtype=2), "x must"), (dict(y_dtype=1), "x must"),
          (dict(width=0), "width"), (dict(width=16385), "width"), (dict(rows=-1), "rows"), (dict(rows=(1 << 31) - 65536), "rows"),
          (dict(weight_dtype=4), "weight type"), (dict(post_weight=P, post_dtype=9), "weight type"), (dict(gate_kind=4), "kind"),
          (dict(gate_kind=-1), "kind"), (dict(gate_kind=1, gate_dtype=5, gate=P), "gate type"), (dict(gate_kind=2), "null gate"),
          (dict(x=None), "null"), (dict(ld_x=-1), "stride"), (dict(ld_gate=-1), "stride")]


@pytest.mark.parametrize("kw,msg", COMMON + [(dict(y=None), "y with a weight"), (dict(weight=None, h=None), "h without")])
def test_norm_forward_refusals(kw, msg):
    assert msg in error(_lib.lib().dk_residual_norm_fwd(norm(**kw), None))


@pytest.mark.parametrize("kw,msg", COMMON + [
    (dict(dx=None), "null"), (dict(grad_y=None), "grad_y"), (dict(weight=None), "grad_y"), (dict(residual=None, dresidual=P), "no residual"),
    (dict(weight=None, grad_y=None, dweight=P), "no weight"), (dict(dpost_weight=P), "no post weight"), (dict(dgate=P), "no gate"),
    (dict(dweight=P), "workspace")])
def test_norm_backward_refusals(kw, msg):
    assert msg in error(_lib.lib().dk_residual_norm_bwd(norm(**kw), None, 0, None))


def test_norm_workspace_and_empty():
    L = _lib.lib()
    assert "null" in error(L.dk_residual_norm_fwd(None, None))
    assert L.dk_residual_norm_bwd_workspace(norm()) == 0 and L.dk_residual_norm_bwd_workspace(norm(width=0)) == -1
    need = L.dk_residual_norm_bwd_workspace(norm(dweight=P))
    assert need == 5 * 64 * 4  # a work-group a row here
    both = norm(dweight=P, post_weight=P, post_dtype=2, dpost_weight=P, gate=P, gate_kind=1, dgate=P)
    assert L.dk_residual_norm_bwd_workspace(both) == 2 * need
    assert L.dk_residual_norm_bwd_workspace(norm(gate=P, gate_kind=3, dgate=P)) == 0
    assert "workspace" in error(L.dk_residual_norm_bwd(norm(dweight=P), P, need - 1, None))
    assert "workspace" in error(L.dk_residual_norm_bwd(norm(dweight=P), P + 4, need, None))
    empty = norm(rows=0, x=None, residual=None, y=None, h=None, dx=None, grad_y=None)
    assert L.dk_residual_norm_fwd(empty, None) == 0 and L.dk_residual_norm_bwd(empty, None, 0, None) == 0


# ---- the scaled rotation -------------------------------------------------------------------------

def rope(**kw):
    d = _lib.ScaledRope()
    for f in ("q", "k", "q_out", "k_out", "positions", "inv_freq"):
        setattr(d, f, P)
    d.batch, d.tokens, d.n_heads, d.n_kv_heads, d.head_dim, d.rotary_dim, d.factor = 2, 5, 4, 2, 64, 32, 1.0
    stride = kw.pop("stride", None)
    if stride is not None:
        d.q_stride[1] = stride
    for f, v in kw.items():
        setattr(d, f, v)
    return bytes(d)


@pytest.mark.parametrize("entry", ["dk_scaled_rope_fwd", "dk_scaled_rope_bwd"])
@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=2), "fp16 or bf16"), (dict(head_dim=0), "head_dim"), (dict(head_dim=1025), "head_dim"), (dict(rotary_dim=65), "rotary_dim"),
    (dict(rotary_dim=66), "rotary_dim"), (dict(rotary_dim=-2), "rotary_dim"), (dict(n_heads=0), "heads"), (dict(n_kv_heads=65537), "heads"),
    (dict(batch=-1), "tokens"), (dict(tokens=1 << 23, batch=2), "2^24"), (dict(q=None), "null"), (dict(k_out=None), "null"),
    (dict(positions=None), "positions"), (dict(inv_freq=None), "positions"), (dict(stride=-64), "stride")])
def test_rope_refusals(entry, kw, msg):
    assert msg in error(getattr(_lib.lib(), entry)(rope(**kw), None))


def test_rope_empty():
    L = _lib.lib()
    assert "null" in error(L.dk_scaled_rope_fwd(None, None))
    empty = rope(tokens=0, q=None, k=None, q_out=None, k_out=None, positions=None, inv_freq=None)
    assert L.dk_scaled_rope_fwd(empty, None) == 0 and L.dk_scaled_rope_bwd(empty, None) == 0


# ---- 4-bit linears -------------------------------------------------------------------------------

def lin(back=0, x=P, dt=0, ldx=64, w=P, meta=P, group=32, sdt=0, bias=None, bdt=0, y=P, ydt=0, ldy=64, m=100, n=64, k=64, copy=0, work=None,
        wb=0):
    return _lib.lib().dk_int4_linear(back, x, dt, ldx, w, meta, group, sdt, bias, bdt, y, ydt, ldy, m, n, k, copy, work, wb, None)


@pytest.mark.parametrize("back", [0, 1])
@pytest.mark.parametrize("kw,msg", [
    (dict(m=-1), "2^23"), (dict(n=1 << 23), "2^23"), (dict(m=1 << 22, n=1 << 15), "2^37"), (dict(m=1 << 22, k=1 << 15), "2^37"), (dict(k=0), "2^20"),
    (dict(k=(1 << 20) + 1), "2^20"), (dict(dt=2), "x must"), (dict(ydt=1), "x must"), (dict(sdt=2), "scales"), (dict(bias=P, bdt=7), "bias"),
    (dict(group=16), "group"), (dict(group=48), "group"), (dict(group=1 << 21), "group"), (dict(y=None), "null"), (dict(x=None), "null"),
    (dict(w=None), "null"), (dict(meta=None), "null"), (dict(ldy=63), "overlap"), (dict(w=P + 8), "aligned"), (dict(meta=P + 2), "aligned"),
    (dict(ldx=-1), "stride"), (dict(ldx=1 << 22), "2^22"), (dict(x=P + 2), "copy"), (dict(ldx=65), "copy"), (dict(k=63, n=63), "copy"),
    (dict(copy=1), "workspace")])
def test_linear_refusals(back, kw, msg):
    assert msg in error(lin(back, **kw))


def test_linear_refusals_of_the_backward():
    assert "bias" in error(lin(1, bias=P))
    assert "no terms" in error(lin(1, n=0))


def test_linear_workspace_and_empty():
    L = _lib.lib()
    assert L.dk_int4_linear_workspace(0, 0, -1, 8, 8) == -1 and L.dk_int4_linear_workspace(0, 0, 5, 8, 0) == -1
    assert L.dk_int4_linear_workspace(0, 0, 0, 8, 8) == 0 and L.dk_int4_linear_workspace(0, 0, 5, 64, 64) == 0
    assert L.dk_int4_linear_workspace(0, 1, 100, 64, 63) == 100 * 64 * 2 and L.dk_int4_linear_workspace(1, 1, 5, 65, 64) == 5 * 72 * 2
    assert L.dk_int4_linear_workspace(0, 1, 5, 64, 63) == 0  # few tokens are read as they are
    plan = (ctypes.c_int32 * 4)()
    assert L.dk_int4_linear_plan(0, 16, 64, 18944, plan) == 0 and plan[3] > 1
    need = L.dk_int4_linear_workspace(0, 0, 16, 64, 18944)
    assert need == plan[3] * 16 * 64 * 4
    args = dict(m=16, n=64, k=18944, ldx=18944)
    assert "workspace" in error(lin(0, **args, work=P, wb=need - 1)) and "workspace" in error(lin(0, **args, work=P + 8, wb=need))
    assert "2^23" in error(L.dk_int4_linear_plan(0, 0, 64, 64, plan)) and "2^23" in error(L.dk_int4_linear_plan(0, 4, 64, 64, None))
    assert lin(0, m=0, x=None, y=None) == 0 and lin(0, n=0, x=None, y=None) == 0 and lin(1, m=0, x=None, y=None) == 0
