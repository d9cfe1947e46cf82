"""No-GPU checks of the layer's operators: struct mirrors, and refusals before anything touches a device."""
import ctypes as C
import os

import pytest
import torch

import nsa_from_scratch_b200 as nsa
from nsa_from_scratch_b200 import _lib as L
from test_cpu_boundary import _struct_fields

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ARG, UNSUPPORTED = -1, -2


@pytest.mark.parametrize("mirror,name", [
    (L.NormArgs, "nsa_norm_args"), (L.NormBwdArgs, "nsa_norm_bwd_args"), (L.RopeAxesArgs, "nsa_rope_axes_args"), (L.LinearArgs, "nsa_linear_args"),
    (L.LinearBwdArgs, "nsa_linear_bwd_args"), (L.GatedMlpArgs, "nsa_gated_mlp_args"), (L.GatedMlpBwdArgs, "nsa_gated_mlp_bwd_args")])
def test_struct_mirrors(mirror, name):
    header = open(os.path.join(ROOT, "include", "nsa_b200.h")).read()
    assert [f[0] for f in mirror._fields_] == [f.split("[")[0] for f in _struct_fields(header, name)]


def refused(rc, code, text):
    assert rc == code and text.encode() in L.load().nsa_last_error(), (rc, L.load().nsa_last_error())


def test_c_entry_points_refuse():
    lib = L.load()
    for fn in ("nsa_rms_norm", "nsa_rms_norm_bwd", "nsa_rope_axes", "nsa_linear", "nsa_linear_bwd", "nsa_gated_mlp", "nsa_gated_mlp_bwd"):
        refused(getattr(lib, fn)(None, None), ARG, "NULL argument block")
    for fn in ("nsa_linear_ws_bytes", "nsa_linear_bwd_ws_bytes", "nsa_gated_mlp_ws_bytes", "nsa_gated_mlp_bwd_ws_bytes"):
        refused(getattr(lib, fn)(None), ARG, "NULL argument block")
    n = L.NormArgs(rows=2, hidden=8, x_dtype=0, res_dtype=0, w_dtype=0, y_dtype=0, eps=1e-6)
    refused(lib.nsa_rms_norm(C.byref(n), None), ARG, "NULL pointer")
    n.w_dtype = 1
    refused(lib.nsa_rms_norm(C.byref(n), None), UNSUPPORTED, "weight dtype")
    n.w_dtype, n.hidden = 0, 0
    refused(lib.nsa_rms_norm(C.byref(n), None), ARG, "bad sizes")
    n.hidden, n.residual = 8, 16
    refused(lib.nsa_rms_norm(C.byref(n), None), ARG, "both be given")
    n.residual, n.y_dtype = None, 4
    refused(lib.nsa_rms_norm(C.byref(n), None), UNSUPPORTED, "result dtype")
    n.y_dtype, n.eps = 0, float("nan")
    refused(lib.nsa_rms_norm(C.byref(n), None), ARG, "eps")
    n.eps, n.rows = 1e-6, 0
    assert lib.nsa_rms_norm(C.byref(n), None) == 0                                  # nothing to do
    refused(lib.nsa_quantize_rows_fp8(1, 1, 1, 2, 8, 0, 1, None), ARG, "format")
    refused(lib.nsa_quantize_rows_fp8(1, None, 1, 2, 8, 0, 2, None), ARG, "NULL")
    r = L.RopeAxesArgs(B=1, T=4, H=2, Hkv=1, D=64, n_axes=2, sections=(C.c_int32 * 8)(16, 16), x_dtype=0, y_dtype=0)
    refused(lib.nsa_rope_axes(C.byref(r), None), ARG, "NULL pointer")
    r.sections = (C.c_int32 * 8)(16, 15)
    refused(lib.nsa_rope_axes(C.byref(r), None), ARG, "add up to 31")
    r.n_axes = 9
    refused(lib.nsa_rope_axes(C.byref(r), None), ARG, "9 axes")
    r.D = 63
    refused(lib.nsa_rope_axes(C.byref(r), None), UNSUPPORTED, "even")
    a = L.LinearArgs(M=4, N=8, K=8, dtype=0, y_dtype=0, act=0)
    refused(lib.nsa_linear(C.byref(a), None), ARG, "NULL pointer")
    a.act = 4
    refused(lib.nsa_linear(C.byref(a), None), ARG, "activation")
    refused(lib.nsa_linear_ws_bytes(C.byref(a)), ARG, "activation")
    a.act, a.y_dtype = 0, 1
    refused(lib.nsa_linear(C.byref(a), None), UNSUPPORTED, "result dtype")
    a.y_dtype, a.dtype = 0, 4
    refused(lib.nsa_linear(C.byref(a), None), UNSUPPORTED, "operand dtype")
    a.dtype, a.x, a.w, a.y = 2, 16, 16, 16
    refused(lib.nsa_linear(C.byref(a), None), ARG, "scales")
    a.dtype, a.K = 0, 0
    refused(lib.nsa_linear(C.byref(a), None), ARG, "bad sizes")
    b = L.LinearBwdArgs(dy=16, x=16, w=16, M=4, N=8, K=8, dtype=0, has_act=1, ws=16)
    refused(lib.nsa_linear_bwd(C.byref(b), None), ARG, "NULL pointer")              # no slope beside an activation
    b.slope = 16
    refused(lib.nsa_linear_bwd(C.byref(b), None), ARG, "workspace")
    m = L.GatedMlpArgs(x=16, wg=16, wu=16, wd=16, y=16, ws=16, M=4, N=8, F=16, dtype=0, act=1)
    refused(lib.nsa_gated_mlp(C.byref(m), None), ARG, "workspace")
    m.p = 16
    refused(lib.nsa_gated_mlp(C.byref(m), None), ARG, "p, s, low and h")
    m.dtype = 4
    refused(lib.nsa_gated_mlp(C.byref(m), None), UNSUPPORTED, "dtype")


def test_c_entry_points_refuse_misaligned_pointers():
    """Off its elements' alignment no kernel can read a pointer; the host says so before anything is launched."""
    lib, A = L.load(), 1 << 20
    norm = dict(x=A, weight=A, y=A, rstd=A, rows=2, hidden=8, x_dtype=0, res_dtype=4, w_dtype=4, y_dtype=0, eps=1e-6, residual=A, h=A)
    for name, at in (("x", A + 1), ("weight", A + 2), ("y", A + 1), ("h", A + 2), ("residual", A + 2), ("rstd", A + 2)):
        refused(lib.nsa_rms_norm(C.byref(L.NormArgs(**{**norm, name: at})), None), ARG, "aligned")
    back = dict(dy=A, h=A, weight=A, rstd=A, dx=A, ws=A, ws_bytes=1 << 20, rows=2, hidden=8, x_dtype=0, res_dtype=0, w_dtype=4)
    for name, at in (("dy", A + 1), ("h", A + 1), ("dweight", A + 2), ("dx", A + 1), ("ws", A + 16)):
        refused(lib.nsa_rms_norm_bwd(C.byref(L.NormBwdArgs(**{**back, name: at})), None), ARG, "aligned")
    refused(lib.nsa_quantize_rows_fp8(A + 1, A, A, 2, 8, 0, 2, None), ARG, "aligned")
    refused(lib.nsa_quantize_rows_fp8(A, A, A + 2, 2, 8, 0, 2, None), ARG, "aligned")
    rope = dict(q=A, k=A, v=A, q_out=A, k_out=A, v_out=A, positions=A, inv_freq=A, B=1, T=4, H=2, Hkv=1, D=64, n_axes=1,
                sections=(C.c_int32 * 8)(32), pos64=1, x_dtype=4, y_dtype=0)
    for name, at in (("q", A + 2), ("k_out", A + 1), ("positions", A + 4), ("inv_freq", A + 4)):
        refused(lib.nsa_rope_axes(C.byref(L.RopeAxesArgs(**{**rope, name: at})), None), ARG, "aligned")
    lin = dict(x=A, w=A, y=A, M=4, N=8, K=8, dtype=0, y_dtype=0, act=0)
    for name, at in (("x", A + 1), ("w", A + 1), ("bias", A + 1), ("y", A + 1), ("residual", A + 1)):
        refused(lib.nsa_linear(C.byref(L.LinearArgs(**{**lin, name: at})), None), ARG, "aligned")
    refused(lib.nsa_linear(C.byref(L.LinearArgs(**{**lin, "dtype": 2, "x_scale": A + 2, "w_scale": A})), None), ARG, "aligned")
    lb = dict(dy=A, x=A, w=A, dx=A, M=4, N=8, K=8, dtype=0, ws=A, ws_bytes=1 << 30)
    for name, at in (("dy", A + 1), ("dx", A + 1), ("ws", A + 128)):
        refused(lib.nsa_linear_bwd(C.byref(L.LinearBwdArgs(**{**lb, name: at})), None), ARG, "aligned")
    m = dict(x=A, wg=A, wu=A, wd=A, y=A, ws=A, ws_bytes=1 << 30, M=4, N=8, F=16, dtype=0, act=1)
    for name, at in (("x", A + 1), ("wd", A + 1), ("y", A + 1), ("ws", A + 16)):
        refused(lib.nsa_gated_mlp(C.byref(L.GatedMlpArgs(**{**m, name: at})), None), ARG, "aligned")
    mb = dict(dy=A, x=A, wg=A, wu=A, wd=A, p=A, s=A, low=A, h=A, dx=A, ws=A, ws_bytes=1 << 30, M=4, N=8, F=16, dtype=0)
    for name, at in (("dy", A + 1), ("p", A + 2), ("dx", A + 1), ("ws", A + 16)):
        refused(lib.nsa_gated_mlp_bwd(C.byref(L.GatedMlpBwdArgs(**{**mb, name: at})), None), ARG, "aligned")


def test_no_cpu_path():
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(8, 8, dtype=torch.bfloat16)
    for call in (lambda: nsa.rms_norm(x, w[0]), lambda: nsa.rms_norm_fp8(x, w[0]), lambda: nsa.quantize_rows_to_fp8(x), lambda: nsa.linear(x, w),
                 lambda: nsa.gated_mlp(x, w, w, w)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="CUDA"):
        q = torch.zeros(1, 2, 1, 8)
        nsa.rope_axes_to_heads(q, q, q, torch.zeros(1, 1, 2, dtype=torch.int64), torch.zeros(4), (4,))


def test_torch_side_shares_the_cxx_runtime():
    """A module that brings a C++ runtime of its own into torch's process crashes at its first formatted message."""
    from nsa_from_scratch_b200 import build
    L.torch_ops()
    assert b"libstdc++.so.6" in open(build.TORCH_LIB, "rb").read()


def test_rope_frequencies():
    f = nsa.rope_frequencies(64, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and float(f[0]) == 1.0 and abs(float(f[16]) - 0.01) < 1e-15
    with pytest.raises(ValueError):
        nsa.rope_frequencies(7)
