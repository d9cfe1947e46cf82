"""No-GPU checks of the layer's operators at the ends of their sizes: what a call plans for a contraction of 2^30 terms, read off
its workspace, and the sizes that are refused."""
import ctypes as C

import pytest

from nsa_from_scratch_b200 import _lib as L
from test_layer_ops_boundary import ARG, refused

A = 1 << 20                     # any 256-byte aligned address: nothing is read
MOST = 2 ** 31 - 2 ** 16
FP32 = 4


def scratch(fn, args, without):
    """Bytes of workspace that the products of `without` take."""
    lib = L.load()
    with_ = getattr(lib, fn)(C.byref(args))
    for name in without:
        setattr(args, name, None)
    rest = getattr(lib, fn)(C.byref(args))
    assert with_ >= 0 and rest >= 0, lib.nsa_last_error()
    return with_ - rest


# 64 elements a step, at most 2^18 steps a part: 2^30 terms make 64 parts of fp32 sums; the sizes are multiples of 8 and aligned
@pytest.mark.parametrize("tokens,parts", [(1 << 30, 64), (MOST, 128), ((1 << 28) + 64, 17)])
def test_weight_gradient_over_many_tokens(tokens, parts):
    a = L.LinearBwdArgs(dy=A, x=A, w=A, dw=A, M=tokens, N=8, K=16, dtype=0)
    assert scratch("nsa_linear_bwd_ws_bytes", a, ["dw"]) >= parts * 8 * 16 * FP32
    b = L.GatedMlpBwdArgs(dy=A, x=A, wg=A, wu=A, wd=A, p=A, s=A, low=A, h=A, dwg=A, dwu=A, dwd=A, M=tokens, N=8, F=16, dtype=1)
    assert scratch("nsa_gated_mlp_bwd_ws_bytes", b, ["dwg", "dwu", "dwd"]) >= parts * 8 * 16 * FP32


def test_gradients_of_wide_layers_over_many_tokens():
    """Beside dx, whose tiles are many, dw's few would be formed whole, each over the whole contraction."""
    a = L.LinearBwdArgs(dy=A, x=A, w=A, dx=A, dw=A, M=1 << 28, N=136, K=136, dtype=0)
    assert scratch("nsa_linear_bwd_ws_bytes", a, ["dw"]) >= 16 * 136 * 136 * FP32


@pytest.mark.parametrize("size", [(1 << 30) + 8, MOST])
@pytest.mark.parametrize("dtype,per", [(0, 64), (2, 128)])
def test_long_rows(size, dtype, per):
    K = size // 16 * 16
    parts = -(-K // per // (1 << 18))
    a = L.LinearArgs(x=A, w=A, y=A, x_scale=A if dtype else None, w_scale=A if dtype else None, M=40, N=8, K=K, dtype=dtype, y_dtype=0, act=0)
    assert L.load().nsa_linear_ws_bytes(C.byref(a)) >= parts * 40 * 8 * FP32


def test_ordinary_sizes_are_split_as_before():
    """Up to 2^22 steps the cheapest of up to 16 ways is free to be any."""
    for tokens in (1 << 10, 1 << 20, 1 << 24):
        a = L.LinearBwdArgs(dy=A, x=A, w=A, dw=A, M=tokens, N=8, K=16, dtype=0)
        assert 0 < scratch("nsa_linear_bwd_ws_bytes", a, ["dw"]) <= 16 * 8 * 16 * FP32


@pytest.mark.parametrize("size", [MOST + 1, 2 ** 31 - 255, 2 ** 31 - 1])
def test_sizes_beyond_the_last(size):
    lib = L.load()
    lin, lb = dict(x=A, w=A, y=A, dtype=0, y_dtype=0), dict(dy=A, x=A, w=A, dx=A, dw=A, ws=A, ws_bytes=1 << 60, dtype=0)
    mlp = dict(x=A, wg=A, wu=A, wd=A, y=A, ws=A, ws_bytes=1 << 60, dtype=0, act=1)
    mb = dict(dy=A, x=A, wg=A, wu=A, wd=A, p=A, s=A, low=A, h=A, dx=A, ws=A, ws_bytes=1 << 60, dtype=0)
    for which in "MNK":
        s = {**dict(M=8, N=8, K=8), which: size}
        for fn, args in (("nsa_linear", L.LinearArgs(**lin, **s)), ("nsa_linear_bwd", L.LinearBwdArgs(**lb, **s))):
            refused(getattr(lib, fn)(C.byref(args), None), ARG, "bad sizes")
            refused(getattr(lib, fn + "_ws_bytes")(C.byref(args)), ARG, "bad sizes")
    for which in "MNF":
        s = {**dict(M=8, N=8, F=8), which: size}
        for fn, args in (("nsa_gated_mlp", L.GatedMlpArgs(**mlp, **s)), ("nsa_gated_mlp_bwd", L.GatedMlpBwdArgs(**mb, **s))):
            refused(getattr(lib, fn)(C.byref(args), None), ARG, "bad sizes")
            refused(getattr(lib, fn + "_ws_bytes")(C.byref(args)), ARG, "bad sizes")
    n = L.NormArgs(x=A, weight=A, y=A, rows=1, hidden=size, x_dtype=0, res_dtype=0, w_dtype=0, y_dtype=0, eps=1e-6)
    refused(lib.nsa_rms_norm(C.byref(n), None), ARG, "bad sizes")
    nb = L.NormBwdArgs(dy=A, h=A, weight=A, rstd=A, dx=A, ws=A, ws_bytes=1 << 60, rows=1, hidden=size, x_dtype=0, res_dtype=0, w_dtype=0)
    refused(lib.nsa_rms_norm_bwd(C.byref(nb), None), ARG, "bad sizes")
    refused(lib.nsa_rms_norm_bwd_ws_bytes(1, size), ARG, "bad sizes")
    refused(lib.nsa_quantize_rows_fp8(A, A, A, 1, size, 0, 2, None), ARG, "bad sizes")
    r = L.RopeAxesArgs(q=A, k=A, v=A, q_out=A, k_out=A, v_out=A, positions=A, inv_freq=A, B=1, T=size, H=1, Hkv=1, D=64, n_axes=1, sections=(C.c_int32 * 8)(32), x_dtype=0, y_dtype=0)
    refused(lib.nsa_rope_axes(C.byref(r), None), ARG, "bad sizes")
