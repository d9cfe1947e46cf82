"""The layer's operators (norm, multi-axis rotary embedding, projections, gated feed-forward block) against their formulas in
64 bits.

Tolerances are worst-case bounds, formed element by element from the same data: `half` is the relative error of one rounding
to the result's type (half a step); a sum of n products in fp32 is off by at most n * 2^-23 times the sum of their magnitudes
(2^-23 rather than 2^-24 per addition: the tensor cores may cut where the CPU rounds); exp and division are good to 2^-20."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
FN = 2.0 ** -20
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24, torch.float8_e4m3fn: 2.0 ** -4, torch.float8_e5m2: 2.0 ** -3}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}            # half a step of the subnormals


@pytest.fixture(scope="module")
def nsa():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import nsa_from_scratch_b200 as m
    return m


def randn(*shape, seed=0, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()


def within(got, ref, tol, what=""):
    """Everywhere |got - ref| <= tol; infinities and NaN in the same places."""
    got, ref, tol = got.detach().double(), ref.detach().double(), torch.as_tensor(tol, dtype=torch.float64, device=got.device).expand(ref.shape)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    assert torch.equal(got[~fin & ~torch.isnan(ref)], ref[~fin & ~torch.isnan(ref)]), what
    over = ((got - ref).abs() - tol)[fin]
    if over.numel():
        worst = float(over.max())
        assert worst <= 0, f"{what}: {worst:.3e} over the bound, {float((over > 0).double().mean()):.2e} of the values"


def act64(z, name):
    if name is None:
        return z
    if name == "relu":
        return torch.relu(z)
    return torch.nn.functional.silu(z) if name == "silu" else torch.nn.functional.gelu(z, approximate="tanh")


def slope64(z, name):
    z = z.detach().requires_grad_(True)
    with torch.enable_grad():
        return torch.autograd.grad(act64(z, name).sum(), z)[0].detach() if name else torch.ones_like(z)


def slope_error(z, dz, name):
    """How far act' may be off where its argument is off by dz (|act''| <= 0.8; relu jumps where the sign may change)."""
    if name is None:
        return torch.zeros_like(z)
    return (z.abs() <= dz).double() if name == "relu" else 0.8 * dz + 4 * FN


# ---------------------------------------------------------------- norm

NORM_SHAPES = [(1, 8), (3, 64), (5, 67), (2, 1), (8, 4096), (300, 768), (7, 1024), (33, 1032), (4, 8192), (3, 16384), (2, 16392), (2, 16385), (700, 4096)]


def norm_inputs(shape, dtype, rdtype, wdtype, seed):
    x = randn(*shape, seed=seed, dtype=dtype)
    res = None if rdtype is None else randn(*shape, seed=seed + 1, std=3.0, dtype=rdtype)
    w = (1 + randn(shape[-1], seed=seed + 2, std=0.3, dtype=torch.float32)).to(wdtype)
    return x, res, w


def norm64(x, res, w, eps):
    h = x.double() if res is None else (x.double() + res.double()).to(torch.float32).to(res.dtype).double()
    r = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    return h, r, h * r * w.double()


@pytest.mark.parametrize("shape", NORM_SHAPES)
@pytest.mark.parametrize("dtype,rdtype,wdtype", [
    (torch.bfloat16, None, torch.bfloat16), (torch.bfloat16, torch.bfloat16, torch.float32), (torch.float16, torch.float16, torch.float16),
    (torch.bfloat16, torch.float32, torch.bfloat16), (torch.float32, torch.float32, torch.float32), (torch.float32, None, torch.float32)])
def test_rms_norm(nsa, shape, dtype, rdtype, wdtype):
    eps = 1e-6
    x, res, w = norm_inputs(shape, dtype, rdtype, wdtype, seed=shape[0] * 7 + shape[1])
    out = nsa.rms_norm(x, w, residual=res, eps=eps)
    h, r, y = norm64(x, res, w, eps)
    got = out
    if res is not None:
        got, gh = out
        assert gh.dtype == res.dtype and torch.equal(gh.double(), h)
    assert got.dtype == dtype
    rel = shape[1] * U + 4 * FN
    within(got, y, (HALF[dtype] + rel) * y.abs() + TINY[dtype], "y")


@pytest.mark.parametrize("fmt", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("shape", [(1, 8), (3, 67), (9, 4096), (260, 768), (2, 16385)])
@pytest.mark.parametrize("dtype,rdtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, None), (torch.float32, torch.float32)])
def test_rms_norm_fp8(nsa, shape, dtype, rdtype, fmt):
    x, res, w = norm_inputs(shape, dtype, rdtype, dtype, seed=shape[1])
    out = nsa.rms_norm_fp8(x, w, residual=res, fmt=fmt)
    h, r, y = norm64(x, res, w, 1e-6)
    q, scale = out[:2]
    assert q.dtype == fmt and scale.dtype == torch.float32 and scale.shape == shape[:-1] and len(out) == (2 if res is None else 3)
    if res is not None:
        assert torch.equal(out[2].double(), h)
    rel = shape[1] * U + 4 * FN
    top = 448.0 if fmt == torch.float8_e4m3fn else 57344.0
    sref = y.abs().amax(-1).clamp_min(1e-12) / top
    within(scale, sref, (rel + 2.0 ** -22) * sref, "scale")
    sub = 2.0 ** -10 if fmt == torch.float8_e4m3fn else 2.0 ** -17                       # half a step of the subnormals
    within(q.double() * scale.double()[..., None], y, (HALF[fmt] + 2 * rel + FN) * y.abs() + sub * scale.double()[..., None] * (1 + FN), "y")


@pytest.mark.parametrize("n", [8, 67, 4096])
def test_quantize_rows(nsa, n):
    x = randn(21, n, seed=n, std=5.0)
    x[3] = 0
    x[4, 1] = float("nan")
    q, s = nsa.quantize_rows_to_fp8(x)
    ref = x.double().abs().amax(-1).clamp_min(1e-12) / 448
    ok = torch.arange(21) != 4
    within(s[ok], ref[ok], ref[ok] * 2.0 ** -22, "scale")
    assert torch.isnan(s[4]) and torch.isnan(q[4].float()).all()
    assert float(q[3].float().abs().max()) == 0 and float(s[3]) > 0
    back = q.double() * s.double()[:, None]
    within(back[ok], x[ok], (2.0 ** -4 + FN) * x[ok].double().abs() + 2.0 ** -10 * (1 + FN) * s[ok].double()[:, None], "x")


@pytest.mark.parametrize("shape", [(1, 8), (5, 67), (2, 1), (8, 4096), (700, 768), (1200, 1032), (3, 16384), (2, 16392), (1001, 4096)])
@pytest.mark.parametrize("dtype,rdtype,wdtype", [
    (torch.bfloat16, None, torch.bfloat16), (torch.float16, torch.float16, torch.float32), (torch.bfloat16, torch.float32, torch.float32),
    (torch.float32, torch.float32, torch.float32)])
def test_rms_norm_backward(nsa, shape, dtype, rdtype, wdtype):
    eps = 1e-5
    x, res, w = norm_inputs(shape, dtype, rdtype, wdtype, seed=shape[0] + shape[1])
    dy = randn(*shape, seed=11, dtype=dtype)
    dh = None if res is None else randn(*shape, seed=12, dtype=rdtype)
    leaves = [t.requires_grad_(True) for t in (x, res, w) if t is not None]
    out = nsa.rms_norm(x, w, residual=res, eps=eps)
    grads = torch.autograd.grad(out, leaves, dy if res is None else (dy, dh))
    again = torch.autograd.grad(nsa.rms_norm(x, w, residual=res, eps=eps), leaves, dy if res is None else (dy, dh))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    h, r, y = norm64(x.detach(), None if res is None else res.detach(), w.detach(), eps)
    n, u = h * r, dy.double() * w.detach().double()
    dx = r * (u - n * (u * n).mean(-1, keepdim=True))
    size = r * (u.abs() + n.abs() * (u * n).abs().mean(-1, keepdim=True))
    if dh is not None:
        dx, size = dx + dh.double(), size + dh.double().abs()
    rel = 2 * shape[1] * U + 8 * FN
    for g, t in zip(grads[:-1], (x, res)):
        assert g.dtype == t.dtype
        within(g, dx, HALF[t.dtype] * dx.abs() + rel * size + TINY[t.dtype], "dx")
    dw, mag = (dy.double() * n).sum(0), (dy.double() * n).abs().sum(0)
    assert grads[-1].dtype == wdtype
    within(grads[-1], dw, HALF[wdtype] * dw.abs() + ((shape[0] + shape[1]) * U + 8 * FN) * mag + TINY[wdtype], "dw")


def test_rms_norm_one_gradient_only(nsa):
    """Only one of the two results is used: the other's gradient is absent, not zero-filled by the caller."""
    x, res, w = norm_inputs((6, 256), torch.bfloat16, torch.bfloat16, torch.bfloat16, seed=3)
    x.requires_grad_(True)
    y, h = nsa.rms_norm(x, w, residual=res)
    g = torch.randn_like(h)
    assert torch.equal(torch.autograd.grad(h, x, g, retain_graph=True)[0], g)
    a, = torch.autograd.grad(y, x, g, retain_graph=True)
    b, = torch.autograd.grad((y, h), x, (g, torch.zeros_like(h)))
    assert torch.equal(a, b)


def test_rms_norm_difference_quotient(nsa):
    """fp32 kernels throughout: the directional derivative against central differences of the 64-bit formula."""
    x, res, w = norm_inputs((5, 136), torch.float32, torch.float32, torch.float32, seed=4)
    dy, dh, v = (randn(5, 136, seed=s, dtype=torch.float32) for s in (5, 6, 7))
    x.requires_grad_(True)
    g, = torch.autograd.grad(nsa.rms_norm(x, w, residual=res), x, (dy, dh))

    def loss(t):
        h = x.detach().double() + t * v.double() + res.double()
        return float((h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.double() * dy.double()).sum() + (h * dh.double()).sum())

    t = 1e-4                                                  # the quotient's own error is t^2 times a third derivative
    want = (loss(t) - loss(-t)) / (2 * t)
    assert abs(float((g.double() * v.double()).sum()) - want) <= 1e-4 * float((g.double() * v.double()).abs().sum())


def test_rms_norm_zero_and_non_finite_rows(nsa):
    x = randn(6, 520, seed=8)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    w = randn(520, seed=9)
    _, _, y = norm64(x, None, w, 1e-6)
    got = nsa.rms_norm(x, w)
    within(got, y, (2.0 ** -8 + 2.0 ** -12) * y.abs().nan_to_num(0), "y")
    assert float(got[1].abs().max()) == 0
    q, s = nsa.rms_norm_fp8(x, w)
    assert float(q[1].float().abs().max()) == 0 and torch.isnan(s[3]) and torch.isfinite(s[[0, 1, 4, 5]]).all()


# ---------------------------------------------------------------- rotary embedding

def rope64(q, k, v, pos, inv, sections):
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    ang = torch.stack([pos[a].double() * inv[j].double() for j, a in enumerate(axis)], -1)[:, :, None]     # [B,T,1,D/2]

    def turn(x):
        a, c = x.double().chunk(2, -1)
        return torch.cat((a * ang.cos() - c * ang.sin(), c * ang.cos() + a * ang.sin()), -1).transpose(1, 2)

    def size(x):
        a, c = x.double().abs().chunk(2, -1)
        return torch.cat((a + c, a + c), -1).transpose(1, 2)

    return [turn(q), turn(k), v.double().transpose(1, 2)], [size(q), size(k), 0 * v.double().transpose(1, 2)]


ROPE = [
    # B, T, H, Hkv, D, sections, far
    (1, 1, 4, 2, 64, (8, 12, 12), 100000), (2, 37, 3, 1, 128, (16, 24, 24), 5000), (1, 130, 2, 2, 32, (16,), 1 << 20), (3, 5, 5, 1, 6, (1, 2), 50),
    (8, 1, 64, 4, 128, (16, 24, 24), 65536), (1, 67, 2, 1, 80, (10, 10, 10, 10), 300), (1, 9, 1, 1, 256, (0, 100, 28), 9), (1, 4, 1, 1, 2, (1,), 10)]


@pytest.mark.parametrize("case", ROPE)
@pytest.mark.parametrize("xdt,ydt,pdt", [(torch.bfloat16, torch.bfloat16, torch.int64), (torch.float32, torch.float16, torch.int32),
                                         (torch.float16, torch.float16, torch.int64), (torch.float32, torch.bfloat16, torch.int64)])
@pytest.mark.parametrize("packed", [True, False])
def test_rope_axes(nsa, case, xdt, ydt, pdt, packed):
    B, T, H, Hkv, D, sections, far = case
    g = torch.Generator().manual_seed(T)
    pos = torch.randint(-far, far, (len(sections), B, T), generator=g).to(pdt).cuda()
    inv = nsa.rope_frequencies(D, 10000.0)
    x = randn(B, T, H + 2 * Hkv, D, seed=T + D, dtype=xdt)
    q, k, v = x.split([H, Hkv, Hkv], 2)
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = nsa.rope_axes_to_heads(q, k, v, pos, inv, sections, dtype=ydt)
    ref, size = rope64(q.detach(), k.detach(), v.detach(), pos, inv, sections)
    for o, r, s in zip(out, ref, size):
        assert o.dtype == ydt and o.is_contiguous()
        within(o, r, HALF[ydt] * r.abs() + FN * s + TINY[ydt], "out")
    with torch.no_grad():
        for a, b in zip(out, nsa.rope_axes_to_heads(q, k, v, pos, inv, sections, dtype=ydt)):
            assert torch.equal(a, b)
    do = [randn(*o.shape, seed=40 + i, dtype=ydt) for i, o in enumerate(out)]
    grads = torch.autograd.grad(out, (q, k, v), do)
    back, bsize = rope64(*(d.transpose(1, 2) for d in do), -pos, inv, sections)
    for gr, r, s in zip(grads, back, bsize):
        assert gr.dtype == xdt
        within(gr, r.transpose(1, 2), HALF[xdt] * r.abs().transpose(1, 2) + FN * s.transpose(1, 2) + TINY[xdt], "grad")


def test_rope_axes_one_axis_is_rope_to_heads(nsa):
    """One axis at positions 0..T-1 and the tables of `rope_cache`: the same rotation to fp32 rounding of the tables."""
    from nsa_from_scratch_b200 import ops
    B, T, H, D = 2, 70, 3, 64
    q = randn(B, T, H, D, seed=1, dtype=torch.float32)
    cos, sin = nsa.rope_cache(T, D, 10000.0, "cuda")
    want = ops.rope_to_heads(q, cos, sin, torch.float16)
    pos = torch.arange(T, device="cuda").expand(1, B, T)
    got = nsa.rope_axes_to_heads(q, q, q, pos, nsa.rope_frequencies(D), (D // 2,), dtype=torch.float16)
    # the tables' angles are fp32 products: off by 2^-23 of an angle below 70
    tol = 2 * 2.0 ** -11 * want.double().abs() + 70 * 2.0 ** -22 * 2 * float(q.abs().max()) + 2.0 ** -24
    within(got[0], want, tol)
    within(got[1], want, tol)
    assert torch.equal(got[2], q.transpose(1, 2).to(torch.float16))


# ---------------------------------------------------------------- projections

def linear64(x, w, bias, act, res):
    """(y, z, |error of z|) of fp32 sums."""
    z = x.double() @ w.double().T
    dz = (x.shape[-1] + 2) * U * (x.double().abs() @ w.double().abs().T)
    if bias is not None:
        z = z + bias.double()
        dz = dz + U * bias.double().abs()
    y = act64(z, act)
    return (y if res is None else y + res.double()), z, dz + U * z.abs()


SIZES = [(1, 1, 1), (1, 64, 64), (2, 40, 72), (3, 33, 67), (5, 264, 520), (8, 96, 1000), (16, 128, 256), (17, 72, 136), (31, 200, 264), (33, 512, 128), (64, 136, 4096),
         (65, 64, 64), (128, 256, 192), (129, 264, 72), (257, 520, 264), (300, 33, 67), (513, 1024, 768), (1000, 200, 1001), (130, 2048, 4096), (4, 4096, 2048)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype,bias,act,res", [(torch.bfloat16, False, None, False), (torch.bfloat16, True, "silu", True), (torch.float16, True, "gelu_tanh", False),
                                                (torch.float16, False, "relu", True)])
def test_linear(nsa, M, N, K, dtype, bias, act, res):
    x, w = randn(M, K, seed=M + K, dtype=dtype), randn(N, K, seed=N, std=K ** -0.5, dtype=dtype)
    b = randn(N, seed=5, dtype=dtype) if bias else None
    r = randn(M, N, seed=6, dtype=dtype) if res else None
    y = nsa.linear(x, w, b, activation=act, residual=r)
    ref, z, dz = linear64(x, w, b, act, r)
    assert y.dtype == dtype
    fwd = 1.2 * dz + 4 * FN * (z.abs() + 1) * (act is not None) + 2 * U * ref.abs()
    within(y, ref, HALF[dtype] * ref.abs() + (1 + HALF[dtype]) * fwd + TINY[dtype], "y")


def linear_backward_bounds(x, w, b, act, dy, dtype):
    half, tiny = HALF[dtype], TINY[dtype]
    _, z, zerr = linear64(x, w, b, act, None)
    s = slope64(z, act)
    serr = slope_error(z, zerr, act)
    if act is not None:
        # act' is kept as q |q| 2^-28: half a step of q is 2^-15, its square root good to 2^-20
        root = (s.abs() + serr).sqrt()
        serr = serr + 2 * root * (2.0 ** -15 + FN * root) + (2.0 ** -15 + FN * root) ** 2
    g = dy.double() * s
    gerr = (half * g.abs() + tiny) * (act is not None) + (1 + half) * dy.double().abs() * serr
    out = {}
    for name, a, c, n in (("dx", g, w.double(), w.shape[0]), ("dw", g.T, x.double(), x.shape[0])):
        err = gerr if name == "dx" else gerr.T
        ref, mag = a @ c, (a.abs() + err) @ c.abs()
        tol = (1 + half) * (err @ c.abs() + (n + 2) * U * mag) + half * ref.abs() + tiny
        out[name] = ref, tol
    ref = g.sum(0)
    # the bias gradient sums what stands before the rounding, but a bound with it holds too
    out["db"] = ref, (1 + half) * (gerr.sum(0) + (x.shape[0] + 2) * U * (g.abs() + gerr).sum(0)) + half * ref.abs() + tiny
    return out


@pytest.mark.parametrize("M,N,K", [s for s in SIZES if s[0] * s[1] * s[2] < 1 << 29])
@pytest.mark.parametrize("dtype,bias,act,res", [(torch.bfloat16, True, None, True), (torch.bfloat16, True, "silu", False), (torch.float16, True, "gelu_tanh", True),
                                                (torch.float16, False, "relu", True), (torch.bfloat16, False, None, False)])
def test_linear_backward(nsa, M, N, K, dtype, bias, act, res):
    x, w = randn(M, K, seed=M + K, dtype=dtype), randn(N, K, seed=N, std=K ** -0.5, dtype=dtype)
    b = randn(N, seed=5, dtype=dtype) if bias else None
    r = randn(M, N, seed=6, dtype=dtype) if res else None
    dy = randn(M, N, seed=7, dtype=dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None]
    grads = torch.autograd.grad(nsa.linear(x, w, b, activation=act, residual=r), leaves, dy)
    again = torch.autograd.grad(nsa.linear(x, w, b, activation=act, residual=r), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    want = linear_backward_bounds(x.detach(), w.detach(), None if b is None else b.detach(), act, dy, dtype)
    within(grads[0], *want["dx"], "dx")
    within(grads[1], *want["dw"], "dw")
    if bias:
        within(grads[2], *want["db"], "db")
    if res:
        assert torch.equal(grads[-1], dy)


@pytest.mark.parametrize("M,N,K", [(1, 64, 128), (3, 33, 67), (7, 96, 1024), (40, 72, 80), (64, 256, 4096), (130, 264, 528), (257, 512, 1040), (300, 130, 200)])
@pytest.mark.parametrize("fmt,dtype,bias,act,res", [(torch.float8_e4m3fn, torch.bfloat16, True, None, True), (torch.float8_e5m2, torch.float16, False, "silu", False),
                                                    (torch.float8_e4m3fn, torch.float16, False, None, False)])
def test_linear_fp8(nsa, M, N, K, fmt, dtype, bias, act, res):
    x, xs = nsa.quantize_rows_to_fp8(randn(M, K, seed=M, std=2.0), fmt=fmt)
    w, ws = nsa.quantize_rows_to_fp8(randn(N, K, seed=N, std=K ** -0.5), fmt=fmt)
    b = randn(N, seed=5, dtype=dtype) if bias else None
    r = randn(M, N, seed=6, dtype=dtype) if res else None
    y = nsa.linear_fp8(x, w, xs, ws, b, activation=act, residual=r, dtype=dtype)
    # fp32 sums of products of the stored values; the tensor cores add fp8 products with no fewer than 13 fraction bits kept
    # below the largest of a group of 32, hence the wider unit
    xd, wd = x.double() * xs.double()[:, None], w.double() * ws.double()[:, None]
    z, mag = xd @ wd.T, xd.abs() @ wd.abs().T
    dz = (K * U + 2.0 ** -13 + 4 * U) * mag
    if b is not None:
        z = z + b.double()
    ref = act64(z, act) if r is None else act64(z, act) + r.double()
    fwd = 1.2 * dz + 4 * FN * (z.abs() + 1) + 2 * U * ref.abs()
    assert y.dtype == dtype
    within(y, ref, HALF[dtype] * ref.abs() + (1 + HALF[dtype]) * fwd + TINY[dtype], "y")


# ---------------------------------------------------------------- gated feed-forward block

MLP_SIZES = [(1, 8, 8), (1, 1, 1), (2, 64, 136), (3, 33, 67), (4, 512, 1376), (16, 128, 264), (33, 264, 72), (130, 256, 192), (257, 136, 520), (600, 768, 1024), (129, 100, 273)]


def mlp_weights(N, F, dtype):
    return (randn(F, N, seed=1, std=N ** -0.5, dtype=dtype), randn(F, N, seed=2, std=N ** -0.5, dtype=dtype), randn(N, F, seed=3, std=F ** -0.5, dtype=dtype))


def mlp_products(x, wg, wu):
    g, u = x.double() @ wg.double().T, x.double() @ wu.double().T
    n = (x.shape[-1] + 2) * U
    return g, u, n * (x.double().abs() @ wg.double().abs().T), n * (x.double().abs() @ wu.double().abs().T)


@pytest.mark.parametrize("M,N,F", MLP_SIZES)
@pytest.mark.parametrize("dtype,act,res", [(torch.bfloat16, "silu", True), (torch.float16, "gelu_tanh", False), (torch.bfloat16, "relu", False), (torch.float16, None, True)])
def test_gated_mlp(nsa, M, N, F, dtype, act, res):
    half, tiny = HALF[dtype], TINY[dtype]
    x, (wg, wu, wd) = randn(M, N, seed=M, dtype=dtype), mlp_weights(N, F, dtype)
    r = randn(M, N, seed=6, dtype=dtype) if res else None
    y = nsa.gated_mlp(x, wg, wu, wd, activation=act, residual=r)
    g, u, ge, ue = mlp_products(x, wg, wu)
    a = act64(g, act)
    ae = 1.2 * ge + 4 * FN * (g.abs() + 1) * (act is not None)
    h = a * u
    he = (1 + half) * (ae * (u.abs() + ue) + a.abs() * ue + 2 * U * h.abs()) + half * h.abs() + tiny      # rounded to 16 bits in between
    ref = h @ wd.double().T
    err = he @ wd.double().abs().T + (F + 2) * U * ((h.abs() + he) @ wd.double().abs().T)
    if r is not None:
        ref = ref + r.double()
    within(y, ref, half * ref.abs() + (1 + half) * (err + 2 * U * ref.abs()) + tiny, "y")


@pytest.mark.parametrize("M,N,F", MLP_SIZES)
@pytest.mark.parametrize("dtype,act,res", [(torch.bfloat16, "silu", True), (torch.float16, "gelu_tanh", False), (torch.float16, "relu", True), (torch.bfloat16, None, False)])
def test_gated_mlp_backward(nsa, M, N, F, dtype, act, res):
    half, tiny = HALF[dtype], TINY[dtype]
    x, ws = randn(M, N, seed=M, dtype=dtype), mlp_weights(N, F, dtype)
    r = randn(M, N, seed=6, dtype=dtype) if res else None
    dy = randn(M, N, seed=7, dtype=dtype)
    leaves = [t.requires_grad_(True) for t in (x, *ws, r) if t is not None]
    grads = torch.autograd.grad(nsa.gated_mlp(x, *ws, activation=act, residual=r), leaves, dy)
    again = torch.autograd.grad(nsa.gated_mlp(x, *ws, activation=act, residual=r), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    xd, wg, wu, wd, dyd = (t.detach().double() for t in (x, *ws, dy))
    g, u, ge, ue = mlp_products(xd, wg, wu)
    a, s = act64(g, act), slope64(g, act)
    ae, se = 1.2 * ge + 4 * FN * (g.abs() + 1) * (act is not None), slope_error(g, ge, act)
    dh = dyd @ wd
    dhe = (N + 2) * U * (dyd.abs() @ wd.abs())

    def product(*fs, half=half, tiny=tiny):
        """(product, its error) of factors given with theirs, rounded to 16 bits."""
        v, hi = 1.0, 1.0
        for f, e in fs:
            v, hi = v * f, hi * (f.abs() + e)
        err = hi - v.abs() + 4 * U * hi
        return v, (1 + half) * err + half * v.abs() + tiny

    def kept(*fs):
        """... to 24 bits."""
        return product(*fs, half=2.0 ** -16, tiny=0.0)

    # act(g) and act'(g) u are kept in 24 bits, act(g) u in 16
    dg, dge = product((dh, dhe), kept((u, ue), (s, se)))
    du, due = product((dh, dhe), kept((a, ae)))
    h, he = product((a, ae), (u, ue))

    def contract(pairs, n):
        ref = sum(p @ q for p, _, q, _ in pairs)
        err = sum((p.abs() + pe) @ (q.abs() + qe) * (1 + (n + 2) * U) - p.abs() @ q.abs() for p, pe, q, qe in pairs)
        return ref, (1 + half) * err + half * ref.abs() + tiny

    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    within(grads[0], *contract([(dg, dge, wg, zero), (du, due, wu, zero)], 2 * F), "dx")
    within(grads[1], *contract([(dg.T, dge.T, xd, zero)], M), "dwg")
    within(grads[2], *contract([(du.T, due.T, xd, zero)], M), "dwu")
    within(grads[3], *contract([(dyd.T, zero, h, he)], M), "dwd")
    if res:
        assert torch.equal(grads[-1], dy)


def test_gated_mlp_difference_quotient(nsa):
    """The gradients' projections on a direction against central differences of the 64-bit formula; 16-bit roundings leave
    3 * 2^-11 of the magnitudes summed (two intermediate roundings and the gradient's own)."""
    M, N, F = 24, 64, 136
    x, ws = randn(M, N, seed=1, dtype=torch.float16), mlp_weights(N, F, torch.float16)
    dy = randn(M, N, seed=7, dtype=torch.float16)
    leaves = [t.requires_grad_(True) for t in (x, *ws)]
    grads = torch.autograd.grad(nsa.gated_mlp(x, *ws), leaves, dy)
    base = [t.detach().double() for t in leaves]
    for i, g in enumerate(grads):
        v = randn(*g.shape, seed=50 + i, dtype=torch.float32).double()

        def loss(t):
            p = [b + t * v if j == i else b for j, b in enumerate(base)]
            return float(((act64(p[0] @ p[1].T, "silu") * (p[0] @ p[2].T)) @ p[3].T * dy.double()).sum())

        t = 1e-5
        want = (loss(t) - loss(-t)) / (2 * t)
        assert abs(float((g.double() * v).sum()) - want) <= 3 * 2.0 ** -11 * float((g.double() * v).abs().sum()) + 1e-6


# ---------------------------------------------------------------- few tiles, long contractions

@pytest.mark.parametrize("M,N,K", [(129, 136, 1024), (200, 1160, 1000), (256, 1024, 1024), (300, 264, 2056), (150, 33, 999), (512, 520, 776), (256, 128, 320),
                                   (257, 2048, 4096), (1024, 1024, 1024), (131, 1, 8192)])
def test_few_tiles(nsa, M, N, K):
    """Shapes whose contraction is split over the CTAs of a cluster, evenly or not, with ragged tiles and rows off the
    16-byte grid: every epilogue, the gradients (operands of the other majorness) and fp8."""
    test_linear(nsa, M, N, K, torch.bfloat16, True, "silu", True)
    test_linear(nsa, M, N, K, torch.float16, False, None, False)
    test_linear_fp8(nsa, M, N, K, torch.float8_e4m3fn, torch.bfloat16, True, None, True)
    test_linear_fp8(nsa, M, N, K, torch.float8_e5m2, torch.float16, False, "silu", False)
    test_linear_backward(nsa, M, N, K, torch.float16, True, "gelu_tanh", True)
    test_linear_backward(nsa, M, N, K, torch.bfloat16, False, None, False)


@pytest.mark.parametrize("M,N,K", [(1500, 2051, 200), (512, 2304, 2048), (700, 1530, 1100), (260, 4104, 1024), (2050, 999, 333)])
def test_more_tiles_than_clusters(nsa, M, N, K):
    """The same where the tiles no longer fit one round of clusters: whole or joined, off the 16-byte grid too."""
    test_linear(nsa, M, N, K, torch.float16, True, "gelu_tanh", True)
    test_linear(nsa, M, N, K, torch.bfloat16, False, None, False)
    test_linear_fp8(nsa, M, N, K, torch.float8_e4m3fn, torch.float16, True, None, True)
    test_linear_backward(nsa, M, N, K, torch.bfloat16, True, "silu", True)


@pytest.mark.parametrize("M,N,F", [(700, 1000, 1377), (1100, 520, 2200)])
def test_more_tiles_than_clusters_of_a_gated_block(nsa, M, N, F):
    test_gated_mlp(nsa, M, N, F, torch.bfloat16, "silu", True)
    test_gated_mlp_backward(nsa, M, N, F, torch.float16, "silu", False)


@pytest.mark.parametrize("M,N,F", [(129, 1024, 264), (200, 256, 700), (300, 2056, 136), (256, 768, 2048), (150, 999, 33)])
def test_few_tiles_of_a_gated_block(nsa, M, N, F):
    test_gated_mlp(nsa, M, N, F, torch.bfloat16, "silu", True)
    test_gated_mlp(nsa, M, N, F, torch.float16, None, False)
    test_gated_mlp_backward(nsa, M, N, F, torch.float16, "gelu_tanh", False)
    test_gated_mlp_backward(nsa, M, N, F, torch.bfloat16, "relu", True)


# ---------------------------------------------------------------- refusals

def test_refusals(nsa):
    x, w, sq = randn(4, 64), randn(64), randn(64, 64)
    e4 = torch.zeros(4, 64, device="cuda", dtype=torch.float8_e4m3fn)
    s4, s64 = torch.ones(4, device="cuda"), torch.ones(64, device="cuda")
    for exc, call in [
        (ValueError, lambda: nsa.rms_norm(x, w[:32])), (TypeError, lambda: nsa.rms_norm(x, w.half())), (TypeError, lambda: nsa.rms_norm(x.double(), w.double())),
        (ValueError, lambda: nsa.rms_norm(x, w, residual=x[:2])), (TypeError, lambda: nsa.rms_norm(x.float(), w, residual=x)),
        (ValueError, lambda: nsa.rms_norm_fp8(x, w, fmt=torch.bfloat16)), (RuntimeError, lambda: nsa.rms_norm(x, w, eps=-1.0)),
        (RuntimeError, lambda: nsa.rms_norm(x, w.cpu())),
        (TypeError, lambda: nsa.linear(x.float(), sq.float())), (TypeError, lambda: nsa.linear(x, sq.half())), (ValueError, lambda: nsa.linear(x, sq[:, :32])),
        (ValueError, lambda: nsa.linear(x, sq, w[:3])), (ValueError, lambda: nsa.linear(x, sq, w.float())), (ValueError, lambda: nsa.linear(x, sq, activation="gelu")),
        (ValueError, lambda: nsa.linear(x, sq, residual=x[:1])), (ValueError, lambda: nsa.linear(x, sq, residual=x.float())),
        (TypeError, lambda: nsa.linear_fp8(x, sq, s4, s64)), (ValueError, lambda: nsa.linear_fp8(e4, e4, s64, s4)), (TypeError, lambda: nsa.linear_fp8(e4, e4, s4, s4, dtype=torch.float32)),
        (ValueError, lambda: nsa.linear_fp8(e4, e4, s4, s4.half())), (TypeError, lambda: nsa.linear_fp8(e4, e4.view(torch.float8_e5m2), s4, s4)),
        (ValueError, lambda: nsa.gated_mlp(x, sq, sq, sq[:32])), (TypeError, lambda: nsa.gated_mlp(x, sq, sq, sq.half())), (ValueError, lambda: nsa.gated_mlp(x, sq, sq, sq, activation="tanh")),
    ]:
        with pytest.raises(exc):
            call()
    q, pos, inv = randn(1, 3, 2, 64), torch.zeros(2, 1, 3, dtype=torch.int64, device="cuda"), nsa.rope_frequencies(64)
    for exc, call in [
        (ValueError, lambda: nsa.rope_axes_to_heads(q, q, q, pos, inv, (16, 15))), (ValueError, lambda: nsa.rope_axes_to_heads(q, q, q, pos, inv, (32,))),
        (ValueError, lambda: nsa.rope_axes_to_heads(q, q, q, pos.float(), inv, (16, 16))), (ValueError, lambda: nsa.rope_axes_to_heads(q, q, q, pos, inv[:3], (16, 16))),
        (TypeError, lambda: nsa.rope_axes_to_heads(q, q.half(), q, pos, inv, (16, 16))), (TypeError, lambda: nsa.rope_axes_to_heads(q, q, q, pos, inv, (16, 16), dtype=torch.float32)),
        (ValueError, lambda: nsa.rope_axes_to_heads(q, q[:, :2], q, pos, inv, (16, 16))), (ValueError, lambda: nsa.rope_axes_to_heads(q[0], q, q, pos, inv, (16, 16))),
    ]:
        with pytest.raises(exc):
            call()


def test_empty(nsa):
    """No rows: empty results, and gradients of the weights that are zero."""
    x = randn(0, 64).requires_grad_(True)
    w, sq = randn(64).requires_grad_(True), randn(64, 64).requires_grad_(True)
    for y, leaves in ((nsa.rms_norm(x, w), (x, w)), (nsa.linear(x, sq, w, activation="silu"), (x, sq, w)), (nsa.gated_mlp(x, sq, sq, sq), (x, sq))):
        assert y.shape == (0, 64)
        for g, t in zip(torch.autograd.grad(y, leaves, torch.empty_like(y)), leaves):
            assert g.shape == t.shape and float(g.float().abs().sum()) == 0
    q, s = nsa.rms_norm_fp8(x, w)
    assert q.shape == (0, 64) and s.shape == (0,)
    assert nsa.linear_fp8(q, q.new_zeros(8, 64), s, s.new_ones(8)).shape == (0, 8)
    p = randn(1, 0, 2, 64)
    assert nsa.rope_axes_to_heads(p, p, p, torch.zeros(1, 1, 0, dtype=torch.int64, device="cuda"), nsa.rope_frequencies(64), (32,))[0].shape == (1, 2, 0, 64)


def test_more_rows_than_32_bits_count(nsa):
    """The products' sizes are 32-bit numbers: more rows are refused, not wrapped."""
    x, w = torch.empty(1 << 31, 1, device="cuda", dtype=torch.bfloat16), randn(8, 1)
    for call in (lambda: nsa.linear(x, w), lambda: nsa.gated_mlp(x, w, w, w.T.contiguous()),
                 lambda: nsa.linear_fp8(x.view(torch.float8_e4m3fn)[:, :1].contiguous(), w.to(torch.float8_e4m3fn), torch.empty(1 << 31, device="cuda"), torch.ones(8, device="cuda"))):
        with pytest.raises(ValueError, match="32-bit"):
            call()
