"""NaN and infinities on their way through the products and back: they reach every result and gradient that the formulas
carry them to, and no other.  Where they arrive is taken from the formulas in 64 bits; everything else equals, bit for bit,
what the same call gives without them (a row of a product is formed without looking at the others)."""
import pytest
import torch

from test_gpu_layer_ops import act64, randn

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def nsa():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import nsa_from_scratch_b200 as m
    return m


def same_elsewhere(got, clean, ref, what):
    nan, fin = torch.isnan(ref), torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), nan), (what, int(torch.isnan(got).sum()), int(nan.sum()))
    assert torch.equal(got[~fin & ~nan].double(), ref[~fin & ~nan]), what
    assert torch.equal(got[fin], clean[fin]), what


def slope(z, name):
    """act' by its formula, silu' = s + z s (1 - s) and the tanh gelu's: NaN at infinite arguments."""
    if name is None:
        return torch.ones_like(z)
    k = 1.0 if name == "silu" else 2 * (2 / torch.pi) ** 0.5
    a = z if name == "silu" else k * (z + 0.044715 * z ** 3)
    s = torch.sigmoid(a)
    return s + z * s * (1 - s) * (1.0 if name == "silu" else k * (1 + 3 * 0.044715 * z * z))


# rows, hidden, F: few rows; joined sums (up to 128 rows, off the 16-byte grid); a cluster's sums; whole tiles
MLP = [(5, 64, 136), (24, 72, 264), (100, 136, 520), (90, 33, 67), (256, 768, 512), (300, 100, 1001), (4000, 72, 1000)]


@pytest.mark.parametrize("M,N,F", MLP)
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, "silu"), (torch.float16, "gelu_tanh"), (torch.float16, None)])
@pytest.mark.parametrize("where,value", [("x", NAN), ("x", INF), ("w_gate", NAN), ("w_up", NAN)])
def test_gated_mlp(nsa, M, N, F, dtype, act, where, value):
    if value == INF and act is None:
        act = "silu"                     # without one the factors are infinite, and whether sums of them are NaN hangs on the others' roundings
    ts = {"x": randn(M, N, seed=1, dtype=dtype), "w_gate": randn(F, N, seed=2, std=N ** -0.5, dtype=dtype), "w_up": randn(F, N, seed=3, std=N ** -0.5, dtype=dtype),
          "w_down": randn(N, F, seed=4, std=F ** -0.5, dtype=dtype)}
    dy = randn(M, N, seed=5, dtype=dtype)

    def step():
        leaves = [t.detach().clone().requires_grad_(True) for t in ts.values()]
        y = nsa.gated_mlp(*leaves, activation=act)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    clean = step()
    ts[where][min(3, ts[where].shape[0] - 1), min(7, N - 1)] = value
    x, wg, wu, wd = (t.double() for t in ts.values())
    g, u = x @ wg.T, x @ wu.T
    p, s = act64(g, act), slope(g, act)
    dh = dy.double() @ wd
    dg, du = dh * (s * u), dh * p
    ref = ((p * u) @ wd.T, dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.double().T @ (p * u))
    assert any(torch.isnan(t).any() for t in ref[1:])
    for a, b, r, name in zip(step(), clean, ref, ("y", "dx", "dwg", "dwu", "dwd")):
        same_elsewhere(a, b, r, name)


LINEAR = [(5, 64, 136), (24, 264, 72), (100, 136, 520), (90, 33, 67), (256, 512, 768), (300, 1001, 100), (4000, 1000, 72)]


@pytest.mark.parametrize("M,N,K", LINEAR)
@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, "silu"), (torch.float16, "gelu_tanh"), (torch.float16, None)])
@pytest.mark.parametrize("where,value", [("x", NAN), ("x", INF), ("w", NAN), ("bias", NAN), ("bias", INF)])
def test_linear(nsa, M, N, K, dtype, act, where, value):
    ts = {"x": randn(M, K, seed=1, dtype=dtype), "w": randn(N, K, seed=2, std=K ** -0.5, dtype=dtype), "bias": randn(N, seed=3, dtype=dtype)}
    dy = randn(M, N, seed=5, dtype=dtype)

    def step():
        leaves = [t.detach().clone().requires_grad_(True) for t in ts.values()]
        y = nsa.linear(*leaves, activation=act)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    clean = step()
    if where == "bias":
        ts["bias"][min(7, N - 1)] = value
    else:
        ts[where][min(3, ts[where].shape[0] - 1), min(7, K - 1)] = value
    x, w, b = (t.double() for t in ts.values())
    z = x @ w.T + b
    dz = dy.double() * slope(z, act)
    ref = (act64(z, act), dz @ w, dz.T @ x, dz.sum(0))
    for a, c, r, name in zip(step(), clean, ref, ("y", "dx", "dw", "db")):
        same_elsewhere(a, c, r, name)
