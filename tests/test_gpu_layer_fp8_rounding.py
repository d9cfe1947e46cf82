"""The fp8 results are round(y / scale), the quotient itself: values that lie between two fp8 numbers to the last bit go to
the even one."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nsa():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import nsa_from_scratch_b200 as m
    return m


def rows(n, dtype, fmt, seed):
    """Rows of random fp8 numbers and the midpoints between neighbours, times a scale of their own; the first column holds the
    largest fp8 number, so that the scale is known.  A few columns are small, zero or subnormal after the division."""
    g = torch.Generator().manual_seed(seed)
    table = torch.arange(256, dtype=torch.uint8).view(fmt).float()
    table = table[torch.isfinite(table) & (table >= 0)].sort().values
    both = torch.cat((table, (table[1:] + table[:-1]) / 2))
    pick = both[torch.randint(len(both), (400, n), generator=g)] * torch.where(torch.rand(400, n, generator=g) < 0.5, -1.0, 1.0)
    pick[:, 0] = table[-1]
    scale = torch.exp2(torch.rand(400, 1, generator=g) * 20 - 10)
    return (pick * scale).clamp(-table[-1] * scale, table[-1] * scale).to(dtype)


@pytest.mark.parametrize("fmt", [torch.float8_e4m3fn, torch.float8_e5m2])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [264, 1003, 4096])
def test_quotient_is_rounded_once(nsa, n, dtype, fmt):
    x = rows(n, dtype, fmt, seed=n)
    if dtype == torch.float16:
        x = (x / 1024 if fmt == torch.float8_e5m2 else x / 64)
    q, s = nsa.quantize_rows_to_fp8(x.cuda(), fmt=fmt)
    top = torch.finfo(fmt).max
    want_s = x.float().abs().amax(-1) / top
    assert torch.equal(s.cpu(), want_s)
    want = (x.float() / want_s[:, None]).clamp(-top, top).to(fmt)
    nan = torch.isnan(want.float())                             # infinities of fp16 over themselves; NaN's sign bit is no value
    assert torch.equal(torch.isnan(q.cpu().float()), nan)
    assert torch.equal(q.cpu().view(torch.uint8)[~nan], want.view(torch.uint8)[~nan]), int((q.cpu().float() != want.float())[~nan].sum())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fmt", [torch.float8_e4m3fn, torch.float8_e5m2])
def test_extreme_rows(nsa, dtype, fmt):
    """Scales at both ends of the range, and rows with infinities: finite values over an infinite scale are 0."""
    top = torch.finfo(fmt).max
    base = torch.linspace(-1, 1, 72)
    x = torch.stack([base * 1e-38, base * 3e-12, base * 1e-20, base * 3.3e38, base * 1e30, torch.zeros(72)]).to(dtype)
    q, s = nsa.quantize_rows_to_fp8(x.cuda(), fmt=fmt)
    want_s = x.float().abs().amax(-1).clamp_min(1e-12) / top
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu().float(), (x.float() / want_s[:, None]).clamp(-top, top).to(fmt).float())
    x[0, 5] = float("inf")
    q, s = nsa.quantize_rows_to_fp8(x.cuda(), fmt=fmt)
    assert torch.isinf(s[0]) and torch.isnan(q[0].float()).cpu().equal(torch.arange(72) == 5) and float(q[0].float().nan_to_num(0).abs().max()) == 0
