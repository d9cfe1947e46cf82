"""Gradients of a weight and a bias over 2^30 tokens: the contraction's length in bytes passes 32 bits, and its parts are
added exactly here (small whole numbers in a few rows, zeros elsewhere)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1 << 30, (1 << 30) + (1 << 24) + 40])
def test_weight_gradient(tokens):
    import nsa_from_scratch_b200 as nsa
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 72 << 30:
        pytest.skip("needs 72 GB of device memory")
    g = torch.Generator().manual_seed(0)
    x, dy = torch.zeros(tokens, 8, device="cuda", dtype=torch.bfloat16), torch.zeros(tokens, 8, device="cuda", dtype=torch.bfloat16)
    at = torch.cat((torch.randint(tokens, (500,), generator=g), torch.tensor([0, 1, (1 << 24) - 1, 1 << 24, (1 << 29) + 63, (1 << 30) - 1, tokens - 1]))).unique().cuda()
    fx, fd = (torch.randint(-3, 4, (len(at), 8), generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    x[at], dy[at] = fx, fd
    w, b = torch.eye(8, device="cuda", dtype=torch.bfloat16).requires_grad_(True), torch.zeros(8, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    y = nsa.linear(x, w, b)
    assert torch.equal(y[at], fx) and float(y[1 << 28:(1 << 28) + 4096].abs().sum()) == float(x[1 << 28:(1 << 28) + 4096].abs().sum())
    dw, db = torch.autograd.grad(y, (w, b), dy)
    assert torch.equal(dw.double(), (fd.double().T @ fx.double()).to(torch.bfloat16).double())
    assert torch.equal(db.double(), fd.double().sum(0).to(torch.bfloat16).double())
    del x, dy, y
    torch.cuda.empty_cache()
