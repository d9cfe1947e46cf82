"""What a decoder block keeps between its calls: the frequencies of its rotary embedding, and its cache."""
import pytest
import torch

from test_gpu_layer_block import make_block, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nsa():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import nsa_from_scratch_b200 as m
    return m


def test_second_stream_right_behind_the_first_call(nsa):
    """The first call waits on a busy stream; a second one on another stream has its frequencies all the same."""
    x = randn(1, 70, 192, seed=1)
    pos = torch.arange(70, device="cuda").view(1, 1, 70)
    with torch.no_grad():
        want = make_block(nsa, sections=None)(x, pos)
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        block = make_block(nsa, sections=None)
        with torch.cuda.stream(a):
            junk = [torch.full((32,), 777.0, device="cuda", dtype=torch.float64) for _ in range(64)]   # what the memory holds before
        torch.cuda.synchronize()
        del junk
        with torch.cuda.stream(a):
            torch.cuda._sleep(1 << 28)                        # about 0.15 s
            first = block(x, pos)
        with torch.cuda.stream(b):
            second = block(x, pos)
        torch.cuda.synchronize()
    assert torch.equal(first, want) and torch.equal(second, want)


def test_changed_base(nsa):
    x = randn(1, 70, 192, seed=1)
    pos = torch.arange(70, device="cuda").view(1, 1, 70)
    block, other = make_block(nsa, sections=None), make_block(nsa, sections=None)
    other.rope_base = 500.0
    with torch.no_grad():
        first = block(x, pos)
        block.rope_base = 500.0
        assert torch.equal(block(x, pos), other(x, pos))
        block.rope_base = 10000.0
        assert torch.equal(block(x, pos), first) and not torch.equal(first, other(x, pos))
