"""Learned pooling and decoding: the cache keeps window means, so a module with learned pooling has no decoding, and says so."""
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


def learned_block(nsa):
    cfg = nsa.NSAConfig(block_size_c=32, stride_c=16, top_k=8, window_size=96, select_per_group=True, pool="learned")
    torch.manual_seed(0)
    return nsa.NSABlock(192, 4, 64, cfg, 344, n_kv_heads=2).to(device="cuda", dtype=torch.bfloat16)


def test_decoding_is_refused(nsa):
    block = learned_block(nsa)
    x = randn(1, 100, 192, seed=1)
    with torch.no_grad():
        assert torch.isfinite(block(x)).all()                             # prefill has it
        with pytest.raises(NotImplementedError, match="learned"):
            block.new_cache(1, 128)
        cache = make_block(nsa, sections=None).new_cache(1, 128)          # a cache of window means
        with pytest.raises(NotImplementedError, match="learned"):
            block(x, cache=cache)
        assert cache.length == 0                                          # untouched
