"""Learned pooling and decoding, without a GPU: the cache keeps window means, so decoding a learned-pool configuration against
it would attend other keys than prefill does."""
import pytest

import nsa_from_scratch_b200 as nsa


def test_cache_of_learned_pooling_is_refused():
    with pytest.raises(NotImplementedError, match="learned"):
        nsa.KVCache(1, 1, 64, 64, nsa.NSAConfig(pool="learned"), device="cpu")
    assert nsa.KVCache(1, 1, 64, 64, nsa.NSAConfig(), device="cpu").length == 0
