"""What the attention layer and the manager refuse about windows, without a GPU:
before anything is appended, and whatever the cache holds."""

import pytest
import torch

from polarquant_kv.inference import CompressedMultiHeadAttention, KVCacheManager, PolarQuantConfig


def test_a_window_over_tracked_weights_leaves_the_cache_as_it_was():
    m = KVCacheManager(PolarQuantConfig(enable_compression=False), 20, 1, 1, 32, "cpu")
    m.track_weights = True                     # (kept for compressed caches; the refusal comes first)
    layer = CompressedMultiHeadAttention(PolarQuantConfig(), 64, 2, 1, window=4)
    for _ in range(2):
        with pytest.raises(ValueError, match="not tracked"):
            layer(torch.zeros(1, 3, 64), m)
        assert m.seq_len == m.next_position == 0 and m._key_cache is None
