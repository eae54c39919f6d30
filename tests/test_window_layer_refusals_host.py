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


def test_sinks_go_with_a_window():
    with pytest.raises(ValueError, match="sinks=2 go with a window"):
        CompressedMultiHeadAttention(PolarQuantConfig(), 64, 2, sinks=2)
    m = KVCacheManager(PolarQuantConfig(enable_compression=False), 20, 1, 1, 32, "cpu")
    with pytest.raises(ValueError, match="sinks=2 go with a window"):
        m.attend(torch.zeros(1, 1, 1, 32), sinks=2)


def test_positions_without_an_embedding():
    layer = CompressedMultiHeadAttention(PolarQuantConfig(enable_compression=False), 64, 2, 1)
    with pytest.raises(ValueError, match="rotary embedding"):
        layer(torch.zeros(1, 3, 64), positions=torch.arange(3))


@pytest.mark.parametrize("cached", [0, 3])
@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-3), dict(window=2.5), dict(window=3, sinks=-1),
                                dict(window=3, sinks=0.5)])
def test_windows_of_an_uncompressed_cache(kw, cached):
    m = KVCacheManager(PolarQuantConfig(enable_compression=False), 20, 1, 1, 32, "cpu")
    m.append(torch.zeros(1, 1, cached, 32), torch.zeros(1, 1, cached, 32))
    with pytest.raises(ValueError, match="window="):
        m.attend(torch.zeros(1, 1, 1, 32), **kw)
