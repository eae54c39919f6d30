"""The attention layer behind a window, without a GPU: the mask, and what is refused."""

import pytest
import torch

from polarquant_kv.inference import CompressedMultiHeadAttention, KVCacheManager, PolarQuantConfig, _hidden


@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 0), (3, 2), (5, 1), (100, 7)])
def test_what_a_row_sees(window, sinks):
    pos = torch.arange(12)
    hidden = _hidden(pos, pos[4:9], window, sinks)
    for i, p in enumerate(range(4, 9)):
        for t in range(12):
            assert bool(hidden[i, t]) == (not (t <= p and (t > p - window or t < sinks)))
    assert torch.equal(_hidden(pos, pos, None, 0), torch.ones(12, 12, dtype=torch.bool).triu(1))


def test_layer_without_a_cache():
    torch.manual_seed(0)
    layer = CompressedMultiHeadAttention(PolarQuantConfig(enable_compression=False), 32, 2, 1, window=3, sinks=1)
    x = torch.randn(1, 9, 32)
    with torch.no_grad():
        out = layer(x)
        # what a token does not see does not move it
        y = x.clone()
        y[:, 2:5] += 1.0
        assert torch.equal(layer(y)[:, :2], out[:, :2]) and torch.equal(layer(y)[:, 7:], out[:, 7:])
        assert not torch.allclose(layer(y)[:, 2:7], out[:, 2:7], atol=1e-4)
        y = x.clone()
        y[:, 0] += 1.0                                   # the sink
        assert not torch.allclose(layer(y)[:, 8], out[:, 8], atol=1e-5)


def test_uncompressed_cache_by_steps():
    torch.manual_seed(0)
    config = PolarQuantConfig(enable_compression=False)
    layer = CompressedMultiHeadAttention(config, 64, 2, 1, window=4, sinks=2)
    m = KVCacheManager(config, 20, 1, 1, 32, "cpu")
    x = torch.randn(1, 11, 64)
    with torch.no_grad():
        parts = [layer(x[:, a:b], m) for a, b in ((0, 6), (6, 7), (7, 11))]
        assert torch.allclose(torch.cat(parts, 1), layer(x), atol=2e-3)


def test_refusals():
    for kw in (dict(window=0), dict(window=4, sinks=-1), dict(window=4, causal=False)):
        with pytest.raises(ValueError, match="window"):
            CompressedMultiHeadAttention(PolarQuantConfig(), 64, 2, **kw)
    m = KVCacheManager(PolarQuantConfig(enable_compression=False), 20, 1, 1, 32, "cpu")
    with pytest.raises(ValueError, match="window"):
        m.attend(torch.zeros(1, 1, 1, 32), causal=False, window=3)
    with pytest.raises(ValueError, match="both be"):
        m.append_rotary(torch.zeros(1, 1, 1, 32), torch.zeros(1, 1, 1, 32), torch.zeros(1, 1, 2, 32), None)
