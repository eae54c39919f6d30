"""KVCacheManager with tracked weights, without a GPU: its bookkeeping, with the
encoders, attention calls and eviction stood in for."""

import pytest
import torch

from polarquant_kv import attention, quantizer
from polarquant_kv.inference import KVCacheManager, PolarQuantConfig

B, H, D = 2, 2, 64


@pytest.fixture
def manager(monkeypatch):
    def encode(kv, R, cache, start, jl_rot=None):
        cache.ensure(start + kv.shape[2])
        cache.seq_len = max(cache.seq_len, start + kv.shape[2])

    def weights(q, keys, R, start, causal=True, jl_rot=None, previous=None, into=None):
        into[:, :, :keys.seq_len] = previous[:, :, :keys.seq_len] + 1.0

    monkeypatch.setattr(quantizer, "compress_pq", encode)
    monkeypatch.setattr(attention, "attention_weights", weights)
    monkeypatch.setattr(attention, "prefill_attention", lambda q, *a, **kw: torch.zeros_like(q, dtype=torch.float16))
    return KVCacheManager(PolarQuantConfig(), 1000, B, H, D, "cpu", page_tokens=64, track_weights=True)


def kv(T):
    return torch.randn(B, H, T, D), torch.randn(B, H, T, D)


def test_a_failed_call_adds_no_weight(manager, monkeypatch):
    manager.append(*kv(10))
    q = torch.randn(B, 4, 10, D)
    manager.attend(q)
    before = manager.weights.clone()

    def fail(*a, **kw):
        raise torch.cuda.OutOfMemoryError("out of memory")

    with monkeypatch.context() as m:
        m.setattr(attention, "prefill_attention", fail)
        with pytest.raises(torch.cuda.OutOfMemoryError):
            manager.attend(q)
    assert torch.equal(manager.weights, before)
    manager.attend(q)
    assert torch.equal(manager.weights, before + 1.0)
