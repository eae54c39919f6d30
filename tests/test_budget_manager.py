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


def modes():
    yield torch.inference_mode
    yield torch.no_grad
    yield torch.enable_grad


@pytest.mark.parametrize("first", list(modes()), ids=lambda m: m.__name__)
@pytest.mark.parametrize("then", list(modes()), ids=lambda m: m.__name__)
def test_calls_in_different_modes(manager, monkeypatch, first, then):
    """Weights, positions and page tables outlive the mode of the call that made them."""
    from polarquant_kv import eviction
    from polarquant_kv.types import PagedPQCache

    def evict(keys, values, weights, keep, sink=0, recent=0, positions=None):
        new = []
        for c in (keys, values):
            n = PagedPQCache(B, H, D, 4, c.codebooks, "cpu", 64, tables=False)
            n.reserve(keep)
            n.seq_len = keep
            new.append(n)
        return eviction.Eviction(*new, kept=torch.zeros(1), weights=weights[:, :, :keep].clone(),
                                 positions=positions[:, :, :keep].clone())

    monkeypatch.setattr(eviction, "evict", evict)
    with first():
        manager.append(*kv(20))                                  # leaves room in the first page's slots
        manager.attend(torch.randn(B, 4, 20, D))
    with then():
        manager.append(*kv(1))
        manager.append(*kv(1100 - 200))                          # past the table's first width
    with first():
        manager.evict(100, 0, 0)
    with then():
        manager.append(*kv(3))
        manager.append(*kv(60))
    assert manager.seq_len == 163 and manager.next_position == 984
    assert torch.equal(manager.positions[0, 0], torch.cat([torch.arange(100), torch.arange(921, 984)]).int())
    assert not manager.weights[:, :, 20:].any() and bool((manager.weights[:, :, :20] == 1.0).all())
    assert all(not t.is_inference() for t in (manager.weights, manager.positions, *(c.table for c in manager.get_kv())))


def test_append_that_cannot_keep_its_weights_changes_nothing(manager, monkeypatch):
    manager.append(*kv(10))

    def fail(T):
        raise RuntimeError("no room")

    with monkeypatch.context() as m:
        m.setattr(manager, "_track", fail)
        with pytest.raises(RuntimeError):
            manager.append(*kv(5))
    assert manager.seq_len == manager.next_position == 10 and all(c.seq_len == 10 for c in manager.get_kv())


def test_reordered_tables_in_different_modes():
    from polarquant_kv.types import PagedPQCache
    with torch.inference_mode():
        c = PagedPQCache(B, H, D, 4, torch.zeros(16), "cpu", 64, jl_dim=D, max_pages=4)
        c.ensure(60)
        c.select_batch(torch.tensor([1, 0]))
    c.ensure(130)
    assert len(c.groups) == 3 and all(
        int(c.table[0, p]) == g.data_ptr() and int(c.sign_table[0, p]) == s.data_ptr()
        for p, (g, s) in enumerate(zip(c.groups, c.sign_groups)))


def test_uncompressed_cache_in_different_modes():
    m = KVCacheManager(PolarQuantConfig(enable_compression=False), 8, B, H, D, "cpu")
    with torch.inference_mode():
        m.append(*kv(2))
    k, v = kv(3)
    m.append(k, v)
    assert torch.equal(m.get_kv()[0][:, :, 2:], k.half())
