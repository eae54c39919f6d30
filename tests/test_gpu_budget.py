"""A cache that lives under a budget, as a program runs it: projections turned by
their positions, appended, attended to with the weights kept, cut to a budget
again and again while the sequence grows. Against float64 on the cached bytes.

Attention outputs carry the bar of the attention tests (2e-3, cosine 0.9999);
weights the tolerance derived in test_gpu_weights; which positions stay follows
from the manager's own weights, so it has to be equal."""

import math

import numpy as np
import pytest
import torch

from polarquant_kv import inference, rotary
from polarquant_kv.inference import CompressedMultiHeadAttention, KVCacheManager, PolarQuantConfig

from test_gpu_evict import want_kept
from test_gpu_weights import decoded, exact

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def attend64(q, mgr, causal=True):
    """(output, weights of the call, bound) of q [B, Hq, Sq, d] on the manager's cache."""
    kc, vc = (c.to_contiguous() for c in mgr.get_kv())
    S, Sq, G = kc.seq_len, q.shape[2], q.shape[1] // kc.num_heads
    total, tol, w = exact(q, kc, mgr.R, S - Sq, causal or Sq == 1, mgr.jl_rot)
    out = w @ decoded(vc).repeat_interleave(G, 1) @ mgr.R.double()
    return out, total, tol


def agree(out, want):
    err = (out.double() - want).abs().max().item()
    cos = torch.nn.functional.cosine_similarity(out.double().flatten(), want.flatten(), 0).item()
    assert err <= 2e-3 and cos >= 0.9999, (err, cos)


@pytest.mark.parametrize("bits,qjl,d", [(4, False, 128), (2, True, 64), (4, True, 128)])
def test_decoding_under_a_budget(bits, qjl, d):
    B, Hq, H, keep, sink, recent = 2, 4, 2, 96, 4, 16
    cfg = PolarQuantConfig(n_bits=bits, enable_qjl=qjl, jl_dim=d)
    mgr = KVCacheManager(cfg, 400, B, H, d, DEV, page_tokens=64, track_weights=True)
    g = torch.Generator(device=DEV).manual_seed(3)
    emb = rotary.RotaryEmbedding(d, base=500.0, scaling={"type": "linear", "factor": 2.0})
    weights = torch.zeros(B, H, 0, dtype=torch.float64, device=DEV)      # in 64 bits, beside the manager's
    bound = weights.clone()
    positions = torch.zeros(B, H, 0, dtype=torch.int64, device=DEV)
    appended = 0
    for T in [130, 1, 1, 37, 1] + [1] * 6 + [200, 1]:
        qkv = [torch.randn(B, n, T, d, generator=g, device=DEV).half() for n in (Hq, H, H)]
        assert mgr.next_position == appended
        at = torch.arange(appended, appended + T, device=DEV)
        q, k = emb(1.5 * qkv[0], qkv[1], at)
        mgr.append(k, qkv[2])
        appended += T
        zeros = torch.zeros(B, H, T, dtype=torch.float64, device=DEV)
        weights, bound = torch.cat([weights, zeros], 2), torch.cat([bound, zeros], 2)
        positions = torch.cat([positions, at.expand(B, H, T)], 2)
        out = mgr.attend(q)
        want, total, tol = attend64(q, mgr)
        agree(out, want)
        weights += total
        bound += tol + weights * 2.0 ** -24                  # and the addition's own rounding
        assert bool(((mgr.weights.double() - weights).abs() <= bound).all())
        assert torch.equal(mgr.positions.long(), positions)
        if mgr.seq_len > keep + 32:
            w32 = mgr.weights.clone()
            before = [c.to_contiguous() for c in mgr.get_kv()]
            S = mgr.seq_len
            r = mgr.evict(keep, sink, recent)
            kept = want_kept(w32.reshape(-1, S).cpu().numpy(), keep, sink, recent).reshape(B, H, keep)
            assert np.array_equal(r.kept.cpu().numpy(), kept) and mgr.seq_len == keep and mgr.next_position == appended
            idx = torch.from_numpy(kept).long().to(DEV)
            weights, bound, positions = (torch.gather(t, 2, idx) for t in (weights, bound, positions))
            for a, b in zip(before, mgr.get_kv()):
                rows = torch.gather(a.blocks, 2, idx[..., None].expand(B, H, keep, a.blocks.shape[-1]))
                assert torch.equal(b.to_contiguous().blocks, rows)
            assert mgr.evict(keep, sink, recent) is None
    assert appended > 370 and mgr.seq_len <= 400
    mgr.reset()
    assert mgr.next_position == mgr.seq_len == 0
    mgr.append(qkv[1][:, :, :1], qkv[2][:, :, :1])
    assert not mgr.weights.any() and not mgr.positions.any()


def test_layer_with_rotary_and_tracking_equals_its_parts():
    torch.manual_seed(0)
    emb = rotary.RotaryEmbedding(64, rot_dim=32, interleaved=True)
    layer = CompressedMultiHeadAttention(PolarQuantConfig(), 256, 4, 2, rotary=emb).to(DEV)
    mgr = KVCacheManager(PolarQuantConfig(), 512, 2, 2, 64, DEV, track_weights=True)
    plain = KVCacheManager(PolarQuantConfig(), 512, 2, 2, 64, DEV)
    xs = torch.randn(2, 90, 256, device=DEV)
    with torch.no_grad():
        for a, b in ((0, 70), (70, 71), (71, 90)):
            x = xs[:, a:b]
            got = layer(x, mgr)
            assert torch.equal(got, layer(x, plain))          # keeping the weights changes no output
            q = layer.q_proj(x).reshape(2, b - a, 4, 64).transpose(1, 2).half()
            q = emb(q, None, torch.arange(a, b, device=DEV))[0]
            want = attend64(q, mgr)[0].transpose(1, 2).reshape(2, b - a, 256).half().float()
            agree(got, layer.o_proj(want).double())
    # each of 4 query heads' 90 rows gives weight 1, over 2 kv heads
    assert torch.allclose(mgr.weights.sum(-1), torch.full((2, 2), 180.0, device=DEV), rtol=1e-4)
    assert plain.weights is None and plain.positions is None


def test_layer_without_a_cache_trains_through_rotary():
    """The layer runs and every projection gets a gradient (the rotation's own
    gradients are tested against the formula and differences beside it)."""
    torch.manual_seed(1)
    layer = CompressedMultiHeadAttention(PolarQuantConfig(enable_compression=False), 128, 2, 1,
                                         rotary=rotary.RotaryEmbedding(64)).to(DEV)
    x = torch.randn(2, 17, 128, device=DEV)
    out = layer(x)
    (out.square().sum()).backward()
    grads = [p.grad.clone() for p in layer.parameters()]
    assert all(torch.isfinite(g).all() and g.abs().max() > 0 for g in grads)


def test_manager_refusals():
    with pytest.raises(ValueError):
        KVCacheManager(PolarQuantConfig(enable_compression=False), 64, 1, 1, 64, DEV, track_weights=True)
    mgr = KVCacheManager(PolarQuantConfig(), 64, 1, 1, 64, DEV)
    with pytest.raises(ValueError):
        mgr.evict(8, 0, 0)
    mgr = KVCacheManager(PolarQuantConfig(), 64, 1, 1, 64, DEV, track_weights=True)
    for kw in (dict(keep=0, sink=0, recent=0), dict(keep=10, sink=4, recent=7)):
        with pytest.raises(ValueError):
            mgr.evict(**kw)
    assert mgr.evict(10, 2, 2) is None and mgr.weights is None
    with pytest.raises(ValueError):
        CompressedMultiHeadAttention(PolarQuantConfig(), 128, 2, rotary=rotary.RotaryEmbedding(32))
    assert math.isclose(rotary.RotaryEmbedding(32).amplitude, 1.0) and inference.PolarQuantConfig().n_bits == 4
