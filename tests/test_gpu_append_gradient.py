"""Derivatives through the query that append_rotary turns: those of
rotary.apply_rotary, to the bit."""

import pytest
import torch
from torch.autograd import forward_ad

import window_ref
from polarquant_kv import append, quantizer, rotary, rotation
from polarquant_kv.inference import KVCacheManager, PolarQuantConfig

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
B, HQ, H, T, D = 2, 4, 2, 19, 64


def make(sections, page):
    q, k, v = (torch.randn(B, T, n, D, device=DEV).transpose(1, 2) for n in (HQ, H, H))
    R = rotation.generate_rotation_matrix(D, device=DEV)
    caches = [quantizer.allocate_paged_cache(B, H, D, 4, DEV, page_tokens=64) if page else
              quantizer.allocate_cache(B, H, T, D, 4, DEV) for _ in range(4)]
    axes = None if sections is None else rotary.axis_of_pairs(sections)
    positions = torch.randint(0, 1000, (B, T) if axes is None else (len(sections), B, T), device=DEV)
    freqs = rotary.rotary_frequencies(48)[0].to(DEV)
    return q, k, v, caches, R, positions, freqs, dict(axes=axes, interleaved=axes is not None, amplitude=1.25)


@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("sections", [None, (10, 14)])
def test_gradient_and_tangent(sections, page):
    q, k, v, caches, R, positions, freqs, how = make(sections, page)
    plain = append.append_rotary(k, v, *caches[:2], R, positions, freqs, query=q, **how)
    x = q.clone().requires_grad_(True)
    out = append.append_rotary(k, v, *caches[2:], R, positions, freqs, query=x, **how)
    assert torch.equal(out.detach(), plain)
    for a, b in zip(caches[:2], caches[2:]):        # the caches get the same
        assert a.seq_len == b.seq_len == T
        assert torch.equal(window_ref.rows_of(a)[0], window_ref.rows_of(b)[0])
    y = q.clone().requires_grad_(True)
    want = rotary.apply_rotary(y, None, positions, freqs, **how)[0]
    g = torch.randn_like(want)
    assert torch.equal(torch.autograd.grad(out, x, g)[0], torch.autograd.grad(want, y, g)[0])
    with torch.no_grad():
        out = append.append_rotary(k, v, *caches[2:], R, positions, freqs, query=x, starts=0, **how)
        assert torch.equal(out, plain) and out.grad_fn is None
    with forward_ad.dual_level():
        t = torch.randn_like(q)
        out = append.append_rotary(k, v, *caches[2:], R, positions, freqs, query=forward_ad.make_dual(q, t), starts=0, **how)
        want = rotary.apply_rotary(t, None, positions, freqs, **how)[0]
        assert torch.equal(forward_ad.unpack_dual(out).tangent, want)


def test_through_the_manager():
    q, k, v, _, R, positions, _, _ = make(None, 0)
    e = rotary.RotaryEmbedding(D)
    q = q.requires_grad_(True)
    m = KVCacheManager(PolarQuantConfig(), 100, B, H, D, DEV)
    out = m.append_rotary(q, k.requires_grad_(True), v, e, positions)
    g = torch.randn_like(out)
    got = torch.autograd.grad(out, q, g)[0]
    assert torch.equal(got, torch.autograd.grad(e(q, None, positions)[0], q, g)[0])
