"""Attention behind a window for queries far from 1: rotated and scaled they pass
what fp16 holds, in single tokens and in chunks, with and without signs. Keys are
small enough for logits of a few units, so that the bounds of window_ref are sharp."""

import pytest
import torch

import test_gpu_window as window_tests
import window_ref
from polarquant_kv import attention, quantizer, rotation

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(Sq, d, Hkv, G, bits, qjl, page, size, scale, S=300, seed=0):
    """Queries of 2 `size`, keys that give logits of about 3."""
    B = 2
    g = torch.Generator(device=DEV).manual_seed(seed)
    R = rotation.generate_rotation_matrix(d, seed=42, device=DEV)
    jl = torch.randn(d, d, generator=g, device=DEV) if qjl else None
    small = 1.5 / (size * scale * d ** 0.5)
    caches = []
    for which in ("keys", "values"):
        x = torch.randn(B, Hkv, S, d, generator=g, device=DEV) * (small if which == "keys" else 1.0)
        p = jl if which == "keys" else None
        c = quantizer.allocate_paged_cache(B, Hkv, d, bits, DEV, page_tokens=page, jl_dim=d if qjl and p is not None else 0) \
            if page else None
        caches.append(quantizer.compress_pq(x, R, bits, cache=c, jl_rot=p))
    q = 2.0 * size * torch.randn(B, Hkv * G, Sq, d, generator=g, device=DEV)
    if jl is not None:
        jl = jl * small         # a correction of the keys' size
    return q, caches[0], caches[1], R, jl


SHAPES = [(64, 2, 7, 4, False, 0), (128, 2, 4, 4, False, 64), (128, 1, 8, 2, False, 0), (64, 2, 3, 4, True, 0),
          (128, 2, 6, 2, True, 64), (128, 1, 12, 4, True, 0)]


@pytest.mark.parametrize("size,scale", [(1e3, None), (1e4, None), (1e3, 1.0), (1e4, 1.0), (3e4, 1.0), (1e-4, 3e8),
                                        (1e18, 1e-4), (1e30, 1e-4)])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "d{}_{}x{}_b{}_{}_p{}".format(*s))
@pytest.mark.parametrize("Sq", [1, 19, 190])
def test_large_queries(Sq, shape, size, scale):
    d, Hkv, G, bits, qjl, page = shape
    q, keys, values, R, jl = make(Sq, d, Hkv, G, bits, qjl, page, min(size, 3e4), d ** -0.5 if scale is None else scale)
    if size > 3e4:      # (radii are fp16: the rest is in the scale)
        q = q * (size / 3e4)
        scale = scale * (3e4 / size)
        assert torch.isfinite(q).all()
    elif size >= 1.0:
        q = q.clamp(-65504, 65504).half() if size < 3e4 else q
    B = 2
    at, n = window_tests.per_sequence([300 - Sq, 5], B), window_tests.per_sequence([Sq, max(1, Sq - 3)], B)
    want, bound = window_ref.window_attention(q, keys, values, R, 64, 3, at, n, scale=scale, p_rot=jl)
    assert float(bound.max()) < 0.05
    got = attention.window_attention(q, keys, values, R, 64, sinks=3, starts=at, counts=n, scale=scale, jl_rot=jl,
                                     out_dtype=torch.float32)
    window_ref.check(got, want, bound)


@pytest.mark.parametrize("Sq", [1, 24])
@pytest.mark.parametrize("d,qjl", [(64, False), (128, False), (128, True)])
def test_sizes_side_by_side(d, qjl, Sq):
    """Rows and heads of very different sizes in one matrix operand: small ones keep their bits."""
    q, keys, values, R, jl = make(Sq, d, 2, 4, 4, qjl, 0, 1.0, 1.0)
    sizes = torch.tensor([1.0, 2.0 ** 17, 2.0 ** -9, 2.0 ** 30, 0.0, 2.0 ** 12], device=DEV)
    q = q * sizes[(torch.arange(8, device=DEV)[:, None] + torch.arange(Sq, device=DEV)) % 6][None, :, :, None]
    at, n = window_tests.per_sequence([300 - Sq, 5], 2), window_tests.per_sequence(Sq, 2)
    want, bound = window_ref.window_attention(q, keys, values, R, 64, 3, at, n, scale=1.0, p_rot=jl)
    got = attention.window_attention(q, keys, values, R, 64, sinks=3, starts=at, scale=1.0, jl_rot=jl, out_dtype=torch.float32)
    window_ref.check(got, want, bound)


@pytest.mark.parametrize("Sq", [1, 24])
@pytest.mark.parametrize("d,bits", [(64, 4), (128, 2)])
def test_large_projections(d, bits, Sq):
    """Signs whose projections alone pass what fp16 holds."""
    q, keys, values, R, jl = make(Sq, d, 2, 4, bits, True, 0, 1.0, 1.0)
    jl = jl / float(jl.abs().max()) * 2.0 ** 26
    at, n = window_tests.per_sequence([300 - Sq, 5], 2), window_tests.per_sequence(Sq, 2)
    want, bound = window_ref.window_attention(q, keys, values, R, 64, 3, at, n, scale=1.0, p_rot=jl)
    got = attention.window_attention(q, keys, values, R, 64, sinks=3, starts=at, scale=1.0, jl_rot=jl, out_dtype=torch.float32)
    window_ref.check(got, want, bound)


@pytest.mark.parametrize("power", [-140, -125, -118, -100, -60])
@pytest.mark.parametrize("Sq", [1, 24])
@pytest.mark.parametrize("d", [64, 128])
def test_tiny_projections(d, Sq, power):
    """Signs whose projections are far below everything else."""
    q, keys, values, R, jl = make(Sq, d, 2, 4, 4, True, 0, 1.0, 1.0)
    jl = torch.ldexp(jl, torch.tensor(float(power), device=DEV))
    at, n = window_tests.per_sequence([300 - Sq, 5], 2), window_tests.per_sequence(Sq, 2)
    want, bound = window_ref.window_attention(q, keys, values, R, 64, 3, at, n, scale=1.0, p_rot=jl)
    got = attention.window_attention(q, keys, values, R, 64, sinks=3, starts=at, scale=1.0, jl_rot=jl, out_dtype=torch.float32)
    window_ref.check(got, want, bound)
