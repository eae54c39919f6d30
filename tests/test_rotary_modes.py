"""Rotary positions under the modes of torch.autograd, without a GPU: the launch
is stood in for by the formula in torch operations that know nothing of
derivatives, as the launch knows nothing of them."""

import pytest
import torch
from torch.autograd import forward_ad

from polarquant_kv import _lib, rotary


def formula(x, positions, freqs, interleaved, m, inverse):
    n = freqs.numel()
    t = positions.double()[:, None] * freqs
    c, s = torch.cos(t).to(x.dtype), torch.sin(t).to(x.dtype) * (-1 if inverse else 1)
    ia = torch.arange(n) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else n)
    a, b = x[..., ia], x[..., ib]
    y = x.clone()
    y[..., ia], y[..., ib] = m * (a * c - b * s), m * (a * s + b * c)
    return y


@pytest.fixture
def launches(monkeypatch):
    """Counts the launches; each sees plain numbers, no tangent and no graph."""
    count = []

    def turn(q, k, positions, freqs, interleaved, amplitude, inverse):
        count.append(1)
        assert k is None or q.dtype == k.dtype
        bare = [None if x is None else torch.from_numpy(x.detach().numpy().copy()) for x in (q, k)]
        return tuple(None if x is None else formula(x, positions, freqs, interleaved, amplitude, inverse) for x in bare)

    monkeypatch.setattr(rotary, "_turn", turn)
    monkeypatch.setattr(_lib, "require_device", lambda *t: None)
    return count


def inputs(dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, tq, tk = (torch.randn(2, h, 5, 8, generator=g, dtype=torch.float64).to(dtype) for h in (3, 1, 3, 1))
    return q, k, tq, tk, torch.arange(7, 12), rotary.rotary_frequencies(6)[0]


@pytest.fixture
def doubles(monkeypatch):
    """float64 stands for the float32 that the kernels take."""
    monkeypatch.setattr(rotary, "_code", lambda t: 0)


@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_mode_tangents(launches, doubles, interleaved):
    q, k, tq, tk, pos, f = inputs()
    how = dict(interleaved=interleaved, amplitude=1.25)

    def want(x):
        return formula(x, pos, f, interleaved, 1.25, False)

    with forward_ad.dual_level():
        dq, dk = forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk)
        for a, b in ((dq, dk), (dq, k), (q, dk), (dq, None)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad):
                    out = rotary.apply_rotary(a, b, pos, f, **how)
                for x, y, t, moves in ((q, out[0], tq, a is dq), (k, out[1], tk, b is dk)):
                    if y is None:
                        assert b is None
                        continue
                    p = forward_ad.unpack_dual(y)
                    assert torch.equal(p.primal, want(x))
                    got = torch.zeros_like(x) if p.tangent is None else p.tangent
                    assert torch.equal(got, want(t) if moves else torch.zeros_like(x))
    before = len(launches)
    rotary.apply_rotary(q, k, pos, f, **how)
    assert len(launches) == before + 1                         # nothing to differentiate: the launch alone


def test_tangent_of_another_type(launches):
    q, k, tq, tk, pos, f = inputs(torch.float32)
    with forward_ad.dual_level():
        out = rotary.apply_rotary(forward_ad.make_dual(q, tq.double()), forward_ad.make_dual(k, tk.bfloat16()), pos, f)
        got = [forward_ad.unpack_dual(y).tangent for y in out]
    assert torch.equal(got[0], formula(tq, pos, f, False, 1.0, False))
    assert torch.equal(got[1], formula(tk.bfloat16().float(), pos, f, False, 1.0, False))


def test_tangent_on_another_device_is_refused(launches, doubles):
    """(forward_ad takes such a pair; the launch would read a foreign address)"""
    q, k, tq, tk, pos, f = inputs()
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="several devices"):
            rotary.apply_rotary(q, forward_ad.make_dual(k, tk.to("meta")), pos, f)


def test_tangents_of_gradients_and_gradients_of_tangents(launches, doubles):
    q, k, tq, tk, pos, f = inputs()
    q1 = q.clone().requires_grad_(True)
    back = lambda x: formula(x, pos, f, False, 1.0, True)
    with forward_ad.dual_level():                               # the gradient is linear in what comes in
        y, _ = rotary.apply_rotary(q1, None, pos, f)
        g, = torch.autograd.grad(y, q1, forward_ad.make_dual(q, tq))
        p = forward_ad.unpack_dual(g)
        assert torch.equal(p.primal, back(q)) and torch.equal(p.tangent, back(tq))
    t1 = tq.clone().requires_grad_(True)
    with forward_ad.dual_level():
        y, _ = rotary.apply_rotary(forward_ad.make_dual(q, t1), k, pos, f)
        g, = torch.autograd.grad(forward_ad.unpack_dual(y).tangent, t1, tk.expand_as(tq).contiguous())
    assert torch.equal(g, back(tk.expand_as(tq)))
    assert torch.autograd.gradcheck(lambda a, b: rotary.apply_rotary(a, b, pos, f, amplitude=1.25),
                                    (q1, k.clone().requires_grad_(True)), check_forward_ad=True)


def test_embedding_used_in_inference_mode_first(launches):
    """What the embedding keeps from a call outlives its mode."""
    q, k, _, _, pos, _ = inputs(torch.float32)
    with torch.inference_mode():
        emb = rotary.RotaryEmbedding(8)
        emb(q.clone(), k.clone(), pos)
    assert not emb.frequencies.is_inference()
    q1 = q.clone().requires_grad_(True)
    y, _ = emb(q1, k, pos)
    g, = torch.autograd.grad(y, q1, torch.ones_like(y))
    assert torch.equal(g, formula(torch.ones_like(q), pos, emb.frequencies, False, 1.0, True))
