"""pqkv_rotary_axes through rotary.apply_rotary(axes=...) against the formula in
64 bits. Tolerance: as for one axis, the fraction of a turn is rounded to 32 bits
once, and everything after it adds up to less than 2^-20 of |x_a| + |x_b|; the
result is rounded once more to its type. Positions of up to 2^33 are turned
here, at which the angle's own roundings in 64 bits count too."""

import pytest
import torch
from torch.autograd import forward_ad

from polarquant_kv import rotary

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def plain(x, positions, axes, freqs, interleaved, m, inverse=False):
    n = freqs.numel()
    at = positions if positions.dim() == 3 else positions[:, None].expand(-1, x.shape[0], -1)
    t = torch.stack([at[a].double() * freqs[i] for i, a in enumerate(axes)], -1)[:, None]     # [B, 1, T, pairs]
    c, s = torch.cos(t), torch.sin(t) * (-1 if inverse else 1)
    x = x.detach().double()
    y, size = x.clone(), torch.zeros_like(x)
    ia = torch.arange(n, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else n)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = m * (a * c - b * s), m * (a * s + b * c)
    # the angle t itself: frequency / (2 pi) (the constant's rounding and the product's), the
    # product with the position, and the one here, each half a step of 64 bits: 4 x 2^-53 |t|
    size[..., ia] = size[..., ib] = abs(m) * (a.abs() + b.abs()) * (2.0 ** -20 + 2.0 ** -51 * t.abs())
    return y, size


def check(got, x, positions, axes, freqs, interleaved, m=1.0, inverse=False):
    want, size = plain(x, positions, axes, freqs, interleaved, m, inverse)
    t = got.dtype
    assert got.shape == x.shape and t == x.dtype
    tol = size + torch.clamp(torch.finfo(t).eps / 2 * (want.abs() + size), min=SMALLEST[t])
    tol[..., 2 * freqs.numel():] = 0.0
    assert bool(((got.double() - want).abs() <= tol).all())


# B, Hq, Hkv, T, d, sections, spread, interleaved, dtype, one row of positions for all sequences
CASES = [
    (1, 1, 1, 1, 64, (16, 16), False, False, torch.float16, False),
    (8, 32, 8, 1, 128, (16, 24, 24), False, False, torch.float16, False),
    (2, 14, 2, 33, 64, (14, 14), False, True, torch.float32, False),
    (3, 5, 5, 257, 128, (24, 20, 20), True, False, torch.bfloat16, True),
    (2, 3, 1, 19, 80, (1, 0, 2), False, False, torch.float16, False),      # an axis without pairs
    (1, 2, 1, 2100, 128, (22, 21, 21), True, True, torch.bfloat16, False),
    (1, 2, 2, 5, 1024, (300, 212), False, False, torch.float32, True),     # the widest head
    (2, 4, 2, 9, 64, (5,), False, False, torch.float32, False),
]
ids = ["B{}_Hq{}_Hkv{}_T{}_d{}_{}_{}".format(*c[:7]) for c in CASES]


def make(case, seed=1):
    B, Hq, Hkv, T, d, sections, spread, inter, dtype, shared = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(B, T, Hq, d, generator=g, device=DEV).to(dtype).transpose(1, 2)
    k = torch.randn(B, T, Hkv, d, generator=g, device=DEV).to(dtype).transpose(1, 2)
    axes = rotary.axis_of_pairs(sections, spread)
    shape = (len(sections), T) if shared else (len(sections), B, T)
    positions = torch.randint(0, 2 ** 33, shape, generator=g, device=DEV)
    positions[:, ..., :1] = 0
    return q, k, positions, axes, rotary.rotary_frequencies(2 * len(axes))[0].to(DEV), inter


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_forward_and_gradient(case):
    q, k, pos, axes, freqs, inter = make(case)
    q.requires_grad_(True), k.requires_grad_(True)
    qo, ko = rotary.apply_rotary(q, k, pos, freqs, interleaved=inter, amplitude=1.25, axes=axes)
    check(qo.detach(), q, pos, axes, freqs, inter, 1.25)
    check(ko.detach(), k, pos, axes, freqs, inter, 1.25)
    gq, gk = torch.randn_like(qo), torch.randn_like(ko)
    dq, dk = torch.autograd.grad((qo, ko), (q, k), (gq, gk))
    check(dq, gq, pos, axes, freqs, inter, 1.25, True)
    check(dk, gk, pos, axes, freqs, inter, 1.25, True)
    # only the keys' gradient
    qo, ko = rotary.apply_rotary(q.detach(), k, pos, freqs, interleaved=inter, axes=axes)
    check(torch.autograd.grad(ko, k, gk)[0], gk, pos, axes, freqs, inter, 1.0, True)
    alone, none = rotary.apply_rotary(q.detach(), None, pos, freqs, interleaved=inter, axes=axes)
    assert none is None and torch.equal(alone, qo)


def test_gradient_against_differences():
    q, k, pos, axes, freqs, inter = make((1, 2, 1, 3, 64, (3, 2, 2), True, True, torch.float32, False))
    gq = torch.randn_like(q)
    f = lambda x: (rotary.apply_rotary(x, None, pos, freqs, interleaved=inter, axes=axes)[0].double() * gq).sum()  # noqa: E731
    x = q.clone().requires_grad_(True)
    grad = torch.autograd.grad(rotary.apply_rotary(x, None, pos, freqs, interleaved=inter, axes=axes)[0], x, gq)[0]
    step = torch.randn_like(q)
    # linear, so a difference over a step of any size is the gradient's product with it, up to
    # the roundings of 2 x 384 values of about 1 (each 2^-22) and of x + step itself
    assert abs(float(f(q + step) - f(q)) - float((grad.double() * step).sum())) <= 2 * 384 * 2.0 ** -21


def test_second_derivatives_and_tangents():
    q, k, pos, axes, freqs, inter = make(CASES[2])
    x = q.clone().requires_grad_(True)
    y = rotary.apply_rotary(x, None, pos, freqs, interleaved=inter, axes=axes)[0]
    g = torch.randn_like(y).requires_grad_(True)
    dx = torch.autograd.grad(y, x, g, create_graph=True)[0]
    dg = torch.autograd.grad(dx, g, q)[0]
    check(dg, q, pos, axes, freqs, inter)
    with forward_ad.dual_level():
        t = torch.randn_like(q)
        out = rotary.apply_rotary(forward_ad.make_dual(q, t), k, pos, freqs, interleaved=inter, axes=axes)[0]
        check(forward_ad.unpack_dual(out).tangent, t, pos, axes, freqs, inter)


def test_equal_axes_are_one_axis():
    q, k, _, axes, freqs, inter = make(CASES[1])
    pos = torch.arange(1000, 1000 + 8, device=DEV)[:, None]
    want = rotary.apply_rotary(q, k, pos, freqs, interleaved=inter)
    got = rotary.apply_rotary(q, k, pos.expand(3, 8, 1), freqs, interleaved=inter, axes=axes)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    emb, flat = rotary.RotaryEmbedding(128, sections=(16, 24, 24)), rotary.RotaryEmbedding(128)
    line = torch.arange(5, 6, device=DEV)
    assert all(torch.equal(a, b) for a, b in zip(emb(q, k, line), flat(q, k, line)))
    assert all(torch.equal(a, b) for a, b in zip(emb(q, k, line.expand(3, 8, 1)), flat(q, k, line)))


def test_strided_positions_and_a_captured_call():
    q, k, pos, axes, freqs, inter = make(CASES[3])
    wide = torch.empty(pos.shape[1], pos.shape[0], dtype=torch.int64, device=DEV)
    wide.copy_(pos.t())
    want = rotary.apply_rotary(q, k, pos, freqs, interleaved=inter, axes=axes)
    got = rotary.apply_rotary(q, k, wide.t(), freqs, interleaved=inter, axes=list(axes))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = rotary.apply_rotary(q, k, pos.to(torch.int64).repeat(2, 1)[:3], freqs, interleaved=inter, axes=axes)
    assert torch.equal(got[0], want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rotary.apply_rotary(q, k, pos, freqs, interleaved=inter, axes=axes)
    for _ in range(3):
        pos += 17
        graph.replay()
        kept = [x.clone() for x in got]
        want = rotary.apply_rotary(q, k, pos, freqs, interleaved=inter, axes=axes)
        torch.cuda.synchronize()
        assert torch.equal(kept[0], want[0]) and torch.equal(kept[1], want[1])


def test_refusals():
    q, k, pos, axes, freqs, inter = make(CASES[1])
    for kw, words in ((dict(axes=axes[:-1]), "axes for"), (dict(axes=axes[:-1] + (3,)), "positions must be"),
                      (dict(axes=axes[:-1] + (-1,)), "numbers of axes"), (dict(axes=axes[:-1] + (256,)), "numbers of axes"),
                      (dict(axes=axes[:-1] + (0.5,)), "numbers of axes"), (dict(positions=pos[:2]), "positions must be"), (dict(positions=pos[0, 0]), "positions must be"),
                      (dict(positions=pos[:, :, None]), "positions must be"), (dict(positions=pos.double()), "integers")):
        with pytest.raises(ValueError, match=words):
            rotary.apply_rotary(q, k, kw.get("positions", pos), freqs, axes=kw.get("axes", axes))
