"""pqkv_rotary through polarquant_kv.rotary against the formula in 64 bits.

Tolerance, from the roundings: the fraction of a turn is rounded to 32 bits
once (at most 2^-26 of a turn, 2 pi 2^-26 radians), sine and cosine are within
4 ulp of values up to 1 (2^-22), the amplitude, its product with them, the two
products and their sum round by 2^-24 each (5 of them): per unit of
m (|x_a| + |x_b|) less than 2 pi 2^-26 + 2^-22 + 5 2^-24 < 2^-20. The result
is rounded once more to its type: half a step, or half the smallest step below
the normal range."""

import math

import pytest
import torch

from polarquant_kv import rotary

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def plain(x, positions, freqs, interleaved, m, inverse=False):
    """(result, bound per element without the last rounding) in 64 bits."""
    n = freqs.numel()
    pos = positions.double()
    pos = pos.view(1, 1, -1, 1) if pos.dim() == 1 else pos[:, None, :, None]
    t = pos * freqs
    c, s = torch.cos(t), torch.sin(t) * (-1 if inverse else 1)
    x = x.detach().double()
    y, size = x.clone(), torch.zeros_like(x)
    ia = torch.arange(n, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else n)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = m * (a * c - b * s), m * (a * s + b * c)
    size[..., ia] = size[..., ib] = abs(m) * (a.abs() + b.abs()) * 2.0 ** -20
    return y, size


def check(got, x, positions, freqs, interleaved, m, inverse=False):
    want, size = plain(x, positions, freqs, interleaved, m, inverse)
    t = got.dtype
    assert got.is_contiguous() and got.shape == x.shape and t == x.dtype
    tol = size + torch.clamp(torch.finfo(t).eps / 2 * (want.abs() + size), min=SMALLEST[t])
    tol[..., 2 * freqs.numel():] = 0.0                     # the rest of the head is copied
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (err - tol).max().item()


CASES = [
    # B, Hq, Hkv, T, d, rot, interleaved, dtype, start
    (1, 1, 1, 1, 64, 64, False, torch.float16, 0),
    (8, 32, 8, 1, 128, 128, False, torch.float16, 131071),
    (1, 14, 2, 1, 64, 64, True, torch.bfloat16, 1000003),
    (2, 14, 2, 33, 64, 48, True, torch.float32, 0),
    (2, 3, 1, 257, 128, 128, False, torch.bfloat16, 7),
    (1, 5, 5, 1030, 64, 32, False, torch.float16, 2 ** 31),
    (3, 4, 2, 17, 80, 80, False, torch.float16, 5),       # half of it is no multiple of the vector
    (2, 4, 2, 19, 128, 42, True, torch.float32, 11),      # odd pair count, scalar items
    (1, 2, 1, 9, 66, 2, False, torch.bfloat16, 3),        # one pair
    (1, 2, 2, 5, 1024, 1024, False, torch.float32, 3),    # the widest head
    (1, 64, 8, 2100, 128, 128, False, torch.bfloat16, 0), # several tokens per workgroup
    (2, 70, 1, 3, 64, 16, True, torch.float16, 0),
]
ids = ["B{}_Hq{}_Hkv{}_T{}_d{}_rot{}_{}_{}".format(*c[:6], "pairs" if c[6] else "halves", str(c[7])[6:]) for c in CASES]


def make(case, seed=1):
    B, Hq, Hkv, T, d, rot, inter, dtype, start = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(B, T, Hq, d, generator=g, device=DEV).to(dtype).transpose(1, 2)
    k = torch.randn(B, T, Hkv, d, generator=g, device=DEV).to(dtype).transpose(1, 2)
    freqs = rotary.rotary_frequencies(rot)[0].to(DEV)
    return q, k, torch.arange(start, start + T, device=DEV), freqs, inter


@pytest.mark.parametrize("case", CASES, ids=ids)
def test_forward_and_gradient(case):
    q, k, pos, freqs, inter = make(case)
    for m in (1.0, 1.25):
        q1, k1 = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
        qo, ko = rotary.apply_rotary(q1, k1, pos, freqs, interleaved=inter, amplitude=m)
        check(qo, q, pos, freqs, inter, m)
        check(ko, k, pos, freqs, inter, m)
        gq, gk = torch.randn_like(qo), torch.randn_like(ko)
        dq, dk = torch.autograd.grad((qo, ko), (q1, k1), (gq, gk))
        check(dq.contiguous(), gq, pos, freqs, inter, m, inverse=True)
        check(dk.contiguous(), gk, pos, freqs, inter, m, inverse=True)


def test_gradient_against_differences():
    """The map is linear, so (f(x + e v) - f(x - e v)) / 2e = f(v) up to the
    roundings of f at |x| + e |v|: with e = 1 the difference is exact to them."""
    q, k, pos, freqs, inter = make(CASES[3])
    q1 = q.clone().requires_grad_(True)
    out, _ = rotary.apply_rotary(q1, None, pos, freqs, interleaved=True, amplitude=0.75)
    w = torch.randn_like(out)
    grad, = torch.autograd.grad(out, q1, w)
    v = torch.randn_like(q)
    plus = rotary.apply_rotary(q + v, None, pos, freqs, interleaved=True, amplitude=0.75)[0].double()
    minus = rotary.apply_rotary(q - v, None, pos, freqs, interleaved=True, amplitude=0.75)[0].double()
    by_difference = ((plus - minus) / 2 * w.double()).sum()
    by_gradient = (grad.double() * v.double()).sum()
    # each element off by at most 2^-19 of its pair's size, times |w|; 8 = the largest |x| + |v| drawn, twice
    bound = 2.0 ** -19 * 8 * w.double().abs().sum()
    assert abs(by_difference - by_gradient) <= bound


def test_queries_alone_keys_alone_and_unused_outputs():
    q, k, pos, freqs, _ = make(CASES[4])
    out, none = rotary.apply_rotary(q, None, pos, freqs)
    assert none is None
    both_q, both_k = rotary.apply_rotary(q, k, pos, freqs)
    assert torch.equal(out, both_q)
    q1, k1 = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    qo, ko = rotary.apply_rotary(q1, k1, pos, freqs)
    g = torch.randn_like(ko)
    dk, = torch.autograd.grad(ko, k1, g, retain_graph=True)          # no gradient arrives at q
    check(dk.contiguous(), g, pos, freqs, False, 1.0, inverse=True)
    g = torch.randn_like(qo)
    dq, = torch.autograd.grad(qo, q1, g)
    check(dq.contiguous(), g, pos, freqs, False, 1.0, inverse=True)
    qo, ko = rotary.apply_rotary(q, k1, pos, freqs)                  # a query that needs no gradient
    dk, = torch.autograd.grad((qo.float().sum() + ko.float().sum()), k1)
    check(dk.contiguous(), torch.ones_like(k), pos, freqs, False, 1.0, inverse=True)


def test_positions_of_each_sequence_and_integer_types():
    q, k, _, freqs, inter = make(CASES[4])
    B, T = q.shape[0], q.shape[2]
    pos = torch.randint(0, 200000, (B, T), device=DEV)
    for p in (pos, pos.int(), pos.t().contiguous().t()):
        qo, ko = rotary.apply_rotary(q, k, p, freqs)
        check(qo, q, pos, freqs, inter, 1.0)
        check(ko, k, pos, freqs, inter, 1.0)
    neg = -pos[0]
    check(rotary.apply_rotary(q, None, neg, freqs)[0], q, neg, freqs, inter, 1.0)


def test_strides_offsets_and_expanded_inputs():
    dtype, d = torch.float16, 64
    freqs = rotary.rotary_frequencies(d)[0].to(DEV)
    big = torch.randn(2, 9, 5, 70, device=DEV).to(dtype)
    pos = torch.arange(9, device=DEV)
    views = [big[..., 1:65].transpose(1, 2),                 # rows off a 16-byte boundary
             big[..., :64].transpose(1, 2),                  # 140-byte rows
             big[:, ::2, :, :64].transpose(1, 2),
             torch.randn(2, 5, d, 9, device=DEV).to(dtype).transpose(2, 3)]   # no dense last dimension
    for v in views:
        p = pos[:v.shape[2]]
        check(rotary.apply_rotary(v, None, p, freqs)[0], v, p, freqs, False, 1.0)
    one = torch.randn(1, 1, 9, d, device=DEV, dtype=torch.float32, requires_grad=True)
    wide = one.expand(2, 5, 9, d)                            # shared heads: the gradient adds up over them
    f32 = rotary.apply_rotary(wide, None, pos, freqs)[0]
    check(f32, wide, pos, freqs, False, 1.0)
    g = torch.randn_like(f32)
    got, = torch.autograd.grad(f32, one, g)
    want, size = plain(g, pos, freqs, False, 1.0, inverse=True)
    err = (got.double() - want.sum((0, 1), keepdim=True)).abs()
    assert bool((err <= 2 * size.sum((0, 1), keepdim=True) + 1e-30).all())


def test_nan_and_infinity_stay_in_their_pair():
    q, _, pos, freqs, _ = make(CASES[4])
    q = q.contiguous()
    q[0, 0, 3, 5], q[1, 2, 200, 64] = float("nan"), float("inf")
    out = rotary.apply_rotary(q, None, pos, freqs)[0]
    bad = ~torch.isfinite(out)
    want = torch.zeros_like(bad)
    want[0, 0, 3, [5, 69]] = True
    want[1, 2, 200, [0, 64]] = True
    assert torch.equal(bad, want) and bool(torch.isnan(out[0, 0, 3, [5, 69]]).all())


def test_empty_calls():
    freqs = rotary.rotary_frequencies(64)[0].to(DEV)
    for shape in ((0, 2, 3, 64), (2, 2, 0, 64), (2, 0, 3, 64)):
        q = torch.zeros(shape, device=DEV, dtype=torch.float16)
        out, k = rotary.apply_rotary(q, q, torch.arange(shape[2], device=DEV), freqs)
        assert out.shape == q.shape and k.shape == q.shape


def test_refusals_on_the_device():
    q, k, pos, freqs, _ = make(CASES[1])
    for bad in (pos.float(), pos[:0], pos.expand(2, 1)):
        with pytest.raises(ValueError):
            rotary.apply_rotary(q, k, bad, freqs)
    with pytest.raises(ValueError):
        rotary.apply_rotary(q, k, pos, freqs.float())
    with pytest.raises(ValueError):
        rotary.apply_rotary(q, k, pos, torch.cat([freqs, freqs]))
    with pytest.raises(TypeError):
        rotary.apply_rotary(q.double(), None, pos, freqs)
    with pytest.raises(ValueError):
        rotary.apply_rotary(q, k, pos.cpu(), freqs)


def test_on_another_stream_and_captured():
    q, k, pos, freqs, inter = make(CASES[4])
    q, k = q.contiguous(), k.contiguous()
    emb = rotary.RotaryEmbedding(128, scaling={"type": "linear", "factor": 2.0})
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = emb(q, k, pos)[0]
    s.synchronize()
    check(got, q, pos, emb.frequencies.to(DEV), inter, 1.0)
    # forward and backward in a graph, replayed over new inputs beside eager work
    q1, k1 = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    w = torch.randn_like(q)
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(emb(q1, k1, pos)[0], q1, w)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo, ko = emb(q1, k1, pos)
        dq, = torch.autograd.grad(qo, q1, w)
    for i in range(4):
        with torch.no_grad():
            q1.copy_(torch.randn_like(q))
            w.copy_(torch.randn_like(q))
        graph.replay()
        eager = emb(q1.detach(), k1.detach(), pos)
        torch.cuda.synchronize()
        assert torch.equal(qo, eager[0]) and torch.equal(ko, eager[1])
        check(dq.contiguous(), w, pos, emb.frequencies.to(DEV), inter, 1.0, inverse=True)


def test_turning_by_a_sum_of_positions():
    """Scores depend on the difference of positions only."""
    d = 64
    freqs = rotary.rotary_frequencies(d)[0].to(DEV)
    q, k = torch.randn(1, 1, 1, d, device=DEV), torch.randn(1, 1, 1, d, device=DEV)

    def score(a, b):
        x = rotary.apply_rotary(q, None, torch.tensor([a], device=DEV), freqs)[0].double()
        y = rotary.apply_rotary(k, None, torch.tensor([b], device=DEV), freqs)[0].double()
        return (x * y).sum().item()

    size = (q.abs().double().view(2, -1).sum(0) * k.abs().double().view(2, -1).sum(0)).sum().item()
    assert math.isclose(score(5, 2), score(500005, 500002), abs_tol=4 * 2.0 ** -20 * size)


def test_gradient_of_the_gradient():
    """f is linear in x, so d/dx of <grad f, u> is 0 and d/dg of it is f(u)."""
    q, _, pos, freqs, _ = make(CASES[3])
    q = q.requires_grad_(True)
    out = rotary.apply_rotary(q, None, pos, freqs, interleaved=True, amplitude=1.5)[0]
    g = torch.randn_like(out).requires_grad_(True)
    dq, = torch.autograd.grad(out, q, g, create_graph=True)
    u = torch.randn_like(dq)
    dg, = torch.autograd.grad(dq, g, u)
    check(dg.contiguous(), u, pos, freqs, True, 1.5)
