"""The attention layer with positions given: on one axis and several, without a
cache and with an uncompressed one against the formula in 64 bits, with a compressed
one against the manager's calls."""

import pytest
import torch

from polarquant_kv import rotary
from polarquant_kv.inference import CompressedMultiHeadAttention, KVCacheManager, PolarQuantConfig

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
B, T, HQ, H, D = 2, 21, 4, 2, 64
SECTIONS = {"one": None, "three": (12, 10, 10)}


def make(sections, compressed, window, sinks):
    torch.manual_seed(3)
    e = rotary.RotaryEmbedding(D, sections=sections)
    layer = CompressedMultiHeadAttention(PolarQuantConfig(enable_compression=compressed), HQ * D, HQ, H, rotary=e,
                                         window=window, sinks=sinks).to(DEV)
    x = torch.randn(B, T, HQ * D, device=DEV)
    shape = (B, T) if sections is None else (len(sections), B, T)
    return layer, e, x, torch.randint(0, 5000, shape, device=DEV)


def heads(layer, x):
    return [p(x).reshape(B, -1, n, D).transpose(1, 2).half()
            for p, n in ((layer.q_proj, HQ), (layer.k_proj, H), (layer.v_proj, H))]


def formula(layer, e, x, positions, window, sinks):
    """(output, bound): the heads' outputs are rounded to fp16 once (2^-11 of each), what is before and after in
    32 bits is off by less than 2^-14 of the norms it sums (256 and 64 terms, weights below 1)."""
    q, k, v = heads(layer, x)
    axes = [0] * (D // 2) if e.axes is None else list(e.axes)
    at = (positions[None] if e.axes is None else positions)[torch.tensor(axes, device=DEV)]       # [pairs, B, T]
    t = (at.permute(1, 2, 0).double() * e.frequencies.to(DEV))[:, None]
    turned = []
    for y in (q, k):
        a, b = y.double().chunk(2, -1)
        y = torch.cat((a * t.cos() - b * t.sin(), a * t.sin() + b * t.cos()), -1)
        turned.append(y.half().double())
    q, k, v = turned[0], turned[1].repeat_interleave(HQ // H, 1), v.double().repeat_interleave(HQ // H, 1)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) / D ** 0.5
    i = torch.arange(T, device=DEV)
    hidden = i[None] > i[:, None]
    if window is not None:
        hidden = hidden | ((i[None] <= i[:, None] - window) & (i[None] >= sinks))
    s = s.masked_fill(hidden, float("-inf"))
    # (a turned state that rounds the other way moves a logit by 2^-11 of its products)
    ds = torch.matmul(q.abs(), k.abs().transpose(2, 3).contiguous()).masked_fill(hidden, 0.0) / D ** 0.5 * 2.0 ** -10
    w = torch.softmax(s, -1)
    out = torch.matmul(w, v)
    off = torch.matmul(w * 2 * ds.amax(-1, keepdim=True), v.abs()) + out.abs() * 2.0 ** -11 + 2.0 ** -14 * torch.matmul(w, v.abs())
    flat = lambda y: y.transpose(1, 2).reshape(B, T, -1)  # noqa: E731
    W = layer.o_proj.weight.double()
    return flat(out) @ W.t(), flat(off + 2.0 ** -14 * out.abs()) @ W.abs().t()


@pytest.mark.parametrize("window,sinks", [(None, 0), (6, 2)])
@pytest.mark.parametrize("sections", SECTIONS)
@torch.no_grad()
def test_the_formula(sections, window, sinks):
    layer, e, x, positions = make(SECTIONS[sections], False, window, sinks)
    want, bound = formula(layer, e, x, positions, window, sinks)
    m = KVCacheManager(PolarQuantConfig(enable_compression=False), 40, B, H, D, DEV)
    steps = torch.cat([layer(x[:, a:b], m, positions=positions[..., a:b]) for a, b in ((0, 9), (9, 10), (10, T))], 1)
    for got in (layer(x, None, positions=positions), steps):
        assert bool(((got.double() - want).abs() <= bound).all())
    assert not bool(((layer(x).double() - want).abs() <= bound).all())       # positions make a difference
    # the ones after those cached are the default
    line = torch.arange(T, device=DEV)
    assert torch.equal(layer(x), layer(x, None, positions=line))


@pytest.mark.parametrize("window,sinks", [(None, 0), (6, 2)])
@pytest.mark.parametrize("sections", SECTIONS)
@torch.no_grad()
def test_a_compressed_cache(sections, window, sinks):
    layer, e, x, positions = make(SECTIONS[sections], True, window, sinks)
    mine, other = (KVCacheManager(PolarQuantConfig(), 40, B, H, D, DEV) for _ in range(2))
    for a, b in ((0, 9), (9, 10), (10, T)):
        got = layer(x[:, a:b], mine, positions=positions[..., a:b])
        q, k, v = heads(layer, x[:, a:b])
        if window is None:
            q, k = e(q, k, positions[..., a:b])
            other.append(k, v)
            out = other.attend(q)
        else:
            q = other.append_rotary(q, k, v, e, positions[..., a:b])
            out = other.attend(q, window=window, sinks=sinks)
        assert torch.equal(got, layer.o_proj(out.transpose(1, 2).reshape(B, b - a, -1).float()))
