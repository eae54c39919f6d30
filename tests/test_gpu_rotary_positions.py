"""Text of a batch through an embedding on several axes: a row of positions per
sequence, in every entry that takes an embedding."""

import pytest
import torch

import window_ref
from polarquant_kv import rotary
from polarquant_kv.inference import CompressedMultiHeadAttention, KVCacheManager, PolarQuantConfig

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SECTIONS = (12, 10, 10)


@pytest.mark.parametrize("B,T", [(8, 1), (2, 5), (1, 9)])
def test_embedding(B, T):
    q, k = torch.randn(B, 4, T, 64, device=DEV), torch.randn(B, 2, T, 64, device=DEV)
    text = torch.randint(0, 100000, (B, T), device=DEV)
    want = rotary.RotaryEmbedding(64)(q, k, text)
    got = rotary.RotaryEmbedding(64, sections=SECTIONS)(q, k, text)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("B,T", [(8, 1), (2, 17)])
def test_manager_and_layer(B, T):
    flat, several = rotary.RotaryEmbedding(64), rotary.RotaryEmbedding(64, sections=SECTIONS)
    q, k, v = (torch.randn(B, n, T, 64, device=DEV).half() for n in (4, 2, 2))
    text = torch.randint(0, 100000, (B, T), device=DEV)
    blocks, turned, outs = [], [], []
    x = torch.randn(B, T, 256, device=DEV)
    for e in (flat, several):
        m = KVCacheManager(PolarQuantConfig(), 100, B, 2, 64, DEV)
        turned.append(m.append_rotary(q, k, v, e, text))
        blocks.append([window_ref.rows_of(c)[0] for c in m.get_kv()])
        torch.manual_seed(0)
        layer = CompressedMultiHeadAttention(PolarQuantConfig(), 256, 4, 2, rotary=e, window=8).to(DEV)
        with torch.no_grad():
            outs.append(layer(x, KVCacheManager(PolarQuantConfig(), 100, B, 2, 64, DEV), positions=text))
    assert torch.equal(turned[0], turned[1]) and torch.equal(outs[0], outs[1])
    assert all(torch.equal(a, b) for a, b in zip(*blocks))
