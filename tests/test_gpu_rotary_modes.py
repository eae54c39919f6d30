"""pqkv_rotary under the modes of torch.autograd. The map is linear, so a tangent
is the launch's own result for the tangent: equal, not near."""

import pytest
import torch
from torch.autograd import forward_ad

from polarquant_kv import rotary

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_forward_mode_tangents(dtype):
    g = torch.Generator(device=DEV).manual_seed(4)
    q, k, tq, tk = (torch.randn(2, 33, h, 64, generator=g, device=DEV).to(dtype).transpose(1, 2) for h in (6, 2, 6, 2))
    pos, f = torch.arange(90, 123, device=DEV), rotary.rotary_frequencies(48)[0].to(DEV)
    how = dict(interleaved=True, amplitude=1.25)
    y, t = rotary.apply_rotary(q, k, pos, f, **how), rotary.apply_rotary(tq, tk, pos, f, **how)
    with forward_ad.dual_level():
        dq, dk = forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk)
        both = [forward_ad.unpack_dual(x) for x in rotary.apply_rotary(dq, dk, pos, f, **how)]
        for i in range(2):
            assert torch.equal(both[i].primal, y[i]) and torch.equal(both[i].tangent, t[i])
        one = [forward_ad.unpack_dual(x) for x in rotary.apply_rotary(q, dk, pos, f, **how)]
        assert one[0].tangent is None or not one[0].tangent.any()
        assert torch.equal(one[1].tangent, t[1])


def test_embedding_used_in_inference_mode_first():
    emb = rotary.RotaryEmbedding(64)
    q, pos = torch.randn(1, 2, 9, 64, device=DEV), torch.arange(9, device=DEV)
    with torch.inference_mode():
        y = emb(q, None, pos)[0].clone()
    q1 = q.clone().requires_grad_(True)
    out = emb(q1, None, pos)[0]
    assert torch.equal(out, y)
    g, = torch.autograd.grad(out, q1, y)
    assert torch.allclose(g, q, atol=1e-5)                      # turned and turned back


def test_first_call_in_a_capture_is_refused(monkeypatch):
    emb = rotary.RotaryEmbedding(64)
    q, pos = torch.randn(1, 2, 9, 64, device=DEV), torch.arange(9, device=DEV)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before a capture"):
        emb(q, None, pos)
    monkeypatch.undo()
    emb(q, None, pos)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    emb(q, None, pos)
