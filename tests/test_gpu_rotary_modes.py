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
