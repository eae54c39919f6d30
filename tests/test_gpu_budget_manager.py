"""KVCacheManager with tracked weights on the GPU: what outlives a call."""

import pytest
import torch

from polarquant_kv.inference import KVCacheManager, PolarQuantConfig

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_calls_in_different_modes_equal_calls_in_one():
    B, Hq, H, D = 1, 4, 2, 64
    g = torch.Generator(device=DEV).manual_seed(8)
    steps = [[torch.randn(B, n, T, D, generator=g, device=DEV).half() for n in (H, H, Hq)] for T in (90, 1, 70, 1, 40, 1)]
    runs = []
    for modes in ((torch.no_grad,) * 6, (torch.inference_mode, torch.no_grad) * 3, (torch.enable_grad, torch.inference_mode) * 3):
        m = KVCacheManager(PolarQuantConfig(), 400, B, H, D, DEV, page_tokens=64, track_weights=True)
        out = []
        for (k, v, q), mode in zip(steps, modes):
            with mode():
                m.append(k, v)
                out.append(m.attend(q).clone())
                m.evict(100, 4, 16)
        runs.append(out + [m.weights.clone(), m.positions.clone()])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
