"""Attention weights where they can go wrong: queries at any address, numbers that
are not finite, chunks in several passes, workspaces of the least size. Bounds as
derived in test_gpu_weights."""

import pytest
import torch

from polarquant_kv import _lib, attention

from test_gpu_evict import paged_copy
from test_gpu_weights import close, decoded, exact, make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("d,qjl", [(64, False), (128, False), (128, True)])
def test_queries_off_a_16_byte_boundary(dtype, d, qjl):
    q, kc, _, R, jl = make(1, 6, 2, 300, d, 4, qjl, Sq=70)
    q = q.to(dtype)
    want, tol, _ = exact(q, kc, R, 230, jl_rot=jl)
    at_home = attention.attention_weights(q, kc, R, 230, jl_rot=jl)
    close(at_home, want, tol)
    for off in (1, 2, 3, 5):
        room = torch.full((q.numel() + 8,), 7.0, dtype=dtype, device=DEV)
        moved = room[off:off + q.numel()].view_as(q)
        moved.copy_(q)
        assert moved.data_ptr() % 16 != 0 and moved.is_contiguous()
        assert torch.equal(attention.attention_weights(moved, kc, R, 230, jl_rot=jl), at_home)
