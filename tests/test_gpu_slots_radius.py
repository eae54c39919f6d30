"""pqkv_dequantize_slots against pqkv_dequantize with R = I on vectors whose
blocks hold different radii: a vector's radius is its first block's, for every
reader of a cache."""

import pytest
import torch

import window_ref
from polarquant_kv import quantizer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("d,bits", [(64, 4), (64, 2), (128, 4), (128, 2)])
def test_the_first_radius_of_a_vector(d, bits, page):
    B, H, S = 2, 3, 150
    g = torch.Generator(device=DEV).manual_seed(4)
    if page:
        cache = quantizer.allocate_paged_cache(B, H, d, bits, DEV, page_tokens=page)
        cache.ensure(S)
        parts = cache.groups
    else:
        cache = quantizer.allocate_cache(B, H, S, d, bits, DEV)
        parts = [cache.blocks]
    for x in parts:
        x.random_(0, 256, generator=g)
        for j in range(d // 32):                    # finite radii, a block's own
            at = j * window_ref.BLOCK_BYTES[bits] + 1
            x[..., at] = x[..., at] % 0x78
    cache.seq_len = S
    blocks = window_ref.rows_of(cache)[0][:, :, :S].contiguous()
    assert not torch.equal(blocks[..., :2], blocks[..., window_ref.BLOCK_BYTES[bits]:][..., :2])
    # a product of two numbers of 11 and 24 bits in 32 bits: half a step
    want = window_ref.states(blocks, cache.codebooks[:1 << bits], bits)
    got = quantizer.dequantize(cache, None, torch.float32)
    assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -24 + 2.0 ** -149).all())
    assert torch.equal(got, quantizer.dequantize(cache, torch.eye(d, device=DEV), torch.float32))


@pytest.mark.parametrize("H", [1, 3])
def test_blocks_longer_than_the_cache_says(H):
    """Streams lie where the blocks have them, also where max_seq_len is less than their length."""
    B, S, d = 2, 40, 64
    g = torch.Generator(device=DEV).manual_seed(6)
    cache = quantizer.compress_pq(torch.randn(B, H, S, d, generator=g, device=DEV), torch.eye(d, device=DEV), 4)
    whole = quantizer.dequantize(cache, None, torch.float32)
    cache.max_seq_len = cache.seq_len = 25
    assert torch.equal(quantizer.dequantize(cache, None, torch.float32), whole[:, :, :25])
    assert torch.equal(quantizer.dequantize(cache, torch.eye(d, device=DEV), torch.float32), whole[:, :, :25])
    cache.blocks = cache.blocks.transpose(0, 1).contiguous().transpose(0, 1)    # (H = 1: dense, with strides of its own)
    assert torch.equal(quantizer.dequantize(cache, None, torch.float32), whole[:, :, :25])
