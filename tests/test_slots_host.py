"""Which caches are read back as they lie, without a GPU."""

import torch

from polarquant_kv import quantizer
from polarquant_kv.types import PQCache


def test_blocks_at_an_odd_address_take_the_other_way():
    bytes_ = torch.zeros(2 * 8 * 36 + 1, dtype=torch.uint8)
    for first, lies in ((0, True), (1, False)):
        blocks = bytes_[first:first + 2 * 8 * 36].view(1, 2, 8, 36)
        assert (blocks.data_ptr() % 2 == 0) == lies
        cache = PQCache(blocks=blocks, head_dim=64, n_bits=4, seq_len=8, max_seq_len=8, codebooks=torch.zeros(16))
        assert quantizer._lies_in_rows(cache) == lies
