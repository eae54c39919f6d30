"""append_rotary with more items than compute units, so that workgroups go from one
item to the next (two tables of sines and slots in turn, positions an item ahead, a
barrier between them), and several segments of 16 tokens to an item; slots read
back with more vectors than one round of its workgroups. The formula and its
tolerances are test_gpu_append's."""

import random

import pytest
import torch

import test_gpu_append as append_tests
import window_ref
from polarquant_kv import quantizer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def some(n, lo, hi, seed):
    r = random.Random(seed)
    return [r.randint(lo, hi) for _ in range(n)]


# as test_gpu_append.CASES; an item has 32 rows at d = 128, 16 with signs, 64 at d = 64
CASES = {
    "runs": (3, 1, 2, 20003, 21000, 128, 128, 4, False, 1024, torch.bfloat16, False, (16, 24, 24), [997, 0, 5], [20003, 17, 19000]),
    "runs_contiguous": (2, 1, 2, 20000, 20000, 128, 96, 2, False, 0, torch.float16, True, None, 0, None),
    "runs_fp32": (2, 1, 3, 9001, 9100, 128, 128, 4, False, 0, torch.float32, False, None, [99, 3], [9001, 8000]),
    "runs_signs": (2, 1, 2, 6005, 6100, 128, 128, 2, True, 256, torch.float16, False, None, [95, 0], [6005, 5000]),
    "runs_64": (2, 1, 2, 20007, 20010, 64, 48, 4, False, 0, torch.float32, True, (12, 12), [3, 1], [20007, 12345]),
    "runs_64_signs": (1, 1, 3, 20001, 20001, 64, 64, 4, True, 64, torch.bfloat16, False, None, 0, None),
    "odd_pairs": (1, 1, 3, 9001, 9001, 128, 42, 4, False, 0, torch.float16, False, None, 0, None),
    "five_tokens": (6000, 1, 3, 5, 16, 128, 128, 4, False, 0, torch.float16, False, None, some(6000, -3, 17, 1), some(6000, 0, 5, 2)),
    "one_token": (20000, 2, 1, 1, 4, 128, 128, 2, False, 0, torch.bfloat16, True, None, some(20000, 0, 4, 3), None),
    "three_tokens_signs": (7000, 1, 2, 3, 7, 64, 64, 4, True, 0, torch.float16, False, (20, 12), some(7000, 0, 5, 4), some(7000, 0, 3, 5)),
}


@pytest.mark.parametrize("name", CASES)
def test_slots_hold_the_turned_vectors(name):
    B, Hq, Hkv, T, S, d, rot, bits, qjl, page, dtype, inter, sections, starts, counts = CASES[name]
    if isinstance(starts, list):
        # tokens whose slot there is no room for count as not there
        n = [T] * B if counts is None else list(counts)
        n = [min(c, S - s) if 0 <= s < S else 0 for c, s in zip(n, starts)]
        starts = [s if 0 <= s < S else (-1 if s < 0 else S) for s in starts]
        counts = n
    case = (B, Hq, Hkv, T, S, d, rot, bits, qjl, page, dtype, inter, sections, starts, counts)
    append_tests.test_slots_hold_the_turned_vectors(case)


@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("d,bits", [(128, 4), (64, 2)])
def test_many_slots_read_back(d, bits, page):
    B, H, S = 1, 3, 100003 if d == 64 else 50001
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(B, H, S, d, generator=g, device=DEV).half()
    R = torch.eye(d, device=DEV)
    cache = quantizer.allocate_paged_cache(B, H, d, bits, DEV, page_tokens=page) if page else None
    cache = quantizer.compress_pq(x, R, bits, cache=cache)
    for n in (S, S - 7):
        blocks = window_ref.rows_of(cache)[0][:, :, :n].contiguous()
        want = window_ref.states(blocks, cache.codebooks[:1 << bits], bits)
        got = quantizer.dequantize(cache, None, torch.float32, n)
        assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -24).all())
        half = quantizer.dequantize(cache, None, torch.float16, n)
        assert torch.equal(half, got.half())
