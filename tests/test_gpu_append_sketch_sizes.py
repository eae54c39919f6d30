"""Signs of projections of any size: multiplied by a power of two, a sketch gives the
signs that it gave (test_gpu_append's tolerance counts in its own units)."""

import pytest
import torch

import test_gpu_append as append_tests
from polarquant_kv import append

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("power", [-60, -20, -7, 6, 9, 30, 90])
@pytest.mark.parametrize("d,T,bits,dtype", [(64, 40, 4, torch.float32), (128, 3, 2, torch.float16), (128, 40, 4, torch.bfloat16)])
def test_a_sketch_of_any_size(d, T, bits, dtype, power):
    case = (2, 1, 2, T, T, d, d, bits, True, 0, dtype, False, None, 0, None)
    q, k, v, keys, values, R, P, positions, freqs, _ = append_tests.make(case)
    P = P * 2.0 ** power
    P[5] *= 2.0 ** 12                     # a row of its own size
    P[7] = 0.0
    append.append_rotary(k, v, keys, values, R, positions, freqs, starts=0, jl_rot=P)
    e = append_tests.check_vectors(keys.blocks, append_tests.turned(k, positions, freqs, None, False, 1.0), R, keys.codebooks, bits)
    bits_ = ((keys.qjl_signs[..., None].int() >> torch.arange(8, device=DEV).int()) & 1).flatten(-2)
    assert bool((bits_[..., 7] == 1).all())                 # a projection of 0 counts as positive
    rows = [i for i in range(d) if i != 7]
    pe = e @ P[rows].double().t()
    unsure = pe.abs() <= P[rows].double().abs().sum(-1) * append_tests.OFF
    assert bool(((bits_[..., rows] == (pe >= 0)) | unsure).all())
    assert float(unsure.double().mean()) < 0.01
