"""Selection at the border of every number of keys that a thread holds."""

import numpy as np
import pytest
import torch

from polarquant_kv import eviction

from test_gpu_evict import DEV, laws, want_kept

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("steps", [2, 4, 8, 12, 16, 20, 24, 28, 32, 48, 64])
def test_select_at_the_border_of_a_step(steps):
    for S in (1024 * steps - 1, 1024 * steps, 1024 * steps + 1):
        for name, w in laws(2, S, steps):
            if name in ("ties", "odd"):
                for keep in (1, S // 3, S - 1, S):
                    got = eviction.select_positions(torch.from_numpy(w).to(DEV).view(1, 2, S), keep)[0].cpu().numpy()
                    assert np.array_equal(got, want_kept(w, keep, 0, 0)), (name, S, keep)
