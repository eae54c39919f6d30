"""The first row's position at the ends of its type, refused before any launch."""

import pytest
import torch

from polarquant_kv import _lib, attention
from test_window_host import c_call


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("Sq", [0, 1, 7])
@pytest.mark.parametrize("start", [2 ** 63 - 1, 2 ** 63 - 7, -2 ** 63, 101])
def test_refused(start, Sq, paged):
    assert c_call(paged, start=start, Sq=Sq) == _lib.ERR_INVALID
    assert b"not all in the cache" in _lib.lib().pqkv_last_error()


def test_a_start_that_is_no_whole_number():
    dev = torch.device("cpu")
    assert attention.row_starts(5.0, 1, 2, dev) == (5, None)
    for bad in (2.5, -0.5):
        with pytest.raises(ValueError, match="whole number"):
            attention.row_starts(bad, 1, 2, dev)
