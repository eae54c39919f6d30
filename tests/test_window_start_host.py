"""The first row's position at the ends of its type, refused before any launch."""

import pytest

from polarquant_kv import _lib
from test_window_host import c_call


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("Sq", [0, 1, 7])
@pytest.mark.parametrize("start", [2 ** 63 - 1, 2 ** 63 - 7, -2 ** 63, 101])
def test_refused(start, Sq, paged):
    assert c_call(paged, start=start, Sq=Sq) == _lib.ERR_INVALID
    assert b"not all in the cache" in _lib.lib().pqkv_last_error()
