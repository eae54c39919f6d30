"""Rotary positions on several axes without a GPU: the pairs' axes, and what the
C entry point refuses."""

import ctypes

import pytest
import torch

from polarquant_kv import _lib, rotary


def test_axis_of_pairs():
    assert rotary.axis_of_pairs([2, 1, 3]) == (0, 0, 1, 2, 2, 2)
    assert rotary.axis_of_pairs((4,)) == (0,) * 4 and rotary.axis_of_pairs((4,), True) == (0,) * 4
    assert rotary.axis_of_pairs((2, 2, 2), True) == (0, 1, 2) * 2
    assert rotary.axis_of_pairs((5, 2, 1), True) == (0, 1, 2, 0, 1, 0, 0, 0)
    for s in ((24, 20, 20), (16, 24, 24)):
        assert [rotary.axis_of_pairs(s).count(a) for a in range(3)] == list(s)
    assert [rotary.axis_of_pairs((24, 20, 20), True).count(a) for a in range(3)] == [24, 20, 20]
    for bad, spread in (([], False), ([0, 0], False), ([3, -1], False), ([1, 3], True), ([2, 2, 4], True), ([1] * 257, False)):
        with pytest.raises(ValueError, match="sections"):
            rotary.axis_of_pairs(bad, spread)


def test_embedding_sections():
    e = rotary.RotaryEmbedding(64, 48, sections=(8, 8, 8))
    assert e.axes == rotary.axis_of_pairs((8, 8, 8)) and e.n_axes == 3
    assert e.positions_by_axis(torch.arange(4)).shape == (3, 4)
    assert rotary.RotaryEmbedding(64).positions_by_axis(torch.arange(4)).shape == (4,)
    with pytest.raises(ValueError, match="pairs"):
        rotary.RotaryEmbedding(64, sections=(8, 8))


def c_call(axes=bytes(8), n_axes=2, by_axis=5, rot=16, **over):
    a = dict(dtype=_lib.F16, d=16, T=5, B=1)
    a.update(over)
    strides = (ctypes.c_int64 * 3)(80, 80, 16)
    return _lib.lib().pqkv_rotary_axes(16, strides, 16, 1, None, None, None, 0, a["dtype"], 16, by_axis, 5, n_axes, axes,
                                       16, a["B"], a["T"], a["d"], rot, 0, 1.0, 0, None)


@pytest.mark.parametrize("over,status", [
    (dict(axes=None), _lib.ERR_INVALID), (dict(n_axes=0), _lib.ERR_INVALID), (dict(n_axes=257), _lib.ERR_INVALID),
    (dict(by_axis=-1), _lib.ERR_INVALID), (dict(axes=bytes([0] * 7 + [2])), _lib.ERR_INVALID),
    (dict(rot=0), _lib.ERR_INVALID), (dict(rot=2048, axes=bytes(1024)), _lib.ERR_INVALID),
    (dict(rot=18, axes=bytes(9)), _lib.ERR_UNSUPPORTED), (dict(dtype=3), _lib.ERR_UNSUPPORTED),
    (dict(B=-1), _lib.ERR_INVALID),
])
def test_refused_before_any_launch(over, status):
    assert c_call(**over) == status
    assert _lib.lib().pqkv_last_error().startswith(b"rotary_axes")


def test_nothing_to_do():
    assert c_call(T=0) == _lib.OK
