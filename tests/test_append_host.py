"""Appending with the rotation on the way, without a GPU: what the C entry points
refuse before any launch."""

import ctypes

import pytest

from polarquant_kv import _lib

ST = (ctypes.c_int64 * 3)(640, 320, 64)


def c_call(paged=False, **over):
    a = dict(k=16, ks=ST, v=16, vs=ST, q=None, qs=None, qo=None, Hq=0, dtype=_lib.F16, pos=16, by_axis=0, by_row=5,
             n_axes=1, axes=None, freqs=16, rot=64, inter=0, amplitude=1.0, R=16, kcb=16, vcb=16, n_bits=4, p_rot=None,
             m=0, B=2, Hkv=2, T=5, d=64, start=95, starts=None, counts=None, S=100)
    a.update({n: x for n, x in over.items() if n in a})
    tail = [over.get("kb", 16), over.get("vb", 16)]
    if paged:
        tail += [over.get("page_tokens", 64), over.get("max_pages", 2)]
    fn = _lib.lib().pqkv_append_rotary_paged if paged else _lib.lib().pqkv_append_rotary
    return fn(*a.values(), *tail, over.get("signs"), None)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("over,status", [
    (dict(B=-1), _lib.ERR_INVALID), (dict(T=-1), _lib.ERR_INVALID), (dict(Hq=-1), _lib.ERR_INVALID),
    (dict(d=96), _lib.ERR_UNSUPPORTED), (dict(rot=66), _lib.ERR_UNSUPPORTED), (dict(rot=3), _lib.ERR_UNSUPPORTED),
    (dict(dtype=3), _lib.ERR_UNSUPPORTED), (dict(n_bits=3), _lib.ERR_UNSUPPORTED),
    (dict(amplitude=float("nan")), _lib.ERR_INVALID), (dict(p_rot=16, m=64), _lib.ERR_INVALID),
    (dict(signs=16), _lib.ERR_INVALID), (dict(signs=16, p_rot=16, m=32), _lib.ERR_UNSUPPORTED),
    (dict(start=96), _lib.ERR_INVALID), (dict(start=-1), _lib.ERR_INVALID), (dict(start=2 ** 62), _lib.ERR_INVALID),
    (dict(start=-2 ** 63), _lib.ERR_INVALID), (dict(axes=bytes(32), n_axes=0), _lib.ERR_INVALID),
    (dict(axes=bytes([1] * 32)), _lib.ERR_INVALID), (dict(axes=bytes(32), by_axis=-1), _lib.ERR_INVALID),
    (dict(by_row=-1), _lib.ERR_INVALID), (dict(pos=None), _lib.ERR_INVALID), (dict(freqs=None), _lib.ERR_INVALID),
    (dict(Hq=1), _lib.ERR_INVALID), (dict(pos=12), _lib.ERR_INVALID), (dict(starts=12), _lib.ERR_INVALID),
    (dict(counts=12), _lib.ERR_INVALID), (dict(k=17), _lib.ERR_INVALID), (dict(k=None), _lib.ERR_INVALID),
    (dict(vs=None), _lib.ERR_INVALID), (dict(R=None), _lib.ERR_INVALID), (dict(R=18), _lib.ERR_INVALID),
    (dict(kcb=None), _lib.ERR_INVALID), (dict(kb=None), _lib.ERR_INVALID),
    (dict(B=1 << 20, T=1 << 10, starts=16), _lib.ERR_UNSUPPORTED),
])
def test_refused_before_any_launch(over, status, paged):
    assert c_call(paged, **over) == status
    assert _lib.lib().pqkv_last_error().startswith(b"append_rotary")


def test_pages_and_nothing_to_do():
    assert c_call(True, page_tokens=96) == _lib.ERR_INVALID and c_call(True, max_pages=1) == _lib.ERR_INVALID
    assert c_call(kb=17) == _lib.ERR_INVALID and c_call(signs=18, p_rot=16, m=64) == _lib.ERR_INVALID
    for paged in (False, True):
        assert c_call(paged, B=0) == _lib.OK and c_call(paged, T=0, start=100) == _lib.OK
        assert c_call(paged, Hkv=0, k=None) == _lib.OK
