"""Attention behind a window without a GPU: what the C entry points and the
Python call refuse before any launch."""

import pytest
import torch

from polarquant_kv import _lib, attention
from polarquant_kv.types import PagedPQCache, PQCache

D = 64


def c_call(paged=False, **over):
    a = dict(q=16, q_dtype=_lib.F16, R=16, k=16, v=16, kcb=16, vcb=16, n_bits=4, qjl=None, p_rot=None, m=0, B=2, Hq=8,
             Hkv=2, Sq=1, start=99, starts=None, counts=None, window=10, sinks=0, S=100, d=64, scale=0.1, out=16,
             out_dtype=_lib.F32, ws=16, ws_bytes=1 << 40)
    a.update(over)
    head = [a[n] for n in ("q", "q_dtype", "R", "k", "v")]
    if paged:
        head += [over.get("page_tokens", 64), over.get("max_pages", 2)]
    fn = _lib.lib().pqkv_window_attn_paged if paged else _lib.lib().pqkv_window_attn
    rest = ("kcb", "vcb", "n_bits", "qjl", "p_rot", "m", "B", "Hq", "Hkv", "Sq", "start", "starts", "counts", "window",
            "sinks", "S", "d", "scale", "out", "out_dtype", "ws", "ws_bytes")
    return fn(*head, *[a[n] for n in rest], None)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("over,status", [
    (dict(B=0), _lib.ERR_INVALID), (dict(Hq=7), _lib.ERR_INVALID), (dict(Sq=-1), _lib.ERR_INVALID),
    (dict(window=0), _lib.ERR_INVALID), (dict(sinks=-1), _lib.ERR_INVALID), (dict(S=-1), _lib.ERR_INVALID),
    (dict(start=100), _lib.ERR_INVALID), (dict(start=-1), _lib.ERR_INVALID), (dict(start=90, Sq=11), _lib.ERR_INVALID),
    (dict(start=2 ** 62), _lib.ERR_INVALID),
    (dict(d=96), _lib.ERR_UNSUPPORTED), (dict(n_bits=3), _lib.ERR_UNSUPPORTED), (dict(q_dtype=2), _lib.ERR_UNSUPPORTED),
    (dict(out_dtype=2), _lib.ERR_UNSUPPORTED), (dict(p_rot=16, m=64), _lib.ERR_INVALID),
    (dict(qjl=16, p_rot=16, m=32), _lib.ERR_UNSUPPORTED), (dict(scale=0.0), _lib.ERR_INVALID),
    (dict(scale=float("inf")), _lib.ERR_INVALID), (dict(q=None), _lib.ERR_INVALID), (dict(out=None), _lib.ERR_INVALID),
    (dict(R=20), _lib.ERR_INVALID), (dict(k=None), _lib.ERR_INVALID), (dict(vcb=None), _lib.ERR_INVALID),
    (dict(starts=12), _lib.ERR_INVALID), (dict(counts=12), _lib.ERR_INVALID), (dict(ws=None), _lib.ERR_WORKSPACE),
    (dict(ws_bytes=1000), _lib.ERR_WORKSPACE), (dict(ws=24), _lib.ERR_INVALID),
    (dict(B=40000), _lib.ERR_UNSUPPORTED), (dict(Sq=2, start=0, Hq=600), _lib.ERR_UNSUPPORTED),
    (dict(Sq=2, start=0, Hq=260, qjl=16, p_rot=16, m=64), _lib.ERR_UNSUPPORTED),
])
def test_refused_before_any_launch(over, status, paged):
    assert c_call(paged, **over) == status
    assert _lib.lib().pqkv_last_error().startswith(b"window_attn")


def test_pages_and_lengths():
    assert c_call(True, page_tokens=96) == _lib.ERR_INVALID
    assert c_call(True, max_pages=1) == _lib.ERR_INVALID
    assert c_call(S=1 << 24, starts=16) == _lib.ERR_UNSUPPORTED
    assert c_call(Sq=0, q=None) == _lib.OK and c_call(Sq=0, start=100, out=None) == _lib.OK


def test_workspace():
    L = _lib.lib()
    f = L.pqkv_window_attn_workspace_bytes
    assert f(0, 8, 2, 1, 100, 64, 10, 0, 0) == 0 and f(1, 8, 2, 1, 100, 64, 0, 0, 0) == 0 and f(1, 7, 2, 1, 100, 64, 9, 0, 0) == 0
    # a window's workspace does not grow with the cache
    assert f(8, 32, 8, 1, 1 << 20, 128, 4096, 4, 0) == f(8, 32, 8, 1, 1 << 23, 128, 4096, 4, 0)
    assert f(1, 8, 2, 1, 1 << 20, 64, 2 ** 31 - 1, 2 ** 31 - 1, 0) >= 4 * 8 * 64
    for Sq in (2, 1000):
        assert f(2, 8, 2, Sq, 5000, 64, 100, 4, 0) > 0 and f(2, 8, 2, Sq, 5000, 64, 100, 4, 1) > 0
    # few rows behind a long window are split: partials; many are not
    assert f(1, 8, 2, 8, 9000, 64, 8000, 4, 0) > 4 * 8 * 8 * 64 > 256 == f(8, 32, 8, 4000, 9000, 64, 8000, 4, 0)


def caches(paged, bits=4, **more):
    out = []
    for _ in range(2):
        if paged:
            c = PagedPQCache(1, 2, D, bits, torch.zeros(16), "cpu", 64)
            c.ensure(8)
            c.seq_len = 8
        else:
            c = PQCache(blocks=torch.zeros(1, 2, 8, 36 if bits == 4 else 20, dtype=torch.uint8), head_dim=D, n_bits=bits,
                        seq_len=8, max_seq_len=8, codebooks=torch.zeros(16))
        out.append(c)
    return out


@pytest.mark.parametrize("paged", [False, True])
def test_python_refuses(paged):
    kc, vc = caches(paged)
    q, R = torch.zeros(1, 4, 1, D), torch.eye(D)
    call = lambda window=3, query=q, k=kc, v=vc, **kw: attention.window_attention(query, k, v, R, window, **kw)  # noqa: E731
    for kw, words in ((dict(query=q[0]), "must be"), (dict(window=0), "at least 1"), (dict(window=2.5), "at least 1"),
                      (dict(sinks=-1), "at least"), (dict(query=torch.zeros(1, 3, 1, D)), "multiple"),
                      (dict(query=torch.zeros(2, 4, 1, D)), "batch"), (dict(v=caches(paged, 2)[1]), "width"),
                      (dict(jl_rot=torch.eye(D)), "no signs"), (dict(), "device tensors")):
        with pytest.raises(ValueError, match=words):
            call(**kw)


def test_starts_and_counts():
    dev = torch.device("cpu")
    assert attention.row_starts(5, 1, 2, dev) == (5, None)
    start, t = attention.row_starts(torch.tensor([3, 4], dtype=torch.int32), 1, 2, dev)
    assert start == 0 and t.dtype == torch.int64 and t.tolist() == [3, 4]
    for bad in (torch.tensor([3]), torch.tensor([1.0, 2.0]), torch.tensor([True, False]), torch.zeros(2, 2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="starts"):
            attention.row_starts(bad, 1, 2, dev)
        with pytest.raises(ValueError, match="counts"):
            attention.row_counts(bad, 2, dev)
    assert attention.row_counts(None, 2, dev) is None
    with pytest.raises(ValueError, match="counts"):
        attention.row_counts(3, 2, dev)
    for f in (lambda: attention.row_starts(torch.tensor([1, 2]), 1, 2, torch.device("cuda:0")),
              lambda: attention.row_counts(torch.tensor([1, 2]), 2, torch.device("cuda:0"))):
        with pytest.raises(ValueError, match="are on cpu"):
            f()
