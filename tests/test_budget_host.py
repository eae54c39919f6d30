"""A cache under a budget and rotary positions, without a GPU: what the C entry
points and the Python calls refuse before any launch, and the frequencies."""

import ctypes
import math

import pytest
import torch

from polarquant_kv import _lib, attention, eviction, rotary
from polarquant_kv.types import PagedPQCache, PQCache

FAKE = 0x1000  # never dereferenced: every call below fails validation first
INV, UNS, WS = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED, _lib.ERR_WORKSPACE


def _status(rc, expect):
    assert rc == expect, (rc, _lib.lib().pqkv_last_error())
    assert _lib.lib().pqkv_last_error()


def _decode(**kw):
    a = dict(q=FAKE, qt=1, R=FAKE, k=FAKE, v=FAKE, kcb=FAKE, vcb=FAKE, bits=4, qjl=None, p=None, m=0, B=1, Hq=8, Hkv=2,
             S=16, S_max=16, d=128, scale=0.088, out=FAKE, ot=1, wi=None, wis=0, wo=FAKE, wos=16, ws=FAKE,
             wsb=1 << 24)
    a.update(kw)
    return _lib.lib().pqkv_decode_attn_weights(*a.values(), None)


@pytest.mark.parametrize("kw,expect", [
    (dict(wo=None), INV), (dict(wos=15), INV), (dict(wi=0x9000, wis=15), INV), (dict(wo=FAKE + 2), INV),
    (dict(wi=FAKE + 16, wis=16), INV),                      # overlaps weights_out without being it
    (dict(wi=FAKE, wis=17, wos=16, B=2), INV),              # the same start, other rows
    (dict(ws=None), WS), (dict(wsb=64), WS), (dict(ws=FAKE + 4), INV),
    (dict(bits=3), UNS), (dict(d=96), UNS), (dict(Hq=7), INV), (dict(scale=0.0), INV), (dict(S=17), INV),
    (dict(B=0), INV), (dict(S=-1), INV), (dict(S=1 << 24, S_max=1 << 24, wos=1 << 24), UNS),
    (dict(Hq=2050, Hkv=2), UNS), (dict(qjl=FAKE), INV), (dict(qjl=FAKE, p=FAKE, m=64), UNS), (dict(q=None), INV),
    (dict(R=FAKE + 4), INV), (dict(qt=2), UNS)])
def test_decode_weights_refusals(kw, expect):
    _status(_decode(**kw), expect)


def test_decode_weights_workspace_covers_the_logits():
    L = _lib.lib()
    base, more = L.pqkv_decode_workspace_bytes(2, 8, 2, 1000, 128), \
        L.pqkv_decode_attn_weights_workspace_bytes(2, 8, 2, 1000, 128)
    assert more >= base + 2 * 8 * 1024 * 4
    assert L.pqkv_decode_attn_weights_workspace_bytes(0, 8, 2, 1000, 128) == 0


def _weights(**kw):
    a = dict(q=FAKE, qt=1, R=FAKE, k=FAKE, cb=FAKE, bits=4, qjl=None, p=None, m=0, B=1, Hq=8, Hkv=2, Sq=4, q_start=12,
             S=16, S_max=16, d=128, scale=0.088, causal=1, wi=None, wis=0, wo=FAKE, wos=16, ws=FAKE, wsb=1 << 24)
    a.update(kw)
    return _lib.lib().pqkv_attn_weights(*a.values(), None)


@pytest.mark.parametrize("kw,expect", [
    (dict(q_start=13), INV),                                # the last query is past the cache
    (dict(q_start=-1), INV), (dict(Sq=-1), INV), (dict(S=17), INV), (dict(Hq=7), INV), (dict(d=96), UNS),
    (dict(bits=3), UNS), (dict(qt=2), UNS), (dict(wo=None), INV), (dict(wos=15), INV), (dict(wi=FAKE + 4, wis=16), INV),
    (dict(ws=None), WS), (dict(wsb=256), WS), (dict(ws=FAKE + 8), INV), (dict(q=None), INV), (dict(k=None), INV),
    (dict(cb=None), INV), (dict(scale=math.nan), INV), (dict(qjl=FAKE), INV), (dict(p=FAKE, m=128), INV),
    (dict(qjl=FAKE, p=FAKE, m=64), UNS), (dict(R=FAKE + 8), INV), (dict(Hq=2050, Hkv=2), UNS)])
def test_attn_weights_refusals(kw, expect):
    _status(_weights(**kw), expect)


def test_attn_weights_nothing_to_do():
    assert _weights(S=0, S_max=0, q_start=0, Sq=0, wo=None) == 0
    assert _weights(Sq=0, wi=FAKE, wis=16) == 0              # in place: the weights stay as they are
    assert _lib.lib().pqkv_attn_weights_workspace_bytes(1, 8, 3, 4, 16, 128, 0) == 0
    # the partials of a long chunk over a long cache stay bounded
    for qjl in (0, 1):
        n = _lib.lib().pqkv_attn_weights_workspace_bytes(8, 32, 8, 8192, 131072, 128, qjl)
        assert n < (1 << 30) + (1 + qjl) * 8 * 32 * 8192 * 128 * 4


def test_paged_calls_check_the_table():
    L = _lib.lib()
    args = [FAKE, 1, FAKE, FAKE, 64, 1, FAKE, 4, None, None, 0, 1, 8, 2, 4, 96, 100, 128, 0.1, 1, None, 0, FAKE, 100,
            FAKE, 1 << 24, None]
    _status(L.pqkv_attn_weights_paged(*args), INV)           # 100 positions, one page of 64
    args[4] = 100
    _status(L.pqkv_attn_weights_paged(*args), INV)           # not a power of two
    args = [FAKE, 1, FAKE, FAKE, FAKE, 64, 1, FAKE, FAKE, 4, None, None, 0, 1, 8, 2, 100, 128, 0.1, FAKE, 1, None, 0,
            FAKE, 100, FAKE, 1 << 24, None]
    _status(L.pqkv_decode_attn_weights_paged(*args), INV)


def test_select_refusals():
    L = _lib.lib()

    def call(w=FAKE, ws=100, n=2, S=100, keep=50, sink=4, recent=10, kept=FAKE):
        return L.pqkv_evict_select(w, ws, n, S, keep, sink, recent, kept, None)

    for kw in (dict(keep=13), dict(keep=101), dict(sink=-1), dict(recent=-1), dict(ws=99), dict(w=None), dict(kept=None),
               dict(n=-1), dict(S=-1, keep=0), dict(w=FAKE + 2), dict(kept=FAKE + 1)):
        _status(call(**kw), INV)
    assert call(n=0) == 0
    assert call(S=0, keep=0) == 0 and call(sink=0, recent=0, keep=0) == 0


def test_gather_refusals():
    L = _lib.lib()
    R = _lib.RowArray

    def call(src=R(FAKE, None, 7200, 0, 0), dst=R(FAKE, None, 3600, 0, 0), size=72, n=1, streams=2, S=100, keep=50,
             fill=50, kept=FAKE):
        return L.pqkv_gather_rows(n, ctypes.byref(src), ctypes.byref(dst), _lib.int_array([size]), kept, streams, S,
                                  keep, fill, None)

    for kw, expect in ((dict(fill=49), INV), (dict(kept=None), INV), (dict(size=70), UNS), (dict(size=0), UNS),
                       (dict(src=R(FAKE, None, 7196, 0, 0)), INV), (dict(dst=R(FAKE, None, 3596, 0, 0)), INV),
                       (dict(src=R(FAKE + 2, None, 7200, 0, 0)), INV), (dict(src=R(None, None, 7200, 0, 0)), INV),
                       (dict(src=R(None, FAKE, 0, 64, 1)), INV),     # 100 positions, one page of 64
                       (dict(dst=R(None, FAKE, 0, 64, 1), fill=65), INV),
                       (dict(dst=R(FAKE, FAKE, 4604, 64, 1)), INV), (dict(dst=R(FAKE + 8, FAKE, 4608, 64, 1)), INV),
                       (dict(dst=R(FAKE, FAKE, 4608 - 16, 64, 1)), INV), (dict(n=7), INV), (dict(n=-1), INV),
                       (dict(streams=-1), INV), (dict(S=-1), INV), (dict(streams=1 << 40), UNS)):
        _status(call(**kw), expect)
    assert call(n=0) == 0 and call(streams=0) == 0 and call(keep=0, fill=0) == 0


def _rot(**kw):
    st = (ctypes.c_int64 * 3)(1024, 128, 128)
    a = dict(q=FAKE, qs=st, qo=FAKE, Hq=8, k=FAKE, ks=st, ko=FAKE, Hkv=2, dt=1, pos=FAKE, ps=0, f=FAKE, B=1, T=1, d=128,
             rot=128, inter=0, amp=1.0, inv=0)
    a.update(kw)
    return _lib.lib().pqkv_rotary(*a.values(), None)


@pytest.mark.parametrize("kw,expect", [
    (dict(rot=127), UNS), (dict(rot=130), UNS), (dict(rot=0), UNS), (dict(d=1026, rot=2), UNS), (dict(dt=3), UNS),
    (dict(amp=math.inf), INV), (dict(q=None), INV), (dict(ko=None), INV), (dict(pos=None), INV), (dict(f=None), INV),
    (dict(B=-1), INV), (dict(Hkv=-1), INV), (dict(q=FAKE + 1), INV), (dict(pos=FAKE + 4), INV), (dict(ps=-1), INV),
    (dict(qs=None), INV), (dict(Hq=65535), UNS)])
def test_rotary_refusals(kw, expect):
    _status(_rot(**kw), expect)


def test_rotary_nothing_to_do():
    assert _rot(T=0) == 0 and _rot(B=0) == 0 and _rot(Hq=0, Hkv=0) == 0


def test_python_calls_refuse_host_tensors_and_bad_shapes():
    x = torch.zeros(1, 2, 3, 8)
    f, _ = rotary.rotary_frequencies(8)
    with pytest.raises(ValueError, match="device tensors"):
        rotary.apply_rotary(x, None, torch.arange(3), f)
    with pytest.raises(ValueError, match="B, H, T, d"):
        rotary.apply_rotary(x[0], None, torch.arange(3), f)
    with pytest.raises(ValueError, match="does not match"):
        rotary.apply_rotary(x, x[:, :, :2], torch.arange(3), f)
    with pytest.raises(ValueError, match="float16"):
        rotary.apply_rotary(x, x.half(), torch.arange(3), f)
    with pytest.raises(ValueError, match="device tensors"):
        eviction.select_positions(torch.zeros(1, 2, 8), 4)
    with pytest.raises(ValueError, match="float32"):
        eviction.select_positions(torch.zeros(1, 2, 8, dtype=torch.float64), 4)
    c = PQCache(blocks=torch.zeros(1, 2, 8, 36, dtype=torch.uint8), head_dim=64, n_bits=4, seq_len=8, max_seq_len=8,
                codebooks=torch.zeros(16))
    p = PagedPQCache(1, 2, 64, 4, torch.zeros(16), "cpu", page_tokens=64)
    w = torch.zeros(1, 2, 8)
    with pytest.raises(ValueError, match="both"):
        eviction.evict(c, p, w, 4)
    with pytest.raises(ValueError, match="float32"):
        eviction.evict(c, c, w[:, :, :7], 4)
    with pytest.raises(ValueError, match="int32"):
        eviction.evict(c, c, w, 4, positions=w)
    with pytest.raises(ValueError, match="device tensors"):
        eviction.evict(c, c, w, 4)
    q = torch.zeros(1, 4, 64)
    with pytest.raises(ValueError, match="device tensors"):
        attention.decode_attention_weights(q, c, c, torch.eye(64))
    with pytest.raises(ValueError, match="B, Hq, Sq, d"):
        attention.attention_weights(q, c, torch.eye(64), 0)
    mixed = PQCache(blocks=torch.zeros(1, 8 * 56, dtype=torch.uint8), head_dim=64, n_bits=(4, 2), seq_len=8,
                    max_seq_len=8, codebooks=torch.zeros(2, 16))
    with pytest.raises(ValueError, match="width"):
        attention.decode_attention_weights(q, mixed, mixed, torch.eye(64))
    with pytest.raises(ValueError, match="width"):
        attention.attention_weights(q.unsqueeze(2), mixed, torch.eye(64), 7)


def test_row_strides():
    t = torch.zeros(2, 3, 10)
    assert eviction._check_rows(t[:, :, :7], "t").stride() == (30, 10, 1) and eviction._row_stride(t[:, :, :7]) == 10
    assert eviction._check_rows(t[:, :2], "t").is_contiguous()            # heads of another tensor between
    assert eviction._check_rows(t[:, :, ::2], "t").is_contiguous()
    assert eviction._check_rows(t[:1, :1].expand(2, 3, 10), "t").is_contiguous()
    assert eviction._row_stride(t[:1, :2]) == 10 and eviction._row_stride(t[:, :1]) == 30
    assert eviction._row_stride(t[:1, :1, :4]) >= 4


def test_reserved_pages():
    c = PagedPQCache(2, 3, 64, 2, torch.zeros(16), "cpu", page_tokens=64, jl_dim=64, tables=False)
    pools = c.reserve(200)
    assert len(c.groups) == len(c.sign_groups) == 4 and c.capacity == 256 and c.max_pages == 4
    for pool, groups, table, n in zip(pools, (c.groups, c.sign_groups), (c.table, c.sign_table), (20, 8)):
        assert pool.shape == (2, 3, 4, 64, n) and table.shape == (6, 4) and table.is_contiguous()
        assert all(g.data_ptr() == pool[0, 0, p].data_ptr() and g.shape == (2, 3, 64, n) for p, g in enumerate(groups))
        # as the writer of the pages writes it
        table.copy_(torch.arange(24).view(6, 4) * (64 * n) + pool.data_ptr())
    with pytest.raises(ValueError):
        c.reserve(10)
    before = c.table.clone(), c.sign_table.clone()
    c.ensure(257)                                             # grows on by page groups
    assert len(c.groups) == 5 and torch.equal(c.table[:, :4], before[0]) and torch.equal(c.sign_table[:, :4], before[1])
    e = PagedPQCache(1, 1, 64, 4, torch.zeros(16), "cpu", page_tokens=64)
    assert e.reserve(0) == [] and e.capacity == 0


@pytest.mark.parametrize("pages", [(3, 16), (16, 3), (1, 3), (5, 7)])
def test_tables_of_two_caches_get_one_width(pages):
    """The kernels walk both tables with one row stride, whatever the caches'
    tables were made for (an evicted cache's have as many pages as it needs)."""
    cb = torch.zeros(16)
    keys, values = (PagedPQCache(2, 2, 64, 4, cb, "cpu", 64, 0, n) for n in pages)
    for c in (keys, values):
        c.ensure(c.max_pages * 64)
        c.seq_len = 40
    rows = [c.table.clone() for c in (keys, values)]
    attention.check_paged(2, 4, 64, keys, values)
    assert keys.max_pages == values.max_pages == max(pages)
    for c, old in zip((keys, values), rows):
        assert c.table.shape == (4, max(pages)) and torch.equal(c.table[:, :old.shape[1]], old)


def test_frequencies_plain_and_linear():
    f, m = rotary.rotary_frequencies(8, 10000.0)
    assert f.dtype == torch.float64 and m == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    g, m = rotary.rotary_frequencies(8, 10000.0, {"type": "linear", "factor": 4})
    assert torch.equal(g, f / 4) and m == 1.0


def test_frequencies_larger_base_keeps_the_fastest_and_stretches_the_slowest():
    f, _ = rotary.rotary_frequencies(64)
    g, m = rotary.rotary_frequencies(64, scaling={"type": "base", "factor": 8.0})
    assert g[0] == f[0] and m == 1.0
    assert math.isclose(g[-1].item(), f[-1].item() / 8, rel_tol=1e-12)
    assert rotary.rotary_frequencies(2, scaling={"type": "base", "factor": 8.0})[0].tolist() == [1.0]


def test_frequencies_bands():
    n, low, high = 8192.0, 1.0, 4.0
    f, _ = rotary.rotary_frequencies(128, 500000.0)
    g, m = rotary.rotary_frequencies(128, 500000.0, {"type": "bands", "factor": 8.0, "original": n})
    assert m == 1.0
    for a, b in zip(f.tolist(), g.tolist()):
        turns = n * a / (2 * math.pi)
        if turns >= high:
            want = a
        elif turns <= low:
            want = a / 8
        else:
            s = (turns - low) / (high - low)
            want = (1 - s) * a / 8 + s * a
        assert math.isclose(b, want, rel_tol=1e-12)
    assert torch.equal(g[:20], f[:20]) and torch.allclose(g[-5:], f[-5:] / 8, rtol=1e-15)


def test_frequencies_yarn():
    n, base, dim, factor = 4096.0, 10000.0, 128, 16.0
    f, _ = rotary.rotary_frequencies(dim, base)
    g, m = rotary.rotary_frequencies(dim, base, {"type": "yarn", "factor": factor, "original": n})
    assert math.isclose(m, 0.1 * math.log(16.0) + 1.0)
    ratio = (g / f).tolist()
    turns = (n * f / (2 * math.pi)).tolist()
    assert all(r == 1.0 for r, t in zip(ratio, turns) if t > 40) and all(
        math.isclose(r, 1 / factor) for r, t in zip(ratio, turns) if t < 0.8)
    assert all(a >= b for a, b in zip(ratio, ratio[1:]))       # a ramp
    lo = math.floor(dim * math.log(n / (2 * math.pi * 32)) / (2 * math.log(base)))
    hi = math.ceil(dim * math.log(n / (2 * math.pi)) / (2 * math.log(base)))
    i = (lo + hi) // 2
    r = (i - lo) / (hi - lo)
    assert math.isclose(ratio[i], 1 - r + r / factor, rel_tol=1e-12)
    assert rotary.rotary_frequencies(dim, scaling={"type": "yarn", "factor": 2, "original": n, "amplitude": 1.5})[1] == 1.5


@pytest.mark.parametrize("args", [
    (7,), (0,), (8, 0.0), (8, 1e4, {"type": "stretch", "factor": 2}), (8, 1e4, {"type": "linear"}),
    (8, 1e4, {"type": "linear", "factor": 0.5}), (8, 1e4, {"type": "linear", "factor": math.inf}),
    (8, 1e4, {"type": "linear", "factor": 2, "original": 4}), (8, 1e4, {"type": "yarn", "factor": 2}),
    (8, 1e4, {"type": "bands", "factor": 2, "original": 4, "low": 4, "high": 4}),
    (8, 1e4, {"type": "yarn", "factor": 2, "original": 0}), (8, 1.0, {"type": "yarn", "factor": 2, "original": 9})])
def test_frequencies_refusals(args):
    with pytest.raises(ValueError):
        rotary.rotary_frequencies(*args)


def test_embedding_refuses_more_than_the_head():
    with pytest.raises(ValueError):
        rotary.RotaryEmbedding(64, rot_dim=66)
