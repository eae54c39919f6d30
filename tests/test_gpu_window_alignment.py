"""Inputs and outputs of the operators behind a window that start off a 16-byte
boundary, strided last dimensions, and page tables of different widths."""

import math

import pytest
import torch

import test_gpu_append as append_tests
import test_gpu_window as window_tests
import window_ref
from polarquant_kv import _lib, append, attention, quantizer, rotary, rotation

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def off(x, n):
    """The values of x, `n` elements behind an aligned address, contiguous."""
    room = torch.empty(x.numel() + n, dtype=x.dtype, device=x.device)
    y = room[n:].view(x.shape)
    y.copy_(x)
    assert y.is_contiguous() and y.data_ptr() % 16
    return y


@pytest.mark.parametrize("n", [1, 2, 3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("Sq,d,qjl", [(1, 64, False), (1, 128, True), (23, 64, False), (23, 128, True), (300, 128, False)])
def test_queries(Sq, d, qjl, dtype, n):
    q, keys, values, R, jl = window_tests.make(2, 8, 2, Sq, 400, d, 4, qjl, 0, dtype=dtype)
    call = lambda x: attention.window_attention(x, keys, values, R, 90, sinks=3, jl_rot=jl, out_dtype=torch.float32)  # noqa: E731
    assert torch.equal(call(off(q, n)), call(q))


@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,Sq,d", [(2, 1, 64), (90, 1, 128), (2, 23, 128), (2, 300, 64), (3, 1200, 128)])
def test_outputs(B, Sq, d, dtype, n):
    Hq, Hkv, S, W = 8, 2, 1300, 40
    q, keys, values, R, _ = window_tests.make(B, Hq, Hkv, Sq, S, d, 4, False, 0)
    want = attention.window_attention(q, keys, values, R, W, starts=S - Sq, out_dtype=dtype)
    room = torch.full((want.numel() + n + 8,), 7.0, dtype=dtype, device=DEV)
    lib = _lib.lib()
    need = lib.pqkv_window_attn_workspace_bytes(B, Hq, Hkv, Sq, S, d, W, 0, 0)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    _lib.check(lib.pqkv_window_attn(
        q.data_ptr(), _lib.F16, R.data_ptr(), keys.blocks.data_ptr(), values.blocks.data_ptr(), keys.codebooks.data_ptr(),
        values.codebooks.data_ptr(), 4, None, None, 0, B, Hq, Hkv, Sq, S - Sq, None, None, W, 0, S, d, 1.0 / math.sqrt(d),
        room[n:].data_ptr(), _lib.dtype_code(dtype), ws.data_ptr(), need, _lib.stream_of(q)))
    assert torch.equal(room[n:n + want.numel()].view(want.shape), want)
    assert bool((room[:n] == 7.0).all()) and bool((room[n + want.numel():] == 7.0).all())


# d, rot, dtype, interleaved, T, qjl
APPENDS = [(128, 128, torch.float16, False, 40, False), (128, 96, torch.bfloat16, True, 3, True),
           (64, 64, torch.float32, False, 33, False), (64, 48, torch.float16, True, 1, True)]


@pytest.mark.parametrize("how", ["off", "strided", "rotation"])
@pytest.mark.parametrize("d,rot,dtype,inter,T,qjl", APPENDS)
def test_appended(d, rot, dtype, inter, T, qjl, how):
    case = (2, 4, 2, T, 64, d, rot, 4, qjl, 0, dtype, inter, None, 0, None)
    q, k, v, keys, values, R, P, positions, freqs, _ = append_tests.make(case)
    if how == "off":
        q, k, v = (off(x.contiguous(), n) for x, n in ((q, 1), (k, 2), (v, 3)))
    elif how == "strided":
        q, k, v = (x.repeat_interleave(2, -1)[..., ::2] for x in (q, k, v))
        assert k.stride(-1) == 2
    else:
        R, P = off(R, 1), None if P is None else off(P, 2)
    got = append.append_rotary(k, v, keys, values, R, positions, freqs, query=q, starts=7, interleaved=inter, jl_rot=P)
    assert torch.equal(got, rotary.apply_rotary(q, None, positions, freqs, interleaved=inter)[0])
    for c, x in ((keys, append_tests.turned(k, positions, freqs, None, inter, 1.0)), (values, v.double())):
        e = append_tests.check_vectors(c.blocks[:, :, 7:7 + T], x, R, c.codebooks, 4)
        if c.qjl_signs is not None:
            append_tests.check_signs(c.qjl_signs[:, :, 7:7 + T], e, P)


@pytest.mark.parametrize("wider", [0, 1])
@pytest.mark.parametrize("given", [False, True])
def test_tables_of_different_widths(given, wider):
    B, H, d, T = 2, 2, 64, 70
    R = rotation.generate_rotation_matrix(d, device=DEV)
    pair = [quantizer.allocate_paged_cache(B, H, d, 4, DEV, page_tokens=64, jl_dim=0) for _ in range(2)]
    twin = [quantizer.allocate_paged_cache(B, H, d, 4, DEV, page_tokens=64, jl_dim=0) for _ in range(2)]
    pair[wider]._widen(64)
    freqs = rotary.rotary_frequencies(d)[0].to(DEV)
    k, v = (torch.randn(B, H, T, d, device=DEV).half() for _ in range(2))
    starts = torch.tensor([100, 3], device=DEV) if given else 100
    for caches in (pair, twin):
        for c in caches:
            c.ensure(1100 if given else 100)         # 18 pages: the narrower tables grow
        append.append_rotary(k, v, *caches, R, torch.arange(T, device=DEV), freqs, starts=starts)
    assert pair[0].max_pages == pair[1].max_pages == 64
    for a, b in zip(pair, twin):
        n = min(a.capacity, b.capacity)
        assert torch.equal(window_ref.rows_of(a)[0][:, :, :n], window_ref.rows_of(b)[0][:, :, :n])
        a.seq_len = b.seq_len = 170
    q = torch.randn(B, 4, 3, d, device=DEV).half()
    call = lambda c: attention.window_attention(q, *c, R, 80, sinks=2)  # noqa: E731
    assert torch.equal(call(pair), call(twin))
