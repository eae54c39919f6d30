"""pqkv_window_attn and _paged through attention.window_attention against the
formula in 64 bits on the same bytes; tolerances in window_ref.py."""

import pytest
import torch

import window_ref
from polarquant_kv import attention, quantizer, rotation
from polarquant_kv.types import PagedPQCache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(B, Hq, Hkv, Sq, S, d, bits, qjl, page, seed=0, dtype=torch.float16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    R = rotation.generate_rotation_matrix(d, seed=42, device=DEV)
    jl = torch.randn(d, d, generator=g, device=DEV) if qjl else None
    caches = []
    for which in ("keys", "values"):
        x = torch.randn(B, Hkv, S, d, generator=g, device=DEV).half()
        p = jl if which == "keys" else None
        if page:
            c = quantizer.allocate_paged_cache(B, Hkv, d, bits, DEV, page_tokens=page, jl_dim=d if p is not None else 0)
            quantizer.compress_pq(x, R, cache=c, start=0, jl_rot=p)
        else:
            c = quantizer.compress_pq(x, R, bits, jl_rot=p)
        caches.append(c)
    q = (2.0 * torch.randn(B, Hq, Sq, d, generator=g, device=DEV)).to(dtype)
    return q, caches[0], caches[1], R, jl


def per_sequence(x, B):
    return torch.tensor(x if isinstance(x, (list, tuple)) else [x] * B, device=DEV)


def poison(keys, values, starts, counts, window, sinks):
    """NaN radii wherever no row looks, and codes of ones behind them."""
    B, H = keys.batch, keys.num_heads
    S = keys.capacity if isinstance(keys, PagedPQCache) else keys.max_seq_len
    t = torch.arange(S, device=DEV)
    for c in (keys, values):
        for b in range(B):
            start, n = int(starts[b]), int(counts[b])
            n = max(0, min(n, S - start)) if 0 <= start < S else 0
            row = torch.arange(start, start + n, device=DEV)[:, None]
            unseen = ~((t <= row) & ((t > row - window) | (t < sinks))).any(0)
            if isinstance(c, PagedPQCache):
                for p, grp in enumerate(c.groups):
                    grp[b][:, unseen[p * c.page_tokens:(p + 1) * c.page_tokens]] = 255
            else:
                c.blocks[b][:, unseen] = 255
    return keys, values


# B, Hq, Hkv, S, window, sinks, d, bits, qjl, page, starts
ROWS = [
    (1, 1, 1, 1, 1, 0, 64, 4, False, 0, 0),
    (1, 2, 2, 5, 3, 1, 64, 2, False, 0, 4),
    (2, 14, 2, 300, 64, 4, 64, 4, False, 0, [299, 17]),
    (2, 14, 2, 300, 65, 4, 64, 4, True, 64, [298, 64]),
    (3, 8, 2, 517, 100, 70, 128, 4, False, 256, [516, 63, 128]),
    (3, 8, 2, 517, 100, 70, 128, 4, True, 0, [516, 163, 191]),
    (2, 16, 2, 1000, 333, 0, 128, 2, False, 64, [999, 332]),
    (2, 16, 2, 1000, 333, 130, 128, 2, True, 256, [700, 333]),
    (1, 12, 1, 700, 256, 5, 128, 4, False, 0, 699),          # a group of 12: two launches
    (1, 5, 1, 700, 1, 0, 128, 4, True, 64, 640),             # only itself
    (1, 6, 1, 700, 1, 1, 64, 4, True, 0, 700 - 1),
    (1, 3, 1, 129, 10 ** 9, 10 ** 9, 128, 4, False, 0, 128),  # more than the cache
    (4, 7, 7, 2500, 2049, 64, 64, 4, False, 256, [2499, 2048, 64, 0]),
    (2, 32, 8, 9000, 4096, 4, 128, 4, False, 256, [8999, 4100]),
]


@pytest.mark.parametrize("out", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("case", ROWS, ids=lambda c: "B{}_{}-{}_S{}_w{}_s{}_d{}_b{}_{}_p{}".format(*c[:10]))
def test_one_row_per_sequence(case, out):
    B, Hq, Hkv, S, window, sinks, d, bits, qjl, page, starts = case
    q, keys, values, R, jl = make(B, Hq, Hkv, 1, S, d, bits, qjl, page)
    at, n = per_sequence(starts, B), per_sequence(1, B)
    poison(keys, values, at, n, window, sinks)
    want, bound = window_ref.window_attention(q, keys, values, R, window, sinks, at, n, p_rot=jl)
    given = at if isinstance(starts, list) else starts
    got = attention.window_attention(q, keys, values, R, window, sinks=sinks, starts=given, jl_rot=jl, out_dtype=out)
    assert got.dtype == out and got.shape == q.shape
    window_ref.check(got, want, bound)


@pytest.mark.parametrize("out", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("B,Hq,Hkv,d,qjl", [(17, 32, 8, 128, False), (33, 16, 4, 128, True), (40, 14, 2, 64, False)])
def test_many_sequences_in_one_split(B, Hq, Hkv, d, qjl, out):
    # (some of them without a row)
    S, window, sinks = 200, 40, 3
    q, keys, values, R, jl = make(B, Hq, Hkv, 1, S, d, 4, qjl, 0)
    at = torch.arange(B, device=DEV) * 11 % S
    n = (torch.arange(B, device=DEV) % 5 != 3).long()
    poison(keys, values, at, n, window, sinks)
    want, bound = window_ref.window_attention(q, keys, values, R, window, sinks, at, n, p_rot=jl)
    got = attention.window_attention(q, keys, values, R, window, sinks=sinks, starts=at, counts=n, jl_rot=jl,
                                     out_dtype=out)
    window_ref.check(got, want, bound)


# B, Hq, Hkv, Sq, S, window, sinks, d, bits, qjl, page, starts, counts
CHUNKS = [
    (1, 1, 1, 2, 2, 1, 0, 64, 4, False, 0, 0, None),
    (2, 14, 2, 17, 300, 64, 4, 64, 4, False, 0, [283, 0], None),
    (2, 14, 2, 33, 300, 65, 4, 64, 2, True, 64, [200, 64], [33, 7]),
    (1, 8, 2, 257, 600, 100, 70, 128, 4, False, 256, 343, None),
    (3, 8, 2, 70, 517, 100, 0, 128, 4, True, 0, [447, 163, 0], [70, 1, 0]),
    (2, 16, 2, 64, 1000, 333, 130, 128, 2, False, 64, [936, 332], [50, 64]),
    (1, 12, 1, 65, 700, 256, 5, 128, 4, False, 0, 635, None),
    (1, 4, 4, 700, 700, 128, 4, 64, 4, False, 64, 0, None),          # a prompt on itself
    (1, 8, 2, 300, 300, 10 ** 9, 10 ** 9, 128, 4, False, 0, 0, None),
    (2, 5, 1, 40, 3000, 2049, 64, 128, 4, True, 256, [2960, 2048], [40, 39]),   # few rows: split
    (1, 32, 8, 20, 9000, 8000, 4, 128, 4, False, 256, 8980, None),
    (1, 130, 1, 5, 200, 33, 2, 64, 4, False, 0, 195, None),                     # one token in a row block
    (5, 2, 1, 1024, 2048, 512, 1, 64, 4, False, 0, [1024, 1, 77, 500, 1000], [1024, 1023, 130, 512, 0]),
]


@pytest.mark.parametrize("out", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("case", CHUNKS, ids=lambda c: "B{}_{}-{}_Sq{}_S{}_w{}_s{}_d{}_b{}_{}_p{}".format(*c[:11]))
def test_chunks(case, out):
    B, Hq, Hkv, Sq, S, window, sinks, d, bits, qjl, page, starts, counts = case
    q, keys, values, R, jl = make(B, Hq, Hkv, Sq, S, d, bits, qjl, page)
    at, n = per_sequence(starts, B), per_sequence(Sq if counts is None else counts, B)
    poison(keys, values, at, n, window, sinks)
    want, bound = window_ref.window_attention(q, keys, values, R, window, sinks, at, n, p_rot=jl)
    given = at if isinstance(starts, list) else starts
    got = attention.window_attention(q, keys, values, R, window, sinks=sinks, starts=given,
                                     counts=None if counts is None else n, jl_rot=jl, out_dtype=out)
    assert got.dtype == out and got.shape == q.shape
    window_ref.check(got, want, bound)
    for b in range(B):
        assert not got[b, :, int(n[b]):].any()


def test_a_hidden_number_that_is_none_in_an_edge_tile():
    """Sixteen rows of one tile that see different positions of it, each next to NaN."""
    for Sq in (1, 16):
        q, keys, values, R, _ = make(1, 4, 1, Sq, 128, 64, 4, False, 0)
        starts = 90
        for t in (80, 95 if Sq > 1 else 91):         # hidden from the rows below, or from those above by the window
            values.blocks[:, :, t, :2] = 255
            values.blocks[:, :, t, 18:20] = 255
        got = attention.window_attention(q, keys, values, R, 8, starts=starts, out_dtype=torch.float32)
        row = torch.arange(starts, starts + Sq, device=DEV)
        sees = ((80 > row - 8) & (80 <= row)) | ((95 if Sq > 1 else 91) <= row) & ((95 if Sq > 1 else 91) > row - 8)
        assert torch.equal(torch.isnan(got).any(-1)[0, 0], sees)
        assert torch.equal(torch.isfinite(got).all(-1)[0, 0], ~sees)


@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("Sq", [1, 9])
def test_sequences_that_are_not_in_the_cache(page, Sq):
    q, keys, values, R, _ = make(5, 4, 2, Sq, 192, 64, 4, False, page)
    at = torch.tensor([-1, 192, 190, -2 ** 40, 2 ** 40], device=DEV)
    n = torch.full((5,), Sq, device=DEV)
    want, bound = window_ref.window_attention(q, keys, values, R, 50, 2, at, n)
    got = attention.window_attention(q, keys, values, R, 50, sinks=2, starts=at, out_dtype=torch.float32)
    window_ref.check(got, want, bound)
    assert not got[[0, 1, 3, 4]].any() and not got[2, :, 2:].any() and bool(got[2, :, 0].any())
    none = attention.window_attention(q, keys, values, R, 50, starts=at.clamp(0, 100), counts=n - Sq)
    assert not none.any()


def test_a_window_of_everything_is_attention():
    q, keys, values, R, jl = make(2, 8, 2, 40, 500, 128, 4, True, 64)
    whole = attention.prefill_attention(q, keys, values, R, 460, jl_rot=jl, out_dtype=torch.float32)
    got = attention.window_attention(q, keys, values, R, 500, jl_rot=jl, out_dtype=torch.float32)
    assert (got - whole).abs().max() <= 1e-4 * whole.abs().max()
    one = attention.decode_attention(q[:, :, -1], keys, values, R, jl_rot=jl, out_dtype=torch.float32)
    got = attention.window_attention(q[:, :, -1:], keys, values, R, 500, jl_rot=jl, out_dtype=torch.float32)
    assert (got[:, :, 0] - one).abs().max() <= 1e-4 * one.abs().max()


@pytest.mark.parametrize("Sq", [1, 5])
def test_captured_calls_follow_their_starts(Sq):
    q, keys, values, R, _ = make(3, 8, 2, Sq, 700, 128, 4, False, 64)
    at = torch.tensor([600, 5, 100], device=DEV)
    n = torch.tensor([Sq, Sq, max(1, Sq - 2)], device=DEV)
    call = lambda: attention.window_attention(q, keys, values, R, 200, sinks=4, starts=at, counts=n,  # noqa: E731
                                              out_dtype=torch.float32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for step in range(4):
        graph.replay()
        kept = got.clone()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(kept, want)
        q.normal_()
        at += torch.tensor([7, 64, -30], device=DEV)


def test_two_streams_at_once():
    a, b = make(2, 8, 2, 1, 600, 128, 4, False, 0, seed=1), make(2, 8, 2, 33, 600, 128, 4, False, 0, seed=2)
    call = lambda x: attention.window_attention(*x[:4], 100, sinks=3, out_dtype=torch.float32)  # noqa: E731
    want = call(a), call(b)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        got = []
        for s, x in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(call(x))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_positions_behind_two_gigabytes():
    """The last stream of a cache of 4.8 GB, its window in its last positions."""
    B, Hkv, S, d = 2, 4, 1 << 23, 128
    small = make(1, 4, 1, 3, 300, d, 4, False, 0)
    from polarquant_kv.types import PQCache
    big = []
    for c in small[1:3]:
        blocks = torch.zeros(B, Hkv, S, 72, dtype=torch.uint8, device=DEV)
        blocks[1, 3, S - 300:] = c.blocks[0, 0]
        big.append(PQCache(blocks=blocks, head_dim=d, n_bits=4, seq_len=S, max_seq_len=S, codebooks=c.codebooks))
    q = torch.zeros(B, 16, 3, d, dtype=torch.float16, device=DEV)
    q[1, 12:] = small[0][0]
    for n in (1, 3):
        got = attention.window_attention(q[:, :, :n], *big, small[3], 100, starts=S - 3, out_dtype=torch.float32)
        want = attention.window_attention(small[0][:, :, :n], *small[1:4], 100, starts=297, out_dtype=torch.float32)
        # (the tiles start elsewhere, so sums are in another order)
        assert (got[1, 12:] - want[0]).abs().max() <= 1e-5 * want.abs().max()
        assert not got[0].any()


def test_strided_queries_and_rotations():
    q, keys, values, R, _ = make(2, 8, 2, 6, 100, 64, 4, False, 0)
    want = attention.window_attention(q, keys, values, R, 30, sinks=1)
    wide = torch.empty(2, 6, 8, 64, dtype=q.dtype, device=DEV).copy_(q.transpose(1, 2)).transpose(1, 2)
    assert not wide.is_contiguous()
    assert torch.equal(attention.window_attention(wide, keys, values, R.t().contiguous().t(), 30, sinks=1), want)
    assert attention.window_attention(q[:, :, :0], keys, values, R, 30).shape == (2, 8, 0, 64)


@pytest.mark.parametrize("S", [60, 300], ids=["one_split", "splits"])
@pytest.mark.parametrize("d,bits,qjl", [(128, 4, False), (64, 2, False), (128, 4, True)])
def test_queries_of_any_size(S, d, bits, qjl):
    # rows of very different sizes side by side in a matrix operand
    q, keys, values, R, jl = make(2, 8, 2, 24, S, d, bits, qjl, 0, dtype=torch.float32)
    sizes = torch.tensor([0.0, 1e-30, 2.0 ** -6, 1.0, 8.0, 20.0], device=DEV)
    q = q * sizes[torch.arange(24, device=DEV) % 6][:, None]
    at, n = per_sequence([S - 24, 5], 2), per_sequence(24, 2)
    want, bound = window_ref.window_attention(q, keys, values, R, 33, 2, at, n, p_rot=jl)
    window_ref.check(attention.window_attention(q, keys, values, R, 33, sinks=2, starts=at, jl_rot=jl), want, bound)
    q[0, 3, 7] = float("inf")
    q[1, 5, 20, 3] = float("nan")
    got = attention.window_attention(q, keys, values, R, 33, sinks=2, starts=at, jl_rot=jl)
    hit = torch.zeros(2, 8, 24, dtype=torch.bool, device=DEV)
    hit[0, 3, 7] = hit[1, 5, 20] = True
    assert torch.isnan(got[hit]).all()
    window_ref.check(got[~hit], want[~hit], bound[~hit])
