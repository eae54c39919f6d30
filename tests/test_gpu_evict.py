"""Eviction on the GPU: the positions that stay (against a stable sort on the
host: whole numbers, so equal), and the move of their rows (bytes, so equal)."""

import numpy as np
import pytest
import torch

from polarquant_kv import eviction, quantizer
from polarquant_kv.rotation import generate_rotation_matrix
from polarquant_kv.types import PagedPQCache, PQCache, vector_bytes

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def want_kept(w, keep, sink, recent):
    """w [n, S] float32 on the host: the definition, row by row."""
    out = np.empty((w.shape[0], keep), np.int32)
    S = w.shape[1]
    at = np.arange(S)
    forced = (at < sink) | (at >= S - recent)
    for r, row in enumerate(w.astype(np.float64)):
        rank = np.where(np.isnan(row), -np.inf, row)
        nan = np.isnan(row) & ~forced
        # forced first, then by weight, NaN last (below -inf), equal ones by index
        order = np.lexsort((at, -np.where(forced, 0, rank), nan, ~forced))
        out[r] = np.sort(order[:keep])
    return out


SELECT = [
    # n, S, keep, sink, recent
    (1, 1, 1, 0, 0), (3, 2, 1, 0, 0), (2, 63, 20, 4, 8), (2, 64, 64, 0, 0), (1, 65, 33, 0, 1), (5, 1023, 512, 4, 64),
    (4, 1024, 1, 1, 0), (4, 1025, 300, 300, 0), (2, 1025, 300, 0, 300), (2, 4097, 4096, 4, 64), (3, 5000, 4, 0, 0),
    (2, 33333, 10000, 4, 256), (1, 131072, 16384, 4, 1024), (300, 777, 100, 3, 5), (1, 70001, 35000, 0, 0),
    (2, 300, 300, 200, 200),                                  # all of it is protected
]


def laws(n, S, seed):
    g = np.random.default_rng(seed)
    tail = np.exp(2.5 * g.standard_normal((n, S)))
    yield "tail", tail.astype(np.float32)
    yield "ties", (np.floor(tail * 4) / 4 * (tail > 0.5)).astype(np.float32)
    yield "equal", np.full((n, S), 0.125, np.float32)
    yield "zeros", np.where(g.random((n, S)) < 0.5, 0.0, -0.0).astype(np.float32)
    odd = tail.astype(np.float32)
    odd[g.random((n, S)) < 0.2] = np.nan
    odd[g.random((n, S)) < 0.1] = np.inf
    odd[g.random((n, S)) < 0.1] = -np.inf
    odd[g.random((n, S)) < 0.1] *= -1
    odd[g.random((n, S)) < 0.1] = 1e-42                        # below the normal range
    yield "odd", odd
    near = np.float32(1.0) + g.integers(0, 3, (n, S)).astype(np.float32) * np.float32(2.0 ** -23)
    yield "neighbours", near.astype(np.float32)


@pytest.mark.parametrize("case", SELECT, ids=["n{}_S{}_keep{}_sink{}_recent{}".format(*c) for c in SELECT])
def test_select(case):
    n, S, keep, sink, recent = case
    for name, w in laws(n, S, S + keep):
        t = torch.from_numpy(w).to(DEV).view(1, n, S)
        got = eviction.select_positions(t, keep, sink, recent)[0].cpu().numpy()
        assert np.array_equal(got, want_kept(w, keep, sink, recent)), name


def test_select_strided_rows():
    g = torch.Generator(device=DEV).manual_seed(3)
    big = torch.randn(2, 3, 1000, generator=g, device=DEV)
    want = eviction.select_positions(big[:, :, :700].contiguous(), 100, 2, 10)
    assert torch.equal(eviction.select_positions(big[:, :, :700], 100, 2, 10), want)
    assert torch.equal(eviction.select_positions(big.transpose(0, 1)[:, :, :700], 100, 2, 10), want.transpose(0, 1))
    odd = torch.randn(1, 2 * 701 + 1, device=DEV)[0, 1:].view(1, 2, 701)          # rows off a 16-byte boundary
    assert torch.equal(eviction.select_positions(odd, 100), eviction.select_positions(odd.clone(), 100))


def test_select_on_a_stream_and_captured():
    w = torch.rand(2, 4, 3001, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        eviction.select_positions(w, 500, 4, 16)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = eviction.select_positions(w, 500, 4, 16)
    for _ in range(4):
        w.copy_(torch.rand_like(w))
        graph.replay()
        assert torch.equal(kept, eviction.select_positions(w, 500, 4, 16))
        torch.cuda.synchronize()


def random_cache(B, H, S, d, bits, jl, seed, S_max=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    S_max = S if S_max is None else S_max

    def rows(n):
        return torch.randint(0, 256, (B, H, S_max, n), generator=g, device=DEV, dtype=torch.uint8)

    return PQCache(blocks=rows(vector_bytes(d, bits)), head_dim=d, n_bits=bits, seq_len=S, max_seq_len=S_max,
                   codebooks=torch.zeros(16, device=DEV), qjl_signs=rows(d // 8) if jl else None, jl_dim=d if jl else 0)


def paged_copy(c, P):
    """The same rows in pages at shuffled places of one pool."""
    B, H, S, d = c.batch, c.num_heads, c.seq_len, c.head_dim
    n = -(-S // P) + 1
    p = PagedPQCache(B, H, d, c.n_bits, c.codebooks, DEV, page_tokens=P, jl_dim=c.jl_dim)
    slot = torch.randperm(B * H * n).view(B * H, n)
    tables, pools = [], []
    for rows in (c.blocks, c.qjl_signs):
        if rows is None:
            tables.append(None)
            continue
        pool = torch.full((B * H * n, P, rows.shape[-1]), 0xA5, dtype=torch.uint8, device=DEV)
        for s in range(B * H):
            for t in range(0, S, P):
                m = min(P, S - t)
                pool[slot[s, t // P], :m] = rows[s // H, s % H, t:t + m]
        tables.append((pool.data_ptr() + slot * (P * rows.shape[-1])).to(DEV))
        pools.append(pool)
    p.adopt(tables[0], n * P, pools, tables[1])
    p.seq_len = S
    return p


MOVE = [
    # B, H, S, keep, d, bits, jl, page
    (1, 1, 1, 1, 64, 4, False, 0), (2, 3, 300, 100, 128, 4, False, 0), (1, 2, 513, 257, 64, 2, True, 0),
    (2, 2, 1000, 256, 128, 2, True, 64), (1, 8, 700, 699, 64, 4, False, 128), (3, 1, 2000, 1000, 128, 4, True, 256),
    (1, 2, 130, 64, 128, 4, False, 64), (1, 1, 100, 0, 64, 4, False, 64), (2, 2, 50, 0, 64, 4, True, 0),
]


@pytest.mark.parametrize("case", MOVE, ids=["B{}_H{}_S{}_keep{}_d{}_b{}_{}_P{}".format(*c[:6], "qjl" if c[6] else "plain",
                                                                                      c[7]) for c in MOVE])
def test_evict_moves_what_stays(case):
    B, H, S, keep, d, bits, jl, page = case
    kc, vc = random_cache(B, H, S, d, bits, jl, 1, S + 5), random_cache(B, H, S, d, bits, False, 2, S + 5)
    before = kc.blocks.clone(), vc.blocks.clone()
    w = torch.rand(B, H, S + 7, device=DEV)
    pos = torch.randint(0, 10 ** 6, (B, H, S + 3), device=DEV, dtype=torch.int32)
    keys, values = (paged_copy(kc, page), paged_copy(vc, page)) if page else (kc, vc)
    sink, recent = min(2, keep), min(3, max(0, keep - 2))
    r = eviction.evict(keys, values, w, keep, sink=sink, recent=recent, positions=pos)
    kept = want_kept(w[:, :, :S].reshape(-1, S).cpu().numpy(), keep, sink, recent).reshape(B, H, keep)
    assert np.array_equal(r.kept.cpu().numpy(), kept)
    at = torch.from_numpy(kept).long().to(DEV)
    assert torch.equal(r.weights, torch.gather(w, 2, at)) and torch.equal(r.positions, torch.gather(pos, 2, at))
    for old, new in ((kc, r.keys), (vc, r.values)):
        assert new.seq_len == keep and type(new) is type(keys)
        n = new.to_contiguous() if page else new
        for a, b in ((old.blocks, n.blocks), (old.qjl_signs, n.qjl_signs)):
            assert (a is None) == (b is None)
            if a is not None:
                assert torch.equal(b, torch.gather(a, 2, at[..., None].expand(B, H, keep, a.shape[-1])))
        if page:
            assert new.capacity == -(-keep // page) * page
            if keep % page:
                assert not new.groups[-1][:, :, keep % page:].any()
    assert torch.equal(kc.blocks, before[0]) and torch.equal(vc.blocks, before[1])


def test_room_for_more_and_appending_after():
    B, H, S, d = 1, 2, 200, 64
    R = generate_rotation_matrix(d, seed=42, device=DEV)
    kv = torch.randn(B, H, S, d, device=DEV).half()
    for paged in (False, True):
        make = (lambda: quantizer.allocate_paged_cache(B, H, d, 4, DEV, page_tokens=64)) if paged else (
            lambda: quantizer.allocate_cache(B, H, S, d, 4, DEV))
        k, v = (quantizer.compress_pq(kv, R, cache=make()) for _ in range(2))
        r = eviction.evict(k, v, torch.rand(B, H, S, device=DEV), 70, room=None if paged else 100)
        old = [c.to_contiguous().blocks if paged else c.blocks[:, :, :70].clone() for c in (r.keys, r.values)]
        new = torch.randn(B, H, 30, d, device=DEV).half()
        quantizer.compress_pq(new, R, cache=r.keys)
        quantizer.compress_pq(new, R, cache=r.values)
        want = quantizer.compress_pq(new, R).blocks
        for c, o in zip((r.keys, r.values), old):
            assert c.seq_len == 100
            b = c.to_contiguous().blocks if paged else c.blocks
            assert torch.equal(b[:, :, :70], o) and torch.equal(b[:, :, 70:], want)
    with pytest.raises(ValueError):
        eviction.evict(k, v, torch.rand(B, H, S, device=DEV), 70, room=69)


def test_positions_outside_the_cache_give_zeros_and_may_repeat():
    c = random_cache(1, 2, 100, 128, 4, False, 5)
    kept = torch.tensor([[[-1, 5, 5, 99, 100, 2 ** 31 - 1]] * 2], dtype=torch.int32, device=DEV)
    (n,), _ = eviction.gather_positions([c], kept)
    assert torch.equal(n.blocks[:, :, 1:4], c.blocks[:, :, [5, 5, 99]])
    assert not n.blocks[:, :, [0, 4, 5]].any()


@pytest.mark.parametrize("keep,pages", [(130, 16), (190, 4), (64, 1)])
def test_attention_on_tables_of_different_widths(keep, pages):
    """An evicted cache's table has as many pages as it needs; beside values
    whose table was made for more (or for as many as a power of two), both are
    read with one row stride."""
    from polarquant_kv import attention
    g = torch.Generator(device=DEV).manual_seed(9)
    B, Hq, H, d, P = 2, 8, 4, 64, 64
    cb = torch.linspace(-1, 1, 16, device=DEV)
    R = torch.linalg.qr(torch.randn(d, d, generator=g, device=DEV))[0].contiguous()

    def cache(S):
        rows = torch.randint(0, 256, (B, H, S, d // 32, 18), generator=g, device=DEV, dtype=torch.uint8)
        rows[..., :2] = (0.5 + torch.rand(B, H, S, d // 32, generator=g, device=DEV)).half().view(torch.uint8).view(
            B, H, S, d // 32, 2)                                       # a finite radius
        return PQCache(blocks=rows.flatten(3), head_dim=d, n_bits=4, seq_len=S, max_seq_len=S, codebooks=cb)

    old, values = cache(300), cache(keep)
    kept = torch.randint(0, 300, (B, H, keep), generator=g, device=DEV, dtype=torch.int32)
    (paged,), _ = eviction.gather_positions([paged_copy(old, P)], kept)
    (flat,), _ = eviction.gather_positions([old], kept)
    assert paged.max_pages == -(-keep // P)
    wide = PagedPQCache(B, H, d, 4, cb, DEV, page_tokens=P, max_pages=pages)
    wide.ensure(keep)
    for p, group in enumerate(wide.groups):
        group[:, :, :min(P, keep - p * P)] = values.blocks[:, :, p * P:(p + 1) * P]
    wide.seq_len = keep
    q = torch.randn(B, Hq, d, generator=g, device=DEV).half()
    out, w = attention.decode_attention_weights(q, paged, wide, R)
    want, w_flat = attention.decode_attention_weights(q, flat, values, R)
    assert torch.equal(out, want) and torch.equal(w, w_flat)
    assert torch.equal(attention.decode_attention(q, paged, wide, R), want)
    assert paged.max_pages == wide.max_pages


def test_rows_that_are_views():
    c = random_cache(2, 2, 60, 64, 4, False, 6)
    kept = torch.arange(0, 60, 3, device=DEV, dtype=torch.int32).expand(2, 2, 20)
    big = torch.randn(2, 2, 2, 90, device=DEV)
    views = [big[:, 0], big[:, 1, :, :70], big[:, :, 0, ::2][:, :, :45].repeat(1, 1, 2)[:, :, :60].transpose(0, 1),
             torch.arange(60, device=DEV, dtype=torch.int32).expand(2, 2, 60)]
    _, moved = eviction.gather_positions([c], kept, views)
    for v, m in zip(views, moved):
        assert torch.equal(m, torch.gather(v, 2, kept.long())) and m.dtype == v.dtype


def test_rows_into_pages_of_a_table():
    """pqkv_gather_rows into pages that lie anywhere (a result with a table and
    no base): rows keep .. fill - 1 are zeros, the last page's rest is left alone."""
    from polarquant_kv import _lib
    B, H, S, keep, P, fill = 1, 3, 500, 150, 64, 170
    c = random_cache(B, H, S, 64, 4, False, 8)
    n, size = -(-fill // P), P * 36
    pool = torch.full((H * n + 2, P, 36), 0xA5, dtype=torch.uint8, device=DEV)
    slot = torch.randperm(H * n).view(H, n) + 1
    table = (pool.data_ptr() + slot * size).to(DEV)
    kept = torch.stack([torch.randperm(S)[:keep].sort().values for _ in range(H)]).int().to(DEV)
    src = _lib.RowArray(c.blocks.data_ptr(), None, S * 36, 0, 0)
    dst = _lib.RowArray(None, table.data_ptr(), 0, P, n)
    _lib.check(_lib.lib().pqkv_gather_rows(1, (_lib.RowArray * 1)(src), (_lib.RowArray * 1)(dst), _lib.int_array([36]),
                                           kept.data_ptr(), H, S, keep, fill, _lib.stream_of(kept)))
    rows = pool[slot.flatten().to(DEV)].view(H, n * P, 36)
    want = torch.gather(c.blocks[0], 1, kept.long()[..., None].expand(H, keep, 36))
    assert torch.equal(rows[:, :keep], want) and not rows[:, keep:fill].any() and bool((rows[:, fill:] == 0xA5).all())
    assert bool((pool[[0, -1]] == 0xA5).all())


def test_caches_past_four_gigabytes():
    """Byte offsets of one stream past 2^32: 4-bit rows of 72 bytes, 61 million
    positions (the page-free cache is 4.4 GB)."""
    S = 61_000_000
    blocks = torch.zeros(1, 1, S, 72, dtype=torch.uint8, device=DEV)
    picks = torch.tensor([0, 1, 29_826_161, 29_826_162, 59_652_323, 59_652_324, S - 1], device=DEV)
    blocks[0, 0, picks] = torch.arange(1, 8, device=DEV, dtype=torch.uint8)[:, None]
    c = PQCache(blocks=blocks, head_dim=128, n_bits=4, seq_len=S, max_seq_len=S, codebooks=torch.zeros(16, device=DEV))
    (n,), _ = eviction.gather_positions([c], picks.int().view(1, 1, -1))
    assert torch.equal(n.blocks[0, 0], torch.arange(1, 8, device=DEV, dtype=torch.uint8)[:, None].expand(7, 72))


def test_refusals_on_the_device():
    c = random_cache(1, 2, 100, 64, 4, False, 7)
    w = torch.rand(1, 2, 100, device=DEV)
    for kw in (dict(keep=101), dict(keep=5, sink=4, recent=2), dict(keep=-1), dict(keep=5, sink=-1)):
        with pytest.raises(ValueError):
            eviction.evict(c, c, w, **kw)
    kept = torch.zeros(1, 2, 3, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        eviction.gather_positions([c], kept.long())
    with pytest.raises(ValueError):
        eviction.gather_positions([c], kept[:, :1])
    with pytest.raises(ValueError):
        eviction.gather_positions([], kept)
    with pytest.raises(ValueError):
        eviction.gather_positions([c], kept, [w.double()])
    with pytest.raises(ValueError):
        eviction.gather_positions([c] * 7, kept)
    other = random_cache(1, 2, 90, 64, 4, False, 7)
    with pytest.raises(ValueError):
        eviction.evict(c, other, w, 50)
    short = PQCache(blocks=c.blocks, head_dim=64, n_bits=4, seq_len=100, max_seq_len=200, codebooks=c.codebooks)
    with pytest.raises(ValueError):
        eviction.gather_positions([short], kept)
