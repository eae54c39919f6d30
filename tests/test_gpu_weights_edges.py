"""Attention weights where they can go wrong: queries at any address, numbers that
are not finite, chunks in several passes, workspaces of the least size. Bounds as
derived in test_gpu_weights."""

import pytest
import torch

from polarquant_kv import _lib, attention
from polarquant_kv.lloyd_max import padded_codebook_torch
from polarquant_kv.qjl import generate_jl_matrix, rotated_jl_matrix
from polarquant_kv.rotation import generate_rotation_matrix
from polarquant_kv.types import PagedPQCache, PQCache

from test_gpu_evict import paged_copy
from test_gpu_weights import close, decoded, exact, make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("d,qjl", [(64, False), (128, False), (128, True)])
def test_queries_off_a_16_byte_boundary(dtype, d, qjl):
    q, kc, _, R, jl = make(1, 6, 2, 300, d, 4, qjl, Sq=70)
    q = q.to(dtype)
    want, tol, _ = exact(q, kc, R, 230, jl_rot=jl)
    at_home = attention.attention_weights(q, kc, R, 230, jl_rot=jl)
    close(at_home, want, tol)
    for off in (1, 2, 3, 5):
        room = torch.full((q.numel() + 8,), 7.0, dtype=dtype, device=DEV)
        moved = room[off:off + q.numel()].view_as(q)
        moved.copy_(q)
        assert moved.data_ptr() % 16 != 0 and moved.is_contiguous()
        assert torch.equal(attention.attention_weights(moved, kc, R, 230, jl_rot=jl), at_home)


def visible64(q, kc, R, q_start, causal=True):
    """[B, Hkv, S] float64: each row's softmax over the positions that it sees, and
    nothing from it for the others, whatever it holds."""
    B, Hq, Sq, d = q.shape
    H, S = kc.num_heads, kc.seq_len
    x = (q.double() @ R.double().t() * d ** -0.5) @ decoded(kc).repeat_interleave(Hq // H, 1).transpose(2, 3)
    seen = torch.ones(Sq, S, dtype=torch.bool, device=DEV)
    if causal:
        seen = torch.arange(S, device=DEV) <= torch.arange(q_start, q_start + Sq, device=DEV)[:, None]
    w = torch.softmax(x.masked_fill(~seen, float("-inf")), -1).masked_fill(~seen, 0.0)
    return w.view(B, H, -1, S).sum(2)


def same(got, want, rel):
    """NaN in the same places; near elsewhere."""
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (torch.isnan(got).sum(), torch.isnan(want).sum())
    a, b = torch.nan_to_num(got.double()), torch.nan_to_num(want)
    assert bool(((a - b).abs() <= rel * b + 1e-37).all()), ((a - b).abs() - rel * b).max().item()


def spoil(cache, b, h, t, value):
    cache.blocks[b, h, t].view(-1, 18)[:, :2] = torch.tensor([value], device=DEV).half().view(torch.uint8)


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("S,at", [(65, 64), (65, 3), (1000, 999), (1000, 500), (4097, 4096), (1, 0)])
@pytest.mark.parametrize("paged", [False, True])
def test_decode_weights_with_a_key_that_is_not_a_number(S, at, paged):
    """One NaN logit makes all weights of its rows NaN, wherever it stands among
    the splits, and no others."""
    q, kc, vc, R, _ = make(2, 14, 2, S, 128, 4, False)
    _, clean = attention.decode_attention_weights(q, kc, vc, R)
    spoil(kc, 1, 0, at, NAN)
    k, v = (paged_copy(c, 64) if paged else c for c in (kc, vc))
    out, w = attention.decode_attention_weights(q, k, v, R)
    assert bool(torch.isnan(w[1, 0]).all()) and bool(torch.isnan(out[1, :7]).all())
    keep = torch.ones(2, 2, dtype=torch.bool, device=DEV)
    keep[1, 0] = False
    assert torch.equal(w[keep], clean[keep]) and bool(torch.isfinite(out[0]).all() and torch.isfinite(out[1, 7:]).all())


@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_decode_weights_with_a_query_that_is_not_a_number(value):
    q, kc, vc, R, _ = make(2, 8, 2, 900, 64, 4, False)
    _, clean = attention.decode_attention_weights(q, kc, vc, R)
    q[0, 5, 17] = value
    _, w = attention.decode_attention_weights(q, kc, vc, R)
    assert bool(torch.isnan(w[0, 1]).all())
    assert torch.equal(w[0, 0], clean[0, 0]) and torch.equal(w[1], clean[1])


@pytest.mark.parametrize("heads", [9, 11, 13, 17])
def test_groups_that_divide_into_uneven_launches(heads):
    q, kc, vc, R, _ = make(1, 2 * heads, 2, 700, 128, 4, False)
    want, tol, _ = exact(q.unsqueeze(2), kc, R)
    out, w = attention.decode_attention_weights(q, kc, vc, R)
    close(w, want, tol)
    assert torch.equal(out, attention.decode_attention(q, kc, vc, R))


def test_callers_page_tables_of_different_widths():
    """The caller's tables are read as they are at each call."""
    q, kc, vc, R, _ = make(1, 4, 2, 150, 64, 4, False)
    want, w = attention.decode_attention_weights(q, kc, vc, R)
    kp, vp = paged_copy(kc, 64), paged_copy(vc, 64)
    wide = torch.nn.functional.pad(vp.table, (0, 5))
    vp.adopt(wide, vp.capacity, vp._adopted[1])
    vp.seq_len = 150
    narrow = kp.table
    for i in range(2):
        out, got = attention.decode_attention_weights(q, kp, vp, R)
        assert torch.equal(out, want) and torch.equal(got, w) and kp.table is narrow and vp.table is wide
        assert torch.equal(attention.decode_attention(q, kp, vp, R), want)
        a, b = (attention.prefill_attention(q.unsqueeze(2), k, v, R, 149) for k, v in ((kp, vp), (kc, vc)))
        assert torch.equal(a, b)
        moved = torch.cat([g.reshape(-1) for g in kp._adopted[1]])         # the owner moves its pages
        narrow += moved.data_ptr() - kp._adopted[1][0].data_ptr()
        kp._adopted = (kp._adopted[0], [moved.view_as(kp._adopted[1][0])])


CHUNKS = [
    # Hq, Hkv, Sq, q_start, S, d
    (4, 2, 33, 0, 33, 64), (14, 2, 65, 190, 255, 128), (8, 8, 16, 113, 129, 64), (12, 4, 40, 100, 600, 128),
    (2, 1, 1100, 100, 1200, 64), (32, 8, 300, 700, 1000, 128),
]


@pytest.mark.parametrize("case", CHUNKS, ids=["Hq{}_Hkv{}_Sq{}_at{}_S{}_d{}".format(*c) for c in CHUNKS])
def test_chunk_weights_with_a_key_that_is_not_a_number(case):
    Hq, Hkv, Sq, q_start, S, d = case
    q, kc, _, R, _ = make(2, Hq, Hkv, S, d, 4, False, Sq=Sq)
    total, tol, _ = exact(q, kc, R, q_start, causal=False)
    rel = (tol / total).max()                                    # one factor bounds every element's error
    clean = attention.attention_weights(q, kc, R, q_start)
    end = q_start + Sq
    places = {0, q_start, end - 1, end - 2, min(end // 2 + 1, end - 1)} | {t for t in (end, end + 3, end + 40, S - 1) if t < S}
    for at in sorted(places):
        other = make(2, Hq, Hkv, S, d, 4, False, Sq=Sq)[1]
        spoil(other, 1, Hkv - 1, at, NAN)
        got = attention.attention_weights(q, other, R, q_start)
        same(got, visible64(q, other, R, q_start), rel)
        if at >= end:                                            # no row sees it
            assert torch.equal(got, clean)
        got = attention.attention_weights(q, other, R, q_start, causal=False)
        same(got, visible64(q, other, R, q_start, False), rel)


@pytest.mark.parametrize("value", [NAN, INF])
@pytest.mark.parametrize("case", CHUNKS, ids=["Hq{}_Hkv{}_Sq{}_at{}_S{}_d{}".format(*c) for c in CHUNKS])
def test_chunk_weights_with_a_query_that_is_not_a_number(case, value):
    """A row that is not a number spoils the positions that it sees and no others."""
    Hq, Hkv, Sq, q_start, S, d = case
    q, kc, _, R, _ = make(2, Hq, Hkv, S, d, 4, False, Sq=Sq)
    total, tol, _ = exact(q, kc, R, q_start, causal=False)
    rel = (tol / total).max()
    for row in sorted({0, Sq // 2, Sq - 1}):
        broken = q.clone()
        broken[1, Hq - 1, row, 5] = value
        got = attention.attention_weights(broken, kc, R, q_start)
        assert bool(torch.isnan(got[1, Hkv - 1, :q_start + row + 1]).all())
        assert not torch.isnan(got[1, Hkv - 1, q_start + row + 1:]).any()
        same(got, visible64(broken, kc, R, q_start), rel)
        assert bool(torch.isnan(attention.attention_weights(broken, kc, R, q_start, causal=False)[1, Hkv - 1]).all())


@pytest.mark.parametrize("value", [NAN, INF, 60000.0])
@pytest.mark.parametrize("qjl", [False, True])
def test_chunk_weights_do_not_depend_on_keys_that_no_row_sees(value, qjl):
    """Later positions in the same block of tokens: equal, not near."""
    q, kc, _, R, jl = make(2, 12, 4, 600, 128, 4, qjl, Sq=43)
    clean = attention.attention_weights(q, kc, R, 100, jl_rot=jl)
    for at in (143, 144, 150, 255, 256, 599):
        _, other, _, _, _ = make(2, 12, 4, 600, 128, 4, qjl, Sq=43)
        for h in range(4):
            spoil(other, 1, h, at, value)
        assert torch.equal(attention.attention_weights(q, other, R, 100, jl_rot=jl), clean)


PASSES = [
    # B, Hq, Hkv, Sq, q_start, d, qjl, rows of a pass with the least workspace
    (4, 14, 2, 2400, 0, 64, False, 16384), (4, 14, 2, 2400, 37, 64, True, 8192), (8, 3, 1, 2800, 100, 128, True, 4096),
]


def rows_with_peaks(B, Hq, Hkv, Sq, q_start, d, qjl, rows, dev):
    """Keys of one length in random directions; the first and last rows of each
    pass of `rows` rows look at one key each, the others at all alike:
    (queries, cache, R, jl_rot, [(row, its key)])."""
    G, S = Hq // Hkv, q_start + Sq
    assert G * Sq > rows and (rows % G or G == 1)
    g = torch.Generator().manual_seed(rows)
    blocks = torch.randint(0, 256, (B, Hkv, S, d // 32, 18), generator=g, dtype=torch.uint8)
    blocks[..., :2] = torch.tensor([8.0]).half().view(torch.uint8)
    signs = torch.randint(0, 256, (B, Hkv, S, d // 8), generator=g, dtype=torch.uint8).to(dev) if qjl else None
    kc = PQCache(blocks=blocks.flatten(3).to(dev), head_dim=d, n_bits=4, seq_len=S, max_seq_len=S,
                 codebooks=padded_codebook_torch(d, 4, dev), qjl_signs=signs, jl_dim=d if qjl else 0)
    R = generate_rotation_matrix(d, seed=42, device=dev)
    jl = rotated_jl_matrix(generate_jl_matrix(d, d, seed=43), R.cpu().numpy(), dev) if qjl else None
    q = (0.25 * torch.randn(B, Hq, Sq, d, generator=g)).half().to(dev)
    keys, peaks = decoded(kc), []
    for edge in list(range(rows, G * Sq, rows)) + [G * Sq]:
        for r in range(edge - 2, min(edge + 2, G * Sq)):
            at = 5 + 17 * len(peaks)
            assert at <= q_start + r // G                        # the row sees it
            k = keys[:, :, at] @ R.double()                      # in the queries' space
            q[:, r % G::G, r // G] = (14 * d ** 0.5 * k / k.square().sum(-1, keepdim=True)).half()
            peaks.append((r, at))
    return q, kc, R, jl, peaks


@pytest.mark.parametrize("case", PASSES, ids=["B{}_Hq{}_Hkv{}_Sq{}_at{}_d{}_{}".format(*c[:6], "qjl" if c[6] else "plain")
                                              for c in PASSES])
def test_rows_at_the_border_of_two_passes(case, monkeypatch):
    """Every row counts once."""
    B, Hq, Hkv, Sq, q_start, d, qjl, rows = case
    G, S = Hq // Hkv, q_start + Sq
    q, kc, R, jl, peaks = rows_with_peaks(*case, DEV)
    want, tol, w = exact(q, kc, R, q_start, jl_rot=jl)
    w = w.view(B, Hkv, G, Sq, S)
    for r, at in peaks:                                          # one lost or counted twice would be seen there
        assert bool((w[:, :, r % G, r // G, at] > 2 * tol[:, :, at]).all())
    del w
    whole = attention.attention_weights(q, kc, R, q_start, jl_rot=jl)
    close(whole, want, tol)
    monkeypatch.setattr(_lib, "workspace", lambda best, least, device: torch.empty(least(), dtype=torch.uint8, device=device))
    close(attention.attention_weights(q, kc, R, q_start, jl_rot=jl), want, tol)
    previous = torch.rand(B, Hkv, S + 3, device=DEV)
    into = previous.clone()
    apart = attention.attention_weights(q, kc, R, q_start, jl_rot=jl, previous=previous)
    attention.attention_weights(q, kc, R, q_start, jl_rot=jl, previous=into, into=into)
    assert torch.equal(into[:, :, :S], apart) and torch.equal(into[:, :, S:], previous[:, :, S:])
    # (each pass's addition to a sum of at most want + 1 rounds by half a step)
    close(apart, want + previous[:, :, :S].double(), tol + 8 * (want + 1.0) * 2.0 ** -24)


def test_no_room_for_the_workspace_of_one_pass(monkeypatch):
    q, kc, _, R, _ = make(4, 14, 2, 2400, 64, 4, False, Sq=2400)
    want, tol, _ = exact(q, kc, R, 0)
    least, real, refused = _lib.lib().pqkv_attn_weights_workspace_least_bytes(4, 14, 2, 2400, 2400, 64, 0), torch.empty, []

    def empty(*size, **kw):
        if len(size) == 1 and size[0] > least:
            refused.append(size[0])
            raise torch.cuda.OutOfMemoryError("out of memory")
        return real(*size, **kw)

    monkeypatch.setattr(torch, "empty", empty)
    got = attention.attention_weights(q, kc, R, 0)
    assert refused
    close(got, want, tol)


def test_tables_are_not_replaced_within_a_capture(monkeypatch):
    q, kc, vc, R, _ = make(1, 4, 2, 150, 64, 4, False)
    want, w = attention.decode_attention_weights(q, kc, vc, R)
    pair = []
    for c, pages in ((kc, 3), (vc, 7)):
        p = PagedPQCache(1, 2, 64, 4, c.codebooks, DEV, page_tokens=64, max_pages=pages)
        p.ensure(150)
        for i, group in enumerate(p.groups):
            n = min(64, 150 - 64 * i)
            group[:, :, :n] = c.blocks[:, :, 64 * i:64 * i + n]
        p.seq_len = 150
        pair.append(p)
    before = pair[0].table
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before a capture"):
        attention.decode_attention_weights(q, *pair, R)
    assert pair[0].table is before
    monkeypatch.undo()
    for capturing in (False, True):                              # widths are one after the first call
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
        out, got = attention.decode_attention_weights(q, *pair, R)
        assert torch.equal(out, want) and torch.equal(got, w)
