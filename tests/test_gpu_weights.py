"""Attention weights of cached positions against the definition in 64 bits on
the decoded bytes of the cache, and the decode output beside them.

Tolerance: a logit is a sum of d products (and d signed projections with QJL)
whose terms carry a relative error below 2^-21 (queries rotated in 32 bits,
split operands) and which is accumulated in 32 bits in some order, at most
2^-24 of the sum of the terms' sizes per addition. With A the largest sum of
sizes over a call's scores, a logit is off by at most
e = (2^-21 + 2 d 2^-24) A, a weight by a factor within exp(2 e) (numerator and
denominator) of its own, and the sums over rows, at most n terms, add n 2^-24
relative. Rotating the query first sums d products again: another d 2^-24 A."""

import math

import numpy as np
import pytest
import torch

from oracle import oracle as O
from polarquant_kv import attention, quantizer
from polarquant_kv.lloyd_max import padded_codebook_torch
from polarquant_kv.qjl import generate_jl_matrix, rotated_jl_matrix
from polarquant_kv.rotation import generate_rotation_matrix
from polarquant_kv.types import PagedPQCache, PQCache

from test_gpu_evict import paged_copy

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def decoded(cache):
    """Rotated states [B, H, S, d] of a contiguous cache, float64."""
    d, bits, S = cache.head_dim, cache.n_bits, cache.seq_len
    x = cache.blocks[:, :, :S].reshape(*cache.blocks.shape[:2], S, d // 32, -1)
    r = x[..., 0, :2].contiguous().view(torch.float16).double()
    parts = [(x[..., 2:] >> (bits * j)) & ((1 << bits) - 1) for j in range(8 // bits)]
    code = torch.stack(parts, -1).flatten(3).long()
    return cache.codebooks.double()[code] * r


def exact(q, kc, R, q_start=None, causal=True, jl_rot=None, scale=None):
    """(weights [B, Hkv, S], their bound per element, softmax [B, Hq, Sq, S]) of q [B, Hq, Sq, d]."""
    B, Hq, Sq, d = q.shape
    H, S = kc.num_heads, kc.seq_len
    G = Hq // H
    scale = d ** -0.5 if scale is None else scale
    k = decoded(kc).repeat_interleave(G, 1)
    qr = q.double() @ R.double().t() * scale
    x = qr @ k.transpose(2, 3)
    # |q_rot| <= sum |q| |R|: the sizes of both products' terms
    size = ((q.double().abs() @ R.double().abs().t() * scale) @ k.abs().transpose(2, 3)).amax().item()
    if jl_rot is not None:
        signs = kc.qjl_signs[:, :, :S]
        bits = (signs[..., None] >> torch.arange(8, device=DEV, dtype=torch.uint8)) & 1
        sign = (bits.flatten(3).double() * 2 - 1) * (signs != 255).any(-1, keepdim=True)
        p = qr @ jl_rot.double().t() / d
        x = x + p @ sign.repeat_interleave(G, 1).transpose(2, 3)
        size += (q.double().abs() @ R.double().abs().t() * scale @ jl_rot.double().abs().t() / d).sum(-1).amax().item()
    if q_start is not None and causal:
        at = torch.arange(q_start, q_start + Sq, device=DEV)
        x = x.masked_fill(torch.arange(S, device=DEV) > at[:, None], float("-inf"))
    w = torch.softmax(x, -1)
    total = w.view(B, H, G * Sq, S).sum(2)
    e = (2.0 ** -21 + 3 * d * 2.0 ** -24) * size
    return total, total * (math.exp(2 * e) - 1 + (G * Sq + 64) * 2.0 ** -24) + 1e-37, w


def close(got, want, tol):
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), ((err - tol).max().item(), err.max().item())
    # and as a whole far nearer than the worst case of every element
    assert (err.norm() / want.norm().clamp(min=1e-30)).item() < 2e-5


def make(B, Hq, Hkv, S, d, bits, qjl, seed=1, Sq=None, own_values=False, S_max=None, qscale=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    R = generate_rotation_matrix(d, seed=42, device=DEV)
    jl_rot = rotated_jl_matrix(generate_jl_matrix(d, d, seed=43), R.cpu().numpy(), DEV) if qjl else None
    k = torch.from_numpy(O.synth_kv(B, Hkv, S, d, seed, "channel")).to(DEV)
    v = torch.from_numpy(O.synth_kv(B, Hkv, S, d, seed + 1)).to(DEV)
    S_max = S if S_max is None else S_max
    kc = quantizer.allocate_cache(B, Hkv, S_max, d, bits, DEV, jl_dim=d if qjl else 0)
    vc = quantizer.allocate_cache(B, Hkv, S_max, d, bits, DEV)
    quantizer.compress_pq(k, R, cache=kc, jl_rot=jl_rot)
    quantizer.compress_pq(v, R, cache=vc)
    if qjl and S > 3:
        kc.qjl_signs[:, :, 2] = 255                        # a zero residual
    if not own_values:
        vc.codebooks = kc.codebooks
    else:
        vc.codebooks = padded_codebook_torch(d, bits, DEV) * 1.5
    shape = (B, Hq, d) if Sq is None else (B, Hq, Sq, d)
    q = (qscale * torch.randn(*shape, generator=g, device=DEV)).half()
    return q, kc, vc, R, jl_rot


DECODE = [
    # B, Hq, Hkv, S, d, bits, qjl
    (1, 1, 1, 1, 64, 4, False), (1, 14, 2, 512, 64, 4, False), (2, 32, 8, 1000, 128, 4, False),
    (1, 8, 8, 63, 128, 2, False), (2, 4, 2, 64, 64, 2, True), (1, 12, 4, 65, 128, 4, True), (1, 5, 1, 3001, 128, 4, True),
    (3, 12, 2, 777, 64, 2, False), (1, 16, 2, 4099, 128, 4, False), (1, 20, 1, 300, 64, 4, True),
    (1, 64, 8, 9001, 128, 2, True), (8, 32, 8, 257, 128, 4, False), (1, 24, 1, 130, 128, 4, False),
]
dec_ids = ["B{}_Hq{}_Hkv{}_S{}_d{}_b{}_{}".format(*c[:6], "qjl" if c[6] else "plain") for c in DECODE]


@pytest.mark.parametrize("case", DECODE, ids=dec_ids)
def test_decode_weights(case):
    B, Hq, Hkv, S, d, bits, qjl = case
    for own in (False, True):
        q, kc, vc, R, jl_rot = make(*case, own_values=own, S_max=S + 11)
        want, tol, _ = exact(q.unsqueeze(2), kc, R, jl_rot=jl_rot)
        out, w = attention.decode_attention_weights(q, kc, vc, R, jl_rot=jl_rot, out_dtype=torch.float32)
        assert w.shape == (B, Hkv, S) and w.dtype == torch.float32
        close(w, want, tol)
        assert torch.equal(out, attention.decode_attention(q, kc, vc, R, jl_rot=jl_rot, out_dtype=torch.float32))
        out2, w2 = attention.decode_attention_weights(q, kc, vc, R, jl_rot=jl_rot, out_dtype=torch.float32)
        assert torch.equal(out, out2) and torch.equal(w, w2)
        page = 64 if S < 500 else 256
        kp, vp = paged_copy(kc, page), paged_copy(vc, page)
        outp, wp = attention.decode_attention_weights(q, kp, vp, R, jl_rot=jl_rot, out_dtype=torch.float32)
        assert torch.equal(out, outp) and torch.equal(w, wp)


def test_decode_weights_accumulate_in_place_and_apart():
    q, kc, vc, R, _ = make(2, 8, 2, 700, 128, 4, False)
    _, w = attention.decode_attention_weights(q, kc, vc, R)
    room = torch.full((2, 2, 1003), -7.0, device=DEV)      # 1003: rows off a 16-byte boundary
    room[:, :, :700] = torch.rand(2, 2, 700, device=DEV)
    before = room.clone()
    _, got = attention.decode_attention_weights(q, kc, vc, R, previous=room, into=room)
    assert got.data_ptr() == room.data_ptr() and torch.equal(got, before[:, :, :700] + w)
    assert torch.equal(room[:, :, 700:], before[:, :, 700:])
    _, fresh = attention.decode_attention_weights(q, kc, vc, R, previous=before[:, :, :700])
    assert torch.equal(fresh, got)
    into = torch.empty(2, 2, 800, device=DEV)
    attention.decode_attention_weights(q, kc, vc, R, previous=before, into=into)
    assert torch.equal(into[:, :, :700], got)
    for bad in (into.transpose(0, 1), into[:, :, ::2], into[:, :, :699], into.double()):
        with pytest.raises(ValueError):
            attention.decode_attention_weights(q, kc, vc, R, into=bad)
    with pytest.raises(RuntimeError):                       # rows of the same memory, shifted
        attention.decode_attention_weights(q, kc, vc, R, previous=room[:, :, 1:701], into=room)


def test_decode_weights_of_an_empty_cache():
    q, kc, vc, R, _ = make(2, 4, 2, 5, 64, 4, False)
    kc.seq_len = vc.seq_len = 0
    out, w = attention.decode_attention_weights(q, kc, vc, R)
    assert w.shape == (2, 2, 0) and not out.any()
    into = torch.full((2, 2, 9), 3.0, device=DEV)
    attention.decode_attention_weights(q, kc, vc, R, into=into)
    assert bool((into == 3.0).all())


def test_decode_weights_peaked_logits():
    """One key far ahead: its weight is G, the others' next to nothing; and
    logits that leave exp's range."""
    q, kc, vc, R, _ = make(1, 4, 1, 400, 128, 4, False, qscale=40.0)
    want, tol, _ = exact(q.unsqueeze(2), kc, R)
    _, w = attention.decode_attention_weights(q, kc, vc, R)
    assert bool(((w.double() - want).abs() <= tol).all()) and bool(torch.isfinite(w).all())
    assert abs(w.sum().item() - 4.0) < 1e-4


CHUNK = [
    # B, Hq, Hkv, Sq, q_start, d, bits, qjl
    (1, 1, 1, 1, 0, 64, 4, False), (1, 4, 2, 2, 0, 64, 4, False), (1, 8, 2, 33, 0, 128, 4, False),
    (2, 14, 2, 65, 190, 64, 4, False), (1, 12, 4, 257, 1000, 128, 2, True), (1, 6, 1, 100, 255, 128, 4, True),
    (2, 8, 8, 16, 700, 64, 2, False), (1, 32, 8, 32, 5000, 128, 4, False), (1, 20, 1, 31, 30, 64, 4, True),
    (1, 2, 2, 1030, 0, 128, 4, False), (1, 16, 1, 300, 511, 64, 2, True), (3, 3, 1, 1, 256, 128, 4, False),
    (1, 9, 1, 513, 3, 64, 4, False), (1, 2, 1, 2100, 100, 64, 4, False),
]
chunk_ids = ["B{}_Hq{}_Hkv{}_Sq{}_at{}_d{}_b{}_{}".format(*c[:7], "qjl" if c[7] else "plain") for c in CHUNK]


@pytest.mark.parametrize("case", CHUNK, ids=chunk_ids)
def test_chunk_weights(case):
    B, Hq, Hkv, Sq, q_start, d, bits, qjl = case
    S = q_start + Sq
    q, kc, vc, R, jl_rot = make(B, Hq, Hkv, S, d, bits, qjl, Sq=Sq, S_max=S + 3)
    prev = torch.rand(B, Hkv, S + 5, device=DEV)
    kp = paged_copy(kc, 64 if S < 1000 else 256)
    for causal in (True, False):
        want, tol, _ = exact(q, kc, R, q_start, causal, jl_rot)
        w = attention.attention_weights(q, kc, R, q_start, causal=causal, jl_rot=jl_rot)
        close(w, want, tol)
        assert torch.equal(w, attention.attention_weights(q, kp, R, q_start, causal=causal, jl_rot=jl_rot))
        keep = prev.clone()
        got = attention.attention_weights(q, kc, R, q_start, causal=causal, jl_rot=jl_rot, previous=keep, into=keep)
        assert torch.equal(got, prev[:, :, :S] + w) and torch.equal(keep[:, :, S:], prev[:, :, S:])


def test_chunk_weights_earlier_queries_and_float_queries():
    """Queries that stand before the cache's end: positions after them get
    nothing from them."""
    q, kc, vc, R, _ = make(1, 4, 2, 600, 128, 4, False, Sq=40)
    want, tol, _ = exact(q, kc, R, 100, True)
    w = attention.attention_weights(q, kc, R, 100)
    close(w, want, tol)
    assert not w[:, :, 140:].any()
    f = attention.attention_weights(q.float(), kc, R, 100)
    assert torch.equal(f, w)
    s = attention.attention_weights(q, kc, R, 100, scale=0.3)
    want, tol, _ = exact(q, kc, R, 100, True, scale=0.3)
    close(s, want, tol)


def test_chunk_weights_nothing_to_add():
    q, kc, vc, R, _ = make(1, 4, 2, 90, 64, 4, False, Sq=4)
    none = attention.attention_weights(q[:, :, :0], kc, R, 90)
    assert none.shape == (1, 2, 90) and not none.any()
    prev = torch.rand(1, 2, 95, device=DEV)
    assert torch.equal(attention.attention_weights(q[:, :, :0], kc, R, 90, previous=prev), prev[:, :, :90])
    kc.seq_len = 0
    assert attention.attention_weights(q[:, :, :0], kc, R, 0).shape == (1, 2, 0)
    kc.seq_len = 90
    with pytest.raises(RuntimeError):
        attention.attention_weights(q, kc, R, 87)           # the last query is past the cache


def test_chunk_of_one_row_agrees_with_decode():
    q, kc, vc, R, jl_rot = make(2, 8, 2, 1200, 128, 4, True)
    _, w = attention.decode_attention_weights(q, kc, vc, R, jl_rot=jl_rot)
    c = attention.attention_weights(q.unsqueeze(2), kc, R, 1199, jl_rot=jl_rot)
    want, tol, _ = exact(q.unsqueeze(2), kc, R, jl_rot=jl_rot)
    assert bool(((w - c).double().abs() <= 2 * tol).all())


def test_long_chunk_in_passes():
    """A shape whose partials need more than one pass over the rows (the
    workspace holds at most 256 MB of them): passes add up to one another."""
    B, Hq, Hkv, Sq, d = 1, 64, 1, 600, 64
    S = 262144
    g = torch.Generator(device=DEV).manual_seed(9)
    blocks = torch.randint(0, 256, (B, Hkv, S, 36), generator=g, device=DEV, dtype=torch.uint8)
    blocks.view(B, Hkv, S, 2, 18)[..., :2] = torch.tensor([8.0], device=DEV).half().view(torch.uint8)
    kc = PQCache(blocks=blocks, head_dim=d, n_bits=4, seq_len=S, max_seq_len=S,
                 codebooks=padded_codebook_torch(d, 4, DEV))
    R = generate_rotation_matrix(d, seed=42, device=DEV)
    q = torch.randn(B, Hq, Sq, d, generator=g, device=DEV).half()
    w = attention.attention_weights(q, kc, R, S - Sq)
    assert abs(w.double().sum().item() - Hq * Sq) < 1e-4 * Hq * Sq
    part = torch.zeros(B, Hkv, S, device=DEV)
    for i in range(0, Sq, 150):                              # the same rows in calls of their own
        part = attention.attention_weights(q[:, :, i:i + 150], kc, R, S - Sq + i, previous=part)
    # other grouping of the same additions: 600 x 64 terms
    assert bool(((w - part).double().abs() <= part.double() * 38400 * 2.0 ** -23).all())


def test_on_another_stream_and_captured():
    q, kc, vc, R, _ = make(1, 8, 2, 900, 128, 4, False)
    qc = torch.randn(1, 8, 20, 128, device=DEV).half()
    acc = torch.zeros(1, 2, 1000, device=DEV)

    def step():
        out, _ = attention.decode_attention_weights(q, kc, vc, R, previous=acc, into=acc)
        w = attention.attention_weights(qc, kc, R, 880)
        return out, w

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    s.synchronize()
    acc.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, w = step()
    want = torch.zeros_like(acc)
    for _ in range(4):
        q.copy_(torch.randn_like(q))
        qc.copy_(torch.randn_like(qc))
        graph.replay()
        o, _ = attention.decode_attention_weights(q, kc, vc, R, previous=want, into=want)
        torch.cuda.synchronize()
        assert torch.equal(out, o) and torch.equal(acc, want)
        assert torch.equal(w, attention.attention_weights(qc, kc, R, 880))


def test_calls_on_two_streams_at_once():
    """Each call has its own workspace: calls that overlap give what they give alone."""
    work = [make(2, 16, 4, 3000 + 500 * i, 128, 4, bool(i), seed=5 + i) for i in range(2)]
    chunk = [torch.randn(2, 16, 70, 128, device=DEV).half() for _ in work]

    def step(i):
        q, kc, vc, R, jl = work[i]
        out, w = attention.decode_attention_weights(q, kc, vc, R, jl_rot=jl)
        return out, w, attention.attention_weights(chunk[i], kc, R, kc.seq_len - 70, jl_rot=jl, previous=w)

    alone = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(5):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(step(i))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_unequal_widths_and_missing_signs_are_refused():
    q, kc, vc, R, _ = make(1, 4, 2, 50, 64, 4, False)
    _, k2, _, _, _ = make(1, 4, 2, 50, 64, 2, False)
    with pytest.raises(ValueError):
        attention.decode_attention_weights(q, kc, k2, R)
    with pytest.raises(ValueError):
        attention.decode_attention_weights(q, kc, vc, R, jl_rot=R)
    with pytest.raises(ValueError):
        attention.attention_weights(q.unsqueeze(2), kc, R, 49, jl_rot=R)
    with pytest.raises(TypeError):
        attention.decode_attention_weights(q.bfloat16(), kc, vc, R)
    assert isinstance(paged_copy(kc, 64), PagedPQCache) and np.isfinite(kc.codebooks.cpu().numpy()).all()
