"""pqkv_append_rotary and _paged through append.append_rotary against the formula
in 64 bits.

Tolerance of a direction y_j / r, from the roundings: two splits into 22 bits
(2^-21 of |R_j| |x| = r, by Cauchy), 3 x 128 fp32 sums (a random walk of half
steps, 4 standard deviations: 4 sqrt(384) 2^-25 < 2^-18.7), the turn (2^-20
(|x_a| + |x_b|), less than 2^-19.5 of the norm), the quotient 2^-23: less than
2^-17 in all. So a code's centroid is at most 2 x 2^-17 further from the direction
than the nearest one, a radius within 2^-17 + 2^-11 (its rounding to fp16), and a
sign may only differ where |(P e)_i| is below what errors of 2^-17 in each of e's
coordinates can do, |P_i|_1 2^-17."""

import pytest
import torch

import window_ref
from polarquant_kv import append, quantizer, rotary, rotation
from polarquant_kv.types import PagedPQCache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
OFF = 2.0 ** -17


def turned(x, positions, freqs, axes, interleaved, m):
    """x [B, H, T, d] float64; positions [B, T] or [A, B, T]."""
    n = freqs.numel()
    at = [positions if axes is None else positions[axes[i]] for i in range(n)]
    t = torch.stack([(p.double() if p.dim() == 2 else p.double()[None].expand(x.shape[0], -1)) * freqs[i]
                     for i, p in enumerate(at)], -1)[:, None]
    x = x.double().clone()
    ia = torch.arange(n, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else n)
    a, b = x[..., ia], x[..., ib]
    x[..., ia], x[..., ib] = m * (a * t.cos() - b * t.sin()), m * (a * t.sin() + b * t.cos())
    return x


def codes_of(blocks, bits):
    x = blocks.reshape(*blocks.shape[:-1], -1, window_ref.BLOCK_BYTES[bits])
    r = x[..., :2].contiguous().view(torch.float16)
    assert torch.equal(r.view(torch.int16), r[..., :1, :].view(torch.int16).expand_as(r))    # one radius in every block
    parts = [(x[..., 2:] >> (bits * j)) & ((1 << bits) - 1) for j in range(8 // bits)]
    return r[..., 0, 0].double(), torch.stack(parts, -1).flatten(-3).long()


def check_vectors(blocks, x, R, codebook, bits):
    """Blocks [..., bytes] hold x [..., d] (float64); returns the residuals in units of the radius."""
    y = x @ R.double().t()
    r = y.norm(dim=-1)
    got_r, code = codes_of(blocks, bits)
    assert bool(((got_r - r).abs() <= r * (OFF + 2.0 ** -11) + 2.0 ** -25).all())
    cb = codebook.double().flatten()[:1 << bits]
    u = y / r[..., None]
    gap = (u[..., None] - cb).abs()
    mine = gap.gather(-1, code[..., None])[..., 0]
    assert bool((mine <= gap.amin(-1) + 2 * OFF).all())
    # and hardly ever not the nearest one at all: 15 borders 2 OFF wide of a range of 0.4
    assert float((mine > gap.amin(-1)).double().mean()) <= 15 * 2 * OFF / 0.4
    return u - cb[code]


def check_signs(signs, e, P):
    bits = ((signs[..., None].int() >> torch.arange(8, device=signs.device).int()) & 1).flatten(-2).bool()
    pe = e @ P.double().t()
    unsure = pe.abs() <= P.double().abs().sum(-1) * OFF
    assert bool(((bits == (pe >= 0)) | unsure).all())
    assert float(unsure.double().mean()) < 0.01


# B, Hq, Hkv, T, S, d, rot, bits, qjl, page, dtype, interleaved, sections, starts, counts
CASES = [
    (1, 1, 1, 1, 1, 64, 64, 4, False, 0, torch.float16, False, None, 0, None),
    (8, 32, 8, 1, 300, 128, 128, 4, False, 256, torch.float16, False, None, [299, 0, 17, 64, 255, 256, 128, 5], None),
    (3, 4, 2, 1, 70, 128, 128, 2, True, 64, torch.bfloat16, True, (20, 22, 22), [69, 3, 0], None),
    (5, 2, 1, 3, 100, 64, 48, 4, True, 0, torch.float32, False, None, [97, 0, 10, 60, 33], [3, 2, 1, 0, 3]),
    (2, 14, 2, 33, 300, 64, 48, 2, False, 0, torch.float32, True, None, 267, None),
    (2, 14, 2, 509, 1500, 64, 64, 4, True, 64, torch.float16, False, (16, 16), [991, 3], [509, 100]),
    (1, 8, 8, 257, 600, 128, 96, 4, False, 256, torch.bfloat16, False, (24, 16, 8), 100, None),
    (2, 7, 7, 20, 64, 128, 42, 4, True, 0, torch.float16, False, None, [44, 0], None),       # odd pair count
    (2, 3, 3, 16, 40, 128, 128, 4, False, 0, torch.float16, True, (30, 34), 24, None),
    (1, 40, 40, 5, 5, 64, 2, 4, False, 0, torch.float32, False, None, 0, None),              # one pair
    (3, 4, 1, 1000, 1024, 128, 128, 2, False, 1024, torch.float16, False, None, [24, 0, 7], [1000, 999, 17]),
    (70, 2, 2, 2, 9, 64, 64, 4, True, 0, torch.bfloat16, False, None, 7, None),
]


def make(case, seed=3):
    B, Hq, Hkv, T, S, d, rot, bits, qjl, page, dtype, inter, sections, starts, counts = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda n: torch.randn(B, T, n, d, generator=g, device=DEV).to(dtype).transpose(1, 2)  # noqa: E731
    q, k, v = rand(Hq), rand(Hkv), rand(Hkv)
    k, v = k * 3, v * 0.01
    R = rotation.generate_rotation_matrix(d, seed=42, device=DEV)
    P = torch.randn(d, d, generator=g, device=DEV) if qjl else None
    caches = []
    for jl in (d if qjl else 0, 0):
        if page:
            c = quantizer.allocate_paged_cache(B, Hkv, d, bits, DEV, page_tokens=page, jl_dim=jl)
            c.ensure(S)
            for grp in c.groups + c.sign_groups:
                grp.random_(0, 256, generator=g)
        else:
            c = quantizer.allocate_cache(B, Hkv, S, d, bits, DEV, jl_dim=jl)
            c.blocks.random_(0, 256, generator=g)
            if jl:
                c.qjl_signs.random_(0, 256, generator=g)
        c.seq_len = S if isinstance(starts, list) else 0
        caches.append(c)
    freqs = rotary.rotary_frequencies(rot)[0].to(DEV)
    axes = None if sections is None else rotary.axis_of_pairs(sections)
    shape = (B, T) if axes is None else (len(sections), B, T)
    positions = torch.randint(0, 100000, shape, generator=g, device=DEV)
    return q, k, v, caches[0], caches[1], R, P, positions, freqs, axes


def expand(x, B, default=None):
    return torch.tensor(x if isinstance(x, list) else [default if x is None else x] * B, device=DEV)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "B{}_{}-{}_T{}_S{}_d{}_rot{}_b{}_{}_p{}".format(*c[:10]))
def test_slots_hold_the_turned_vectors(case):
    B, Hq, Hkv, T, S, d, rot, bits, qjl, page, dtype, inter, sections, starts, counts = case
    q, k, v, keys, values, R, P, positions, freqs, axes = make(case)
    before = [[None if x is None else x.clone() for x in window_ref.rows_of(c)] for c in (keys, values)]
    at, n = expand(starts, B), expand(counts, B, T)
    m = 1.25
    got = append.append_rotary(k, v, keys, values, R, positions, freqs, query=q,
                               starts=at if isinstance(starts, list) else starts,
                               counts=None if counts is None else n, interleaved=inter, amplitude=m, axes=axes, jl_rot=P)
    plain = rotary.apply_rotary(q, None, positions, freqs, interleaved=inter, amplitude=m, axes=axes)[0]
    assert torch.equal(got, plain)
    t = torch.arange(T, device=DEV)
    b, t = torch.nonzero(t < n[:, None], as_tuple=True)
    slot = at[b] + t
    for which, x, old in (("keys", turned(k, positions, freqs, axes, inter, m), before[0]), ("values", v.double(), before[1])):
        c = keys if which == "keys" else values
        blocks, signs = window_ref.rows_of(c)
        e = check_vectors(blocks[b, :, slot], x[b, :, t], R, c.codebooks, bits)
        if signs is not None:
            check_signs(signs[b, :, slot], e, P)
        # everything else as it was
        for new, was in ((blocks, old[0]), (signs, old[1])):
            if new is not None:
                was[b, :, slot] = new[b, :, slot]
                assert torch.equal(new, was)
        assert c.seq_len == (S if isinstance(starts, list) else starts + T)


def test_like_turning_and_compressing():
    """In 32 bits nothing is rounded between the two, so the codes are those of both calls but for borders."""
    case = (2, 4, 2, 100, 100, 128, 128, 4, True, 0, torch.float32, False, None, 0, None)
    q, k, v, keys, values, R, P, positions, freqs, _ = make(case)
    append.append_rotary(k, v, keys, values, R, positions, freqs, starts=0, jl_rot=P)
    kt = rotary.apply_rotary(q, k, positions, freqs)[1]
    for x, c, p in ((kt, keys, P), (v.contiguous(), values, None)):
        want = quantizer.compress_pq(x, R, 4, jl_rot=p)
        (r0, c0), (r1, c1) = codes_of(c.blocks, 4), codes_of(want.blocks, 4)
        assert float((c0 != c1).double().mean()) <= 15 * 4 * OFF / 0.4
        assert bool(((r0 - r1).abs() <= r1 * (2 * OFF + 2.0 ** -10)).all())


@pytest.mark.parametrize("qjl", [False, True])
@pytest.mark.parametrize("bits", [4, 2])
def test_zeros_and_numbers_that_are_none(bits, qjl):
    case = (1, 1, 2, 40, 40, 64, 64, bits, qjl, 0, torch.float32, False, None, 0, None)
    q, k, v, keys, values, R, P, positions, freqs, _ = make(case)
    k, v = k.contiguous(), v.contiguous()
    fine = append.append_rotary(k, v, keys, values, R, positions, freqs, starts=0, jl_rot=P, query=q)
    clean = keys.blocks.clone(), values.blocks.clone()
    bad = {1: float("nan"), 5: float("inf"), 17: -float("inf")}
    k[:, :, 3] = v[:, :, 3] = 0.0
    for t, x in bad.items():
        k[:, :, t, 7] = v[:, :, t, 60] = x
    k[:, :, 20] *= 1e30
    v[:, :, 20] *= 1e-20
    k[:, :, 21] *= 1e-35
    append.append_rotary(k, v, keys, values, R, positions, freqs, starts=0, jl_rot=P)
    zero = quantizer.compress_pq(torch.zeros(1, 2, 1, 64, device=DEV), R, bits, jl_rot=P)
    for c, was in ((keys, clean[0]), (values, clean[1])):
        r, code = codes_of(c.blocks, bits)
        for t in bad:
            assert torch.isnan(r[:, :, t]).all() and not code[:, :, t].any()
        assert torch.equal(c.blocks[:, :, 3:4], zero.blocks)
        rest = [t for t in range(40) if t not in (*bad, 3, 20, 21)]
        assert torch.equal(c.blocks[:, :, rest], was[:, :, rest])
    (r, code), (_, was) = codes_of(keys.blocks, bits), codes_of(clean[0], bits)
    assert (r[:, :, 20] == 65504).all() and float((code[:, :, 20] != was[:, :, 20]).double().mean()) < 0.02
    assert torch.equal(keys.blocks[:, :, 21:22], zero.blocks)                # a norm below 1e-30 counts as zero
    (r, code), (_, was) = codes_of(values.blocks, bits), codes_of(clean[1], bits)
    assert not r[:, :, 20].any() and float((code[:, :, 20] != was[:, :, 20]).double().mean()) < 0.02
    if qjl:
        assert torch.equal(keys.qjl_signs[:, :, 3:4], zero.qjl_signs)
    assert fine is not None


def test_a_codebook_of_its_own_and_one_without_order():
    case = (1, 1, 2, 64, 64, 128, 128, 4, False, 0, torch.float16, False, None, 0, None)
    q, k, v, keys, values, R, P, positions, freqs, _ = make(case)
    values.codebooks = (values.codebooks * 1.3).contiguous()
    keys.codebooks = keys.codebooks.flip(0).contiguous()
    append.append_rotary(k, v, keys, values, R, positions, freqs, starts=0)
    check_vectors(keys.blocks, turned(k, positions, freqs, None, False, 1.0), R, keys.codebooks, 4)
    check_vectors(values.blocks, v.double(), R, values.codebooks, 4)


@pytest.mark.parametrize("page", [0, 64])
def test_slots_that_there_is_no_room_for(page):
    case = (5, 2, 2, 4, 128, 64, 64, 4, True, page, torch.float16, False, None, [-1, 126, 128, -2 ** 40, 2 ** 40], None)
    q, k, v, keys, values, R, P, positions, freqs, _ = make(case)
    before = [[None if x is None else x.clone() for x in window_ref.rows_of(c)] for c in (keys, values)]
    append.append_rotary(k, v, keys, values, R, positions, freqs, starts=expand(case[13], 5), jl_rot=P)
    for c, x, old in ((keys, turned(k, positions, freqs, None, False, 1.0), before[0]), (values, v.double(), before[1])):
        blocks, signs = window_ref.rows_of(c)
        check_vectors(blocks[1, :, 126:], x[1, :, :2], R, c.codebooks, 4)
        for new, was in ((blocks, old[0]), (signs, old[1])):
            if new is not None:
                was[1, :, 126:] = new[1, :, 126:]
                assert torch.equal(new, was)
    none = torch.zeros(5, dtype=torch.int64, device=DEV)
    append.append_rotary(k, v, keys, values, R, positions, freqs, starts=none, counts=none - 3, jl_rot=P)
    assert torch.equal(window_ref.rows_of(keys)[0], before[0][0])


@pytest.mark.parametrize("T", [1, 40])
def test_a_cache_without_a_page(T):
    g = torch.Generator(device=DEV).manual_seed(7)
    q, k, v = (torch.randn(2, h, T, 128, generator=g, device=DEV).half() for h in (4, 2, 2))
    R = rotation.generate_rotation_matrix(128, seed=42, device=DEV)
    keys, values = (quantizer.allocate_paged_cache(2, 2, 128, 4, DEV, page_tokens=64) for _ in range(2))
    freqs, _ = rotary.rotary_frequencies(128)
    freqs, positions = freqs.to(DEV), torch.arange(T, device=DEV)
    out = append.append_rotary(k, v, keys, values, R, positions, freqs, query=q, starts=expand([0, 3], 2))
    assert torch.equal(out, rotary.apply_rotary(q, None, positions, freqs)[0])
    assert keys.capacity == values.capacity == keys.seq_len == 0


def test_captured_appends_follow_their_starts():
    case = (3, 4, 2, 1, 200, 128, 128, 4, False, 64, torch.float16, False, None, [10, 63, 150], None)
    q, k, v, keys, values, R, P, positions, freqs, _ = make(case)
    other = make(case)[3:5]
    at = expand(case[13], 3)
    args = (R, positions, freqs)
    append.append_rotary(k, v, keys, values, *args, query=q, starts=at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = append.append_rotary(k, v, keys, values, *args, query=q, starts=at)
    append.append_rotary(k, v, *other, *args, query=q, starts=at)
    for _ in range(4):
        for x in (k, v, q):
            x.normal_()
        at += 7
        positions += 7
        graph.replay()
        kept = got.clone()
        want = append.append_rotary(k, v, *other, *args, query=q, starts=at)
        torch.cuda.synchronize()
        assert torch.equal(kept, want)
        for a, b in zip((keys, values), other):
            assert torch.equal(window_ref.rows_of(a)[0], window_ref.rows_of(b)[0])


def test_growing_caches_and_refusals():
    d = 64
    R = rotation.generate_rotation_matrix(d, device=DEV)
    freqs = rotary.rotary_frequencies(d)[0].to(DEV)
    keys, values = (quantizer.allocate_paged_cache(1, 2, d, 4, DEV, page_tokens=64, jl_dim=0) for _ in range(2))
    k = torch.randn(1, 2, 100, d, device=DEV)
    pos = torch.arange(100, device=DEV)
    assert append.append_rotary(k, k, keys, values, R, pos, freqs) is None
    append.append_rotary(k, k, keys, values, R, pos + 100, freqs)
    assert keys.seq_len == values.seq_len == 200 and len(keys.groups) == 4
    check_vectors(window_ref.rows_of(keys)[0][:, :, 100:200], turned(k, (pos + 100)[None], freqs, None, False, 1.0), R,
                  keys.codebooks, 4)
    small = quantizer.allocate_cache(1, 2, 150, d, 4, DEV)
    call = lambda key=k, value=k, kc=small, vc=None, p=pos, f=freqs, **kw: append.append_rotary(  # noqa: E731
        key, value, kc, vc if vc is not None else quantizer.allocate_cache(1, 2, 150, d, 4, DEV), R, p, f, **kw)
    for kw, words in ((dict(starts=51), "slots"), (dict(starts=-1), "slots"), (dict(value=k[:, :, :5]), "match"),
                      (dict(value=k.half()), "one type"), (dict(query=k[:, :, :5]), "match"), (dict(f=freqs.float()), "float64"),
                      (dict(p=pos[:5]), "positions"), (dict(p=pos.float()), "integers"), (dict(key=k[:, :1], value=k[:, :1]), "multiple|kv heads"),
                      (dict(vc=values), "paged"), (dict(vc=quantizer.allocate_cache(1, 2, 150, d, 2, DEV)), "width"),
                      (dict(jl_rot=R), "no signs"), (dict(starts=torch.zeros(2, dtype=torch.int64, device=DEV)), "starts"),
                      (dict(axes=(0,) * 31), "axes for"), (dict(p=pos.cpu()), "device")):
        with pytest.raises(ValueError, match=words):
            call(**kw)
    assert small.seq_len == 0
    call(key=k[:, :, :0], value=k[:, :, :0], p=pos[:0])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before"):
        with torch.cuda.graph(graph):
            append.append_rotary(k, k, keys, values, R, pos, freqs)


@pytest.mark.parametrize("out", [torch.float16, torch.float32], ids=["f16", "f32"])
@pytest.mark.parametrize("d,bits,page", [(64, 4, 0), (64, 2, 64), (128, 4, 256), (128, 2, 0)])
def test_slots_read_back(d, bits, page, out):
    """The values of slots: to the bit what the product with a unit matrix gives."""
    case = (2, 3, 3, 70, 150, d, d, bits, False, page, torch.float16, False, None, [80, 3], None)
    q, k, v, keys, values, R, P, positions, freqs, _ = make(case)
    for c in (keys, values):                        # radii of every kind among random bytes
        blocks = c.groups[0] if page else c.blocks
        for t, bits16 in enumerate((0x0000, 0x8000, 0x7C00, 0xFC00, 0x7E01, 0x0001, 0x7BFF, 0xFBFF)):
            for j in range(d // 32):
                at = j * window_ref.BLOCK_BYTES[bits]
                blocks[:, :, t, at], blocks[:, :, t, at + 1] = bits16 & 255, bits16 >> 8
        S = c.capacity if page else 150
        got = quantizer.dequantize(c, None, out, S)
        whole = c.to_contiguous(S) if page else c
        blocks = whole.blocks.contiguous()
        for j in range(1, d // 32):                 # (one radius a vector, as encoders write it)
            at = j * window_ref.BLOCK_BYTES[bits]
            blocks[..., at:at + 2] = blocks[..., :2]
        want = quantizer.dequantize(whole, torch.eye(d, device=DEV), out, S)
        same = (got == want) | (torch.isnan(got) & torch.isnan(want))
        first = torch.zeros_like(same)
        first[..., :32] = True                      # the first block's radius is the vector's
        assert bool((same | ~first).all())
        if not page:
            got = quantizer.dequantize(c, None, out, S)
            assert bool(((got == want) | (torch.isnan(got) & torch.isnan(want))).all())
            assert torch.equal(torch.signbit(got[~torch.isnan(got)]), torch.signbit(want[~torch.isnan(got)]))
        assert torch.equal(quantizer.dequantize(c, None, out, 5).nan_to_num(7.0), got[:, :, :5].nan_to_num(7.0))
        with pytest.raises(ValueError, match="capacity"):
            quantizer.dequantize(c, None, out, S + 1)
