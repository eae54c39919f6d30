"""A serving run behind a window: KVCacheManager and the attention layer with
appends on the way, against the operators and the formula in 64 bits."""

import pytest
import torch

import window_ref
from polarquant_kv import append, attention, quantizer, rotary, rotation
from polarquant_kv.inference import CompressedMultiHeadAttention, KVCacheManager, PolarQuantConfig

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("qjl", [False, True])
@pytest.mark.parametrize("bits", [4, 2])
def test_manager_run(bits, qjl):
    B, Hq, H, D, W, sinks = 2, 6, 2, 64, 50, 3
    config = PolarQuantConfig(n_bits=bits, jl_dim=D, enable_qjl=qjl)
    m = KVCacheManager(config, 400, B, H, D, DEV, page_tokens=64)
    emb = rotary.RotaryEmbedding(D, sections=(12, 10, 10), interleaved=True)
    twin = [quantizer.allocate_paged_cache(B, H, D, bits, DEV, page_tokens=64, jl_dim=jl) for jl in (D if qjl else 0, 0)]
    g = torch.Generator(device=DEV).manual_seed(2)
    at = 0
    for T in (90, 1, 1, 33, 1, 130, 1):
        q, k, v = (torch.randn(B, T, n, D, generator=g, device=DEV).half().transpose(1, 2) for n in (Hq, H, H))
        positions = torch.arange(at, at + T, device=DEV).expand(3, -1) // torch.tensor([[1], [2], [3]], device=DEV)
        qt = m.append_rotary(q, k, v, emb, positions)
        assert torch.equal(qt, emb(q, None, positions)[0])
        # the same appended by itself, as sequences of starts of their own
        for c in twin:
            c.ensure(at + T)
        append.append_rotary(k, v, *twin, m.R, positions, emb.frequencies_on(q.device), axes=emb.axes, interleaved=True,
                             starts=torch.full((B,), at, device=DEV), jl_rot=m.jl_rot)
        at += T
        for mine, other in zip(m.get_kv(), twin):
            other.seq_len = at
            for x, y in zip(window_ref.rows_of(mine), window_ref.rows_of(other)):
                assert (x is None and y is None) or torch.equal(x[:, :, :at], y[:, :, :at])
        assert m.seq_len == m.next_position == at
        out = m.attend(qt, window=W, sinks=sinks)
        start = torch.full((B,), at - T, device=DEV)
        want, bound = window_ref.window_attention(qt, *m.get_kv(), m.R, W, sinks, start, torch.full((B,), T), p_rot=m.jl_rot)
        window_ref.check(out, want, bound)
    with pytest.raises(ValueError, match="window"):
        m.attend(qt, causal=False, window=W)
    tracked = KVCacheManager(PolarQuantConfig(), 400, B, H, D, DEV, track_weights=True)
    tracked.append_rotary(q, k, v, rotary.RotaryEmbedding(D))
    assert tracked.positions[0, 0].tolist() == [0]
    with pytest.raises(ValueError, match="window"):
        tracked.attend(qt, window=W)
    m.reset()
    assert not m.attend(qt, window=W).any()


def test_uncompressed_manager_and_layer():
    """The same layer on an uncompressed cache is the mask's plain form; on a compressed one it is near it."""
    torch.manual_seed(0)
    B, D, W, sinks = 2, 64, 20, 2
    emb = rotary.RotaryEmbedding(D)
    x = torch.randn(B, 60, 4 * D, device=DEV)
    outs = {}
    for compressed in (False, True):
        torch.manual_seed(1)
        config = PolarQuantConfig(enable_compression=compressed)
        layer = CompressedMultiHeadAttention(config, 4 * D, 4, 2, rotary=emb, window=W, sinks=sinks).to(DEV)
        m = KVCacheManager(config, 100, B, 2, D, DEV)
        with torch.no_grad():
            parts = [layer(x[:, a:b], m) for a, b in ((0, 40), (40, 41), (41, 60))]
            outs[compressed] = torch.cat(parts, 1)
            whole = layer(x)
    # a chunk by chunk run sees what the run without a cache sees
    fine = outs[False].float() - whole.float()
    assert fine.norm() <= 2e-3 * whole.norm()               # fp16 states and outputs: 2^-11 each, several times over
    # 4-bit codes: each state is off by about a tenth of its norm (the distortion of 16 levels)
    off = outs[True].float() - whole.float()
    assert 1e-3 * whole.norm() < off.norm() < 0.3 * whole.norm()
    late = layer(x[:, :5], None, positions=torch.arange(7, 12, device=DEV))
    assert late.shape == (B, 5, 4 * D)


def test_a_captured_decode_step():
    """Append and attention of one token per sequence, captured once and replayed as the sequences grow."""
    B, Hq, H, D, W, sinks, S = 3, 8, 2, 128, 40, 4, 256
    R = rotation.generate_rotation_matrix(D, device=DEV)
    freqs = rotary.rotary_frequencies(D)[0].to(DEV)
    pairs = [[quantizer.allocate_paged_cache(B, H, D, 4, DEV, page_tokens=64) for _ in range(2)] for _ in range(2)]
    for c in pairs[0] + pairs[1]:
        c.ensure(S)
        c.seq_len = S
    starts = torch.tensor([5, 60, 100], device=DEV)
    q, k, v = (torch.randn(B, n, 1, D, device=DEV).half() for n in (Hq, H, H))
    g = torch.Generator(device=DEV).manual_seed(0)
    first = torch.randn(B, H, 100, D, generator=g, device=DEV).half()
    for p in pairs:
        for c in p:
            quantizer.compress_pq(first, R, cache=c, start=0)
            c.seq_len = S

    def step(keys, values):
        qt = append.append_rotary(k, v, keys, values, R, starts[:, None], freqs, query=q, starts=starts)
        return attention.window_attention(qt, keys, values, R, W, sinks=sinks, starts=starts, out_dtype=torch.float32)

    step(*pairs[0])
    step(*pairs[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*pairs[0])
    for _ in range(70):
        for x in (q, k, v):
            x.normal_()
        graph.replay()
        kept = got.clone()
        want = step(*pairs[1])
        torch.cuda.synchronize()
        assert torch.equal(kept, want)
        ref, bound = window_ref.window_attention(rotary.apply_rotary(q, None, starts[:, None], freqs)[0], *pairs[1], R, W,
                                                 sinks, starts, [1] * B) if int(starts[0]) % 20 == 5 else (None, None)
        if ref is not None:
            window_ref.check(want, ref, bound)
        starts += 1
