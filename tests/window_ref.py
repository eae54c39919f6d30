"""Attention behind a window in 64 bits, from a cache's bytes (test helper)."""

import math

import torch

BLOCK_BYTES = {4: 18, 2: 10}


def rows_of(cache):
    """(blocks [B, H, S, vector bytes], signs or None) of a contiguous or paged cache, all its room."""
    if hasattr(cache, "groups"):
        whole = cache.to_contiguous(cache.capacity)
        return whole.blocks, whole.qjl_signs
    return cache.blocks, cache.qjl_signs


def states(blocks, codebook, bits):
    """Decoded rotated states [..., d] of blocks [..., vector bytes], float64."""
    x = blocks.reshape(*blocks.shape[:-1], -1, BLOCK_BYTES[bits])
    r = x[..., 0, :2].contiguous().view(torch.float16).double()
    parts = [(x[..., 2:] >> (bits * j)) & ((1 << bits) - 1) for j in range(8 // bits)]
    code = torch.stack(parts, -1).flatten(-3).long()
    return codebook.double().reshape(-1)[code] * r


def window_attention(q, keys, values, R, window, sinks, starts, counts, scale=None, p_rot=None):
    """(out [B, Hq, Sq, d] float64, bound of the error without the last rounding).

    The bound, from the roundings. Chains of n fp32 operations err by at most about
    4 sqrt(n) 2^-24 of the norms (a random walk of n half steps, 4 standard
    deviations); products of parts leave 2^-21 of each term. Queries are rotated (n =
    d), multiplied with the keys (n = d), with signs once more: a logit is off by
    less than e = (8 sqrt(d) 2^-24 + 2^-21) |q| |k| scale < 2^-17.4 |q| |k| scale for d =
    128. Weights are then off by 2 e relative, plus the exponential's and the sums'
    2^-20, and the output by that share of sum w |v| plus the last rotation's
    2^-18 of |o|; |v| and |o| are norms, which bound each coordinate."""
    B, Hq, Sq, d = q.shape
    kb, sb = rows_of(keys)
    vb, _ = rows_of(values)
    H, G = kb.shape[1], Hq // kb.shape[1]
    S = kb.shape[2]
    R = R.double()
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(B, Hq, Sq, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    t = torch.arange(S, device=q.device)
    for b in range(B):
        start, n = int(starts[b]), int(counts[b])
        if not 0 <= start < S:
            continue
        n = max(0, min(n, Sq, S - start))
        if n == 0:
            continue
        row = torch.arange(start, start + n, device=q.device)[:, None]
        seen = (t <= row) & ((t > row - window) | (t < sinks))
        any_seen = seen.any(0)                              # what no row sees is not looked at
        seen = seen[:, any_seen]
        for h in range(H):
            k = states(kb[b, h, any_seen], keys.codebooks, keys.n_bits)
            v = states(vb[b, h, any_seen], values.codebooks, values.n_bits)
            if p_rot is not None:
                s = sb[b, h, any_seen].int()
                sign = ((s[..., None] >> torch.arange(8, device=q.device).int()) & 1).flatten(-2).double() * 2 - 1
                sign = sign * (s != 255).any(-1, keepdim=True)
            for g in range(h * G, h * G + G):
                qr = q[b, g, :n].double() @ R.T * scale
                x = qr @ k.T
                size = qr.norm(dim=-1, keepdim=True) * k.norm(dim=-1)
                if p_rot is not None:
                    pq = qr @ p_rot.double().T / d
                    x = x + pq @ sign.T
                    size = size + 2 * pq.norm(dim=-1, keepdim=True) * math.sqrt(d)
                x = x.masked_fill(~seen, -math.inf)
                e = (size * 2.0 ** -17.4).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
                w = torch.softmax(x, -1)
                # (a weight of 0 hides whatever stands there)
                vn = torch.where(seen[..., None], v, torch.zeros_like(v)) if not bool(torch.isfinite(v).all()) else v
                o = torch.einsum("nt,ntd->nd", w, vn) if vn.dim() == 3 else w @ vn
                out[b, g, :n] = o @ R
                vsum = (w * v.norm(dim=-1).nan_to_num(0.0, 0.0, 0.0)).sum(-1, keepdim=True)
                bound[b, g, :n] = (2 * e + 2.0 ** -19) * vsum + 2.0 ** -18 * o.norm(dim=-1, keepdim=True)
    return out, bound


def check(got, want, bound):
    half_step = torch.finfo(got.dtype).eps / 2
    tol = bound + half_step * (want.abs() + bound) + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -140)
    assert torch.isfinite(got).all()
    off = (got.double() - want).abs() - tol
    worst = int(off.argmax())
    assert float(off.max()) <= 0.0, (float(off.max()), worst, float(got.flatten()[worst]), float(want.flatten()[worst]))
