"""The operators of a serving step on a compressed cache whose attention looks
at a window: their cases, their plain form in elementary torch operations, and
the calls a program makes of this package's kernels for the same.

A case is a dict of plain values; "op" names the operator:

  axes     rotary.apply_rotary with the pairs of a head shared out among
           several axes of positions (time, height, width), and its gradients
  append   append.append_rotary: a step's queries and keys turned, keys and
           values encoded into the cache's slots, every sequence at its own
  window   attention.window_attention on a compressed cache: the last `window`
           positions and the first `sinks`, one query token per sequence or a
           chunk of them, every sequence at its own length

With `own` false, run() computes the plain form; with `own` true it calls the
package. Caches are built here (rotated Gaussian states, polar split, nearest
centroid, packed blocks), so that no input depends on the package.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 32                              # coordinates per block
BLOCK_BYTES = {4: 18, 2: 10}            # fp16 radius + 32 codes
# Lloyd-Max centroids of a unit normal (positive half), scaled by 1 / sqrt(d)
LEVELS = {4: [0.1284, 0.3881, 0.6568, 0.9424, 1.2562, 1.6180, 2.0690, 2.7326], 2: [0.4528, 1.5104]}


# ------------------------------------------------------------------- the cases
#
# sections: pairs per axis, "a,b,c"; spread: dealt out in turn instead of in runs.
# S: slots of the cache; step: how many positions each sequence is behind the one
# before it; pad: how many of a chunk's tokens each sequence has fewer than the one
# before it. Appended codes have 4 bits: a value at the border of two codes may be
# given either, and one returned as the code's value is then off by their distance,
# which at 2 bits is the size of the value itself.

def listed():
    return [
        # One decode step of a serving batch of 8 with time, height and width positions.
        dict(name="axes_step", op="axes", B=8, Hq=32, Hkv=8, T=1, d=128, sections="16,24,24", spread=False,
             interleaved=False, dtype="f16", start=70001, grad=False),
        # A training step on images of 37 x 37 patches: rows and columns, interleaved pairs, part of the head.
        dict(name="axes_image_train", op="axes", B=4, Hq=16, Hkv=16, T=1369, d=64, sections="14,14", spread=False,
             interleaved=True, dtype="f32", start=0, grad=True),
        # The prompt of a video: many query heads, axes dealt out pair by pair.
        dict(name="axes_video_32k", op="axes", B=1, Hq=64, Hkv=8, T=32760, d=128, sections="24,20,20", spread=True,
             interleaved=False, dtype="bf16", start=0, grad=False),
        # One decode step of 8 sequences of different lengths, in pages.
        dict(name="append_step", op="append", B=8, Hq=32, Hkv=8, T=1, S=2048, step=131, pad=0, d=128, page=256,
             sections="64", spread=False, interleaved=False, dtype="f16", start=100000),
        # Chunks of two prompts of a small model, padded to the longer, into a contiguous cache.
        dict(name="append_chunk_padded", op="append", B=2, Hq=14, Hkv=2, T=509, S=1536, step=77, pad=101, d=64, page=0,
             sections="24", spread=False, interleaved=True, dtype="f32", start=0),
        # A long prompt with three axes of positions: the largest append.
        dict(name="append_prompt_32k", op="append", B=1, Hq=32, Hkv=8, T=32768, S=32768, step=0, pad=0, d=128, page=4096,
             sections="16,24,24", spread=False, interleaved=False, dtype="bf16", start=0),
        # One token of a small model behind a short window: launches and host time.
        dict(name="window_step_small", op="window", B=1, Hq=14, Hkv=2, Sq=1, S=2011, step=0, pad=0, window=512, sinks=4,
             d=64, bits=4, qjl=False, page=0, out="f32"),
        # Serving of 16 sequences of different lengths in pages, 2-bit keys with the sign sketch that corrects them.
        dict(name="window_step_paged_qjl", op="window", B=16, Hq=32, Hkv=8, Sq=1, S=16384, step=997, pad=0, window=4096,
             sinks=4, d=128, bits=2, qjl=True, page=256, out="f16"),
        # A full batch of 64 sequences behind windows of 4096: the largest decode step.
        dict(name="window_step_64", op="window", B=64, Hq=32, Hkv=8, Sq=1, S=6144, step=23, pad=0, window=4096, sinks=16,
             d=128, bits=4, qjl=False, page=0, out="f16"),
        # Chunks of odd lengths in the middle of two sequences of a small model, padded, in small pages.
        dict(name="window_chunk_padded", op="window", B=2, Hq=14, Hkv=2, Sq=257, S=3001, step=411, pad=60, window=512,
             sinks=4, d=64, bits=4, qjl=False, page=64, out="f32"),
        # Chunks of four sequences of 16K tokens with corrected 2-bit keys.
        dict(name="window_chunk_qjl", op="window", B=4, Hq=32, Hkv=8, Sq=512, S=16384, step=1500, pad=0, window=4096,
             sinks=4, d=128, bits=2, qjl=True, page=256, out="f16"),
        # A whole prompt behind a window: the largest product.
        dict(name="window_prompt_8k", op="window", B=1, Hq=32, Hkv=8, Sq=8191, S=8191, step=0, pad=0, window=1024,
             sinks=4, d=128, bits=4, qjl=False, page=0, out="f16"),
    ]


# (query heads, kv heads, head dim)
SHAPES = [(14, 2, 64), (32, 8, 128), (64, 8, 128), (32, 32, 128), (16, 16, 64)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(hi, lo + 1))))))


def draw(rng):
    case = _drawn(rng)
    most = [work(c) for c in listed() if c["op"] == case["op"]]
    # no costlier than the operator's largest listed cases
    while any(work(case)[k] > max(w[k] for w in most) for k in ("bytes", "flops")):
        if case["op"] == "window" and case["Sq"] == 1:
            case["B"] = max(1, 3 * case["B"] // 4)
        else:
            name = "Sq" if case["op"] == "window" else "T"
            case[name] = max(2, 3 * case[name] // 4)
            case["pad"] = min(case.get("pad", 0), (case[name] - 1) // case["B"])
    return case


def _sections(rng, pairs):
    n = rng.choice([1, 2, 3])
    cuts = sorted(rng.sample(range(1, pairs), n - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [pairs])]


def _drawn(rng):
    op = rng.choice(["axes", "append", "window"])
    Hq, Hkv, d = rng.choice(SHAPES)
    if op in ("axes", "append"):
        rot = d if rng.random() < 0.5 else 2 * rng.randrange(4, d // 2)
        s = _sections(rng, rot // 2)
        if op == "axes" and len(s) == 1:
            s = [s[0] - s[0] // 2, s[0] // 2]
        # dealt out, every axis but the first has to find its pairs among the first ones
        spread = all(a + len(s) * (s[a] - 1) < sum(s) for a in range(1, len(s))) and rng.random() < 0.7
        c = dict(op=op, B=_log(rng, 1, 16), Hq=Hq, Hkv=Hkv, d=d, sections=",".join(map(str, s)), spread=spread,
                 interleaved=rng.random() < 0.5, dtype=rng.choice(["f16", "bf16", "f32"]),
                 start=rng.choice([0, _log(rng, 1, 1000000)]))
        c["T"] = 1 if rng.random() < 0.3 else _log(rng, 2, 32768 // c["B"])
        if op == "axes":
            c["grad"] = rng.random() < 0.4
            return c
        c["page"] = rng.choice([0, 0, 256, 1024])
        c["pad"] = rng.randrange(0, (c["T"] - 1) // c["B"] + 1) if rng.random() < 0.5 else 0
        c["step"] = rng.choice([0, rng.randrange(1, 64)])
        c["S"] = c["T"] + c["step"] * (c["B"] - 1) + rng.randrange(0, 300)
        return c
    c = dict(op=op, Hq=Hq, Hkv=Hkv, d=d, bits=rng.choice([4, 4, 2]), qjl=rng.random() < 0.3,
             page=rng.choice([0, 0, 64, 256]), out=rng.choice(["f16", "f32"]), window=_log(rng, 16, 8192),
             sinks=rng.choice([0, 4, rng.randrange(1, 200)]))
    if rng.random() < 0.5:
        c.update(B=_log(rng, 1, 64), Sq=1, pad=0)
    else:
        c.update(B=rng.choice([1, 1, 2, 4]), Sq=_log(rng, 2, 4096))
        c["pad"] = rng.randrange(0, (c["Sq"] - 1) // c["B"] + 1) if rng.random() < 0.5 else 0
    c["S"] = c["Sq"] + _log(rng, 1, min(32768, 1048576 // (c["B"] * Hkv)))
    c["step"] = rng.randrange(0, (c["S"] - c["Sq"]) // c["B"] + 1) if rng.random() < 0.7 else 0
    return c


# ------------------------------------------------------------------ the inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _orthogonal(d, seed):
    g = torch.Generator().manual_seed(seed)
    q, r = torch.linalg.qr(torch.randn(d, d, generator=g, dtype=torch.float64))
    return (q * torch.sign(torch.diagonal(r))).float().contiguous().to(DEV)


def _codebook(d, bits):
    half = torch.tensor(LEVELS[bits], dtype=torch.float64) / math.sqrt(d)
    return torch.cat([-half.flip(0), half]).float().to(DEV)


def _blocks(B, H, S, d, bits, g):
    """Encoded states [B, H, S, vector bytes]: Gaussian directions, radii of
    sqrt(d) times a log-normal factor."""
    cb = _codebook(d, bits)
    y = torch.randn(B, H, S, d, generator=g, device=DEV)
    norm = y.norm(dim=-1, keepdim=True)
    code = torch.bucketize(y / norm, (cb[1:] + cb[:-1]) / 2).to(torch.uint8)
    r = norm * torch.exp(0.3 * torch.randn(B, H, S, 1, generator=g, device=DEV))
    return _packed(r.half(), code, bits)


def _packed(r16, code, bits):
    """Blocks [..., vector bytes] of radii [..., 1] and codes [..., d]."""
    lead, nb = code.shape[:-1], code.shape[-1] // BLOCK
    out = torch.empty(*lead, nb, BLOCK_BYTES[bits], dtype=torch.uint8, device=DEV)
    out[..., :2] = r16.contiguous().view(torch.uint8).unsqueeze(-2)
    code = code.view(*lead, nb, -1, 8 // bits)
    packed = code[..., 0]
    for j in range(1, 8 // bits):
        packed = packed | (code[..., j] << (bits * j))
    out[..., 2:] = packed
    return out.flatten(-2)


def _paged(rows, page):
    """[B, H, S, n] as pages [pages, B, H, page, n], zeros behind S."""
    B, H, S, n = rows.shape
    pages = -(-S // page)
    full = torch.zeros(B, H, pages * page, n, dtype=rows.dtype, device=DEV)
    full[:, :, :S] = rows
    return full.view(B, H, pages, page, n).permute(2, 0, 1, 3, 4).contiguous()


def _axes(c):
    """The axis of each pair."""
    s = [int(x) for x in c["sections"].split(",")]
    if not c["spread"]:
        return [a for a, n in enumerate(s) for _ in range(n)]
    out = [0] * sum(s)
    for a in range(1, len(s)):
        for j in range(s[a]):
            out[a + j * len(s)] = a
    return out


def _positions(c):
    """[axes, B, T] positions as a vision-language model gives them: runs of text
    (all axes alike) around frames of 14 x 18 patches (time, row, column); images
    (two axes): rows and columns."""
    n, B, T = c["sections"].count(",") + 1, c["B"], c["T"]
    t = torch.arange(T, device=DEV)
    rows = [c["start"] + t]
    if n == 2:
        side = max(1, math.isqrt(T))
        rows = [c["start"] + t // side, c["start"] + t % side]
    if n == 3:
        text = 17
        in_frames = (t >= text) & (t < T - text)
        i = t - text
        last = c["start"] + text + (T - 2 * text) // 252 + 18
        grid = [i // 252, i // 18 % 14, i % 18]
        flat = torch.where(t < text, c["start"] + t, last + t - (T - text))
        rows = [torch.where(in_frames, c["start"] + text + x, flat) for x in grid]
    behind = torch.arange(B, device=DEV)[:, None] * c.get("step", 3)
    return torch.stack([(r - behind).clamp(min=0) for r in rows])


def _frequencies(rot):
    """Radians a position turns each pair by, in 64 bits."""
    return (10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)).to(DEV)


def _heads(c, n, g):
    """As a projection leaves them: [B, T, H, d], seen as [B, H, T, d]."""
    return torch.randn(c["B"], c["T"], n, c["d"], generator=g, device=DEV).to(DTYPES[c["dtype"]]).transpose(1, 2)


def _axes_inputs(c, seed):
    g, t = _gen(seed), DTYPES[c["dtype"]]
    s = dict(q=_heads(c, c["Hq"], g), k=_heads(c, c["Hkv"], g), positions=_positions(c), axes=_axes(c))
    s["freqs"] = _frequencies(2 * len(s["axes"]))
    if c["grad"]:
        s["gq"] = torch.randn(c["B"], c["Hq"], c["T"], c["d"], generator=g, device=DEV).to(t)
        s["gk"] = torch.randn(c["B"], c["Hkv"], c["T"], c["d"], generator=g, device=DEV).to(t)
    return s


def _starts(c):
    """(first slot, tokens) of each sequence's new tokens."""
    T = c["Sq"] if c["op"] == "window" else c["T"]
    b = torch.arange(c["B"], device=DEV)
    return c["S"] - T - b * c["step"], T - b * c["pad"]


def _append_inputs(c, seed):
    g = _gen(seed)
    B, H, d = c["B"], c["Hkv"], c["d"]
    s = dict(q=_heads(c, c["Hq"], g), k=_heads(c, H, g), v=_heads(c, H, g), positions=_positions(c), axes=_axes(c))
    s["freqs"] = _frequencies(2 * len(s["axes"]))
    s["starts"], s["counts"] = _starts(c)
    s.update(S=c["S"], codebook=_codebook(d, 4), R=_orthogonal(d, seed + 1))
    for name in ("keys", "values"):                             # what the cache holds so far
        s[name] = _blocks(B, H, c["S"], d, 4, g)
        if c["page"]:
            s[name] = _paged(s[name], c["page"])
    return s


def _window_inputs(c, seed):
    g = _gen(seed)
    B, H, d, bits, S = c["B"], c["Hkv"], c["d"], c["bits"], c["S"]
    s = dict(S=S, codebook=_codebook(d, bits), R=_orthogonal(d, seed + 1))
    s["keys"], s["values"] = _blocks(B, H, S, d, bits, g), _blocks(B, H, S, d, bits, g)
    if c["qjl"]:
        s["signs"] = torch.randint(0, 256, (B, H, S, d // 8), generator=g, device=DEV, dtype=torch.uint8)
        s["signs"][:, :, ::97] = 255                     # zero residuals
        s["p_rot"] = torch.randn(d, d, generator=g, device=DEV)
    s["q"] = (2.0 * torch.randn(B, c["Hq"], c["Sq"], d, generator=g, device=DEV)).half()
    s["starts"], s["counts"] = _starts(c)
    if c["page"]:
        for name in ("keys", "values", "signs"):
            if name in s:
                s[name] = _paged(s[name], c["page"])
    return s


def _handles(c, s):
    """The caches as the package's programs hold them."""
    from polarquant_kv.types import PagedPQCache, PQCache
    B, H, d, bits, S, page = c["B"], c["Hkv"], c["d"], c.get("bits", 4), s["S"], c["page"]
    table16 = torch.zeros(16, dtype=torch.float32, device=DEV)
    table16[:1 << bits] = s["codebook"]
    for name in ("keys", "values"):
        signs = s.get("signs") if name == "keys" else None
        jl = d if signs is not None else 0
        if page:
            cache = PagedPQCache(B, H, d, bits, table16, DEV, page_tokens=page, jl_dim=jl)
            cache.ensure(S)
            for p, group in enumerate(cache.groups):
                group.copy_(s[name][p])
                if jl:
                    cache.sign_groups[p].copy_(signs[p])
            cache.seq_len = S
        else:
            cache = PQCache(blocks=s[name], head_dim=d, n_bits=bits, seq_len=S, max_seq_len=S, codebooks=table16,
                            qjl_signs=signs, jl_dim=jl)
        s[name + "_cache"] = cache
    return s


def prepare(case, seed):
    s = {"axes": _axes_inputs, "append": _append_inputs, "window": _window_inputs}[case["op"]](case, seed)
    s["case"] = case
    if own:
        sys.path.insert(0, os.path.join(os.getcwd(), "polarquant-kv_amd"))
        if case["op"] != "axes":
            _handles(case, s)
    if case["op"] == "axes" and case["grad"]:
        s["q"].requires_grad_(True)
        s["k"].requires_grad_(True)
    return s


# -------------------------------------------------------------- the plain forms

def _angles(s):
    """[B, T, pairs] in 64 bits."""
    at = s["positions"][torch.tensor(s["axes"], device=DEV)]            # [pairs, B, T]
    return at.permute(1, 2, 0).double() * s["freqs"]


def _turned(x, cos, sin, interleaved):
    """x [B, H, T, d] in 32 bits, cos / sin [B, 1, T, rot / 2]."""
    rot = 2 * cos.shape[-1]
    y, rest = x[..., :rot], x[..., rot:]
    a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:])
    u, v = a * cos - b * sin, a * sin + b * cos
    y = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((y, rest), -1)


def _plain_axes(s):
    c = s["case"]
    angle = _angles(s).unsqueeze(1)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out = {n: _turned(s[n].detach().float(), cos, sin, c["interleaved"]).to(s[n].dtype) for n in ("q", "k")}
    if c["grad"]:       # the transposed rotation
        for n in ("gq", "gk"):
            out[n] = _turned(s[n].float(), cos, -sin, c["interleaved"]).to(s[n].dtype)
    return out


def _rows(s, name):
    """The array [B, H, S, n] of a cache, gathered from its pages."""
    x = s[name]
    if s["case"]["page"]:
        p, B, H, page, n = x.shape
        x = x.permute(1, 2, 0, 3, 4).reshape(B, H, p * page, n)[:, :, :s["S"]]
    return x


def _states(x, codebook, d, bits):
    """Rotated states r c[code] [B, H, S, d] of blocks, in 32 bits."""
    x = x.reshape(*x.shape[:3], d // BLOCK, BLOCK_BYTES[bits])
    r = x[..., 0, :2].contiguous().view(torch.float16).float()
    shift = torch.arange(0, 8, bits, device=DEV, dtype=torch.uint8)
    code = (x[..., 2:, None] >> shift) & ((1 << bits) - 1)
    return codebook[code.flatten(3).int()] * r


def _plain_append(s):
    c = s["case"]
    B, H, T, d, page = c["B"], c["Hkv"], c["T"], c["d"], c["page"]
    angle = _angles(s).unsqueeze(1)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q = _turned(s["q"].float(), cos, sin, c["interleaved"]).to(s["q"].dtype)
    out = dict(q=q)
    t = torch.arange(T, device=DEV)
    b, t = torch.nonzero(t < s["counts"][:, None], as_tuple=True)       # the tokens that there are
    slot = s["starts"][b] + t
    for name, x in (("keys", _turned(s["k"].float(), cos, sin, c["interleaved"])), ("values", s["v"].float())):
        y = torch.matmul(x[b, :, t], s["R"].t())                        # [tokens, H, d]
        r = y.square().sum(-1, keepdim=True).sqrt()
        mid = (s["codebook"][1:] + s["codebook"][:-1]) / 2
        code = torch.bucketize(y / r, mid).to(torch.uint8)
        rows = _packed(r.half(), code, 4)
        if page:
            s[name][slot // page, b, :, slot % page] = rows
        else:
            s[name][b, :, slot] = rows
        out[name] = _states(_rows(s, name), s["codebook"], d, 4).half()
    return out


def _plain_window(s):
    c = s["case"]
    B, Hq, H, Sq, d, bits, S = c["B"], c["Hq"], c["Hkv"], c["Sq"], c["d"], c["bits"], s["S"]
    W, sinks = c["window"], c["sinks"]
    # the sinks, then every position of a row's window
    first = s["starts"] - W + 1
    n = min(W - 1 + Sq, S)
    first = torch.minimum(first, S - torch.tensor(n, device=DEV)).clamp(min=0)
    at = first[:, None] + torch.arange(n, device=DEV)                                   # [B, n]
    seen = (at >= sinks)
    if sinks:
        head = torch.arange(min(sinks, S), device=DEV).expand(B, -1)
        at, seen = torch.cat((head, at), 1), torch.cat((torch.ones_like(head, dtype=torch.bool), seen), 1)
    row = s["starts"][:, None] + torch.arange(Sq, device=DEV)                           # [B, Sq]
    gap = row[:, :, None] - at[:, None, :]
    seen = seen[:, None, :] & (gap >= 0) & ((gap < W) | (at < sinks)[:, None, :])       # [B, Sq, n]

    def gathered(name):
        x = _rows(s, name)
        return torch.gather(x, 2, at[:, None, :, None].expand(B, H, at.shape[1], x.shape[-1]))

    qr = torch.matmul(s["q"].float(), s["R"].t()).view(B, H, -1, d) / math.sqrt(d)
    x = torch.matmul(qr, _states(gathered("keys"), s["codebook"], d, bits).transpose(2, 3))
    if c["qjl"]:
        signs = gathered("signs")
        sign = ((signs[..., None] >> torch.arange(8, device=DEV, dtype=torch.uint8)) & 1).flatten(3).float() * 2 - 1
        sign = sign * (signs != 255).any(-1, keepdim=True)          # a zero residual has no correction
        x = x + torch.matmul(torch.matmul(qr, s["p_rot"].t()) / d, sign.transpose(2, 3))
    x = x.view(B, Hq, Sq, -1).masked_fill(~seen[:, None], float("-inf"))
    w = torch.softmax(x, -1).view(B, H, -1, at.shape[1])
    out = torch.matmul(torch.matmul(w, _states(gathered("values"), s["codebook"], d, bits)), s["R"]).view(B, Hq, Sq, d)
    there = torch.arange(Sq, device=DEV) < s["counts"][:, None]
    return dict(out=(out * there[:, None, :, None]).to(DTYPES[c["out"]]))


# ------------------------------------------------------------ the package's calls

def _own_axes(s):
    from polarquant_kv import rotary
    c = s["case"]
    q, k = rotary.apply_rotary(s["q"], s["k"], s["positions"], s["freqs"], interleaved=c["interleaved"],
                               axes=s["axes"])
    out = dict(q=q, k=k)
    if c["grad"]:
        out["gq"], out["gk"] = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
    return out


def _own_append(s):
    from polarquant_kv import append, quantizer
    c = s["case"]
    keys, values = s["keys_cache"], s["values_cache"]
    q = append.append_rotary(s["k"], s["v"], keys, values, s["R"], s["positions"], s["freqs"], query=s["q"],
                             starts=s["starts"], counts=s["counts"], interleaved=c["interleaved"], axes=s["axes"])
    # what the slots now stand for
    return dict(q=q, keys=quantizer.dequantize(keys, None, torch.float16, s["S"]),
                values=quantizer.dequantize(values, None, torch.float16, s["S"]))


def _own_window(s):
    from polarquant_kv import attention
    c = s["case"]
    alike = c["step"] == 0 and c["pad"] == 0
    return dict(out=attention.window_attention(
        s["q"], s["keys_cache"], s["values_cache"], s["R"], c["window"], sinks=c["sinks"],
        starts=c["S"] - c["Sq"] if alike else s["starts"], counts=s["counts"] if c["pad"] else None,
        jl_rot=s.get("p_rot"), out_dtype=DTYPES[c["out"]]))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"axes": _own_axes, "append": _own_append, "window": _own_window}[op](state)
    return {"axes": _plain_axes, "append": _plain_append, "window": _plain_window}[op](state)


# ---------------------------------------------------------- what a pass has to do

def work(case):
    c, B = case, case["B"]
    if c["op"] == "axes":
        rot = 2 * len(_axes(c))
        n = B * c["T"] * (c["Hq"] + c["Hkv"]) * (2 if c["grad"] else 1)
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": 2 * n * c["d"] * size + 8 * B * c["T"] * (c["sections"].count(",") + 1), "flops": 3 * n * rot}
    d = c["d"]
    if c["op"] == "append":
        size = 4 if c["dtype"] == "f32" else 2
        tokens = sum(c["T"] - b * c["pad"] for b in range(B))
        vec = d // BLOCK * BLOCK_BYTES[4]
        # queries read and written, keys and values read; the new vectors written; the slots' values
        # written out of all vectors
        data = 2 * B * c["T"] * c["Hq"] * d * size + tokens * 2 * c["Hkv"] * (d * size + vec)
        return {"bytes": data + 2 * B * c["Hkv"] * c["S"] * (vec + 2 * d),
                "flops": 2 * tokens * 2 * c["Hkv"] * d * d}
    vec = d // BLOCK * BLOCK_BYTES[c["bits"]] * 2 + (d // 8 if c["qjl"] else 0)
    read = pairs = 0
    W, sinks = c["window"], c["sinks"]
    for b in range(B):
        start, count = c["S"] - c["Sq"] - b * c["step"], c["Sq"] - b * c["pad"]
        lo = max(0, start - W + 1)
        read += start + count - lo + min(sinks, lo)

        def seen(p):        # pairs of the rows before position p
            full = max(0, p - (W + sinks))                  # rows that see W + sinks positions
            m = p - full
            return full * (W + sinks) + m * (m + 1) // 2

        pairs += seen(start + count) - seen(start)
    size = 4 if c["out"] == "f32" else 2
    return {"bytes": c["Hkv"] * read * vec + B * c["Hq"] * c["Sq"] * d * (2 + size), "flops": 4 * c["Hq"] * pairs * d}


# ------------------------------------------------------------- in 64 bits, apart

def _exact_turned(x, angle, interleaved):
    n = angle.shape[-1]
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)       # complex [B, 1, T, rot / 2]
    x = x.detach().double().clone()
    ia = torch.arange(n, device=DEV) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else n)
    z = torch.complex(x[..., ia], x[..., ib]) * turn
    x[..., ia], x[..., ib] = z.real, z.imag
    return x


def _exact_angle(s):
    angle = torch.empty(*s["positions"].shape[1:], len(s["axes"]), dtype=torch.float64, device=DEV)
    for i, a in enumerate(s["axes"]):
        angle[..., i] = s["positions"][a].double() * s["freqs"][i]
    return angle


def _exact_states(rows, codebook, bits):
    """Decoded states [..., S, d] of blocks, in 64 bits."""
    x = rows.reshape(*rows.shape[:-1], -1, BLOCK_BYTES[bits])
    r = x[..., 0, :2].contiguous().view(torch.float16).double()
    parts = [(x[..., 2:] >> (bits * j)) & ((1 << bits) - 1) for j in range(8 // bits)]
    code = torch.stack(parts, -1).flatten(-3).long()
    return codebook.double()[code] * r


def exact(case, seed):
    c = case
    if c["op"] == "axes":
        s = _axes_inputs(c, seed)
        angle = _exact_angle(s)
        out = {n: _exact_turned(s[n], angle, c["interleaved"]) for n in ("q", "k")}
        if c["grad"]:
            out["gq"], out["gk"] = (_exact_turned(s[n], -angle, c["interleaved"]) for n in ("gq", "gk"))
        return out
    flat = dict(c, page=0)
    if c["op"] == "append":
        s = _append_inputs(flat, seed)
        angle = _exact_angle(s)
        out = dict(q=_exact_turned(s["q"], angle, c["interleaved"]))
        cb, R = s["codebook"].double(), s["R"].double()
        for name, x in (("keys", _exact_turned(s["k"], angle, c["interleaved"])), ("values", s["v"].double())):
            held = _exact_states(s[name], s["codebook"], 4)
            for b in range(c["B"]):
                n, at = int(s["counts"][b]), int(s["starts"][b])
                for h in range(c["Hkv"]):
                    y = x[b, h, :n] @ R.T
                    r = torch.linalg.vector_norm(y, dim=-1, keepdim=True)
                    u = y / r
                    near = torch.searchsorted((cb[1:] + cb[:-1]) / 2, u.contiguous())
                    held[b, h, at:at + n] = cb[near] * r.half().double()
            out[name] = held
        return out
    s = _window_inputs(flat, seed)
    B, Hq, H, d, Sq, W, sinks = c["B"], c["Hq"], c["Hkv"], c["d"], c["Sq"], c["window"], c["sinks"]
    G = Hq // H
    R, scale = s["R"].double(), d ** -0.5
    out = torch.zeros(B, Hq, Sq, d, dtype=torch.float64, device=DEV)
    for b in range(B):
        start, n = int(s["starts"][b]), int(s["counts"][b])
        end, lo = start + n, max(0, start - W + 1)
        at = torch.cat((torch.arange(min(sinks, lo), device=DEV), torch.arange(lo, end, device=DEV)))
        row = torch.arange(start, end, device=DEV)[:, None]
        hidden = (at > row) | ((at <= row - W) & (at >= sinks))
        for h in range(H):
            keys = _exact_states(s["keys"][b, h, at], s["codebook"], c["bits"])
            values = _exact_states(s["values"][b, h, at], s["codebook"], c["bits"])
            if c["qjl"]:
                bits = s["signs"][b, h, at].int()[:, :, None].bitwise_right_shift(torch.arange(8, device=DEV).int()) & 1
                sign = torch.where(bits.view(at.numel(), d) > 0, 1.0, -1.0).double()
                sign[(bits.view(at.numel(), d) > 0).all(-1)] = 0.0
            for g in range(h * G, h * G + G):
                q = s["q"][b, g, :n].double() @ R.T * scale
                x = q @ keys.T
                if c["qjl"]:
                    x += (q @ s["p_rot"].double().T / d) @ sign.T
                x[hidden] = -math.inf
                p = torch.exp(x - x.amax(-1, keepdim=True))
                out[b, g, :n] = p / p.sum(-1, keepdim=True) @ values @ R
    return dict(out=out)
