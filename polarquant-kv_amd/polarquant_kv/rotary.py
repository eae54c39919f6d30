"""Rotary positions of queries and keys (device tensors only).

No counterpart in the reference, whose attention layers have no positions
(src/polarquant_kv_cuda/inference/attention.py:12-92). Positions are an
argument, not the slot a token has in a cache: after an eviction the two
differ.

  rotary_frequencies  radians per position of each pair, in 64 bits, with the
                      usual scalings for contexts longer than trained for
  apply_rotary        q and k turned in one launch (pqkv_rotary), with its
                      gradient
  RotaryEmbedding     both for one head shape; what an attention layer takes
"""

from __future__ import annotations

import functools
import math

import torch
from torch.autograd import forward_ad

from . import _lib


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling: dict | None = None):
    """(frequencies [rot_dim / 2] float64 on the host, amplitude): pair i turns
    by base^(-2 i / rot_dim) radians per position, changed by `scaling`:

      None                                          as they are
      {"type": "linear", "factor": f}               all divided by f
      {"type": "base", "factor": f}                 a larger base, f^(rot_dim / (rot_dim - 2)) times:
                                                    the fastest pair as it is, the slowest divided by f
      {"type": "bands", "factor": f, "original": n, "low": 1, "high": 4}
                                                    by how often a pair turns over n positions: from `high`
                                                    times as it is, up to `low` times divided by f, between
                                                    them a mean weighted linearly in the number of turns
      {"type": "yarn", "factor": f, "original": n, "fast": 32, "slow": 1, "amplitude": None}
                                                    as it is above `fast` turns, divided by f below
                                                    `slow`, a linear ramp over the pair's index between;
                                                    amplitude 0.1 ln f + 1 unless given
    """
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim must be even and positive, got {rot_dim}")
    if not base > 0:
        raise ValueError(f"base must be positive, got {base}")
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    freqs = base ** (-2.0 * i / rot_dim)
    if scaling is None:
        return freqs, 1.0
    known = {"linear": {"factor"}, "base": {"factor"}, "bands": {"factor", "original", "low", "high"},
             "yarn": {"factor", "original", "fast", "slow", "amplitude"}}
    kind = scaling.get("type")
    if kind not in known:
        raise ValueError(f"scaling type must be one of {sorted(known)}, got {kind!r}")
    extra = set(scaling) - known[kind] - {"type"}
    if extra:
        raise ValueError(f"scaling {kind!r} takes no {sorted(extra)}")
    if "factor" not in scaling or ("original" in known[kind] and "original" not in scaling):
        raise ValueError(f"scaling {kind!r} needs {sorted(known[kind] & {'factor', 'original'})}")
    f = float(scaling["factor"])
    if not (f >= 1.0 and math.isfinite(f)):
        raise ValueError(f"scaling factor must be at least 1, got {f}")
    if kind == "linear":
        return freqs / f, 1.0
    if kind == "base":
        if rot_dim == 2:
            return freqs, 1.0
        return (base * f ** (rot_dim / (rot_dim - 2))) ** (-2.0 * i / rot_dim), 1.0
    n = float(scaling["original"])
    if not n > 0:
        raise ValueError(f"scaling original must be positive, got {n}")
    if kind == "bands":
        low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
        if not 0 < low < high:
            raise ValueError(f"scaling needs 0 < low < high, got {low}, {high}")
        turns = n * freqs / (2 * math.pi)
        kept = ((turns - low) / (high - low)).clamp(0.0, 1.0)      # share of the unscaled frequency
        return freqs * (kept + (1.0 - kept) / f), 1.0
    fast, slow = float(scaling.get("fast", 32.0)), float(scaling.get("slow", 1.0))
    if not 0 < slow < fast:
        raise ValueError(f"scaling needs 0 < slow < fast, got {slow}, {fast}")
    if not base > 1:
        raise ValueError(f"yarn scaling needs a base above 1, got {base}")

    def pair_with(turns):              # (fractional) index of the pair that turns so often over n positions
        return rot_dim * math.log(n / (2 * math.pi * turns)) / (2 * math.log(base))

    lo, hi = max(math.floor(pair_with(fast)), 0), min(math.ceil(pair_with(slow)), rot_dim - 1)
    ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    given = scaling.get("amplitude")
    return freqs * (1.0 - ramp + ramp / f), float(given) if given is not None else 0.1 * math.log(f) + 1.0


def _code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return _lib.BF16
    return _lib.dtype_code(t.dtype)


@functools.lru_cache(maxsize=256)
def _int64_3(a: int, b: int, c: int):
    return (_lib.c_int64 * 3)(a, b, c)


def _strides(x: torch.Tensor):
    return _int64_3(*x.stride()[:3])       # (read-only to the call)


def _turn(q, k, positions, freqs, interleaved, amplitude, inverse):
    """The launch: q [B, Hq, T, d] and k [B, Hkv, T, d] (or None) -> contiguous
    turned copies."""
    q = q if q.stride(-1) == 1 or q.numel() == 0 else q.contiguous()
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)    # (half of torch.empty's host time)
    ko, ks, Hkv = None, None, 0
    if k is not None:
        k = k if k.stride(-1) == 1 or k.numel() == 0 else k.contiguous()
        ko = torch.empty_like(k, memory_format=torch.contiguous_format)
        ks, Hkv = _strides(k), k.shape[1]
    B, Hq, T, d = q.shape
    with _lib.on_device(q):
        _lib.check(_lib.lib().pqkv_rotary(
            q.data_ptr(), _strides(q), qo.data_ptr(), Hq, _lib.ptr(k), ks, _lib.ptr(ko), Hkv, _code(q),
            positions.data_ptr(), positions.stride(0) if positions.dim() == 2 else 0, freqs.data_ptr(), B, T, d,
            2 * freqs.numel(), int(interleaved), amplitude, int(inverse), _lib.stream_of(q)))
    return qo, ko


def _has_tangent(*tensors) -> bool:
    """Whether any of them carries a forward-mode derivative."""
    if forward_ad._current_level < 0:          # (none is open: 0.1 us, where asking each tensor takes 1)
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, freqs, interleaved, amplitude, inverse):
        ctx.save_for_backward(positions, freqs)
        ctx.how = (interleaved, amplitude, not inverse)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(positions, freqs)
            ctx.shapes, ctx.dtype = (q.shape, None if k is None else k.shape), q.dtype
        ctx.set_materialize_grads(False)
        return _turn(q, k, positions, freqs, interleaved, amplitude, inverse)

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        # y = M x: the tangent is M times x's (which may be of another type)
        interleaved, amplitude, back = ctx.how
        turn = _Rotary.apply if torch.is_grad_enabled() else _turn
        _lib.require_one_device(tq, tk, *ctx.saved_tensors)            # (make_dual takes any)
        moving = [t.to(ctx.dtype) for t in (tq, tk) if t is not None]
        out = list(turn(*(moving + [None])[:2], *ctx.saved_tensors, interleaved, amplitude, not back))
        return tuple(None if shape is None else moving[0].new_zeros(shape) if t is None else out.pop(0)
                     for t, shape in zip((tq, tk), ctx.shapes))

    @staticmethod
    def backward(ctx, gq, gk):
        # y = M x with M a scaled rotation of each pair, so the gradient is the
        # same turn back: linear in g, and nothing of x is kept for it
        if not ctx.needs_input_grad[0]:
            gq = None
        if not ctx.needs_input_grad[1]:
            gk = None
        if gq is None and gk is None:
            return (None,) * 7
        # (create_graph, or gradients with tangents: differentiable again)
        turn = _Rotary.apply if torch.is_grad_enabled() or _has_tangent(gq, gk) else _turn
        if gq is None:
            out = (None, turn(gk, None, *ctx.saved_tensors, *ctx.how)[0])
        else:
            out = turn(gq, gk, *ctx.saved_tensors, *ctx.how)
        return *out, None, None, None, None, None


def apply_rotary(query: torch.Tensor, key: torch.Tensor | None, positions: torch.Tensor, frequencies: torch.Tensor, *,
                 interleaved: bool = False, amplitude: float = 1.0):
    """query [B, Hq, T, d] and key [B, Hkv, T, d] (or None) with the first
    2 * len(frequencies) coordinates of every head turned by positions *
    frequencies: -> (query, key), contiguous, in the inputs' type (fp16, bf16
    or fp32; one for both). positions: integers [T] or [B, T]; frequencies:
    radians per position, float64 (rotary_frequencies, on the device). Pairs
    are (i, i + rot_dim / 2), or neighbours with interleaved. The inputs may
    have any strides and may be expanded; gradients flow to both, and
    forward-mode tangents (torch.autograd.forward_ad) through them."""
    for name, x in (("query", query), ("key", key)):
        if x is not None and x.dim() != 4:
            raise ValueError(f"{name} must be [B, H, T, d], got {tuple(x.shape)}")
    B, _, T, d = query.shape
    if key is not None:
        if (key.shape[0], key.shape[2], key.shape[3]) != (B, T, d):
            raise ValueError(f"key {tuple(key.shape)} does not match query {tuple(query.shape)}")
        if key.dtype != query.dtype:
            raise ValueError(f"query is {query.dtype}, key {key.dtype}")
    _lib.require_device(query, key, positions, frequencies)
    _lib.require_one_device(query, key, positions, frequencies)
    _code(query)
    if frequencies.dim() != 1 or frequencies.dtype != torch.float64:
        raise ValueError("frequencies must be a float64 vector")
    if not 2 <= 2 * frequencies.numel() <= d:
        raise ValueError(f"{2 * frequencies.numel()} turned coordinates of a head of {d}")
    if positions.dtype.is_floating_point or positions.dtype.is_complex or positions.dtype == torch.bool:
        raise ValueError(f"positions must be integers, got {positions.dtype}")
    if tuple(positions.shape) not in ((T,), (B, T)):
        raise ValueError(f"positions must be [{T}] or [{B}, {T}], got {tuple(positions.shape)}")
    args = (query, key, positions.to(torch.int64).contiguous(), frequencies.contiguous(), bool(interleaved),
            float(amplitude))
    if (torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad))) or \
            _has_tangent(query, key):
        return _Rotary.apply(*args, False)
    return _turn(*args, False)


class RotaryEmbedding:
    """apply_rotary with the frequencies of one head shape: rot_dim (default:
    the whole head) of head_dim coordinates, base, scaling and pairing as
    rotary_frequencies and apply_rotary take them. The first call on a device
    copies the frequencies to it, which a graph capture does not allow: such a
    call is refused there."""

    def __init__(self, head_dim: int, rot_dim: int | None = None, base: float = 10000.0, scaling: dict | None = None,
                 interleaved: bool = False):
        self.head_dim = head_dim
        self.rot_dim = head_dim if rot_dim is None else int(rot_dim)
        if self.rot_dim > head_dim:
            raise ValueError(f"rot_dim {rot_dim} exceeds head_dim {head_dim}")
        self.interleaved = interleaved
        with torch.inference_mode(False):
            self.frequencies, self.amplitude = rotary_frequencies(self.rot_dim, base, scaling)
        self._on: dict = {}            # the frequencies on each device used

    def __call__(self, query: torch.Tensor, key: torch.Tensor | None, positions: torch.Tensor):
        freqs = self._on.get(query.device)
        if freqs is None:
            if query.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"call the embedding on {query.device} once before a capture")
            # they serve later calls, which may be differentiated whatever mode this one runs in
            with torch.inference_mode(False):
                freqs = self._on[query.device] = self.frequencies.to(query.device)
        return apply_rotary(query, key, positions, freqs, interleaved=self.interleaved, amplitude=self.amplitude)


__all__ = ["rotary_frequencies", "apply_rotary", "RotaryEmbedding"]
