"""Appending to a compressed cache with the rotation on the way (device tensors
only).

No counterpart in the reference, whose layers have no positions and whose cache
appends by concatenation (src/polarquant_kv_cuda/inference/kv_cache.py:96-116).
append_rotary is rotary.apply_rotary and two quantizer.compress_pq calls in one:
the turned keys are encoded as they are, without having been rounded and stored in
between, and every sequence has slots of its own (pqkv_append_rotary, _paged).
"""

from __future__ import annotations

import torch

from . import _lib
from .attention import _codebook_tables, check_paged, check_shapes, check_signs, page_tables, row_counts, row_starts
from .rotary import _code, _has_tangent, _strides, apply_rotary, check_axes, position_strides
from .types import PagedPQCache


def append_rotary(key: torch.Tensor, value: torch.Tensor, keys, values, rotation_matrix: torch.Tensor,
                  positions: torch.Tensor, frequencies: torch.Tensor, *, query: torch.Tensor | None = None, starts=None,
                  counts: torch.Tensor | None = None, interleaved: bool = False, amplitude: float = 1.0, axes=None,
                  jl_rot: torch.Tensor | None = None):
    """key and value [B, Hkv, T, d] into the caches `keys` and `values` (both
    PQCache, or both PagedPQCache; one width), the keys turned by positions *
    frequencies on the way; query [B, Hq, T, d] is turned too and returned
    (contiguous, in its type), else None; gradients and forward-mode tangents flow
    through it as through rotary.apply_rotary (not through what is cached). fp16, bf16
    or fp32, one for all; any strides. positions, frequencies, interleaved, amplitude and axes as
    rotary.apply_rotary takes them. jl_rot = P R^T adds the keys' QJL signs.

    starts: the slot of each sequence's first token: a number for all, by default
    seq_len, with which the caches grow (pages are added, seq_len covers the new
    slots), or integers [B] on the device, for sequences of different lengths: the
    kernel reads them, so that a captured call follows them, and neither pages
    (PagedPQCache.ensure) nor seq_len change. counts ([B], device): how many of the T
    tokens each sequence has, in a padded chunk. Tokens past them, or whose slot the
    caches have no room for, are not written."""
    for name, x in (("key", key), ("value", value), ("query", query)):
        if x is not None and x.dim() != 4:
            raise ValueError(f"{name} must be [B, H, T, d], got {tuple(x.shape)}")
    B, Hkv, T, d = key.shape
    if value.shape != key.shape:
        raise ValueError(f"value {tuple(value.shape)} does not match key {tuple(key.shape)}")
    if query is not None and (query.shape[0], query.shape[2], query.shape[3]) != (B, T, d):
        raise ValueError(f"query {tuple(query.shape)} does not match key {tuple(key.shape)}")
    if value.dtype != key.dtype or (query is not None and query.dtype != key.dtype):
        raise ValueError("query, key and value must have one type")
    if frequencies.dim() != 1 or frequencies.dtype != torch.float64:
        raise ValueError("frequencies must be a float64 vector")
    if not 2 <= 2 * frequencies.numel() <= d:
        raise ValueError(f"{2 * frequencies.numel()} turned coordinates of a head of {d}")
    if positions.dtype.is_floating_point or positions.dtype.is_complex or positions.dtype == torch.bool:
        raise ValueError(f"positions must be integers, got {positions.dtype}")
    given_axes = axes
    if axes is not None:
        axes = check_axes(axes, positions, frequencies.numel(), B, T)
    elif tuple(positions.shape) not in ((T,), (B, T)):
        raise ValueError(f"positions must be [{T}] or [{B}, {T}], got {tuple(positions.shape)}")
    dtype = _code(key)
    paged = isinstance(keys, PagedPQCache) or isinstance(values, PagedPQCache)
    if (check_paged if paged else check_shapes)(B, Hkv, d, keys, values, rotation_matrix) != Hkv:
        raise ValueError(f"{Hkv} kv heads, the caches have {keys.num_heads}")
    if keys.mixed or values.mixed or keys.n_bits != values.n_bits:
        raise ValueError("keys and values must be of one and the same width")
    check_signs(jl_rot, keys, d)
    if jl_rot is None and keys.qjl_signs is not None:
        raise ValueError("the key cache keeps QJL signs: pass jl_rot")
    _lib.require_device(key, value, query, positions, frequencies, rotation_matrix, jl_rot)
    _lib.require_one_device(key, value, query, positions, frequencies, rotation_matrix, jl_rot, keys.codebooks,
                            keys.table if paged else keys.blocks, values.codebooks,
                            values.table if paged else values.blocks)
    start, starts = row_starts(keys.seq_len if starts is None else starts, T, B, key.device)
    counts = row_counts(counts, B, key.device)
    if starts is None:
        if start < 0 or (not paged and start + T > keys.max_seq_len):
            raise ValueError(f"slots {start}..{start + T - 1} of a cache of {keys.max_seq_len if not paged else 'pages'}")
        if paged:
            if key.is_cuda and torch.cuda.is_current_stream_capturing() and \
                    start + T > min(keys.capacity, values.capacity):
                raise RuntimeError("a captured append needs its pages before (ensure)")
            keys.ensure(start + T)
            values.ensure(start + T)
            check_paged(B, Hkv, d, keys, values)        # (one width of tables again)
    turned = None
    if query is not None and ((torch.is_grad_enabled() and query.requires_grad) or _has_tangent(query)):
        turned, _ = apply_rotary(query, None, positions, frequencies, interleaved=interleaved, amplitude=amplitude,
                                 axes=given_axes)
        query = None
    k, v, q = (x if x is None or x.stride(-1) == 1 or x.numel() == 0 else x.contiguous() for x in (key, value, query))
    positions = positions.to(torch.int64)
    if axes is None or positions.stride(-1) != 1:
        positions = positions.contiguous()
    freqs = frequencies.contiguous()
    R, P = _lib.dense_f32(rotation_matrix), _lib.dense_f32(jl_rot)
    out = None if q is None else torch.empty_like(q, memory_format=torch.contiguous_format)
    lib = _lib.lib()
    by_axis, by_row, n_axes = position_strides(positions, axes)
    S = min(keys.capacity, values.capacity) if paged else keys.max_seq_len
    kcb, vcb = (keys.codebooks, values.codebooks) if paged else _codebook_tables(keys, values, False, Hkv)
    head = (k.data_ptr(), _strides(k), v.data_ptr(), _strides(v), _lib.ptr(q), None if q is None else _strides(q),
            _lib.ptr(out), 0 if q is None else q.shape[1], dtype, positions.data_ptr(), by_axis, by_row, n_axes, axes,
            freqs.data_ptr(), 2 * freqs.numel(), int(bool(interleaved)), float(amplitude), R.data_ptr(),
            kcb.data_ptr(), vcb.data_ptr(), keys.n_bits, _lib.ptr(P), d if P is not None else 0, B, Hkv, T, d, start,
            _lib.ptr(starts), _lib.ptr(counts), S)
    stream = _lib.stream_of(k)
    with _lib.on_device(k):
        if paged:
            ktab, vtab, stab, max_pages = page_tables(keys, values)
            _lib.check(lib.pqkv_append_rotary_paged(*head, ktab.data_ptr(), vtab.data_ptr(), keys.page_tokens,
                                                    max_pages, stab.data_ptr() if P is not None else None, stream))
        else:
            _lib.check(lib.pqkv_append_rotary(*head, keys.blocks.data_ptr(), values.blocks.data_ptr(),
                                              keys.qjl_signs.data_ptr() if P is not None else None, stream))
    if starts is None:
        for c in (keys, values):
            c.seq_len = max(c.seq_len, start + T)
    return out if turned is None else turned


__all__ = ["append_rotary"]
