"""Eviction: a cache cut to the positions that attention used most.

No counterpart in the reference, whose token importance assigns widths by
position only (src/polarquant_kv_cuda/token_importance.py:17-40). The weights
come from attention.decode_attention_weights and attention.attention_weights,
added up over the steps; here the positions that stay are chosen
(select_positions, pqkv_evict_select) and their keys, values, signs, weights
and positions moved into a new cache in one launch (pqkv_gather_rows). They
keep their order, so the last positions of a cache are its newest ones before
and after.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from .types import PagedPQCache, PQCache, vector_bytes


def _check_budget(S: int, keep: int, sink: int, recent: int) -> None:
    if sink < 0 or recent < 0:
        raise ValueError(f"sink={sink} and recent={recent} must not be negative")
    if not min(S, sink + recent) <= keep <= S:
        raise ValueError(f"keep={keep} must be between sink + recent = {sink + recent} and the {S} positions held")


def _check_rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """t with rows [B, H] one stride apart and dense."""
    if t.is_contiguous():
        return t
    B, H, S = t.shape
    dense = t.stride(2) == 1 or S <= 1
    if not dense or (B > 1 and H > 1 and t.stride(0) != H * t.stride(1)) or _row_stride(t) < S:
        return t.contiguous()
    return t


def _row_stride(t: torch.Tensor) -> int:
    """Elements between consecutive (batch, head) rows of a [B, H, S] tensor."""
    B, H, S = t.shape
    if t.is_contiguous() or B * H <= 1:
        return max(S, 1)
    return t.stride(1) if H > 1 else t.stride(0)


def select_positions(weights: torch.Tensor, keep: int, sink: int = 0, recent: int = 0) -> torch.Tensor:
    """weights [B, H, S] float32 -> int32 [B, H, keep], ascending: the first
    `sink` and last `recent` positions and the heaviest of the others; equal
    weights by the lowest index, NaN below every weight."""
    if weights.dim() != 3 or weights.dtype != torch.float32:
        raise ValueError(f"weights must be [B, H, S] float32, got {tuple(weights.shape)} {weights.dtype}")
    _lib.require_device(weights)
    B, H, S = weights.shape
    _check_budget(S, keep, sink, recent)
    weights = _check_rows(weights, "weights")
    kept = torch.empty(B, H, keep, dtype=torch.int32, device=weights.device)
    with _lib.on_device(weights):
        _lib.check(_lib.lib().pqkv_evict_select(weights.data_ptr(), _row_stride(weights), B * H, S, keep, sink, recent,
                                                kept.data_ptr(), _lib.stream_of(weights)))
    return kept


def _cache_arrays(cache):
    """(fields of pqkv_row_array, row bytes) of a cache's blocks and, with
    signs, of those."""
    vb = vector_bytes(cache.head_dim, cache.n_bits)
    if isinstance(cache, PagedPQCache):
        out = [((0, cache.table.data_ptr(), 0, cache.page_tokens, cache.max_pages), vb)]
        if cache.sign_table is not None:
            out.append(((0, cache.sign_table.data_ptr(), 0, cache.page_tokens, cache.max_pages),
                        cache.jl_dim // 8))
        return out
    out = [((cache.blocks.data_ptr(), 0, cache.max_seq_len * vb, 0, 0), vb)]
    if cache.qjl_signs is not None:
        m8 = cache.qjl_signs.shape[-1]
        out.append(((cache.qjl_signs.data_ptr(), 0, cache.max_seq_len * m8, 0, 0), m8))
    return out


def _empty_like(cache, positions: int, room: int):
    """A cache of the same kind for `positions` positions (a contiguous one of
    `room` positions) whose rows (and, paged, tables) are not yet written, and
    its arrays as _cache_arrays gives them."""
    B, H, d = cache.batch, cache.num_heads, cache.head_dim
    if isinstance(cache, PagedPQCache):
        if positions == 0:
            return PagedPQCache(B, H, d, cache.n_bits, cache.codebooks, cache.device, cache.page_tokens,
                                cache.jl_dim, 1), ()
        new = PagedPQCache(B, H, d, cache.n_bits, cache.codebooks, cache.device, cache.page_tokens, cache.jl_dim,
                           tables=False)
        P, n = cache.page_tokens, -(-positions // cache.page_tokens)
        return new, [((pool.data_ptr(), table.data_ptr(), n * P * pool.shape[-1], P, n), pool.shape[-1])
                     for pool, table in zip(new.reserve(positions), (new.table, new.sign_table))]
    fresh, signs = cache.blocks.new_empty if room == positions else cache.blocks.new_zeros, None
    if cache.qjl_signs is not None:
        signs = fresh((B, H, room, cache.qjl_signs.shape[-1]))
    new = PQCache(blocks=fresh((B, H, room, vector_bytes(d, cache.n_bits))),
                  head_dim=d, n_bits=cache.n_bits, seq_len=0, max_seq_len=room, codebooks=cache.codebooks,
                  qjl_signs=signs, jl_dim=cache.jl_dim)
    return new, _cache_arrays(new)


def _check_cache(cache, name: str, B: int, H: int, device) -> None:
    if cache.mixed:
        raise ValueError(f"{name}: caches of one width per head are not moved")
    if (cache.batch, cache.num_heads) != (B, H):
        raise ValueError(f"{name}: batch {cache.batch} and heads {cache.num_heads}, expected {B} and {H}")
    if isinstance(cache, PagedPQCache):
        if cache.capacity < cache.seq_len:
            raise ValueError(f"{name}: fewer pages than its seq_len needs")
        arrays = [cache.table, cache.sign_table]
    else:
        need = cache.max_seq_len * vector_bytes(cache.head_dim, cache.n_bits)
        if cache.blocks.numel() < B * H * need or not cache.blocks.is_contiguous():
            raise ValueError(f"{name}: blocks must be contiguous and cover the cache's shape")
        if not 0 <= cache.seq_len <= cache.max_seq_len:
            raise ValueError(f"{name}: seq_len {cache.seq_len} outside 0..{cache.max_seq_len}")
        s = cache.qjl_signs
        if s is not None and (s.numel() < B * H * cache.max_seq_len * s.shape[-1] or not s.is_contiguous()):
            raise ValueError(f"{name}: signs must be contiguous and cover the cache's shape")
        arrays = [cache.blocks, s]
    _lib.require_device(*arrays)
    for t in arrays:
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, the kept positions on {device}")


def gather_positions(caches, kept: torch.Tensor, rows=(), room: int | None = None):
    """New caches (of the same kinds, seq_len = keep) with position i of stream
    (b, h) the old position kept[b, h, i], and, for each [B, H, >= S] 4-byte
    tensor in `rows`, the new [B, H, keep] one: one launch for all. caches: at
    most two with signs, four without; contiguous results hold `room` positions
    (default: keep). A kept position outside the cache gives zeros."""
    if kept.dim() != 3 or kept.dtype != torch.int32:
        raise ValueError(f"kept must be [B, H, keep] int32, got {tuple(kept.shape)} {kept.dtype}")
    _lib.require_device(kept, *rows)
    _lib.require_one_device(kept, *rows)
    kept = kept if kept.is_contiguous() else kept.contiguous()
    B, H, keep = kept.shape
    room = keep if room is None else int(room)
    if room < keep:
        raise ValueError(f"room for {room} positions, {keep} are kept")
    if not caches:
        raise ValueError("at least one cache is required")
    S = caches[0].seq_len
    for i, c in enumerate(caches):
        _check_cache(c, f"cache {i}", B, H, kept.device)
        if c.seq_len != S:
            raise ValueError(f"cache {i} holds {c.seq_len} positions, the first one {S}")
    src, dst, sizes, new_rows = [], [], [], []
    with _lib.on_device(kept):
        new, fill = [], keep
        for old in caches:
            c, arrays = _empty_like(old, keep, room)
            if isinstance(c, PagedPQCache):
                if fill not in (keep, c.capacity):
                    raise ValueError("paged caches in one move must share page_tokens")
                fill = c.capacity
            for (a, size), (n, _) in zip(_cache_arrays(old), arrays):
                src += a
                dst += n
                sizes.append(size)
            c.seq_len = keep
            new.append(c)
        held = []                      # copies that the launch reads
        for t in rows:
            if t.dim() != 3 or t.element_size() != 4 or t.shape[:2] != (B, H) or t.shape[2] < S:
                raise ValueError(f"rows must be 4-byte [{B}, {H}, >= {S}] tensors, got {tuple(t.shape)} {t.dtype}")
            t = _check_rows(t, "rows")
            held.append(t)
            n = torch.empty_like(kept, dtype=t.dtype)
            src.extend((t.data_ptr(), 0, 4 * _row_stride(t), 0, 0))
            dst.extend((n.data_ptr(), 0, 4 * keep, 0, 0))
            sizes.append(4)
            new_rows.append(n)
        if len(sizes) > _lib.MAX_GATHER:
            raise ValueError(f"{len(sizes)} arrays in one move, at most {_lib.MAX_GATHER}")
        if keep > 0:
            _lib.check(_lib.lib().pqkv_gather_rows(len(sizes), _lib.row_arrays(src), _lib.row_arrays(dst),
                                                   _lib.int_array(sizes), kept.data_ptr(), B * H, S, keep, fill,
                                                   _lib.stream_of(kept)))
    return new, new_rows


@dataclass
class Eviction:
    """What evict() returns: the new caches, the old index of every position
    they hold, and the weights and positions (None where none were given)
    moved with them."""
    keys: "PQCache | PagedPQCache"
    values: "PQCache | PagedPQCache"
    kept: torch.Tensor                       # int32 [B, H, keep]
    weights: torch.Tensor                    # float32 [B, H, keep]
    positions: "torch.Tensor | None" = None  # int32 [B, H, keep]


def evict(keys, values, weights: torch.Tensor, keep: int, *, sink: int = 0, recent: int = 0,
          positions: torch.Tensor | None = None, room: int | None = None) -> Eviction:
    """Cut keys and values (both PQCache, or both PagedPQCache; one width each) to
    `keep` positions per (batch, head) by weights [B, H, >= seq_len] float32
    (select_positions over the first seq_len). positions: int32 [B, H, >=
    seq_len], moved along. The old caches are left as they are: their memory
    goes back when the caller drops them."""
    B, H, S = keys.batch, keys.num_heads, keys.seq_len
    if isinstance(keys, PagedPQCache) != isinstance(values, PagedPQCache):
        raise ValueError("keys and values must both be paged caches, or both PQCache")
    if values.seq_len != S:
        raise ValueError("keys and values hold different numbers of positions")
    if weights.dim() != 3 or weights.shape[:2] != (B, H) or weights.shape[2] < S or weights.dtype != torch.float32:
        raise ValueError(f"weights must be [{B}, {H}, >= {S}] float32, got {tuple(weights.shape)} {weights.dtype}")
    if positions is not None and positions.dtype != torch.int32:
        raise ValueError(f"positions must be int32, got {positions.dtype}")
    kept = select_positions(weights[:, :, :S], keep, sink, recent)
    rows = [weights] if positions is None else [weights, positions]
    (k, v), moved = gather_positions([keys, values], kept, rows, room)
    return Eviction(keys=k, values=v, kept=kept, weights=moved[0], positions=moved[1] if len(moved) > 1 else None)


__all__ = ["select_positions", "gather_positions", "evict", "Eviction"]
