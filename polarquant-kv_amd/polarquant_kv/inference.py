"""Inference-side cache and attention layer on the compressed format.

Mirrors src/polarquant_kv_cuda/inference/{config,kv_cache,attention}.py of
the reference with the same names and arguments:

  PolarQuantConfig             n_bits, group_size, jl_dim, enable_qjl,
                               enable_compression (config.py)
  KVCacheManager               append / get_kv / reset / seq_len /
                               memory_bytes / compression_ratio (kv_cache.py:14-134)
  CompressedMultiHeadAttention q/k/v/o projections, forward(x, cache_manager)
                               (attention.py:12-95)

Differences, all on purpose:
  - the compressed caches are paged (PagedPQCache): they grow by pages of
    page_tokens positions as the sequence grows, and append encodes the new
    positions straight into their pages through the page table
    (pqkv_encode_paged), never copying what is cached (the reference
    concatenates the whole cache with torch.cat on every append,
    kv_cache.py:96-116), so a decode step costs O(new tokens), not O(S), and
    memory follows the sequence, not max_seq_len (a limit only); attention
    runs the paged decode / chunked-prefill kernels;
  - the layout is block_pq4 / block_pq2 with Lloyd-Max centroids (the
    reference manager stores its per-group min/scale format);
  - with enable_qjl the keys carry the QJL sign sketch and attention adds
    the correction (the reference manager never writes signs, kv_cache.py:112);
  - CompressedMultiHeadAttention applies the causal rule to a multi-token
    chunk on every path (query i of a chunk at positions p0.. sees positions
    <= p0 + i): the compressed cache, the uncompressed cache and no cache.
    The reference calls non-causal SDPA / compressed attention on all three
    (inference/attention.py:63-92), so a chunk's queries see its later
    tokens; causal=False reproduces that;
  - a manager can keep how much attention weight each cached position has
    got (track_weights) and cut its caches to the heaviest ones (evict), so a
    sequence may grow past max_seq_len cached positions;
  - the attention layer can turn its queries and keys by their positions
    (rotary), which the manager counts apart from the slots of its caches.
All GPU work goes through libpqkv_hip.so.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import _lib, attention, quantizer
from .types import PagedPQCache


@dataclass
class PolarQuantConfig:
    n_bits: int = 4
    group_size: int = 32
    jl_dim: int = 64
    enable_qjl: bool = False
    enable_compression: bool = True


class KVCacheManager:
    """Compressed KV cache of one attention layer: up to max_seq_len
    positions per (batch, head), kept in pages of page_tokens positions
    (a power of two, >= 64), filled by prefill (several tokens) and decode
    (one token) appends. With track_weights, attend() also adds up the
    softmax weight that each cached position gets, for evict()."""

    def __init__(self, config: PolarQuantConfig, max_seq_len: int, batch: int, num_heads: int, head_dim: int,
                 device: str = "cuda", rotation_seed: int = 42, page_tokens: int = 256, track_weights: bool = False):
        from .rotation import generate_rotation_matrix
        if config.enable_compression:
            quantizer._validate_params(config.n_bits, config.group_size, head_dim)
            if config.n_bits not in (2, 4):
                raise ValueError(f"the codebook format stores 2- or 4-bit codes, got n_bits={config.n_bits}")
        elif track_weights:
            raise ValueError("weights are kept for compressed caches")
        self.config = config
        self.track_weights = track_weights
        self.page_tokens = int(page_tokens)
        self.max_seq_len = int(max_seq_len)
        self.batch = batch
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.device = device
        self.R = generate_rotation_matrix(head_dim, seed=rotation_seed, device=device)
        self.jl_rot = None
        if config.enable_compression and config.enable_qjl:
            if config.jl_dim != head_dim:
                raise ValueError(f"the QJL sketch here has m = head_dim projections (jl_dim={config.jl_dim}, "
                                 f"head_dim={head_dim})")
            from .qjl import generate_jl_matrix, rotated_jl_matrix
            self.jl_matrix = generate_jl_matrix(config.jl_dim, head_dim, seed=rotation_seed + 1)
            self.jl_rot = rotated_jl_matrix(self.jl_matrix, self.R.cpu().numpy(), device)
        self._keys: PagedPQCache | None = None
        self._values: PagedPQCache | None = None
        self._key_cache: torch.Tensor | None = None
        self._value_cache: torch.Tensor | None = None
        self._seq_len = 0
        self._next_position = 0
        # with track_weights: [batch, num_heads, room] of every slot, room >= seq_len
        self._weights: torch.Tensor | None = None
        self._positions: torch.Tensor | None = None

    # ---- allocation ----
    def _allocate(self):
        if self.config.enable_compression:
            B, H, d, bits = self.batch, self.num_heads, self.head_dim, self.config.n_bits
            self._keys = quantizer.allocate_paged_cache(B, H, d, bits, self.device, page_tokens=self.page_tokens,
                                                        jl_dim=d if self.jl_rot is not None else 0)
            self._values = quantizer.allocate_paged_cache(B, H, d, bits, self.device, page_tokens=self.page_tokens)
        else:
            shape = (self.batch, self.num_heads, self.max_seq_len, self.head_dim)
            with _lib.lasting():
                self._key_cache = torch.zeros(shape, dtype=torch.float16, device=self.device)
                self._value_cache = torch.zeros(shape, dtype=torch.float16, device=self.device)

    @property
    def seq_len(self) -> int:
        return self._seq_len

    @property
    def next_position(self) -> int:
        """Position of the next appended token: how many were appended since
        the last reset, those evicted since among them."""
        return self._next_position

    @property
    def weights(self) -> torch.Tensor | None:
        """[batch, num_heads, seq_len] float32: the attention weight each cached
        position has got (track_weights)."""
        return None if self._weights is None else self._weights[:, :, :self._seq_len]

    @property
    def positions(self) -> torch.Tensor | None:
        """[batch, num_heads, seq_len] int32: where the token of each slot
        stood in its sequence (track_weights)."""
        return None if self._positions is None else self._positions[:, :, :self._seq_len]

    @property
    def memory_bytes(self) -> int:
        """Bytes of the cached positions (K + V, and the QJL signs)."""
        if self._seq_len == 0:
            return 0
        n = self.batch * self.num_heads * self._seq_len
        if not self.config.enable_compression:
            return 2 * n * self.head_dim * 2
        from .types import vector_bytes
        per = 2 * vector_bytes(self.head_dim, self.config.n_bits)
        if self.jl_rot is not None:
            per += self.head_dim // 8
        return n * per

    @property
    def allocated_bytes(self) -> int:
        """Device bytes held: the pages allocated so far (and their tables,
        weights and positions); uncompressed, the max_seq_len-position arrays."""
        if self.config.enable_compression:
            if self._keys is None:
                return 0
            tracked = 0 if self._weights is None else 8 * self._weights.numel()
            return self._keys.memory_bytes() + self._values.memory_bytes() + tracked
        return 0 if self._key_cache is None else 2 * self._key_cache.numel() * 2

    @property
    def compression_ratio(self) -> float:
        if self._seq_len == 0:
            return 0.0
        original = self.batch * self.num_heads * self._seq_len * self.head_dim * 2 * 2   # K + V, fp16
        return original / self.memory_bytes

    # ---- writes ----
    def append(self, key: torch.Tensor, value: torch.Tensor) -> None:
        """key / value [batch, num_heads, new_seq, head_dim] (fp16 or fp32) at
        positions seq_len .. seq_len + new_seq - 1, encoded into their pages
        (pages are added as the positions need them)."""
        if key.shape != value.shape or key.dim() != 4:
            raise ValueError("key and value must both be [batch, num_heads, new_seq, head_dim]")
        B, H, T, d = key.shape
        if (B, H, d) != (self.batch, self.num_heads, self.head_dim):
            raise ValueError(f"shape {tuple(key.shape)} does not match the cache "
                             f"({self.batch}, {self.num_heads}, *, {self.head_dim})")
        if self._seq_len + T > self.max_seq_len:
            raise RuntimeError(f"KV cache full: {self._seq_len} + {T} > {self.max_seq_len}")
        if self._keys is None and self._key_cache is None:
            self._allocate()
        if self.track_weights:                 # (first: if it fails, nothing is in the caches)
            self._track(T)
        if self.config.enable_compression:
            quantizer.compress_pq(key, self.R, cache=self._keys, start=self._seq_len, jl_rot=self.jl_rot)
            quantizer.compress_pq(value, self.R, cache=self._values, start=self._seq_len)
        else:
            self._key_cache[:, :, self._seq_len:self._seq_len + T] = key.to(torch.float16)
            self._value_cache[:, :, self._seq_len:self._seq_len + T] = value.to(torch.float16)
        self._seq_len += T
        self._next_position += T

    def _track(self, T: int) -> None:
        """Slots seq_len .. seq_len + T - 1: no weight yet, and the next positions."""
        S, need = self._seq_len, self._seq_len + T
        room = 0 if self._weights is None else self._weights.shape[2]
        if need > room:
            room = min(max(need, 2 * room, self.page_tokens), self.max_seq_len)
            shape = (self.batch, self.num_heads, room)
            with _lib.lasting():
                w = torch.zeros(shape, dtype=torch.float32, device=self.device)
                p = torch.zeros(shape, dtype=torch.int32, device=self.device)
            if S:
                w[:, :, :S], p[:, :, :S] = self._weights[:, :, :S], self._positions[:, :, :S]
            self._weights, self._positions = w, p
        else:
            self._weights[:, :, S:need] = 0.0
        self._positions[:, :, S:need] = torch.arange(self._next_position, self._next_position + T, dtype=torch.int32,
                                                     device=self.device)

    def get_kv(self):
        """Compressed: the two PagedPQCache objects (seq_len positions valid);
        uncompressed: views of the first seq_len positions."""
        if not self.config.enable_compression:
            if self._key_cache is None:
                return None, None
            return self._key_cache[:, :, :self._seq_len], self._value_cache[:, :, :self._seq_len]
        return self._keys, self._values

    def reset(self) -> None:
        """Forget the cached positions (the pages are kept for reuse)."""
        self._seq_len = 0
        self._next_position = 0
        for c in (self._keys, self._values):
            if c is not None:
                c.seq_len = 0

    def evict(self, keep: int, sink: int = 4, recent: int = 64):
        """Cut the caches to `keep` positions per (batch, head): the first
        `sink`, the last `recent` and those with the most attention weight so
        far, in their order (eviction.evict; needs track_weights). Nothing is
        done when no more than that are cached. Returns the Eviction, whose
        caches, weights and positions are the manager's own from then on, or
        None."""
        if not self.track_weights:
            raise ValueError("evict() needs track_weights")
        if keep < 1 or keep < sink + recent:
            raise ValueError(f"keep={keep} must be at least 1 and sink + recent = {sink + recent}")
        if self._seq_len <= keep:
            return None
        from . import eviction
        with _lib.lasting():
            r = eviction.evict(self._keys, self._values, self._weights, keep, sink=sink, recent=recent,
                               positions=self._positions)
        self._keys, self._values, self._weights, self._positions = r.keys, r.values, r.weights, r.positions
        self._seq_len = keep
        return r

    # ---- reads ----
    def attend(self, query: torch.Tensor, causal: bool = True) -> torch.Tensor:
        """query [batch, q_heads, Sq, head_dim] for the last Sq cached
        positions -> [batch, q_heads, Sq, head_dim] fp16: compressed
        attention (decode for Sq = 1, causal prefill otherwise) with the QJL
        term when the manager keeps signs. With track_weights the queries'
        weights are added to those of the cached positions."""
        if self._seq_len == 0:
            return torch.zeros_like(query, dtype=torch.float16)
        if not self.config.enable_compression:
            k, v = self.get_kv()
            rep = query.shape[1] // k.shape[1]
            k = k.float().repeat_interleave(rep, 1)
            v = v.float().repeat_interleave(rep, 1)
            Sq, S = query.shape[2], k.shape[2]
            s = torch.matmul(query.float(), k.transpose(-1, -2).contiguous()) / math.sqrt(self.head_dim)
            if causal and Sq > 1:
                pos = torch.arange(S, device=query.device)
                qpos = torch.arange(S - Sq, S, device=query.device)
                s = s.masked_fill(pos[None, :] > qpos[:, None], float("-inf"))
            return torch.matmul(torch.softmax(s, -1), v).half()
        Sq = query.shape[2]
        start = self._seq_len - Sq
        if self.track_weights:
            w = self._weights
            if Sq == 1:
                out, _ = attention.decode_attention_weights(query[:, :, 0], self._keys, self._values, self.R,
                                                            jl_rot=self.jl_rot, out_dtype=torch.float16, previous=w,
                                                            into=w)
                return out.unsqueeze(2)
            # the weights last: a call that fails has added none of them
            out = attention.prefill_attention(query, self._keys, self._values, self.R, start, causal=causal,
                                              out_dtype=torch.float16, jl_rot=self.jl_rot)
            attention.attention_weights(query, self._keys, self.R, start, causal=causal, jl_rot=self.jl_rot,
                                        previous=w, into=w)
            return out
        jl = self.jl_matrix if self.jl_rot is not None else None
        return attention.compressed_attention_gpu(query, self._keys, self._values, self.R, jl_matrix=jl,
                                                  causal=causal, q_start=start)


class CompressedMultiHeadAttention(torch.nn.Module):
    """Multi-head (GQA) attention whose KV cache is the compressed one
    (src/polarquant_kv_cuda/inference/attention.py:12-95). rotary
    (rotary.RotaryEmbedding of the head's size): queries and keys turned by
    their positions before the keys are cached."""

    def __init__(self, config: PolarQuantConfig, embed_dim: int, num_heads: int, num_kv_heads: int | None = None,
                 causal: bool = True, rotary=None):
        super().__init__()
        self.config = config
        self.rotary = rotary
        self.causal = causal
        self.embed_dim = embed_dim
        self.num_heads = num_heads
        self.num_kv_heads = num_kv_heads or num_heads
        self.head_dim = embed_dim // num_heads
        if rotary is not None and rotary.head_dim != self.head_dim:
            raise ValueError(f"rotary head_dim {rotary.head_dim}, the layer's {self.head_dim}")
        self.q_proj = torch.nn.Linear(embed_dim, num_heads * self.head_dim, bias=False)
        self.k_proj = torch.nn.Linear(embed_dim, self.num_kv_heads * self.head_dim, bias=False)
        self.v_proj = torch.nn.Linear(embed_dim, self.num_kv_heads * self.head_dim, bias=False)
        self.o_proj = torch.nn.Linear(num_heads * self.head_dim, embed_dim, bias=False)

    def forward(self, x: torch.Tensor, cache_manager: KVCacheManager | None = None) -> torch.Tensor:
        """x [batch, seq_len, embed_dim] -> [batch, seq_len, embed_dim]. With a
        cache manager the new keys and values are appended and the queries
        attend to everything cached (causally unless causal=False)."""
        B, T, _ = x.shape
        q = self.q_proj(x).reshape(B, T, self.num_heads, self.head_dim).transpose(1, 2).half()
        k = self.k_proj(x).reshape(B, T, self.num_kv_heads, self.head_dim).transpose(1, 2).half()
        v = self.v_proj(x).reshape(B, T, self.num_kv_heads, self.head_dim).transpose(1, 2).half()
        if self.rotary is not None:
            start = 0 if cache_manager is None else cache_manager.next_position
            q, k = self.rotary(q, k, torch.arange(start, start + T, device=x.device))
        if cache_manager is not None:
            cache_manager.append(k.contiguous(), v.contiguous())
            out = cache_manager.attend(q.contiguous(), causal=self.causal)
        else:
            rep = self.num_heads // self.num_kv_heads
            kk = k.float().repeat_interleave(rep, 1)
            vv = v.float().repeat_interleave(rep, 1)
            s = torch.matmul(q.float(), kk.transpose(-1, -2).contiguous()) / math.sqrt(self.head_dim)
            if self.causal:
                mask = torch.ones(T, T, dtype=torch.bool, device=x.device).triu(1)
                s = s.masked_fill(mask, float("-inf"))
            out = torch.matmul(torch.softmax(s, -1), vv).half()
        out = out.transpose(1, 2).reshape(B, T, -1)
        return self.o_proj(out.to(self.o_proj.weight.dtype))
