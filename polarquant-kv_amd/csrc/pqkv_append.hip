// Appending keys and values to a cache, the keys turned by their positions on the
// way (pqkv_append_rotary, _paged).
//
// A key x becomes x' (pair (a, b) of its first rot_dim coordinates turned by t =
// position * frequency and scaled, in 32 bits, not rounded in between), y = R x',
// r = |y|, the nearest centroid of each y_j / r, and a block of fp16(r) and codes
// in slot start_b + token of its stream; a value the same without the turn. With
// signs the residual e = y / r - c[code] of a key is projected, bit i = (P_rot e)_i
// >= 0.
//
// Bound by memory for 16-bit inputs: 512 bytes read and 144 written per token and
// kv head (d = 128) beside 2 x 2 d^2 operations. The rotation runs on the matrix
// cores in parts: each vector is scaled by a power of two that puts its largest
// coordinate in [2^12, 2^13), x = x_hi + x_lo in fp16 (22 bits of the largest), R
// the same at 2^8 times its values, and R x = R_hi x_hi + R_lo x_hi + R_hi x_lo in
// 32 bits (what is left out is 2^-22 of a term). Whether a vector is close to a
// border between two codes is decided as exactly as fp32 products would.
//
// Work split: a workgroup (one per compute unit) keeps R's parts in LDS as
// operands and loops over items, runs of up to 64 (sequence, token) rows whose
// sines and cosines it puts into LDS once for all heads. A wave takes 16-vector
// tiles (16 tokens of one head, or with fewer tokens several heads) two at a time:
// every operand read serves both. The contraction runs over pairs: in each
// step of two matrix instructions a lane holds both sides of its eight pairs, so
// the turn needs no exchange, and R's columns are permuted to match; its rows
// are permuted so that a lane ends with 32 (d = 64: 16) neighbouring coordinates of
// one vector, a whole block of codes, which it packs and stores by itself. The
// sign product takes its residuals in that order, too: nothing leaves the lanes.
#include "pqkv_cells.h"
#include "pqkv_device.h"
#include "pqkv_launch.h"

namespace pqkv {

namespace {

constexpr int kAW = 8;                  // waves per workgroup
constexpr float kRScale = 256.0f;       // R's (and P_rot's) factor, 2^8

__device__ __forceinline__ float4_t mfma16(half8_t a, half8_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(half_t x) { return (float)x; }
__device__ __forceinline__ float widen(bf16_t x) { return bf16_to_float(x.bits); }

template <typename T>
struct alignas(16) Octet {
  T v[8];
};

// Sum and maximum over the four lanes of a vector (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float lanes_sum(float x) {
  x += shfl_xor_f(x, 16);
  return x + shfl_xor_f(x, 32);
}
__device__ __forceinline__ float lanes_max(float x) {
  x = fmaxf(x, shfl_xor_f(x, 16));
  return fmaxf(x, shfl_xor_f(x, 32));
}

// x as fp16 parts; x is made opaque, or the compiler may round a product once
// for one part and twice for the other.
__device__ __forceinline__ void split2(float x, half_t *hi, half_t *lo) {
  asm("" : "+v"(x));
  const half_t h = (half_t)x;
  *hi = h;
  *lo = (half_t)(x - (float)h);
}

template <int D, bool QJL>
struct AppendSmem {
  static constexpr int OT = D / 16, KS = D / 32;
  static constexpr int ROW = D / 2 * 8 + 16;      // bytes of a row's sines and cosines: 16 rows' 16-byte reads
                                                  // then fall into different banks
  static constexpr int ROWS = (QJL && D == 128 ? 8192 : 16384) / (D / 2 * 8);   // of an item
  half8_t r[OT][KS][2][64];                       // R's parts as operands: hi, lo
  half8_t p[QJL ? OT : 1][QJL ? KS : 1][2][QJL ? 64 : 1];
  uint2 cells[2][kECellSlots];                    // of the keys' and the values' codebook
  __attribute__((aligned(16))) uint8_t turn[ROWS * ROW];
  float cb[2][16];
  float thr[16];
  int ucell[16], table_ok[2];
};

struct AppendKernelArgs {
  AppendArgs a;
  int tt_shift;                   // tokens of a segment (a run of one sequence's), a power of two up to 16
  int token_blocks, segs;         // segments of a sequence, and in all
  int item_segs, items;
  FastDiv blocks_div, heads_div;  // by token_blocks and Hkv
};

// Coordinate of side s of pair p: the turned pairs, then what is left in pairs.
__device__ __forceinline__ int pair_coord(int p, int s, int rot, int d, bool inter) {
  if (inter) return 2 * p + s;
  const int h = rot / 2;
  return p < h ? p + s * h : rot + (p - h) + s * (d - rot) / 2;
}

template <typename T, int D, bool VEC, bool QJL>
__global__ void __launch_bounds__(kAW * 64, 1) append_kernel(const AppendKernelArgs k) {
  const AppendArgs &a = k.a;
  using SM = AppendSmem<D, QJL>;
  constexpr int OT = SM::OT, KS = SM::KS, NM = KS / 2;
  constexpr int NC = D / 4;                       // coordinates of a vector that a lane ends with
  __shared__ SM sm;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const bool inter = a.interleaved;
  const int nl = a.bits == 4 ? 16 : 4;

  // Operands: row r = n of tile o is coordinate NC (r / 4) + 4 o + r % 4, so that
  // lane group g's results are NC neighbouring ones; element j of step ks is side
  // ks & 1 of pair 8 (4 (ks / 2) + g) + j.
  for (int i = tid; i < OT * KS * 64; i += kAW * 64) {
    const int l = i & 63, ks = (i >> 6) % KS, o = (i >> 6) / KS;
    const float *row = a.R + (NC * ((l & 15) >> 2) + 4 * o + (l & 3)) * D;
    half8_t hi, lo;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      half_t h, w;
      split2(row[pair_coord(8 * (4 * (ks >> 1) + (l >> 4)) + j, ks & 1, a.rot_dim, D, inter)] * kRScale, &h, &w);
      hi[j] = h;
      lo[j] = w;
    }
    sm.r[o][ks][0][l] = hi;
    sm.r[o][ks][1][l] = lo;
    if constexpr (QJL) {
      // residuals stand in a lane in coordinate order: element j of step ks is
      // coordinate NC g + 8 ks + j
      const float *prow = a.p_rot + (NC * ((l & 15) >> 2) + 4 * o + (l & 3)) * D + NC * (l >> 4) + 8 * ks;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        half_t h, w;
        split2(prow[j] * kRScale, &h, &w);
        hi[j] = h;
        lo[j] = w;
      }
      sm.p[o][ks][0][l] = hi;
      sm.p[o][ks][1][l] = lo;
    }
  }
  if (tid < 32) sm.cb[tid >> 4][tid & 15] = (tid & 15) < nl ? (tid < 16 ? a.k_cb : a.v_cb)[tid & 15] : 0.0f;
  __syncthreads();
  build_cell_table<kAW * 64>(sm.cb[0], nl, tid, sm.cells[0], sm.thr, sm.ucell, &sm.table_ok[0]);
  const bool shared_cb = a.k_cb == a.v_cb;
  if (!shared_cb) build_cell_table<kAW * 64>(sm.cb[1], nl, tid, sm.cells[1], sm.thr, sm.ucell, &sm.table_ok[1]);
  const bool ok_k = sm.table_ok[0] != 0, ok_v = sm.table_ok[shared_cb ? 0 : 1] != 0;

  const int tt_mask = (1 << k.tt_shift) - 1;      // tokens of a segment - 1
  const int half = a.rot_dim / 2;

  for (int item = blockIdx.x; item < k.items; item += gridDim.x) {
    const int seg0 = item * k.item_segs;
    const int segs = min(k.item_segs, k.segs - seg0);
    __syncthreads();                              // the last item's table has been read
    for (int i = tid; i < (segs << k.tt_shift) * (D / 2); i += kAW * 64) {
      const int row = i / (D / 2), p = i % (D / 2);
      const int seg = seg0 + (row >> k.tt_shift);
      const int b = (int)k.blocks_div.div((uint32_t)seg);
      const int t = ((seg - b * k.token_blocks) << k.tt_shift) + (row & tt_mask);
      float2 cs = make_float2(1.0f, 0.0f);        // what is not turned
      if (p < half && t < a.T) {
        const int64_t at = (int64_t)b * a.pos_batch_stride + a.axes.of[p] * a.axes.stride + t;
        const double turns = (double)a.positions[at] * (a.freqs[p] * 0.15915494309189533577);   // 1 / (2 pi)
        const float frac = (float)(turns - __builtin_rint(turns));
        float s, c;
        sincospif(2.0f * frac, &s, &c);
        cs = make_float2(a.amplitude * c, a.amplitude * s);
      }
      *(float2 *)(sm.turn + row * SM::ROW + p * 8) = cs;
    }
    __syncthreads();

    const int pairs = segs * a.Hkv;               // (segment, head) pairs of the item
    const int per = 16 >> k.tt_shift;             // of a tile
    const int kind_tiles = (pairs + per - 1) / per, tiles = 2 * kind_tiles;

    struct Where {
      const T *src;
      uint8_t *dst, *sign;
      int row;
      bool ok;
    };
    auto locate = [&](int tile) {
      Where w;
      const bool key = tile < kind_tiles;
      const int q = (key ? tile : tile - kind_tiles) * per + (n >> k.tt_shift);
      const int sl = (int)k.heads_div.div((uint32_t)q), h = q - sl * a.Hkv;
      const int seg = seg0 + sl, b0 = (int)k.blocks_div.div((uint32_t)seg);
      const int t0 = ((seg - b0 * k.token_blocks) << k.tt_shift) + (n & tt_mask);
      w.ok = q < pairs && t0 < a.T;
      const int b = w.ok ? b0 : 0, t = w.ok ? t0 : 0, hh = w.ok ? h : 0;   // (loads of a vector that exists)
      w.row = w.ok ? (sl << k.tt_shift) + (n & tt_mask) : 0;
      const int64_t *st = key ? a.k_stride : a.v_stride;
      w.src = (const T *)(key ? a.k : a.v) + b * st[0] + hh * st[1] + t * st[2];
      const int64_t start = a.starts ? a.starts[b] : a.start;
      w.ok = w.ok && start >= 0 && start < a.S && start + t < a.S && (!a.counts || t < a.counts[b]);
      const int slot = w.ok ? (int)start + t : 0;
      const int64_t stream = (int64_t)b * a.Hkv + hh;
      w.dst = w.sign = nullptr;
      if (w.ok) {
        if (a.k_pages) {
          const int64_t pg = stream * a.max_pages + (slot >> a.page_shift);
          const int in = slot & ((1 << a.page_shift) - 1);
          w.dst = (key ? a.k_pages : a.v_pages)[pg] + (int64_t)in * a.vec_bytes;
          if (QJL && key) w.sign = a.s_pages[pg] + in * (D / 8);
        } else {
          w.dst = (key ? a.k_blocks : a.v_blocks) + (stream * a.S + slot) * a.vec_bytes;
          if (QJL && key) w.sign = a.signs + (stream * a.S + slot) * (D / 8);
        }
      }
      return w;
    };

    // x's parts as operands, and what undoes their power of two and R's
    auto load = [&](const Where &w, bool key, half8_t (&hi)[KS], half8_t (&lo)[KS], float &undo) {
      float x[NM][2][8];
      float top = 0.0f;
#pragma unroll
      for (int m = 0; m < NM; ++m) {
        const int p0 = 8 * (4 * m + g);
        if constexpr (VEC) {
          const int c0 = inter ? 2 * p0 : pair_coord(p0, 0, a.rot_dim, D, false);
          const int c1 = inter ? 2 * p0 + 8 : pair_coord(p0, 1, a.rot_dim, D, false);
          const Octet<T> u = *(const Octet<T> *)(w.src + c0), v = *(const Octet<T> *)(w.src + c1);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            x[m][0][j] = widen(inter ? (j < 4 ? u.v[(2 * j) & 7] : v.v[(2 * j) & 7]) : u.v[j]);
            x[m][1][j] = widen(inter ? (j < 4 ? u.v[(2 * j + 1) & 7] : v.v[(2 * j + 1) & 7]) : v.v[j]);
          }
        } else {
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[m][s][j] = widen(w.src[pair_coord(p0 + j, s, a.rot_dim, D, inter)]);
        }
        if (key) {
          const float4 *tr = (const float4 *)(sm.turn + w.row * SM::ROW + p0 * 8);
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const float4 cs = tr[j >> 1];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float c = e ? cs.z : cs.x, s = e ? cs.w : cs.y;
              const float u = x[m][0][j + e], v = x[m][1][j + e];
              x[m][0][j + e] = u * c - v * s;
              x[m][1][j + e] = u * s + v * c;
            }
          }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[m][s][j]));
      }
      top = lanes_max(top);
      // 2^(12 - exponent): biased 266 - E, held within the normal numbers
      const int E = (int)(__builtin_bit_cast(uint32_t, top) >> 23);
      const int up = min(266 - E, 254);
      const float scale = __builtin_bit_cast(float, (uint32_t)up << 23);
      undo = __builtin_ldexpf(1.0f / kRScale, 127 - up);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          half_t h, l;
          split2(x[ks >> 1][ks & 1][j] * scale, &h, &l);
          hi[ks][j] = h;
          lo[ks][j] = l;
        }
    };

    // Codes of a lane's coordinates: four (two) dwords of 4-bit codes for d = 128
    // (64), half as many of 2-bit ones; e: the residuals in units of the radius.
    auto quantise = [&](const float4_t (&acc)[OT], bool key, float undo, uint32_t (&word)[NC / 8], uint16_t &radius,
                        float (&e)[QJL ? NC : 1]) {
      float ss = 0.0f;
#pragma unroll
      for (int o = 0; o < OT; ++o)
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = __builtin_fmaf(acc[o][i], acc[o][i], ss);
      ss = lanes_sum(ss);
      const float rs = __fsqrt_rn(ss), r = rs * undo;
      // a vector of zeros has direction 0
      const float inv = r <= 1e-30f ? 0.0f : __fdiv_rn(1.0f, rs);
      radius = radius_half_bits(r);
      const float live = inv == 0.0f ? 0.0f : 1.0f;   // (its residual is 0 as well)
      const uint2 *cells = sm.cells[key || shared_cb ? 0 : 1];
      const float *cb = sm.cb[key ? 0 : 1];
#pragma unroll
      for (int i = 0; i < NC / 8; ++i) word[i] = 0;
      // (a lookup needs |direction| <= 1; numbers that are none have index 0)
      const bool plain = (key ? ok_k : ok_v) && ss < __builtin_inff();
      const bool all_plain = __builtin_amdgcn_ballot_w64(!plain) == 0;
#pragma unroll
      for (int o = 0; o < OT; ++o)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = acc[o][i] * inv;
          int c;
          if (all_plain) c = table_code(cells, u);
          else c = u == u ? scan_index_rolled(u, cb, nl) : 0;
          const int at = 4 * o + i;
          if (a.bits == 4) word[at >> 3] |= (uint32_t)c << (4 * (at & 7));
          else word[at >> 4] |= (uint32_t)c << (2 * (at & 15));
          if constexpr (QJL) e[at] = __builtin_fmaf(-live, cb[c], u);
        }
    };

    typedef uint32_t u32a __attribute__((aligned(2)));
    typedef uint32_t u32x2a __attribute__((ext_vector_type(2), aligned(2)));
    typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(2)));
    auto store = [&](const Where &w, const uint32_t (&word)[NC / 8], uint16_t radius) {
      if (!w.ok) return;
      const int bb = a.bits == 4 ? kPq4BlockBytes : kPq2BlockBytes;
      if constexpr (D == 128) {
        uint8_t *p = w.dst + g * bb;
        *(uint16_t *)p = radius;
        if (a.bits == 4) *(u32x4a *)(p + 2) = u32x4a{word[0], word[1], word[2], word[3]};
        else *(u32x2a *)(p + 2) = u32x2a{word[0], word[1]};
      } else {
        uint8_t *p = w.dst + (g >> 1) * bb;
        if ((g & 1) == 0) *(uint16_t *)p = radius;
        if (a.bits == 4) *(u32x2a *)(p + 2 + 8 * (g & 1)) = u32x2a{word[0], word[1]};
        else *(u32a *)(p + 2 + 4 * (g & 1)) = word[0];
      }
    };

    // signs of the residuals e: lane group g's results are projections NC g ..
    auto sketch = [&](const Where &w, const float (&e)[QJL ? NC : 1]) {
      if constexpr (QJL) {
        half8_t eh[KS], el[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            half_t h, l;
            // (residuals are below 2: 2^12 keeps the low parts normal)
            split2(e[8 * ks + j] * 4096.0f, &h, &l);
            eh[ks][j] = h;
            el[ks][j] = l;
          }
        uint32_t bits = 0;
#pragma unroll
        for (int o = 0; o < OT; ++o) {
          float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const half8_t ph = sm.p[o][ks][0][lane], pl = sm.p[o][ks][1][lane];
            acc = mfma16(ph, eh[ks], acc);
            acc = mfma16(pl, eh[ks], acc);
            acc = mfma16(ph, el[ks], acc);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) bits |= acc[i] >= 0.0f ? 1u << (4 * o + i) : 0u;
        }
        if (w.ok) {
          if constexpr (D == 128) *(uint32_t *)(w.sign + 4 * g) = bits;
          else *(uint16_t *)(w.sign + 2 * g) = (uint16_t)bits;
        }
      }
    };

    auto run = [&](auto count, int tile) {
      constexpr int NT = decltype(count)::value;
      Where w[NT];
      half8_t hi[NT][KS], lo[NT][KS];
      float undo[NT];
      bool key[NT];
#pragma unroll
      for (int v = 0; v < NT; ++v) {
        key[v] = tile + kAW * v < kind_tiles;
        w[v] = locate(tile + kAW * v);
      }
#pragma unroll
      for (int v = 0; v < NT; ++v) load(w[v], key[v], hi[v], lo[v], undo[v]);
      float4_t acc[NT][OT];
#pragma unroll
      for (int o = 0; o < OT; ++o) {
#pragma unroll
        for (int v = 0; v < NT; ++v) acc[v][o] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const half8_t rh = sm.r[o][ks][0][lane], rl = sm.r[o][ks][1][lane];
#pragma unroll
          for (int v = 0; v < NT; ++v) acc[v][o] = mfma16(rh, hi[v][ks], acc[v][o]);
#pragma unroll
          for (int v = 0; v < NT; ++v) acc[v][o] = mfma16(rl, hi[v][ks], acc[v][o]);
#pragma unroll
          for (int v = 0; v < NT; ++v) acc[v][o] = mfma16(rh, lo[v][ks], acc[v][o]);
        }
      }
#pragma unroll
      for (int v = 0; v < NT; ++v) {
        uint32_t word[NC / 8];
        uint16_t radius;
        float e[QJL ? NC : 1];
        quantise(acc[v], key[v], undo[v], word, radius, e);
        store(w[v], word, radius);
        if (QJL && key[v]) sketch(w[v], e);
      }
    };
    int tile = wave;
    for (; tile + kAW < tiles; tile += 2 * kAW) run(std::integral_constant<int, 2>{}, tile);
    if (tile < tiles) run(std::integral_constant<int, 1>{}, tile);
  }
}

template <typename T, int D, bool VEC>
hipError_t launch_vec(const AppendKernelArgs &a, int blocks, hipStream_t s) {
  if (a.a.p_rot) append_kernel<T, D, VEC, true><<<blocks, kAW * 64, 0, s>>>(a);
  else append_kernel<T, D, VEC, false><<<blocks, kAW * 64, 0, s>>>(a);
  return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_type(const AppendArgs &a, hipStream_t s) {
  // tokens of a segment: as many as a tile has vectors, or all of fewer
  int tt_shift = 0;
  while (tt_shift < 4 && (1 << tt_shift) < a.T) ++tt_shift;
  const int token_blocks = (a.T + (1 << tt_shift) - 1) >> tt_shift, segs = a.B * token_blocks;
  // segments of an item: as many as give each wave two tiles, fewer where that
  // leaves compute units idle (but whole tiles), within the table's rows
  const int cus = device_compute_units();
  const int per = 16 >> tt_shift;
  const int most = (a.p_rot ? AppendSmem<D, true>::ROWS : AppendSmem<D, false>::ROWS) >> tt_shift;
  int n = (kAW * per + a.Hkv - 1) / a.Hkv;
  const int spread = (segs + cus - 1) / cus, whole = (per + a.Hkv - 1) / a.Hkv;
  if (n > spread) n = spread > whole ? spread : whole;
  if (n > most) n = most;
  const int items = (segs + n - 1) / n;
  const AppendKernelArgs k{a, tt_shift, token_blocks, segs, n, items, FastDiv(token_blocks), FastDiv(a.Hkv)};
  constexpr int SZ = sizeof(T);
  uintptr_t at = (uintptr_t)a.k | (uintptr_t)a.v;
  int64_t el = a.interleaved ? 0 : a.rot_dim / 2;
  for (int i = 0; i < 3; ++i) el |= a.k_stride[i] | a.v_stride[i];
  const int blocks = items < cus ? items : cus;
  const bool vec = at % 16 == 0 && el % 8 == 0;
  static_assert(SZ == 2 || SZ == 4, "eight elements are whole 16-byte pieces");
  return vec ? launch_vec<T, D, true>(k, blocks, s) : launch_vec<T, D, false>(k, blocks, s);
}

}  // namespace

hipError_t launch_append(const AppendArgs &a, int dtype, hipStream_t s) {
  if (a.d == 128) {
    if (dtype == PQKV_F32) return launch_type<float, 128>(a, s);
    if (dtype == PQKV_F16) return launch_type<half_t, 128>(a, s);
    return launch_type<bf16_t, 128>(a, s);
  }
  if (dtype == PQKV_F32) return launch_type<float, 64>(a, s);
  if (dtype == PQKV_F16) return launch_type<half_t, 64>(a, s);
  return launch_type<bf16_t, 64>(a, s);
}

}  // namespace pqkv
