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
// operands (64 KB at d = 128) and loops over items, runs of 16 to 64 (sequence, token)
// rows whose sines and cosines it puts into LDS once for all heads, an item ahead.
// A wave takes one 16-vector tile at a time (16 tokens of one head, or with fewer
// tokens several heads); sixteen waves, four per SIMD, hide each other's waits, and a
// wave's next inputs are requested before it works on these. The contraction runs
// over pairs: in each step of two matrix instructions a lane holds both sides of its
// eight pairs, so the turn needs no exchange, and R's columns are permuted to match;
// its rows are permuted so that a lane ends with 32 (d = 64: 16) neighbouring
// coordinates of one vector, a whole block of codes, which it packs and stores by
// itself. The sign product takes its residuals in that order, too: nothing leaves
// the lanes.
//
// Measured (bf16, d = 128, 32768 tokens of 8 heads): 80-95 us box to box, 172 MB at
// 1.8 to 2.1 TB/s, 51 GFLOP (three products) at 540 to 640 TFLOP/s. Of its cycles the
// vector units issue for 51 % (20 instructions a coordinate: turn, parts, radius, a table
// lookup and a compare), the matrix cores are busy for 31 %, LDS for 42 % (R's 64 KB of
// operands a tile, lookups, sines; 14 % are bank conflicts of the lookups): no one bound,
// the first two share a SIMD's issue. Eight waves of two tiles each took 125; 64 rows to
// an item 88 where 32 take 90 and a step's rows alone 93. The same at 2 bits 79, with
// signs (eight waves, 16 rows to an item) 129 and at 2 bits 127, of fp32 inputs 100 (24
// registers spilled by sixteen waves, so eight), at d = 64 43 us, in replayed graphs.
// One token of 8 sequences takes 16 us: of 33 000 cycles the table of codes is 10 700,
// first loads and R's parts 9 000, the sines 4 100, the tile 10 200. Searching the
// codebook instead, or R's loads ahead of the table, were no faster (19.4 and 15.9).
#include "pqkv_cells.h"
#include "pqkv_device.h"
#include "pqkv_launch.h"

namespace pqkv {

namespace {

// Waves of a workgroup: four per SIMD, which hide each other's waits, where their
// 128 registers are enough (sixteen waves spill 24 registers of 32-bit inputs at d =
// 128, 80 and more where inputs come element by element or with signs).
template <typename T, int D, bool VEC, bool QJL>
constexpr int append_waves() {
  return D == 64 || (VEC && sizeof(T) == 2 && !QJL) ? 16 : 8;
}
constexpr float kRScale = 256.0f;       // R's (and P_rot's) factor, 2^8

__device__ __forceinline__ float4_t mfma16(half8_t a, half8_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(half_t x) { return (float)x; }
__device__ __forceinline__ float widen(bf16_t x) { return bf16_to_float(x.bits); }

// What a kernel only reads, at an address that is the same for all lanes: through
// the scalar cache, so that no vector load is waited for.
template <typename T>
__device__ __forceinline__ T uniform(const T *p) {
  return *(const __attribute__((address_space(4))) T *)(uintptr_t)p;
}

template <typename T>
struct alignas(16) Octet {
  T v[8];
};

// Sum and maximum over the four lanes of a vector (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float lanes_sum(float x) {
  auto p = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  x = __builtin_bit_cast(float, (uint32_t)p[0]) + __builtin_bit_cast(float, (uint32_t)p[1]);
  auto q = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return __builtin_bit_cast(float, (uint32_t)q[0]) + __builtin_bit_cast(float, (uint32_t)q[1]);
}
__device__ __forceinline__ float lanes_max(float x) {
  auto p = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  x = fmaxf(__builtin_bit_cast(float, (uint32_t)p[0]), __builtin_bit_cast(float, (uint32_t)p[1]));
  auto q = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)q[0]), __builtin_bit_cast(float, (uint32_t)q[1]));
}

// x * s (s a power of two) as fp16 parts: one mixed multiply-add each. The high
// part is made opaque, or the compiler may round the product once for it and
// twice for the difference.
__device__ __forceinline__ void split2(float x0, float x1, float s, half2_t *hi, half2_t *lo) {
  half2_t h = {(half_t)(x0 * s), (half_t)(x1 * s)};
  asm("" : "+v"(h));
  *hi = h;
  *lo = half2_t{(half_t)__builtin_fmaf(x0, s, -(float)h[0]), (half_t)__builtin_fmaf(x1, s, -(float)h[1])};
}
__device__ __forceinline__ void split8(const float *x, float s, half8_t *hi, half8_t *lo) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    half2_t h, l;
    split2(x[j], x[j + 1], s, &h, &l);
    (*hi)[j] = h[0];
    (*hi)[j + 1] = h[1];
    (*lo)[j] = l[0];
    (*lo)[j + 1] = l[1];
  }
}

template <int D, bool QJL>
struct AppendSmem {
  static constexpr int OT = D / 16, KS = D / 32;
  static constexpr int ROW = D / 2 * 8 + 16;      // bytes of a row's sines and cosines: 16 rows' 16-byte reads
                                                  // then fall into different banks
  static constexpr int ROWS = D == 64 ? 64 : QJL ? 16 : 32;   // of an item
  // beside P_rot a second codebook has no room for a table: its values are scanned for
  static constexpr int TABLES = QJL && D == 128 ? 1 : 2;
  half8_t r[OT][KS][2][64];                       // R's parts as operands: hi, lo
  half8_t p[QJL ? OT : 1][QJL ? KS : 1][2][QJL ? 64 : 1];
  uint2 cells[TABLES][kECellSlots];               // of the keys' and the values' codebook
  __attribute__((aligned(16))) uint8_t turn[2][ROWS * ROW];   // of an item and the next
  int slot[2][ROWS];                              // of a row's token, or -1: not to be written
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

// RUNS: 16 tokens or more of a sequence (a tile is a run of one head's tokens);
// else a tile holds all tokens of several (sequence, head) pairs.
template <typename T, int D, bool VEC, bool QJL, bool RUNS, int kAW = append_waves<T, D, VEC, QJL>()>
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

  const bool shared_cb = a.k_cb == a.v_cb;
  bool ok_k, ok_v;                                // whether the codebooks have tables
  const int tt_shift = RUNS ? 4 : k.tt_shift, tt_mask = (1 << tt_shift) - 1;   // tokens of a segment
  const int per = 16 >> tt_shift;                 // (segment, head) pairs of a tile
  constexpr int HP = D / 2, RS = kAW * 64 / HP;   // pairs of a row; rows that the threads make at a time
  constexpr int NR = SM::ROWS / RS;               // and how often

  // Sines and cosines of an item's rows. A thread has one pair, and the rows RS
  // apart, whose positions (`ahead`) it loads an item before (loaded with the table
  // they cost a prompt of 32768 tokens 10 of 90 us).
  const int pr = tid % HP, row0 = tid / HP;
  const double freq = pr < a.rot_dim / 2 ? a.freqs[pr] * 0.15915494309189533577 : 0.0;   // 1 / (2 pi)
  const int64_t axis = pr < a.rot_dim / 2 ? a.axes.of[pr] * a.axes.stride : 0;
  auto rows_of = [&](int item) { return min(k.item_segs, k.segs - item * k.item_segs) << tt_shift; };
  auto where = [&](int item, int row, int &b, int &t) {
    const int seg = item * k.item_segs + (row >> tt_shift);
    b = (int)k.blocks_div.div((uint32_t)seg);
    t = ((seg - b * k.token_blocks) << tt_shift) + (row & tt_mask);
  };
  int64_t ahead[NR];
  auto positions = [&](int item) {
    const int rows = rows_of(item);
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      int b, t;
      const int row = row0 + RS * j;
      where(item, row < rows ? row : 0, b, t);    // (a row's number is within the calls: token 0 for those past T)
      ahead[j] = a.positions[(int64_t)b * a.pos_batch_stride + axis + (t < a.T ? t : 0)];
    }
  };
  auto table = [&](int item, int buf) {
    const int rows = rows_of(item);
    if constexpr (!RUNS) {
      for (int row = tid; row < rows; row += kAW * 64) {
        int b, t;
        where(item, row, b, t);
        const int64_t start = a.starts ? a.starts[b] : a.start;
        const bool ok = t < a.T && start >= 0 && start < a.S && start + t < a.S && (!a.counts || t < a.counts[b]);
        sm.slot[buf][row] = ok ? (int)start + t : -1;
      }
    }
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      const int row = row0 + RS * j;
      if (row >= rows) break;
      const double turns = (double)ahead[j] * freq;
      const float frac = (float)(turns - __builtin_rint(turns));
      float s, c;
      sincospif(2.0f * frac, &s, &c);
      // what is not turned has frequency 0, and is not scaled
      const float m = pr < a.rot_dim / 2 ? a.amplitude : 1.0f;
      *(float2 *)(sm.turn[buf] + row * SM::ROW + pr * 8) = make_float2(m * c, m * s);
    }
  };

  // A tile of an item: 16 vectors, `row` the item's row of this lane's, `stream` its
  // (sequence, head), slot where it goes or -1 (RUNS: known here, else with the
  // item's table).
  struct Vec {
    const T *src;
    int row, stream, slot;
  };
  auto locate = [&](int item, int tile, bool key, int kind_tiles, int pairs) {
    Vec w;
    const int seg0 = item * k.item_segs;
    const int64_t *st = key ? a.k_stride : a.v_stride;
    const T *base = (const T *)(key ? a.k : a.v);
    const int tl = key ? tile : tile - kind_tiles;
    if constexpr (RUNS) {                         // the same segment and head for all lanes
      const int sl = (int)k.heads_div.div((uint32_t)tl), h = tl - sl * a.Hkv;
      const int seg = seg0 + sl, b = (int)k.blocks_div.div((uint32_t)seg);
      const int t0 = (seg - b * k.token_blocks) << 4;
      const int64_t start = a.starts ? uniform(a.starts + b) : a.start;
      int64_t count = a.counts ? uniform(a.counts + b) : a.T;
      count = start >= 0 && start < a.S ? min(min(count, (int64_t)a.T), a.S - start) : 0;
      w.row = 16 * sl + n;
      w.stream = b * a.Hkv + h;
      w.slot = t0 + n < count ? (int)start + t0 + n : -1;
      // (a vector past the end reads the segment's first)
      w.src = base + b * st[0] + h * st[1] + (int64_t)(t0 + n < a.T ? t0 + n : t0) * st[2];
    } else {
      const int q = tl * per + (n >> tt_shift);
      const int sl = (int)k.heads_div.div((uint32_t)q), h = q - sl * a.Hkv;
      const int seg = seg0 + sl, b0 = (int)k.blocks_div.div((uint32_t)seg);
      const int t0 = ((seg - b0 * k.token_blocks) << tt_shift) + (n & tt_mask);
      const bool ok = q < pairs && t0 < a.T;
      const int b = ok ? b0 : 0, hh = ok ? h : 0;
      w.row = ok ? (sl << tt_shift) + (n & tt_mask) : -1;
      w.stream = b * a.Hkv + hh;
      w.slot = -1;
      w.src = base + b * st[0] + hh * st[1] + (int64_t)(ok ? t0 : 0) * st[2];
    }
    return w;
  };
  // Its inputs: NM x two octets, sides a and b of eight pairs (interleaved: the 16
  // coordinates as they lie).
  struct Raw {
    Octet<T> x[NM][2];
  };
  int off[NM][2];
#pragma unroll
  for (int m = 0; m < NM; ++m) {
    const int p0 = 8 * (4 * m + g);
    off[m][0] = inter ? 2 * p0 : pair_coord(p0, 0, a.rot_dim, D, false);
    off[m][1] = inter ? 2 * p0 + 8 : pair_coord(p0, 1, a.rot_dim, D, false);
  }
  // (inputs that come element by element are loaded where they are used)
  auto fetch = [&](const Vec &w, Raw &raw) {
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      raw.x[m][0] = *(const Octet<T> *)(w.src + off[m][0]);
      raw.x[m][1] = *(const Octet<T> *)(w.src + off[m][1]);
    }
  };
  // x's parts as operands, and what undoes their power of two and R's.
  auto parts_of = [&](auto turn, auto neighbours, const Raw &raw, const Vec &w, int buf, half8_t (&hi)[KS],
                      half8_t (&lo)[KS], float &undo) {
    float x[KS][8];
    float top = 0.0f;
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      float (&xa)[8] = x[2 * m];
      float (&xb)[8] = x[2 * m + 1];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (!VEC) {
          const int p = 8 * (4 * m + g) + j;
          xa[j] = widen(w.src[pair_coord(p, 0, a.rot_dim, D, inter)]);
          xb[j] = widen(w.src[pair_coord(p, 1, a.rot_dim, D, inter)]);
        } else if constexpr (decltype(neighbours)::value) {
          xa[j] = widen(raw.x[m][j >> 2].v[(2 * j) & 7]);
          xb[j] = widen(raw.x[m][j >> 2].v[(2 * j + 1) & 7]);
        } else {
          xa[j] = widen(raw.x[m][0].v[j]);
          xb[j] = widen(raw.x[m][1].v[j]);
        }
      }
      if constexpr (decltype(turn)::value) {
        const float4 *tr = (const float4 *)(sm.turn[buf] + w.row * SM::ROW + 64 * (4 * m + g));
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float4 cs = tr[j >> 1];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float c = e ? cs.z : cs.x, s = e ? cs.w : cs.y;
            const float u = xa[j + e], v = xb[j + e];
            xa[j + e] = u * c - v * s;
            xb[j + e] = u * s + v * c;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(fmaxf(fabsf(xa[j]), fabsf(xb[j])), top);
    }
    top = lanes_max(top);
    // 2^(12 - exponent): biased 266 - E, held within the normal numbers
    const int up = min(266 - (int)(__builtin_bit_cast(uint32_t, top) >> 23), 254);
    const float scale = __builtin_bit_cast(float, (uint32_t)up << 23);
    undo = __builtin_ldexpf(1.0f / kRScale, 127 - up);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) split8(x[ks], scale, &hi[ks], &lo[ks]);
  };
  auto parts = [&](const Raw &raw, bool key, const Vec &w, int buf, half8_t (&hi)[KS], half8_t (&lo)[KS], float &undo) {
    const std::true_type yes;
    const std::false_type no;
    if (key) {
      if (VEC && inter) parts_of(yes, yes, raw, w, buf, hi, lo, undo);
      else parts_of(yes, no, raw, w, buf, hi, lo, undo);
    } else {
      if (VEC && inter) parts_of(no, yes, raw, w, buf, hi, lo, undo);
      else parts_of(no, no, raw, w, buf, hi, lo, undo);
    }
  };

  // Codes of a lane's coordinates: four (two) dwords of 4-bit codes for d = 128
  // (64), half as many of 2-bit ones; e: the residuals in units of the radius.
  auto quantise = [&](const float4_t (&acc)[OT], bool key, float undo, uint32_t (&word)[NC / 8], uint16_t &radius,
                      float (&e)[QJL ? NC : 1]) {
    float part[4] = {};
#pragma unroll
    for (int o = 0; o < OT; ++o)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[i] = __builtin_fmaf(acc[o][i], acc[o][i], part[i]);
    const float ss = lanes_sum((part[0] + part[1]) + (part[2] + part[3]));
    // 1 / r to an ulp (a sum of squares of at least 2^40, unless all are 0)
    const float rsq = ss > 0.0f ? __builtin_amdgcn_rsqf(ss) : 0.0f;
    const float r = ss * rsq * undo;
    // a vector of zeros has direction 0
    const float inv = r <= 1e-30f ? 0.0f : rsq;
    radius = radius_half_bits(r);
    const float live = inv == 0.0f ? 0.0f : 1.0f;   // (its residual is 0 as well)
    const uint2 *cells = sm.cells[key || shared_cb ? 0 : SM::TABLES - 1];
    const float *cb = sm.cb[key ? 0 : 1];
    // (a lookup needs |direction| <= 1; numbers that are none have index 0)
    const bool plain = (key ? ok_k : ok_v) && ss < __builtin_inff();
    const bool all_plain = __builtin_amdgcn_ballot_w64(!plain) == 0;
    auto codes = [&](auto table, auto bits) {
      constexpr int B = decltype(bits)::value, W = 32 / B;   // codes of a dword
      int c[NC];
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const float u = acc[i >> 2][i & 3] * inv;
        if constexpr (decltype(table)::value) c[i] = table_code(cells, u);
        else c[i] = u == u ? scan_index_rolled(u, cb, nl) : 0;
        if constexpr (QJL) e[i] = __builtin_fmaf(-live, cb[c[i]], u);
      }
#pragma unroll
      for (int i = 0; i < NC / W; ++i) {
        word[i] = 0;
#pragma unroll
        for (int j = W - 1; j >= 0; --j) word[i] = (word[i] << B) + (uint32_t)c[W * i + j];
      }
    };
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 2> two;
    if (all_plain) {
      if (a.bits == 4) codes(std::true_type{}, four);
      else codes(std::true_type{}, two);
    } else {
      if (a.bits == 4) codes(std::false_type{}, four);
      else codes(std::false_type{}, two);
    }
  };

  // A lane's block of codes. RUNS: through buffers over the stream (or the one or two
  // pages that 16 slots lie in), which drop what has no slot: no branch, so that
  // what waits for a load does not wait for the stores after it.
  typedef uint32_t u32a __attribute__((aligned(2)));
  typedef uint32_t u32x2a __attribute__((ext_vector_type(2), aligned(2)));
  typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(2)));
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const int bb = a.bits == 4 ? kPq4BlockBytes : kPq2BlockBytes;
  const int piece = D == 128 ? g * bb : (g >> 1) * bb, codes_at = piece + 2 + (D == 128 ? 0 : a.bits * 2 * (g & 1));
  constexpr int kNowhere = -16;                   // an offset past every buffer's end, all of a store's bytes
  auto put_buffer = [&](uint8_t *base, uint32_t bytes, int at, const uint32_t (&word)[NC / 8], uint16_t radius) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(base, (short)0, (int)bytes, 0x00020000);
    const int ra = at < 0 || (D == 64 && (g & 1)) ? kNowhere : at + piece, ca = at < 0 ? kNowhere : at + codes_at;
    __builtin_amdgcn_raw_buffer_store_b16(radius, r, ra, 0, 0);
    if constexpr (D == 128) {
      if (a.bits == 4) __builtin_amdgcn_raw_buffer_store_b128((u32x4){word[0], word[1], word[2], word[3]}, r, ca, 0, 0);
      else __builtin_amdgcn_raw_buffer_store_b64((u32x2){word[0], word[1]}, r, ca, 0, 0);
    } else {
      if (a.bits == 4) __builtin_amdgcn_raw_buffer_store_b64((u32x2){word[0], word[1]}, r, ca, 0, 0);
      else __builtin_amdgcn_raw_buffer_store_b32(word[0], r, ca, 0, 0);
    }
  };
  // (wave-uniform) the first slot of a run, and its stream
  struct Run {
    int first, stream;
  };
  auto run_of = [&](const Vec &w) {
    return Run{__builtin_amdgcn_readfirstlane(w.slot), __builtin_amdgcn_readfirstlane(w.stream)};
  };
  auto store = [&](const Vec &w, bool key, const uint32_t (&word)[NC / 8], uint16_t radius) {
    if constexpr (RUNS) {
      const Run run = run_of(w);                  // (slots of a run: the first ones have theirs)
      if (a.k_pages) {
        uint8_t *const *pages = (key ? a.k_pages : a.v_pages) + (int64_t)run.stream * a.max_pages;
        const int mask = (1 << a.page_shift) - 1, bytes = (mask + 1) * a.vec_bytes;
        const int pg = max(run.first, 0) >> a.page_shift, pl = min(max(run.first, 0) + 15, a.S - 1) >> a.page_shift;
        const int at = (w.slot & mask) * a.vec_bytes;
        put_buffer(uniform(pages + pg), bytes, w.slot >= 0 && (w.slot >> a.page_shift) == pg ? at : -1, word, radius);
        if (pl != pg) put_buffer(uniform(pages + pl), bytes, w.slot >= 0 && (w.slot >> a.page_shift) != pg ? at : -1, word, radius);
      } else {
        uint8_t *base = (key ? a.k_blocks : a.v_blocks) + ((int64_t)run.stream * a.S + max(run.first, 0)) * a.vec_bytes;
        put_buffer(base, 16 * a.vec_bytes, w.slot >= 0 ? (w.slot - run.first) * a.vec_bytes : -1, word, radius);
      }
    } else {
      if (w.slot < 0) return;
      uint8_t *p;
      if (a.k_pages) {
        p = (key ? a.k_pages : a.v_pages)[(int64_t)w.stream * a.max_pages + (w.slot >> a.page_shift)] +
            (w.slot & ((1 << a.page_shift) - 1)) * a.vec_bytes;
      } else {
        p = (key ? a.k_blocks : a.v_blocks) + ((int64_t)w.stream * a.S + w.slot) * a.vec_bytes;
      }
      if (D == 128 || (g & 1) == 0) *(uint16_t *)(p + piece) = radius;
      p += codes_at;
      if constexpr (D == 128) {
        if (a.bits == 4) *(u32x4a *)p = u32x4a{word[0], word[1], word[2], word[3]};
        else *(u32x2a *)p = u32x2a{word[0], word[1]};
      } else {
        if (a.bits == 4) *(u32x2a *)p = u32x2a{word[0], word[1]};
        else *(u32a *)p = word[0];
      }
    }
  };

  // signs of the residuals e: lane group g's results are projections NC g ..
  auto sketch = [&](const Vec &w, const float (&e)[QJL ? NC : 1]) {
    if constexpr (QJL) {
      half8_t eh[KS], el[KS];
      // (residuals are below 2: 2^12 keeps the low parts normal)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) split8(e + 8 * ks, 4096.0f, &eh[ks], &el[ks]);
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
      const int slot = w.slot;
      if (slot >= 0) {
        uint8_t *p;
        if (a.k_pages)
          p = a.s_pages[(int64_t)w.stream * a.max_pages + (slot >> a.page_shift)] +
              (slot & ((1 << a.page_shift) - 1)) * (D / 8);
        else p = a.signs + ((int64_t)w.stream * a.S + slot) * (D / 8);
        if constexpr (D == 128) *(uint32_t *)(p + 4 * g) = bits;
        else *(uint16_t *)(p + 2 * g) = (uint16_t)bits;
      }
    }
  };

  // A step: a tile of an item for each wave, number `tile` + wave (the item's keys',
  // then its values'; one past its last is the last again, without slots). All waves
  // make the same steps.
  struct Step {
    int item, tile, pairs, kind_tiles, buf;
  };
  auto shape = [&](Step &p) {
    p.tile = 0;
    if (p.item < k.items) p.pairs = min(k.item_segs, k.segs - p.item * k.item_segs) * a.Hkv;
    p.kind_tiles = (p.pairs + per - 1) / per;
  };
  auto after = [&](Step p) {
    p.tile += kAW;
    if (p.tile >= 2 * p.kind_tiles) {
      p.item += gridDim.x;
      p.buf ^= 1;
      shape(p);
    }
    return p;
  };
  Vec w, wn;
  Raw raw;
  half8_t hi[KS], lo[KS];
  float undo;
  auto tile_of = [&](const Step &p) { return min(p.tile + wave, 2 * p.kind_tiles - 1); };
  auto request = [&](const Step &p) {
    const int tile = tile_of(p);
    wn = locate(p.item, tile, tile < p.kind_tiles, p.kind_tiles, p.pairs);
    if constexpr (VEC) fetch(wn, raw);
  };
  auto is_key = [&](const Step &p) { return tile_of(p) < p.kind_tiles; };
  auto take = [&](const Step &p) {                // the requested inputs as operands
    w = wn;
    if constexpr (!RUNS) {
      w.slot = w.row >= 0 ? sm.slot[p.buf][w.row] : -1;
      w.row = max(w.row, 0);
    }
    if (p.tile + wave >= 2 * p.kind_tiles) w.slot = -1;
    parts(raw, is_key(p), w, p.buf, hi, lo, undo);
  };

  // The first step's loads go out before the operands are made.
  Step cur{(int)blockIdx.x, 0, 0, 0, 0};
  shape(cur);
  positions(cur.item);
  request(cur);

  // Operands: row r = n of tile o is coordinate NC (r / 4) + 4 o + r % 4, so that
  // lane group g's results are NC neighbouring ones; element j of step ks is side
  // ks & 1 of pair 8 (4 (ks / 2) + g) + j.
  auto put = [&](half8_t (&to)[OT][KS][2][64], int row, int ks, int gg, const float (&x)[8]) {
    const int o = (row % NC) >> 2, l = 16 * gg + 4 * (row / NC) + (row & 3);
    half8_t hi, lo;
    split8(x, kRScale, &hi, &lo);
    to[o][ks][0][l] = hi;
    to[o][ks][1][l] = lo;
  };
  if constexpr (VEC) {
    // 16 columns a thread: those of two steps
    for (int i = tid; i < D * (D / 16); i += kAW * 64) {
      const int row = i / (D / 16), c = 16 * (i % (D / 16));
      float4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = *(const float4 *)(a.R + row * D + c + 4 * j);
      const float *y = (const float *)x;
      float u[8], v[8];
      if (inter) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u[j] = y[2 * j];
          v[j] = y[2 * j + 1];
        }
        put(sm.r, row, 2 * (c >> 6), (c >> 4) & 3, u);
        put(sm.r, row, 2 * (c >> 6) + 1, (c >> 4) & 3, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u[j] = y[j];
          v[j] = y[8 + j];
        }
        // the pairs and the side of eight columns
        auto place = [&](int c, const float (&x)[8]) {
          const int t = c < a.rot_dim ? c : c - a.rot_dim, h = (c < a.rot_dim ? a.rot_dim : D - a.rot_dim) / 2;
          const int side = t >= h ? 1 : 0;
          const int oct = (t - side * h + (c < a.rot_dim ? 0 : a.rot_dim / 2)) >> 3;
          put(sm.r, row, 2 * (oct >> 2) + side, oct & 3, x);
        };
        place(c, u);
        place(c + 8, v);
      }
    }
  } else {
    for (int i = tid; i < D * KS * 4; i += kAW * 64) {
      const int row = i / (KS * 4), ks = (i >> 2) % KS, gg = i & 3;
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[j] = a.R[row * D + pair_coord(8 * (4 * (ks >> 1) + gg) + j, ks & 1, a.rot_dim, D, inter)];
      put(sm.r, row, ks, gg, x);
    }
  }
  if constexpr (QJL) {
    // residuals stand in a lane in coordinate order: element j of step ks is
    // coordinate NC g + 8 ks + j
    for (int i = tid; i < D * KS * 4; i += kAW * 64) {
      const int row = i / (KS * 4), c = 8 * (i % (KS * 4)), gg = c / NC, ks = (c % NC) >> 3;
      float x[8], top = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = a.p_rot[row * D + c + j];
        top = fmaxf(top, fabsf(x[j]));
      }
      // only the sign of a projection counts: a row (of KS * 4 neighbouring threads) whose
      // largest entry is not from 2^-5 to 2^7 (a sketch's are) is scaled to [2^4, 2^5)
#pragma unroll
      for (int n = 1; n < KS * 4; n *= 2) top = fmaxf(top, __shfl_xor(top, n));
      const int ex = (int)(__builtin_bit_cast(uint32_t, top) >> 23);
      if (ex != 0 && ex != 255 && (ex < 127 - 5 || ex >= 127 + 7)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __builtin_ldexpf(x[j], 131 - ex);
      }
      put(sm.p, row, ks, gg, x);
    }
  }
  if (tid < 32) sm.cb[tid >> 4][tid & 15] = (tid & 15) < nl ? (tid < 16 ? a.k_cb : a.v_cb)[tid & 15] : 0.0f;
  __syncthreads();
  build_cell_table<kAW * 64>(sm.cb[0], nl, tid, sm.cells[0], sm.thr, sm.ucell, &sm.table_ok[0]);
  if (SM::TABLES == 2 && !shared_cb)
    build_cell_table<kAW * 64>(sm.cb[1], nl, tid, sm.cells[SM::TABLES - 1], sm.thr, sm.ucell, &sm.table_ok[1]);
  ok_k = sm.table_ok[0] != 0;
  ok_v = shared_cb ? ok_k : SM::TABLES == 2 && sm.table_ok[1] != 0;

  // A step's inputs are on their way while the one before is worked on; the table of
  // the next item is made before the barrier after which this one's may be
  // overwritten.
  table(cur.item, 0);
  if (cur.item + (int)gridDim.x < k.items) positions(cur.item + gridDim.x);
  __syncthreads();
  for (;;) {
    take(cur);
    const Step nx = after(cur);
    if (nx.item < k.items) request(nx);
    float4_t acc[OT];
#pragma unroll
    for (int o = 0; o < OT; ++o) {
      acc[o] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const half8_t rh = sm.r[o][ks][0][lane], rl = sm.r[o][ks][1][lane];
        acc[o] = mfma16(rh, hi[ks], acc[o]);
        acc[o] = mfma16(rl, hi[ks], acc[o]);
        acc[o] = mfma16(rh, lo[ks], acc[o]);
      }
    }
    uint32_t word[NC / 8];
    uint16_t radius;
    float e[QJL ? NC : 1];
    const bool key = is_key(cur);
    quantise(acc, key, undo, word, radius, e);
    store(w, key, word, radius);
    if (QJL && key) sketch(w, e);
    if (nx.item >= k.items) return;
    if (nx.item != cur.item) {
      table(nx.item, nx.buf);
      if (nx.item + (int)gridDim.x < k.items) positions(nx.item + gridDim.x);
      lds_barrier();
    }
    cur = nx;
  }
}

template <typename T, int D, bool VEC, bool QJL>
hipError_t launch_as(const AppendArgs &a, hipStream_t s) {
  constexpr int AW = append_waves<T, D, VEC, QJL>(), ROWS = AppendSmem<D, QJL>::ROWS;
  // tokens of a segment: as many as a tile has vectors, or all of fewer
  int tt_shift = 0;
  while (tt_shift < 4 && (1 << tt_shift) < a.T) ++tt_shift;
  const int token_blocks = (a.T + (1 << tt_shift) - 1) >> tt_shift, segs = a.B * token_blocks;
  // segments of an item: as many as give each wave four tiles, fewer where that
  // leaves compute units idle (but whole tiles), within the table's rows
  const int cus = device_compute_units(), per = 16 >> tt_shift;
  int n = (2 * AW * per + a.Hkv - 1) / a.Hkv;
  const int spread = (segs + cus - 1) / cus, whole = (per + a.Hkv - 1) / a.Hkv;
  if (n > spread) n = spread > whole ? spread : whole;
  if (n > ROWS >> tt_shift) n = ROWS >> tt_shift;
  const int items = (segs + n - 1) / n, blocks = items < cus ? items : cus;
  const AppendKernelArgs k{a, tt_shift, token_blocks, segs, n, items, FastDiv(token_blocks), FastDiv(a.Hkv)};
  if (tt_shift == 4) append_kernel<T, D, VEC, QJL, true><<<blocks, AW * 64, 0, s>>>(k);
  else append_kernel<T, D, VEC, QJL, false><<<blocks, AW * 64, 0, s>>>(k);
  return hipGetLastError();
}

template <typename T, int D>
hipError_t launch_type(const AppendArgs &a, hipStream_t s) {
  // eight elements at a time where every run of eight starts on 16 bytes
  static_assert(sizeof(T) == 2 || sizeof(T) == 4, "eight elements are whole 16-byte pieces");
  const uintptr_t at = (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.R;
  int64_t el = a.interleaved ? 0 : a.rot_dim / 2;
  for (int i = 0; i < 3; ++i) el |= a.k_stride[i] | a.v_stride[i];
  if (at % 16 == 0 && el % 8 == 0) return a.p_rot ? launch_as<T, D, true, true>(a, s) : launch_as<T, D, true, false>(a, s);
  return a.p_rot ? launch_as<T, D, false, true>(a, s) : launch_as<T, D, false, false>(a, s);
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
