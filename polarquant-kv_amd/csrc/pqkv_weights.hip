// The attention weight that each cached position gets: after a decode call,
// from the logits it wrote (decode_merge_weights_kernel), and for a chunk of query
// tokens (attn_weights_kernel).
#include <type_traits>

#include "pqkv_decode_merge.h"
#include "pqkv_device.h"
#include "pqkv_launch.h"

namespace pqkv {

namespace {

// The same lane position of the four 16-lane groups, combined (gfx950 swaps).
__device__ __forceinline__ float rows4_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = fmaxf(__builtin_bit_cast(float, (uint32_t)p[0]), __builtin_bit_cast(float, (uint32_t)p[1]));
  const uint32_t v = __builtin_bit_cast(uint32_t, x);
  auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)q[0]), __builtin_bit_cast(float, (uint32_t)q[1]));
}
__device__ __forceinline__ float rows4_sum(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = __builtin_bit_cast(float, (uint32_t)p[0]) + __builtin_bit_cast(float, (uint32_t)p[1]);
  const uint32_t v = __builtin_bit_cast(uint32_t, x);
  auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_bit_cast(float, (uint32_t)q[0]) + __builtin_bit_cast(float, (uint32_t)q[1]);
}

// The sum over each 16-lane row, in all of its lanes (row rotations).
template <int N>
__device__ __forceinline__ float row_ror_add(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x120 + N, 0xF, 0xF, true));
}
__device__ __forceinline__ float row16_sum(float x) {
  return row_ror_add<1>(row_ror_add<2>(row_ror_add<4>(row_ror_add<8>(x))));
}

// ---- after a decode call ----
//
// weights[t] = in[t] + sum over the kv head's query heads of exp2(s_t - M) / L,
// with M and L merged from the splits' partials. A workgroup takes 1024
// tokens of one (batch, kv head): it merges the group's partials first (few,
// and in L2), then reads one row of logits per head, four tokens per thread.
// Bound by those rows: 4 (G + 2) bytes per token and kv head. The same launch
// joins the output's splits (decode_merge_body, the workgroups after them),
// which needs nothing of the weights: a launch less. 8 sequences of 32768 tokens,
// 32 query / 8 kv heads: 13 us for 50 MB.
constexpr int kDwTokens = 1024;

template <bool VEC>
__device__ __forceinline__ void decode_weights_body(float2 *ml, const DecodeArgs &a, const DecodeWeights &w,
                                                    uint32_t blk) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t tiles = (uint32_t)(a.S + kDwTokens - 1) / kDwTokens;
  const int64_t bh = blk / tiles;
  const int t0 = (int)(blk - (uint32_t)bh * tiles) * kDwTokens + 4 * tid;
  const int b = (int)(bh / a.Hkv), h = (int)(bh - (int64_t)b * a.Hkv);
  const int64_t row0 = (int64_t)b * a.Hq + (int64_t)h * a.gq;
  // the first heads' logits (and what there was) are on their way while the
  // partials are merged
  constexpr int AHEAD = 4;
  const bool there = t0 < a.S;
  const float *lrow = w.logits + row0 * w.logit_stride + (there ? t0 : 0);
  const float *in = w.in ? w.in + bh * w.in_stride + t0 : nullptr;
  const bool vec = VEC && t0 + 4 <= a.S;
  float4 s[AHEAD], o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int g = 0; g < AHEAD; ++g) s[g] = *(const float4 *)(lrow + (int64_t)min(g, a.gq - 1) * w.logit_stride);
  if (vec && in) o = *(const float4 *)in;
  for (int g = wave; g < a.gq; g += 4) {   // ml: per head of the group M, 1 / L
    const float *p = a.part + (row0 + g) * a.split_stride * (a.d + 2);
    float mx = -INFINITY, L = 0.0f;
    for (int sp = lane; sp < a.split_stride; sp += 64) mx = fmaxf(mx, p[(int64_t)sp * (a.d + 2)]);
    mx = wave_max(mx);
    for (int sp = lane; sp < a.split_stride; sp += 64) {
      // (a split without a number to its maximum has the sum NaN, which stays)
      const float m = p[(int64_t)sp * (a.d + 2)], e = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
      L = __builtin_fmaf(e, p[(int64_t)sp * (a.d + 2) + 1], L);
    }
    L = wave_sum(L);
    if (lane == 0) ml[g] = make_float2(mx, L == 0.0f ? 0.0f : 1.0f / L);
  }
  __syncthreads();
  if (!there) return;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](float4 v, float2 x) {
    sum[0] = __builtin_fmaf(__builtin_amdgcn_exp2f(v.x - x.x), x.y, sum[0]);
    sum[1] = __builtin_fmaf(__builtin_amdgcn_exp2f(v.y - x.x), x.y, sum[1]);
    sum[2] = __builtin_fmaf(__builtin_amdgcn_exp2f(v.z - x.x), x.y, sum[2]);
    sum[3] = __builtin_fmaf(__builtin_amdgcn_exp2f(v.w - x.x), x.y, sum[3]);
  };
#pragma unroll
  for (int g = 0; g < AHEAD; ++g)
    if (g < a.gq) add(s[g], ml[g]);
#pragma unroll 4
  for (int g = AHEAD; g < a.gq; ++g) add(*(const float4 *)(lrow + (int64_t)g * w.logit_stride), ml[g]);
  float *out = w.out + bh * w.out_stride + t0;
  if (vec) {
    *(float4 *)out = make_float4(o.x + sum[0], o.y + sum[1], o.z + sum[2], o.w + sum[3]);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (t0 + j < a.S) out[j] = (in ? in[j] : 0.0f) + sum[j];
}

// MS: the most splits the join's table of their weights holds (1024 of them
// leave room for half as many workgroups).
template <int D, typename TOUT, bool VEC, int MS>
__global__ void __launch_bounds__(256) decode_merge_weights_kernel(const DecodeArgs a, const DecodeWeights w,
                                                                  const float *__restrict__ R,
                                                                  TOUT *__restrict__ out, int weight_blocks) {
  __shared__ union {
    MergeSmem<D, MS> merge;
    float2 ml[kMaxGroupWeights];
  } sm;
  const int blk = blockIdx.x;
  if (blk < weight_blocks) {
    decode_weights_body<VEC>(sm.ml, a, w, (uint32_t)blk);
  } else {
    const int m = blk - weight_blocks;
    decode_merge_body<D, TOUT, true, MS>(sm.merge, a.part, R, out, a.B * a.Hq, a.split_stride, m / (D / 32), m % (D / 32));
  }
}

// ---- of a chunk of query tokens ----
//
// Row r = i G + g of a (batch, kv head) stream is query token i of the
// group's head g. The softmax needs each row's maximum and sum before any
// column can be summed, so the scores are computed twice, by a workgroup that
// decodes its tokens' keys once, keeps them as matrix operands in registers and
// lets the rows pass by:
//   STATS: per row, the maximum and the sum over the workgroup's tokens
//   (attn_stats_kernel joins the token blocks'),
//   sums:  per token, sum over the rows of exp2(s - M) / L
//   (weights_join_kernel joins the row chunks' in order, so nothing depends on
//   which workgroup ends first).
// A causal row at position p meets only the blocks that start at or before p.
//
// Products are v_mfma_f32_16x16x32_f16 on fp32 operands split hi / lo, three of
// them (hi hi + hi lo + lo hi) into one fp32 accumulator. A = 16 tokens' keys
// r c[code], B = 16 rows' queries, so accumulator i of lane (col, grp) is token
// 4 grp + i of row col: a row's statistics reduce over a lane's registers and
// the four lane groups, a column's sum stays in its register until the end.
// Powers of two keep the parts in fp16's range: a row's largest query value at
// 2^8 (queries per row, undone by a factor per lane), the block's largest key at
// 2^8 (per workgroup). With QJL the signs join the same accumulator as +- the
// keys' power of two against the projections (two more products; +-0 where the
// sketch is all ones, a zero residual).
//
// Bound by the products: 8191 tokens of 32 query / 8 kv heads (d = 128) on
// themselves take 700 and 680 us in the two passes, 825 GFLOP of products each, 1.2
// PFLOP/s (a library product of two 8192 x 8192 fp16 matrices reaches 1.13; the
// matrix cores are busy 55 % of the cycles, two other vector instructions stand
// beside each product). With few rows the decoding of the keys and the first loads of
// each workgroup weigh more: 32 rows x 4 heads on 131072 tokens 120 and 133 us (103
// GFLOP, 0.8 PFLOP/s, 30 to 36 %).
constexpr int kWW = 4;      // waves of a workgroup
constexpr int kStage = 32;  // rows of a stage

struct WeightsKernelArgs {
  AttnWeightsArgs a;
  FastDiv group;             // by G
  int xcd_groups;            // > 0: (stream, chunk) groups dealt to the XCDs
};

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) const half8_t lds_chalf8;

template <int D, bool QJL>
struct RowRec {                                    // 16 rows as B operands
  static constexpr int KS = D / 32;
  static constexpr int PARTS = QJL ? 4 : 2;        // q hi, q lo (, projections hi, lo)
  static constexpr int BYTES = KS * PARTS * 1024;  // segment (ks, part): 64 lanes x 16 bytes
};

// Eight values as high and low parts, two at a time (one conversion a pair).
// (x in registers of its own: where it is a product, the conversion may
// otherwise be fused with it and round the unrounded product, while the
// remainder is taken from the rounded one: a step of the high part lost on
// values next to a tie)
typedef float float2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void split_parts(const float (&x)[8], half8_t *hi, half8_t *lo) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float u = x[i], v = x[i + 1];
    asm("" : "+v"(u), "+v"(v));
    const half2_t h = __builtin_convertvector((float2_t){u, v}, half2_t);
    const half2_t l = __builtin_convertvector((float2_t){u - (float)h.x, v - (float)h.y}, half2_t);
    (*hi)[i] = h.x;
    (*hi)[i + 1] = h.y;
    (*lo)[i] = l.x;
    (*lo)[i + 1] = l.y;
  }
}

// The power of two that brings `most` to [2^8, 2^9); 0 if it is zero, subnormal or not finite.
__device__ __forceinline__ int scale_exponent(float most, int largest) {
  const int ex = (int)((__builtin_bit_cast(uint32_t, most) >> 23) & 0xFF);
  return ex == 0 || ex == 255 ? 0 : min(135 - ex, largest);
}

// The address of row r of a pass in a [B][Hq][Sq] arrangement of vectors.
__device__ __forceinline__ int64_t row_vector(const WeightsKernelArgs &k, int64_t stream, int r) {
  const AttnWeightsArgs &a = k.a;
  const int b = (int)(stream / a.Hkv), h = (int)(stream - (int64_t)b * a.Hkv);
  const uint32_t rr = (uint32_t)(min(r, a.rows - 1) + a.row0), tok = k.group.div(rr);
  return ((int64_t)b * a.Hq + h * a.G + (int)(rr - tok * a.G)) * a.Sq + tok;
}

// Eight values of each of a row's parts (queries, projections) -> its share of
// the record: hi and lo, times 2^sh.
template <int D, bool QJL>
__device__ __forceinline__ void put_row(uint8_t *rec, int j, int rl, const float (&x)[QJL ? 2 : 1][8], int sh) {
  using Rec = RowRec<D, QJL>;
  const float sc = __builtin_ldexpf(1.0f, sh);
#pragma unroll
  for (int p = 0; p < (QJL ? 2 : 1); ++p) {
    half8_t hi, lo;
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = x[p][i] * sc;
    split_parts(e, &hi, &lo);
    uint8_t *seg = rec + ((j >> 2) * Rec::PARTS + 2 * p) * 1024 + ((j & 3) * 16 + rl) * 16;
    *(half8_t *)seg = hi;
    *(half8_t *)(seg + 1024) = lo;
  }
}

// With QJL: rotated queries and projections -> records of 16 rows, and each
// row's factor. Rows past the pass's last one are zeros.
template <int D>
__global__ void __launch_bounds__(2 * D) weights_rows_kernel(const WeightsKernelArgs k) {
  constexpr bool QJL = true;
  using Rec = RowRec<D, QJL>;
  __shared__ float most[D / 8][16];
  const AttnWeightsArgs &a = k.a;
  const int tid = threadIdx.x, rl = tid & 15, j = tid >> 4;   // row of the tile; its eight coordinates
  const uint32_t tiles = (uint32_t)a.row_tiles;
  const int64_t stream = blockIdx.x / tiles;
  const int tile = (int)(blockIdx.x - (uint32_t)stream * tiles), r = tile * 16 + rl;
  float x[2][8];
  float mx = 0.0f;
  const int64_t row = row_vector(k, stream, r);
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const float *src = (p ? a.pq : a.q) + row * D + 8 * j;
    const float4 u = *(const float4 *)src, v = *(const float4 *)(src + 4);
    const float e[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[p][i] = r < a.rows ? e[i] : 0.0f;
      mx = fmaxf(mx, fabsf(x[p][i]));
    }
  }
  most[j][rl] = mx;
  __syncthreads();
  for (int i = 0; i < D / 8; ++i) mx = fmaxf(mx, most[i][rl]);
  const int sh = scale_exponent(mx, 100);
  if (j == 0) a.row_factor[stream * tiles * 16 + r] = __builtin_ldexpf(1.0f, -sh);
  put_row<D, QJL>(a.records + (stream * tiles + tile) * Rec::BYTES, j, rl, x, sh);
}

// Without QJL, from the queries themselves (a.x): y = R x on the matrix cores, so
// that the rotated queries are never written. A = R, split hi / lo once per
// workgroup into registers (a wave's D / 4 outputs), B = 16 queries as they lie in
// memory: fp16 queries are their own high part (two products), fp32 ones are scaled
// and split (three). Queries off a 16-byte boundary (ALIGNED false) are read in the
// pieces that their type's alignment allows.
// 32764 x 8 rows (d = 128): 58 us (200 MB, 3.5 TB/s) where rotating first (75)
// and making records of the result (48) took 123.
template <int D, typename T, bool ALIGNED>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : 4) weights_rotate_rows_kernel(const WeightsKernelArgs k, uint32_t n_tiles) {
  using Rec = RowRec<D, false>;
  constexpr int KS = D / 32, OT = D / 64;          // outputs of a wave: OT tiles of 16
  constexpr bool F32 = sizeof(T) == 4;
  __shared__ __align__(16) float ys[2][16][D + 4];
  __shared__ float most[2][4][16];
  const AttnWeightsArgs &a = k.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, grp = lane >> 4;

  // the wave's rows of R, scaled by a power of two of its own
  float4 rv[OT][KS][2];
  float rm = 0.0f;
#pragma unroll
  for (int o = 0; o < OT; ++o)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        rv[o][ks][p] = *(const float4 *)(a.R + (16 * (OT * wave + o) + col) * D + 32 * ks + 8 * grp + 4 * p);
        const float4 u = rv[o][ks][p];
        rm = fmaxf(fmaxf(fmaxf(rm, fabsf(u.x)), fmaxf(fabsf(u.y), fabsf(u.z))), fabsf(u.w));
      }
  const int rsh = scale_exponent(wave_max(rm), 100);
  const float rscale = __builtin_ldexpf(1.0f, rsh), undo = a.q_scale * __builtin_ldexpf(1.0f, -rsh);
  half8_t rh[OT][KS], rl[OT][KS];
#pragma unroll
  for (int o = 0; o < OT; ++o)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const float4 u = rv[o][ks][0], v = rv[o][ks][1];
      const float e[8] = {u.x * rscale, u.y * rscale, u.z * rscale, u.w * rscale,
                          v.x * rscale, v.y * rscale, v.z * rscale, v.w * rscale};
      split_parts(e, &rh[o][ks], &rl[o][ks]);
    }

  struct Operand {
    half8_t h[KS], l[F32 ? KS : 1];
    float undo;
  };
  const uint32_t tiles = (uint32_t)a.row_tiles;
  auto read = [&](const T *src, auto &to) {   // 16 bytes
    if constexpr (ALIGNED) to = *(const std::remove_reference_t<decltype(to)> *)src;
    else __builtin_memcpy(&to, src, 16);
  };
  auto load = [&](uint32_t n) {
    Operand o;
    const int64_t stream = n / tiles;
    const int r = (int)(n - (uint32_t)stream * tiles) * 16 + col;
    const T *src = (const T *)a.x + row_vector(k, stream, r) * D + 8 * grp;
    o.undo = r < a.rows ? undo : 0.0f;             // rows past the last one: zeros
    if constexpr (F32) {
      float4 u[KS][2];
      float mx = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          read(src + 32 * ks + 4 * p, u[ks][p]);
          mx = fmaxf(fmaxf(fmaxf(mx, fabsf(u[ks][p].x)), fmaxf(fabsf(u[ks][p].y), fabsf(u[ks][p].z))), fabsf(u[ks][p].w));
        }
      const int sh = scale_exponent(rows4_max(mx), 100);
      const float sc = __builtin_ldexpf(1.0f, sh);
      o.undo *= __builtin_ldexpf(1.0f, -sh);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const float e[8] = {u[ks][0].x * sc, u[ks][0].y * sc, u[ks][0].z * sc, u[ks][0].w * sc,
                            u[ks][1].x * sc, u[ks][1].y * sc, u[ks][1].z * sc, u[ks][1].w * sc};
        split_parts(e, &o.h[ks], &o.l[ks]);
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) read(src + 32 * ks, o.h[ks]);
    }
    return o;
  };
  uint32_t n = blockIdx.x;
  int buf = 0;
  Operand x = load(n);
  for (; n < n_tiles; n += gridDim.x, buf ^= 1) {
    const Operand now = x;
    if (n + gridDim.x < n_tiles) x = load(n + gridDim.x);
    float4_t acc[OT];
#pragma unroll
    for (int o = 0; o < OT; ++o) acc[o] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int o = 0; o < OT; ++o) {
        acc[o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rl[o][ks], now.h[ks], acc[o], 0, 0, 0);
        if constexpr (F32) acc[o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rh[o][ks], now.l[ks], acc[o], 0, 0, 0);
        acc[o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rh[o][ks], now.h[ks], acc[o], 0, 0, 0);
      }
    // through LDS into the record's order (two buffers: one barrier a tile),
    // the row's largest value beside it
    float mx = 0.0f;
#pragma unroll
    for (int o = 0; o < OT; ++o) {
      const float4_t y = now.undo == 0.0f ? (float4_t){0.f, 0.f, 0.f, 0.f} : acc[o] * now.undo;
      *(float4_t *)&ys[buf][col][16 * (OT * wave + o) + 4 * grp] = y;
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fabsf(y[i]));
    }
    mx = rows4_max(mx);
    if (grp == 0) most[buf][wave][col] = mx;
    __syncthreads();
    const int rr = tid & 15, j = tid >> 4;
    if (j < D / 8) {
      float y[1][8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[0][i] = ys[buf][rr][8 * j + i];
      mx = fmaxf(fmaxf(most[buf][0][rr], most[buf][1][rr]), fmaxf(most[buf][2][rr], most[buf][3][rr]));
      const int sh = scale_exponent(mx, 100);
      if (j == 0) a.row_factor[(int64_t)n * 16 + rr] = __builtin_ldexpf(1.0f, -sh);
      put_row<D, false>(a.records + (int64_t)n * Rec::BYTES, j, rr, y, sh);
    }
  }
}

// TT: 16-token tiles per wave.
template <int D, bool QJL, int TT, bool STATS>
__global__ void __launch_bounds__(64 * kWW, QJL || TT == 4 ? 2 : 3) attn_weights_kernel(const WeightsKernelArgs k) {
  using Rec = RowRec<D, QJL>;
  constexpr int KS = Rec::KS, TOK = 16 * TT * kWW, RT = kStage / 16;
  constexpr int SEGS = RT * Rec::BYTES / 1024;
  __shared__ __attribute__((aligned(16))) uint8_t qb[2][RT * Rec::BYTES];
  __shared__ float2 pair_tab[256];                 // 4-bit: byte -> two centroids; 2-bit: nibble
  __shared__ float red[kWW];
  __shared__ float2 st[STATS ? 2 : 1][kWW][kStage];
  const AttnWeightsArgs &a = k.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;

  // Workgroup -> (stream, chunk, token block), the blocks of one (stream,
  // chunk) group side by side: they read the same rows. With groups enough for
  // every XCD (workgroup n runs on XCD n % 8) a group stays on one, whose L2
  // then holds its rows. Later chunks first: a causal chunk meets more blocks.
  uint32_t blk = blockIdx.x;
  uint32_t gi, tbu;
  if (k.xcd_groups) {
    const uint32_t j = blk >> 3;
    tbu = j % (uint32_t)a.tblocks;
    gi = (j / (uint32_t)a.tblocks) * 8 + (blk & 7);
    if (gi >= (uint32_t)k.xcd_groups) return;
  } else {
    tbu = blk % (uint32_t)a.tblocks;
    gi = blk / (uint32_t)a.tblocks;
  }
  const uint32_t n_streams = (uint32_t)(a.B * a.Hkv);
  const int chunk = a.chunks - 1 - (int)(gi / n_streams), tb = (int)tbu;
  const int64_t stream = gi % n_streams;
  const int t0 = tb * TOK, tw0 = t0 + 16 * TT * wave, tw1 = tw0 + 16 * TT - 1;
  int r_begin = chunk * a.chunk_rows;
  const int r_end = min(r_begin + a.chunk_rows, a.rows);
  if (a.causal) {   // the first row that sees token t0
    const int64_t first = (int64_t)(t0 - a.q_start) * a.G - a.row0;
    if (first >= r_end) {
      if (!STATS && a.chunks == 1)   // no row sees the block: what there was stays
        for (int t = t0 + tid; t < min(t0 + TOK, a.S); t += 64 * kWW)
          a.out[stream * a.out_stride + t] = a.in ? a.in[stream * a.in_stride + t] : 0.0f;
      return;
    }
    if (first > r_begin) r_begin = (int)first;
  }

  const uint8_t *records = a.records + stream * a.row_tiles * (int64_t)Rec::BYTES;
  const __amdgpu_buffer_rsrc_t res = __builtin_amdgcn_make_buffer_rsrc(
      (void *)records, (short)0, (int)((int64_t)a.row_tiles * Rec::BYTES), 0x00020000);
  const float *factor = a.row_factor + stream * a.row_tiles * 16;
  const float2 *stat = a.stat + stream * a.row_tiles * 16;
  auto copy_stage = [&](int s, lds_u8 *__restrict dst) {
    const int at = __builtin_amdgcn_readfirstlane(s * RT * Rec::BYTES);
#pragma unroll
    for (int j = 0; j < SEGS / kWW; ++j) {
      const int sg = wave + kWW * j;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(res, (lds_void *)(dst + 1024 * sg), 16, 16 * lane, at + 1024 * sg, 0, 0);
    }
  };
  const int s0 = r_begin / kStage, s1 = (r_end + kStage - 1) / kStage;
  copy_stage(s0, (lds_u8 *)qb[s0 & 1]);

  // ---- this wave's keys, 16 TT tokens: lane (col, grp) holds coordinates
  // 32 ks + 8 grp .. + 7 of token 16 tt + col; those that no row of the pass sees
  // are zeros, so that they neither set the block's scale nor meet padding rows ----
  const int seen = a.causal ? min(a.S, a.q_start + (int)k.group.div((uint32_t)(a.rows - 1 + a.row0)) + 1) : a.S;
  const int vb = vector_bytes(D, a.bits);
  const uint8_t *kv[TT], *sv[TT];
  float radius[TT], rmax = 0.0f;
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
    const int t = min(tw0 + 16 * tt + col, a.S - 1);
    if (a.k_pages) {
      const int64_t pg = stream * a.max_pages + (t >> a.page_shift);
      const int64_t at = t & ((1 << a.page_shift) - 1);
      kv[tt] = a.k_pages[pg] + at * vb;
      sv[tt] = QJL ? a.s_pages[pg] + at * (D / 8) : nullptr;
    } else {
      kv[tt] = a.k_cache + (stream * a.S_max + t) * vb;
      sv[tt] = QJL ? a.qjl + (stream * a.S_max + t) * (D / 8) : nullptr;
    }
    const float r = half_bits_to_float(*(const uint16_t *)kv[tt]);
    radius[tt] = tw0 + 16 * tt + col < seen ? r : 0.0f;
    rmax = fmaxf(rmax, fabsf(radius[tt]));
  }
  uint32_t code[TT][KS];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint8_t *p = kv[tt] + qs_offset((32 * ks + 8 * grp) * a.bits / 8, a.bits);
      code[tt][ks] = *(const uint16_t *)p;
      if (a.bits == 4) code[tt][ks] |= (uint32_t)((const uint16_t *)p)[1] << 16;
    }
  float cmax = 0.0f;
  for (int i = 0; i < (1 << a.bits); ++i) cmax = fmaxf(cmax, fabsf(a.codebook[i]));
  {
    const int sh = a.bits == 4 ? 4 : 2, m = (1 << a.bits) - 1;
    pair_tab[tid] = make_float2(a.codebook[tid & m], a.codebook[(tid >> sh) & m]);
  }
  rmax = wave_max(rmax);
  if (lane == 0) red[wave] = rmax;
  __syncthreads();
  rmax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const int ksh = max(scale_exponent(rmax * cmax, 14), -24);
  const float kscale = __builtin_ldexpf(1.0f, ksh), kundo = __builtin_ldexpf(1.0f, -ksh);
  half8_t kh[TT][KS], kl[TT][KS], sg[QJL ? TT : 1][KS];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
    const float rs = radius[tt] * kscale;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 c = pair_tab[a.bits == 4 ? (code[tt][ks] >> (8 * i)) & 255 : (code[tt][ks] >> (4 * i)) & 15];
        e[2 * i] = c.x * rs;
        e[2 * i + 1] = c.y * rs;
      }
      split_parts(e, &kh[tt][ks], &kl[tt][ks]);
    }
    if constexpr (QJL) {
      uint32_t w[D / 32];
      bool ones = true;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        __builtin_memcpy(&w[i], sv[tt] + 4 * i, 4);
        ones = ones && w[i] == 0xFFFFFFFFu;
      }
      const half_t one = (half_t)(ones || tw0 + 16 * tt + col >= seen ? 0.0f : kscale);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 8; ++i) sg[tt][ks][i] = (w[ks] >> (8 * grp + i)) & 1u ? one : -one;
    }
  }

  // ---- the rows, a stage at a time ----
  struct RowInfo {
    float f[RT];
    float2 x[RT];
  };
  auto row_info = [&](int s) {
    RowInfo o;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = kStage * s + 16 * rt + col;
      o.f[rt] = factor[r];
      if constexpr (!STATS) o.x[rt] = stat[r];
    }
    return o;
  };
  float csum[TT][4];
#pragma unroll
  for (int tt = 0; tt < TT; ++tt)
#pragma unroll
    for (int i = 0; i < 4; ++i) csum[tt][i] = 0.0f;

  // Stage s out of buf; stage s + 1 (if `more`) is copied into the other buffer
  // meanwhile. (The two are restricted pointers so that the compiler knows the
  // copy apart from the reads: it would wait for it before the first of them.)
  auto compute = [&](int s, const RowInfo &info, const lds_u8 *__restrict buf, lds_u8 *__restrict other, bool more,
                     auto masked) {
    constexpr bool kMasked = decltype(masked)::value;
    if (more) copy_stage(s + 1, other);
    const lds_chalf8 *q = (const lds_chalf8 *)(buf + 16 * lane);
    float4_t acc[RT][TT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) acc[rt][tt] = (float4_t){0.f, 0.f, 0.f, 0.f};
    // step n = (row tile, k-step); its operands are read one step ahead (the
    // fence holds products and reads in place, other work may move)
    half8_t rows[2][Rec::PARTS];
    auto read = [&](int n) {
#pragma unroll
      for (int p = 0; p < Rec::PARTS; ++p) rows[n & 1][p] = q[(n * Rec::PARTS + p) * 64];
    };
    read(0);
#pragma unroll
    for (int n = 0; n < RT * KS; ++n) {
      const int rt = n / KS, ks = n % KS;
      if (n + 1 < RT * KS) read(n + 1);
      __builtin_amdgcn_sched_barrier(0x0676);
      const half8_t bh = rows[n & 1][0], bl = rows[n & 1][1];
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
        acc[rt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl[tt][ks], bh, acc[rt][tt], 0, 0, 0);
        acc[rt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[tt][ks], bl, acc[rt][tt], 0, 0, 0);
        acc[rt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[tt][ks], bh, acc[rt][tt], 0, 0, 0);
      }
      if constexpr (QJL) {
        const half8_t ph = rows[n & 1][2], pl = rows[n & 1][3];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
          acc[rt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(sg[tt][ks], pl, acc[rt][tt], 0, 0, 0);
          acc[rt][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(sg[tt][ks], ph, acc[rt][tt], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float f = info.f[rt] * kundo;
      int last = a.S - 1;   // the last token the lane's row sees
      if (kMasked && a.causal)
        last = min(last, a.q_start + (int)k.group.div((uint32_t)(kStage * s + 16 * rt + col + a.row0)));
      const int rel = last - tw0 - 4 * grp;
      if constexpr (STATS) {
        float m = -INFINITY;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (kMasked && 16 * tt + i > rel) acc[rt][tt][i] = -INFINITY;
            m = fmaxf(m, acc[rt][tt][i]);
          }
        m = rows4_max(m) * f;      // the factor is positive: the maximum stays where it is
        const float ref = kMasked && m == -INFINITY ? 0.0f : m;
        float l = 0.0f;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[rt][tt][i], f, -ref));
        l = rows4_sum(l);
        if (grp == 0) st[s & 1][wave][16 * rt + col] = make_float2(m, l);
      } else {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // (the whole term is dropped: a row that is not a number has 1 / L = NaN)
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[rt][tt][i], f, -info.x[rt].x));
            const float with = __builtin_fmaf(e, info.x[rt].y, csum[tt][i]);
            csum[tt][i] = kMasked && 16 * tt + i > rel ? csum[tt][i] : with;
          }
      }
    }
  };
  // STATS: the four waves' statistics of stage s, joined and written (a maximum
  // of -inf has the sum 0, or NaN where all its logits are that, which stays)
  auto write_stats = [&](int s) {
    const int r = kStage * s + lane;
    if (wave != (s & (kWW - 1)) || lane >= kStage || r < r_begin || r >= r_end) return;
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kWW; ++w) m = fmaxf(m, st[s & 1][w][lane].x);
#pragma unroll
    for (int w = 0; w < kWW; ++w) {
      const float2 x = st[s & 1][w][lane];
      l = __builtin_fmaf(x.y, x.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x.x - m), l);
    }
    a.part[(stream * a.tblocks + tb) * a.rows + r] = make_float2(m, l);
  };
  RowInfo info = row_info(s0);
  for (int s = s0; s < s1; ++s) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");             // stage s has arrived (this wave's part)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // everyone's; stage s - 1 has been read
    const bool more = s + 1 < s1;
    const RowInfo next = row_info(more ? s + 1 : s);
    if (STATS && s > s0) write_stats(s - 1);
    lds_u8 *buf = (lds_u8 *)qb[s & 1], *other = (lds_u8 *)qb[(s + 1) & 1];
    const int p_first = a.q_start + (int)k.group.div((uint32_t)(kStage * s + a.row0));
    const int p_last = a.q_start + (int)k.group.div((uint32_t)(kStage * s + kStage - 1 + a.row0));
    if (tw0 >= a.S || (a.causal && p_last < tw0)) {   // none of the wave's tokens
      if (more) copy_stage(s + 1, other);
      if (STATS && lane < kStage) st[s & 1][wave][lane] = make_float2(-INFINITY, 0.0f);
    } else if (tw1 >= a.S || (a.causal && p_first < tw1)) {
      compute(s, info, buf, other, more, std::true_type{});
    } else {
      compute(s, info, buf, other, more, std::false_type{});
    }
    info = next;
  }
  if constexpr (STATS) {
    __syncthreads();
    write_stats(s1 - 1);
    return;
  }
  // each token's sum over the 16 row columns
#pragma unroll
  for (int tt = 0; tt < TT; ++tt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = row16_sum(csum[tt][i]);
      const int t = tw0 + 16 * tt + 4 * grp + i;
      if (col == 0) {
        if (a.chunks > 1) a.col[((stream * a.chunks + chunk) * a.tblocks + tb) * TOK + t - t0] = v;
        else if (t < a.S)
          a.out[stream * a.out_stride + t] = (a.in ? a.in[stream * a.in_stride + t] : 0.0f) + v;
      }
    }
}

// Joins the token blocks' maxima and sums of RW rows, 256 / RW threads per row;
// rows past the last one get (inf, 0), whose weights are 0.
template <int RW>
__global__ void __launch_bounds__(256) attn_stats_kernel(const WeightsKernelArgs k) {
  constexpr int SUB = 256 / RW;
  __shared__ float2 sub[SUB][RW];
  const AttnWeightsArgs &a = k.a;
  const uint32_t tiles = (uint32_t)a.row_tiles * 16 / RW;
  const int64_t stream = blockIdx.x / tiles;
  const int rl = threadIdx.x % RW, q = threadIdx.x / RW;
  const int r = (int)(blockIdx.x - (uint32_t)stream * tiles) * RW + rl;
  const int rr = min(r, a.rows - 1);
  const int last = a.causal ? min(a.q_start + (int)k.group.div((uint32_t)(rr + a.row0)), a.S - 1) : a.S - 1;
  const int n = last / a.tokens + 1;
  const float2 *p = a.part + stream * a.tblocks * a.rows + rr;
  float m = -INFINITY, l = 0.0f;
  auto join = [&](float2 x) {
    const float mn = fmaxf(m, x.x), ref = mn == -INFINITY ? 0.0f : mn;   // (no maximum: sums of 0, or NaN)
    l = l * __builtin_amdgcn_exp2f(m - ref) + x.y * __builtin_amdgcn_exp2f(x.x - ref);
    m = mn;
  };
#pragma unroll 8
  for (int i = q; i < n; i += SUB) join(p[(int64_t)i * a.rows]);
  sub[q][rl] = make_float2(m, l);
  __syncthreads();
  if (q != 0) return;
#pragma unroll
  for (int i = 1; i < SUB; ++i) join(sub[i][rl]);
  a.stat[stream * a.row_tiles * 16 + r] = r < a.rows ? make_float2(m, 1.0f / l) : make_float2(INFINITY, 0.0f);
}

// out = in + the row chunks' sums of one token, in the chunks' order.
__global__ void __launch_bounds__(256) weights_join_kernel(const AttnWeightsArgs a) {
  const uint32_t tiles = (uint32_t)(a.S + 255) / 256;
  const int64_t stream = blockIdx.x / tiles;
  const int t = (int)(blockIdx.x - (uint32_t)stream * tiles) * 256 + threadIdx.x;
  if (t >= a.S) return;
  const int tb = t / a.tokens;
  int c0 = 0;
  if (a.causal) {   // chunks that end before the first row that sees the block were not computed
    const int64_t first = (int64_t)(tb * a.tokens - a.q_start) * a.G - a.row0;
    if (first >= a.rows) c0 = a.chunks;
    else if (first > 0) c0 = (int)(first / a.chunk_rows);
  }
  float sum = 0.0f;
#pragma unroll 4
  for (int c = c0; c < a.chunks; ++c) sum += a.col[((stream * a.chunks + c) * a.tblocks) * (int64_t)a.tokens + t];
  a.out[stream * a.out_stride + t] = (a.in ? a.in[stream * a.in_stride + t] : 0.0f) + sum;
}

__global__ void __launch_bounds__(256) weights_copy_kernel(const float *in, int64_t in_stride, float *out,
                                                           int64_t out_stride, int S) {
  const uint32_t tiles = (uint32_t)(S + 255) / 256;
  const int64_t stream = blockIdx.x / tiles;
  const int t = (int)(blockIdx.x - (uint32_t)stream * tiles) * 256 + threadIdx.x;
  if (t < S) out[stream * out_stride + t] = in ? in[stream * in_stride + t] : 0.0f;
}

template <int D, bool QJL, int TT>
void launch_passes(const AttnWeightsArgs &a, int64_t streams, hipStream_t s) {
  WeightsKernelArgs k{a, FastDiv((uint32_t)a.G), 0};
  const int64_t groups = streams * a.chunks;
  if (groups % 8 == 0 || groups >= 64) k.xcd_groups = (int)groups;
  const unsigned grid = (unsigned)((k.xcd_groups ? (groups + 7) / 8 * 8 : groups) * a.tblocks);
  const uint32_t tiles = (uint32_t)(streams * a.row_tiles);
  if constexpr (QJL) {
    weights_rows_kernel<D><<<tiles, 2 * D, 0, s>>>(k);
  } else {
    const unsigned blocks = tiles < 1024 ? tiles : 1024;   // (each reads R once)
    auto rotate = [&](auto t, auto aligned) {
      weights_rotate_rows_kernel<D, decltype(t), decltype(aligned)::value><<<blocks, 256, 0, s>>>(k, tiles);
    };
    auto typed = [&](auto t) {
      if ((uintptr_t)a.x % 16 == 0) rotate(t, std::true_type{});
      else rotate(t, std::false_type{});
    };
    if (a.x_dtype == PQKV_F16) typed(half_t{});
    else typed(float{});
  }
  attn_weights_kernel<D, QJL, TT, true><<<grid, 64 * kWW, 0, s>>>(k);
  // few rows of many blocks: more threads per row (128 rows x 8 streams of 1024 blocks 11 us -> 6)
  if (tiles <= 1024 && a.tblocks > 64) attn_stats_kernel<8><<<2 * tiles, 256, 0, s>>>(k);
  else attn_stats_kernel<32><<<tiles / 2, 256, 0, s>>>(k);
  attn_weights_kernel<D, QJL, TT, false><<<grid, 64 * kWW, 0, s>>>(k);
  if (a.chunks > 1)   // (one chunk: the sums are the result)
    weights_join_kernel<<<(unsigned)(streams * ((a.S + 255) / 256)), 256, 0, s>>>(a);
}

template <int D>
void launch_head(const AttnWeightsArgs &a, int64_t streams, hipStream_t s) {
  if (a.pq != nullptr) launch_passes<D, true, 2>(a, streams, s);
  else if (a.tokens == 128) launch_passes<D, false, 2>(a, streams, s);
  else launch_passes<D, false, 4>(a, streams, s);
}

}  // namespace

hipError_t launch_decode_merge_weights(const DecodeArgs &a, const DecodeWeights &w, const float *R, void *out,
                                       int out_dtype, hipStream_t s) {
  if (a.split_stride > kMaxSplits || a.gq > kMaxGroupWeights) return hipErrorInvalidValue;
  const int wb = (int)((int64_t)((a.S + kDwTokens - 1) / kDwTokens) * a.B * a.Hkv);
  const int mb = (a.B * a.Hq + kMergeHeads - 1) / kMergeHeads * (a.d / 32);
  const bool vec = ((uintptr_t)w.out | (uintptr_t)w.in) % 16 == 0 && (w.out_stride | (w.in ? w.in_stride : 0)) % 4 == 0;
#define PQKV_DMW(DD, T, V, M) \
  decode_merge_weights_kernel<DD, T, V, M><<<(unsigned)(wb + mb), 256, 0, s>>>(a, w, R, (T *)out, wb)
#define PQKV_DMW_V(DD, T) \
  if (a.split_stride > 64) { \
    if (vec) PQKV_DMW(DD, T, true, kMaxSplits); \
    else PQKV_DMW(DD, T, false, kMaxSplits); \
  } else if (vec) PQKV_DMW(DD, T, true, 64); \
  else PQKV_DMW(DD, T, false, 64)
  if (a.d == 128 && out_dtype == PQKV_F32) { PQKV_DMW_V(128, float); }
  else if (a.d == 128) { PQKV_DMW_V(128, half_t); }
  else if (out_dtype == PQKV_F32) { PQKV_DMW_V(64, float); }
  else { PQKV_DMW_V(64, half_t); }
#undef PQKV_DMW_V
#undef PQKV_DMW
  return hipGetLastError();
}

hipError_t launch_attn_weights(const AttnWeightsArgs &a, hipStream_t s) {
  const int64_t streams = (int64_t)a.B * a.Hkv;
  if (a.d == 128) launch_head<128>(a, streams, s);
  else launch_head<64>(a, streams, s);
  return hipGetLastError();
}

hipError_t launch_weights_copy(const float *in, int64_t in_stride, float *out, int64_t out_stride, int64_t streams,
                               int S, hipStream_t s) {
  weights_copy_kernel<<<(unsigned)(streams * ((S + 255) / 256)), 256, 0, s>>>(in, in_stride, out, out_stride, S);
  return hipGetLastError();
}

}  // namespace pqkv
