// The attention weight that each cached position gets: after a decode call,
// from the logits it wrote (decode_weights_kernel), and for a chunk of query
// tokens (attn_weights_kernel).
#include "pqkv_device.h"
#include "pqkv_launch.h"

namespace pqkv {

namespace {

// ---- after a decode call ----
//
// weights[t] = in[t] + sum over the kv head's query heads of exp2(s_t - M) / L,
// with M and L merged from the splits' partials. A workgroup takes 1024
// tokens of one (batch, kv head): it merges the group's partials first (few,
// and in L2), then reads one row of logits per head, four tokens per thread.
// Bound by those rows: 4 (G + 2) bytes per token and kv head.
constexpr int kDwTokens = 1024;

template <bool VEC>
__global__ void __launch_bounds__(256) decode_weights_kernel(const DecodeArgs a, const DecodeWeights w) {
  extern __shared__ float2 ml[];   // per head of the group: M, 1 / L
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t tiles = (uint32_t)(a.S + kDwTokens - 1) / kDwTokens;
  const int64_t bh = blockIdx.x / tiles;
  const int t0 = (int)(blockIdx.x - (uint32_t)bh * tiles) * kDwTokens + 4 * tid;
  const int b = (int)(bh / a.Hkv), h = (int)(bh - (int64_t)b * a.Hkv);
  const int64_t row0 = (int64_t)b * a.Hq + (int64_t)h * a.gq;
  for (int g = wave; g < a.gq; g += 4) {
    const float *p = a.part + (row0 + g) * a.split_stride * (a.d + 2);
    float mx = -INFINITY, L = 0.0f;
    for (int sp = lane; sp < a.split_stride; sp += 64) mx = fmaxf(mx, p[(int64_t)sp * (a.d + 2)]);
    mx = wave_max(mx);
    for (int sp = lane; sp < a.split_stride; sp += 64) {
      const float m = p[(int64_t)sp * (a.d + 2)];
      if (m != -INFINITY) L = __builtin_fmaf(__builtin_amdgcn_exp2f(m - mx), p[(int64_t)sp * (a.d + 2) + 1], L);
    }
    L = wave_sum(L);
    if (lane == 0) ml[g] = make_float2(mx, L > 0.0f ? 1.0f / L : 0.0f);
  }
  __syncthreads();
  if (t0 >= a.S) return;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const float *lrow = w.logits + row0 * w.logit_stride + t0;
#pragma unroll 4
  for (int g = 0; g < a.gq; ++g) {
    const float4 s = *(const float4 *)(lrow + (int64_t)g * w.logit_stride);
    const float2 x = ml[g];
    sum[0] = __builtin_fmaf(__builtin_amdgcn_exp2f(s.x - x.x), x.y, sum[0]);
    sum[1] = __builtin_fmaf(__builtin_amdgcn_exp2f(s.y - x.x), x.y, sum[1]);
    sum[2] = __builtin_fmaf(__builtin_amdgcn_exp2f(s.z - x.x), x.y, sum[2]);
    sum[3] = __builtin_fmaf(__builtin_amdgcn_exp2f(s.w - x.x), x.y, sum[3]);
  }
  const float *in = w.in ? w.in + bh * w.in_stride + t0 : nullptr;
  float *out = w.out + bh * w.out_stride + t0;
  if (VEC && t0 + 4 <= a.S) {
    float4 o = in ? *(const float4 *)in : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    o.x += sum[0];
    o.y += sum[1];
    o.z += sum[2];
    o.w += sum[3];
    *(float4 *)out = o;
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (t0 + j < a.S) out[j] = (in ? in[j] : 0.0f) + sum[j];
}

// ---- of a chunk of query tokens ----
//
// Row r = i G + g of a (batch, kv head) stream is query token i of the
// group's head g. The softmax needs each row's maximum and sum before any
// column can be summed, so the scores are computed twice, from keys that a
// workgroup decodes once and keeps: kWeightTokens tokens, against kWeightRows
// rows that pass by.
//   STATS: per row, the maximum and the sum over the workgroup's tokens
//   (attn_stats_kernel joins the token blocks'),
//   sums:  per token, sum over the rows of exp2(s - M) / L
//   (weights_join_kernel joins the row chunks' in order, so nothing depends on
//   which workgroup ends first).
// A causal row at position p meets only the blocks that start at or before p.
template <int D, bool QJL, bool STATS>
__global__ void __launch_bounds__(256) attn_weights_kernel(const AttnWeightsArgs a) {
  constexpr int NR = 8;
  __shared__ __align__(16) float qs[NR][D], ps[QJL ? NR : 1][D];
  __shared__ float red[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t blk = blockIdx.x;
  const int chunk = blk % (uint32_t)a.chunks;
  blk /= (uint32_t)a.chunks;
  const int tb = blk % (uint32_t)a.tblocks;
  const int64_t stream = blk / (uint32_t)a.tblocks;
  const int b = (int)(stream / a.Hkv), h = (int)(stream - (int64_t)b * a.Hkv);
  const int t0 = tb * kWeightTokens, t = t0 + tid;
  int r_begin = chunk * kWeightRows;
  const int r_end = min(r_begin + kWeightRows, a.rows);
  if (a.causal) {   // the first row that sees token t0
    const int64_t first = (int64_t)(t0 - a.q_start) * a.G - a.row0;
    if (first >= r_end) return;
    if (first > r_begin) r_begin = (int)first;
  }
  float c[D], radius = 0.0f;
  uint32_t sg[QJL ? D / 32 : 1];
  bool zero_res = true;
  const int vb = vector_bytes(D, a.bits);
  if (t < a.S) {
    const uint8_t *kv, *sv;
    if (a.k_pages) {
      const int64_t pg = stream * a.max_pages + (t >> a.page_shift);
      const int64_t at = t & ((1 << a.page_shift) - 1);
      kv = a.k_pages[pg] + at * vb;
      sv = QJL ? a.s_pages[pg] + at * (D / 8) : nullptr;
    } else {
      kv = a.k_cache + (stream * a.S_max + t) * vb;
      sv = QJL ? a.qjl + (stream * a.S_max + t) * (D / 8) : nullptr;
    }
    radius = half_bits_to_float(*(const uint16_t *)kv);
    for (int k = 0; k < D; ++k) {
      const int byte = kv[qs_offset(k * a.bits / 8, a.bits)];
      c[k] = a.codebook[(byte >> (k * a.bits % 8)) & ((1 << a.bits) - 1)];
    }
    if constexpr (QJL)
      for (int k = 0; k < D / 32; ++k) {
        uint32_t w = 0;
        for (int j = 0; j < 4; ++j) w |= (uint32_t)sv[4 * k + j] << (8 * j);
        sg[k] = w;
        zero_res = zero_res && w == 0xFFFFFFFFu;
      }
  } else {
    for (int k = 0; k < D; ++k) c[k] = 0.0f;
    if constexpr (QJL)
      for (int k = 0; k < D / 32; ++k) sg[k] = 0;
  }
  float col = 0.0f;
  for (int r0 = r_begin; r0 < r_end; r0 += NR) {
    __syncthreads();
    for (int i = tid; i < NR * D; i += 256) {
      const int r = min(r0 + i / D, r_end - 1) + a.row0;
      const int64_t row = ((int64_t)b * a.Hq + h * a.G + r % a.G) * a.Sq + r / a.G;
      qs[i / D][i % D] = a.q[row * D + i % D];
      if constexpr (QJL) ps[i / D][i % D] = a.pq[row * D + i % D];
    }
    __syncthreads();
    for (int rr = 0; rr < min(NR, r_end - r0); ++rr) {
      const int r = r0 + rr;
      float s = 0.0f;
      for (int k = 0; k < D; ++k) s = __builtin_fmaf(qs[rr][k], c[k], s);
      s *= radius;
      if constexpr (QJL) {
        float x = 0.0f;
        for (int k = 0; k < D; ++k) x += (sg[k / 32] >> (k % 32)) & 1u ? ps[rr][k] : -ps[rr][k];
        s = zero_res ? s : s + x;
      }
      const int pos = a.q_start + (r + a.row0) / a.G;
      const bool valid = t < a.S && (!a.causal || t <= pos);
      if constexpr (STATS) {
        const float v = valid ? s : -INFINITY;
        float m = wave_max(v);
        __syncthreads();
        if (lane == 0) red[wave] = m;
        __syncthreads();
        m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float l = wave_sum(valid ? __builtin_amdgcn_exp2f(v - m) : 0.0f);
        __syncthreads();
        if (lane == 0) red[wave] = l;
        __syncthreads();
        if (tid == 0)
          a.part[(stream * a.tblocks + tb) * a.rows + r] = make_float2(m, red[0] + red[1] + red[2] + red[3]);
      } else {
        const float2 x = a.stat[stream * a.rows + r];
        if (valid) col = __builtin_fmaf(__builtin_amdgcn_exp2f(s - x.x), x.y, col);
      }
    }
  }
  if constexpr (!STATS)
    a.col[((stream * a.chunks + chunk) * a.tblocks + tb) * kWeightTokens + tid] = col;
}

// Joins the token blocks' maxima and sums of one row.
__global__ void __launch_bounds__(256) attn_stats_kernel(const AttnWeightsArgs a) {
  const uint32_t tiles = (uint32_t)(a.rows + 255) / 256;
  const int64_t stream = blockIdx.x / tiles;
  const int r = (int)(blockIdx.x - (uint32_t)stream * tiles) * 256 + threadIdx.x;
  if (r >= a.rows) return;
  const int last = a.causal ? min(a.q_start + (r + a.row0) / a.G, a.S - 1) : a.S - 1;
  const int n = last / kWeightTokens + 1;
  const float2 *p = a.part + stream * a.tblocks * a.rows + r;
  float m = -INFINITY, l = 0.0f;
  for (int i = 0; i < n; ++i) {
    const float2 x = p[(int64_t)i * a.rows];
    const float mn = fmaxf(m, x.x);
    if (mn == -INFINITY) continue;
    l = l * __builtin_amdgcn_exp2f(m - mn) + x.y * __builtin_amdgcn_exp2f(x.x - mn);
    m = mn;
  }
  a.stat[stream * a.rows + r] = make_float2(m, 1.0f / l);
}

// out = in + the row chunks' sums of one token, in the chunks' order.
__global__ void __launch_bounds__(256) weights_join_kernel(const AttnWeightsArgs a) {
  const int64_t stream = blockIdx.x / (uint32_t)a.tblocks;
  const int tb = (int)(blockIdx.x - (uint32_t)stream * a.tblocks);
  const int t = tb * kWeightTokens + threadIdx.x;
  if (t >= a.S) return;
  int c0 = 0;
  if (a.causal) {   // chunks that end before the first row that sees the block were not computed
    const int64_t first = (int64_t)(tb * kWeightTokens - a.q_start) * a.G - a.row0;
    if (first >= a.rows) c0 = a.chunks;
    else if (first > 0) c0 = (int)(first / kWeightRows);
  }
  float sum = 0.0f;
  for (int c = c0; c < a.chunks; ++c) sum += a.col[((stream * a.chunks + c) * a.tblocks + tb) * kWeightTokens + threadIdx.x];
  a.out[stream * a.out_stride + t] = (a.in ? a.in[stream * a.in_stride + t] : 0.0f) + sum;
}

__global__ void __launch_bounds__(256) weights_copy_kernel(const float *in, int64_t in_stride, float *out,
                                                           int64_t out_stride, int S) {
  const uint32_t tiles = (uint32_t)(S + 255) / 256;
  const int64_t stream = blockIdx.x / tiles;
  const int t = (int)(blockIdx.x - (uint32_t)stream * tiles) * 256 + threadIdx.x;
  if (t < S) out[stream * out_stride + t] = in ? in[stream * in_stride + t] : 0.0f;
}

template <int D, bool QJL>
void launch_passes(const AttnWeightsArgs &a, int64_t streams, hipStream_t s) {
  const unsigned grid = (unsigned)(streams * a.tblocks * a.chunks);
  attn_weights_kernel<D, QJL, true><<<grid, 256, 0, s>>>(a);
  attn_stats_kernel<<<(unsigned)(streams * ((a.rows + 255) / 256)), 256, 0, s>>>(a);
  attn_weights_kernel<D, QJL, false><<<grid, 256, 0, s>>>(a);
  weights_join_kernel<<<(unsigned)(streams * a.tblocks), 256, 0, s>>>(a);
}

}  // namespace

hipError_t launch_decode_weights(const DecodeArgs &a, const DecodeWeights &w, hipStream_t s) {
  const unsigned grid = (unsigned)((int64_t)((a.S + kDwTokens - 1) / kDwTokens) * a.B * a.Hkv);
  const size_t lds = (size_t)a.gq * sizeof(float2);
  const bool vec = ((uintptr_t)w.out | (uintptr_t)w.in) % 16 == 0 && (w.out_stride | (w.in ? w.in_stride : 0)) % 4 == 0;
  if (vec) decode_weights_kernel<true><<<grid, 256, lds, s>>>(a, w);
  else decode_weights_kernel<false><<<grid, 256, lds, s>>>(a, w);
  return hipGetLastError();
}

hipError_t launch_attn_weights(const AttnWeightsArgs &a, hipStream_t s) {
  const int64_t streams = (int64_t)a.B * a.Hkv;
  const bool qjl = a.pq != nullptr;
  if (a.d == 128) qjl ? launch_passes<128, true>(a, streams, s) : launch_passes<128, false>(a, streams, s);
  else qjl ? launch_passes<64, true>(a, streams, s) : launch_passes<64, false>(a, streams, s);
  return hipGetLastError();
}

hipError_t launch_weights_copy(const float *in, int64_t in_stride, float *out, int64_t out_stride, int64_t streams,
                               int S, hipStream_t s) {
  weights_copy_kernel<<<(unsigned)(streams * ((S + 255) / 256)), 256, 0, s>>>(in, in_stride, out, out_stride, S);
  return hipGetLastError();
}

}  // namespace pqkv
