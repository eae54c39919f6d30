// The join of a decode call's splits, as the body of a workgroup (its own
// launch in pqkv_decode.hip; with the cached positions' weights in
// pqkv_weights.hip).
#pragma once

#include "pqkv_device.h"
#include "pqkv_launch.h"

namespace pqkv {

// Combine splits, normalise and rotate back: out = R^T (sum_s w_s o_s / L).
// Workgroup (hg, cg): kMergeHeads query heads x 32 output columns. One wave
// per head computes the split weights; every workgroup of a head group forms
// the full normalised o_rot (cheap, L2-resident partials) and then its 32
// outputs from the matching 32 columns of R, staged as [32][D + 4] (16-byte
// reads; each 16-lane phase of them covers all 64 banks).
// ROT = false (R == nullptr): the normalised o_rot itself is the output.
// MS: the most splits.
template <int D, int MS = kMaxSplits>
struct MergeSmem {
  static constexpr int NC = 32;    // output columns per workgroup
  static constexpr int RP = D + 4;
  __align__(16) float rs[NC * RP];    // rs[jj][k] = R[k][c0 + jj]
  __align__(16) float os[kMergeHeads * D];
  float wts[kMergeHeads][MS];
};

template <int D, typename TOUT, bool ROT = true, int MS = kMaxSplits>
__device__ __forceinline__ void decode_merge_body(MergeSmem<D, MS> &sm, const float *__restrict__ part,
                                                  const float *__restrict__ R, TOUT *__restrict__ out, int BHq,
                                                  int splits, int hg, int cg) {
  constexpr int NH = kMergeHeads;
  constexpr int NC = MergeSmem<D>::NC, RP = MergeSmem<D>::RP;
  constexpr int RU = NC * D / 4 / 256;   // R float4 loads per thread
  constexpr int OU = NH * D / 256;       // (head, coordinate) sums per thread
  constexpr int SB = 16;                 // splits whose o values are loaded at once
  auto &rs = sm.rs;
  auto &os = sm.os;
  auto &wts = sm.wts;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int head0 = hg * NH, c0 = cg * NC;
  // Every independent global read goes out before the first wait: the R
  // columns, this wave's split maxima and sums (up to 64 splits), and the
  // first SB splits of the thread's o values.
  float4 rv[RU];
  if constexpr (ROT) {
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int i = tid + 256 * u, k = i / (NC / 4), j4 = i % (NC / 4);
      rv[u] = *(const float4 *)(R + (int64_t)k * D + c0 + 4 * j4);
    }
  }
  const int hq_w = head0 + wave;
  const float *pw = part + (int64_t)min(hq_w, BHq - 1) * splits * (D + 2);
  const float m0 = lane < splits ? pw[(int64_t)lane * (D + 2)] : -INFINITY;
  const float l0 = lane < splits ? pw[(int64_t)lane * (D + 2) + 1] : 0.0f;
  float ov[OU][SB];
#pragma unroll
  for (int u = 0; u < OU; ++u) {
    const int i = tid + 256 * u, hh = i / D, c = i % D;
    const float *p = part + (int64_t)min(head0 + hh, BHq - 1) * splits * (D + 2) + 2 + c;
#pragma unroll
    for (int sp = 0; sp < SB; ++sp) ov[u][sp] = sp < splits ? p[(int64_t)sp * (D + 2)] : 0.0f;
  }
  if constexpr (ROT) {
#pragma unroll
    for (int u = 0; u < RU; ++u) {
      const int i = tid + 256 * u, k = i / (NC / 4), j4 = i % (NC / 4);
      rs[(4 * j4 + 0) * RP + k] = rv[u].x;
      rs[(4 * j4 + 1) * RP + k] = rv[u].y;
      rs[(4 * j4 + 2) * RP + k] = rv[u].z;
      rs[(4 * j4 + 3) * RP + k] = rv[u].w;
    }
  }
  if (hq_w < BHq) {
    float mx = m0;
    for (int sp = lane + 64; sp < splits; sp += 64) mx = fmaxf(mx, pw[(int64_t)sp * (D + 2)]);
    mx = wave_max(mx);
    float L = 0.0f;
    for (int sp = lane; sp < splits; sp += 64) {
      const float ms = sp == lane ? m0 : pw[(int64_t)sp * (D + 2)];
      const float ls = sp == lane ? l0 : pw[(int64_t)sp * (D + 2) + 1];
      const float e = ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms - mx);
      wts[wave][sp] = e;
      L = __builtin_fmaf(e, ls, L);
    }
    L = wave_sum(L);
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    for (int sp = lane; sp < splits; sp += 64) wts[wave][sp] *= inv;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < OU; ++u) {
    const int i = tid + 256 * u, hh = i / D, c = i % D;
    const int hq = head0 + hh;
    float o = 0.0f;
    if (hq < BHq) {
#pragma unroll
      for (int sp = 0; sp < SB; ++sp)
        if (sp < splits) o = __builtin_fmaf(wts[hh][sp], ov[u][sp], o);
      const float *p = part + (int64_t)hq * splits * (D + 2) + 2 + c;
#pragma unroll 8
      for (int sp = SB; sp < splits; ++sp) o = __builtin_fmaf(wts[hh][sp], p[(int64_t)sp * (D + 2)], o);
    }
    os[i] = o;
  }
  __syncthreads();
  if (!ROT && tid < NH * NC) {
    const int hh = tid / NC, jj = tid % NC;
    const int hq = head0 + hh;
    if (hq < BHq) out[(int64_t)hq * D + c0 + jj] = (TOUT)os[hh * D + c0 + jj];
  }
  if (ROT && tid < NH * NC) {
    const int hh = tid / NC, jj = tid % NC;
    const float4 *orow = (const float4 *)(os + hh * D);
    const float4 *rr = (const float4 *)(rs + jj * RP);
    float acc = 0.0f;
#pragma unroll 4
    for (int k4 = 0; k4 < D / 4; ++k4) {
      const float4 a4 = orow[k4], r4 = rr[k4];
      acc = __builtin_fmaf(a4.x, r4.x, acc);
      acc = __builtin_fmaf(a4.y, r4.y, acc);
      acc = __builtin_fmaf(a4.z, r4.z, acc);
      acc = __builtin_fmaf(a4.w, r4.w, acc);
    }
    const int hq = head0 + hh;
    if (hq < BHq) out[(int64_t)hq * D + c0 + jj] = (TOUT)acc;
  }
}

}  // namespace pqkv
