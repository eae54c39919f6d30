// Rotary positions of queries and keys in one launch (pqkv_rotary, pqkv_rotary_axes).
//
// Pair i of a head's first rot_dim coordinates turns by t = position * freq[i]:
//   y_a = m (x_a cos t - x_b sin t),  y_b = m (x_a sin t + x_b cos t)
// with (a, b) = (i, i + rot_dim / 2), or (2i, 2i + 1) interleaved; the other
// coordinates are copied. The gradient is the same with -t.
//
// With several axes of positions (time, height, width) each pair has one of
// them; the table of the pairs' axes comes as a kernel argument, so nothing is
// copied for it and a call can be captured. It is read once per sine and cosine,
// not once per head: 64 + 8 heads x 32760 tokens on three axes (bf16, d = 128) take 238
// us, 1.21 GB at 5.1 TB/s, which is what they take on one and what a copy takes.
//
// The angle is a product in 64 bits, reduced to a fraction of a turn there
// (a position of 10^6 turns the first pair 1.6 10^5 times: in 32 bits the
// fraction would keep 7 bits); sine and cosine of the fraction, the products
// and the sum are in 32 bits, rounded once to the tensors' type.
//
// Bound by the bytes (each input read once, each output written once). A
// workgroup takes a few tokens of one sequence and the heads of them: their
// sines and cosines are computed once into LDS and serve every head. Inputs
// have any strides between tokens, heads and sequences (a projection's
// [B][T][H][d] is read as it is); the outputs are contiguous [B][H][T][d],
// which is what the encoders and attention take, so no transposing copy
// follows. 64 query and 8 key heads x 32768 tokens (d = 128, bf16): 240 us, 5.0
// TB/s, what a copy of 1 GiB moves; 40 heads of 8 single tokens: 3.1 us, the
// launch's own.
#include <type_traits>

#include "pqkv_device.h"
#include "pqkv_launch.h"

namespace pqkv {

namespace {

template <typename T> struct Elem;
template <> struct Elem<float> {
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};
template <> struct Elem<half_t> {
  static __device__ __forceinline__ float up(half_t x) { return (float)x; }
  static __device__ __forceinline__ half_t down(float x) { return (half_t)x; }
};
template <> struct Elem<bf16_t> {
  static __device__ __forceinline__ float up(bf16_t x) { return bf16_to_float(x.bits); }
  // round to nearest even; NaN stays NaN
  static __device__ __forceinline__ bf16_t down(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const uint32_t r = u + 0x7FFFu + ((u >> 16) & 1u);
    return bf16_t{(uint16_t)((x != x ? (u | 0x400000u) : r) >> 16)};
  }
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

struct RotaryKernelArgs {
  RotaryArgs a;
  FastDiv per_head, heads;   // items of a head; heads of a workgroup's share
  int tokens, head_count;    // tokens and heads per workgroup
  int n_rot, n_rest;         // items of the turned and of the copied part
};

struct OneAxis {};

// V elements of each of a pair's two sides per item (of a copied item: V in all).
// AX: OneAxis, or RotaryAxes.
template <typename T, int V, bool INTER, typename AX>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryKernelArgs k, const AX axes) {
  extern __shared__ __align__(8) float2 turn[];   // [tokens][rot_dim / 2]: m cos, m sin
  const RotaryArgs &a = k.a;
  const int half = a.rot_dim / 2;
  const uint32_t tiles = (uint32_t)(a.T + k.tokens - 1) / (uint32_t)k.tokens;
  const int b = (int)(blockIdx.x / tiles), t0 = (int)(blockIdx.x - (uint32_t)b * tiles) * k.tokens;
  const int h0 = blockIdx.y * k.head_count;
  const int nt = min(k.tokens, a.T - t0);
  for (int i = threadIdx.x; i < nt * half; i += 256) {
    const int t = i / half, p = i - t * half;
    int64_t row = (int64_t)b * a.pos_batch_stride;
    if constexpr (!std::is_empty<AX>::value) row += axes.of[p] * axes.stride;
    const double pos = (double)a.positions[row + t0 + t];
    const double turns = pos * (a.freqs[p] * 0.15915494309189533577);   // 1 / (2 pi)
    const float frac = (float)(turns - __builtin_rint(turns));
    float s, c;
    sincospif(2.0f * frac, &s, &c);
    turn[i] = make_float2(a.amplitude * c, a.inverse ? -a.amplitude * s : a.amplitude * s);
  }
  __syncthreads();
  const int nh = min(k.head_count, a.Hq + a.Hkv - h0);
  const uint32_t per_head = (uint32_t)(k.n_rot + k.n_rest);
  const uint32_t items = (uint32_t)nt * k.head_count * per_head;
  typedef Vec<T, V> VT;
  for (uint32_t it = threadIdx.x; it < items; it += 256) {
    const uint32_t row = k.per_head.div(it), c = it - row * per_head;
    const uint32_t t = k.heads.div(row), hh = row - t * k.head_count;
    if ((int)hh >= nh) continue;
    const int h = h0 + (int)hh;
    const bool key = h >= a.Hq;
    const int hx = key ? h - a.Hq : h, H = key ? a.Hkv : a.Hq;
    const int64_t *st = key ? a.k_stride : a.q_stride;
    const T *x = (const T *)(key ? a.k : a.q) + b * st[0] + hx * st[1] + (int64_t)(t0 + t) * st[2];
    T *y = (T *)(key ? a.k_out : a.q_out) + (((int64_t)b * H + hx) * a.T + t0 + t) * a.d;
    if ((int)c >= k.n_rot) {
      const int e = a.rot_dim + ((int)c - k.n_rot) * V;
      *(VT *)(y + e) = *(const VT *)(x + e);
      continue;
    }
    const int p0 = (int)c * V;                          // the item's first pair
    const int e0 = INTER ? 2 * p0 : p0, e1 = INTER ? 2 * p0 + V : p0 + half;
    const VT u = *(const VT *)(x + e0), w = *(const VT *)(x + e1);
    VT yu, yw;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      // interleaved, the pair's two sides are neighbours in the 2 V elements
      const int ia = INTER ? 2 * j : j, ib = INTER ? 2 * j + 1 : V + j;
      const float2 cs = turn[t * half + p0 + j];
      const float xa = Elem<T>::up(ia < V ? u.v[ia] : w.v[ia - V]);
      const float xb = Elem<T>::up(ib < V ? u.v[ib] : w.v[ib - V]);
      const T ya = Elem<T>::down(xa * cs.x - xb * cs.y), yb = Elem<T>::down(xa * cs.y + xb * cs.x);
      if (ia < V) yu.v[ia] = ya; else yw.v[ia - V] = ya;
      if (ib < V) yu.v[ib] = yb; else yw.v[ib - V] = yb;
    }
    *(VT *)(y + e0) = yu;
    *(VT *)(y + e1) = yw;
  }
}

template <typename T, int V, typename AX>
hipError_t launch(const RotaryArgs &a, const AX &axes, hipStream_t s) {
  const int H = a.Hq + a.Hkv, half = a.rot_dim / 2;
  const int n_rot = half / V, n_rest = (a.d - a.rot_dim) / V, per_head = n_rot + n_rest;
  // tokens of a workgroup: as many as leave 2048 workgroups, up to four; heads:
  // all of them, or (few tokens) as many as make an item per thread
  int tokens = 1;
  while (tokens < 4 && (int64_t)a.B * a.T / (2 * tokens) >= 2048) tokens *= 2;
  int heads = H;
  if ((int64_t)a.B * a.T < 1024) {
    heads = (256 + per_head - 1) / per_head;
    if (heads > H) heads = H;
  }
  const RotaryKernelArgs k{a, FastDiv(per_head), FastDiv(heads), tokens, heads, n_rot, n_rest};
  const dim3 grid((unsigned)((int64_t)((a.T + tokens - 1) / tokens) * a.B), (H + heads - 1) / heads);
  const size_t lds = (size_t)tokens * half * sizeof(float2);
  if (a.interleaved) rotary_kernel<T, V, true><<<grid, 256, lds, s>>>(k, axes);
  else rotary_kernel<T, V, false><<<grid, 256, lds, s>>>(k, axes);
  return hipGetLastError();
}

// 16-byte items where every item of every row starts on a 16-byte boundary,
// else an element at a time.
template <typename T, typename AX>
hipError_t launch_type(const RotaryArgs &a, const AX &axes, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.q_out | (uintptr_t)a.k | (uintptr_t)a.k_out;
  int64_t el = a.d | (a.rot_dim / 2);
  for (int i = 0; i < 3; ++i) el |= a.q_stride[i] | (a.Hkv ? a.k_stride[i] : 0);
  return at % 16 == 0 && el % V == 0 ? launch<T, V>(a, axes, s) : launch<T, 1>(a, axes, s);
}

template <typename AX>
hipError_t launch_any(const RotaryArgs &a, const AX &axes, int dtype, hipStream_t s) {
  if (dtype == PQKV_F32) return launch_type<float>(a, axes, s);
  if (dtype == PQKV_F16) return launch_type<half_t>(a, axes, s);
  return launch_type<bf16_t>(a, axes, s);
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs &a, int dtype, hipStream_t s) { return launch_any(a, OneAxis{}, dtype, s); }

hipError_t launch_rotary_axes(const RotaryArgs &a, const RotaryAxes &axes, int dtype, hipStream_t s) {
  return launch_any(a, axes, dtype, s);
}

}  // namespace pqkv
