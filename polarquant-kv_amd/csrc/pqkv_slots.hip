// What the slots of a cache stand for, without a rotation (pqkv_dequantize_slots):
// out[stream][t][j] = r16 c[code_j], contiguous or through the page table.
//
// 144 bytes of a vector pair become 512 (fp16, d = 128), at 3.6 TB/s; what bounds it are
// its vector instructions, 12.5 a coordinate, 81 % of the cycles (the address of a slot in
// its page, the codes, NaN and saturation). A
// thread takes eight coordinates (the codes that one 16-byte store of fp16 needs),
// neighbouring threads neighbouring ones, so that stores and the reads of a vector's
// bytes are dense; the codebook is in LDS, one bank an entry. 8 streams of 32768
// vectors of 128 to fp16: 24 us (86 MB, 3.6 TB/s) where the product with a unit matrix
// took 82 behind a copy out of the pages of 29.
#include "pqkv_device.h"
#include "pqkv_launch.h"

namespace pqkv {

namespace {

// 24 us for the above with two vectors a thread at once and 2048 workgroups that stay, 26
// with one, 25.6 with 4096 workgroups, 33.5 with one in 16384; with eight 24.5, but 5.1
// where 1536 vectors of 64 take 3.4.
constexpr int kAtOnce = 2, kBlocks = 2048;

template <typename T>
struct alignas(16) Eight {
  T v[8];
};

__device__ __forceinline__ void put(float x, float &to) { to = x; }
// fp16 saturates; NaN stays NaN
__device__ __forceinline__ void put(float x, half_t &to) { to = (half_t)(x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x); }

template <typename T, int D, int BITS>
__global__ void __launch_bounds__(256) slots_kernel(const SlotsArgs a, const FastDiv by_s) {
  __shared__ float cb[16];
  if (threadIdx.x < (1 << BITS)) cb[threadIdx.x] = a.codebook[threadIdx.x];
  __syncthreads();
  constexpr int G = D / 8, VB = vector_bytes(D, BITS), PER = 256 / G;    // threads of a vector; vectors of a workgroup at once
  constexpr int U = kAtOnce;
  const int g = threadIdx.x % G;
  // U vectors at a time: their addresses, then their bytes, then their stores
  for (int64_t v0 = (int64_t)blockIdx.x * (U * PER) + threadIdx.x / G; v0 < a.vectors; v0 += (int64_t)gridDim.x * (U * PER)) {
    const uint8_t *p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t v = v0 + u * PER < a.vectors ? v0 + u * PER : v0;
      // (vectors within 32 bits: the number of the stream, and the slot)
      const uint32_t s = by_s.div((uint32_t)v), t = (uint32_t)v - s * by_s.d;
      if (a.pages) p[u] = a.pages[(int64_t)s * a.max_pages + (t >> a.page_shift)] + (t & ((1u << a.page_shift) - 1)) * VB;
      else p[u] = a.blocks + (int64_t)s * a.stride + (int64_t)t * VB;
    }
    uint32_t w[U];
    uint16_t h[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      h[u] = *(const uint16_t *)p[u];            // (the vector's radius is its first block's)
      const uint8_t *codes = p[u] + (g / 4) * block_bytes(BITS) + 2;
      if constexpr (BITS == 4) {
        const uint16_t *q = (const uint16_t *)codes + 2 * (g % 4);
        w[u] = q[0] | (uint32_t)q[1] << 16;
      } else {
        w[u] = ((const uint16_t *)codes)[g % 4];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t v = v0 + u * PER;
      if (v >= a.vectors) break;
      float r = half_bits_to_float(h[u]);
      if (__builtin_isinf(r)) r = __builtin_nanf("");   // (no encoder writes one; a rotation would give NaN)
      Eight<T> o;
#pragma unroll
      for (int j = 0; j < 8; ++j) put(r * cb[(w[u] >> (BITS * j)) & ((1 << BITS) - 1)] + 0.0f, o.v[j]);
      *(Eight<T> *)((T *)a.out + v * D + 8 * g) = o;
    }
  }
}

template <typename T>
hipError_t launch(const SlotsArgs &a, int d, int bits, hipStream_t s) {
  const int64_t per = kAtOnce * 256 / (d / 8), want = (a.vectors + per - 1) / per;
  const unsigned blocks = (unsigned)(want < kBlocks ? want : kBlocks);
  const FastDiv by_s((uint32_t)a.S);
  if (d == 128) {
    if (bits == 4) slots_kernel<T, 128, 4><<<blocks, 256, 0, s>>>(a, by_s);
    else slots_kernel<T, 128, 2><<<blocks, 256, 0, s>>>(a, by_s);
  } else {
    if (bits == 4) slots_kernel<T, 64, 4><<<blocks, 256, 0, s>>>(a, by_s);
    else slots_kernel<T, 64, 2><<<blocks, 256, 0, s>>>(a, by_s);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_slots(const SlotsArgs &a, int d, int bits, int out_dtype, hipStream_t s) {
  return out_dtype == PQKV_F32 ? launch<float>(a, d, bits, s) : launch<half_t>(a, d, bits, s);
}

}  // namespace pqkv
