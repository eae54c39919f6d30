// Eviction: which positions of a cache stay (evict_select_kernel) and the move
// of their vectors into a new cache (gather_rows_kernel).
//
// Selection keeps, per stream, the `keep` positions of the largest weights
// (the first `sink` and last `recent` positions rank above every weight, NaN
// below), equal weights by the lowest index, in ascending order. Weights map to
// unsigned keys of the same order; the keep-th largest key is found digit by
// digit (11 + 11 + 10 bits, most significant first): a histogram of the digit
// over the keys that match the digits found so far, then the bin that holds
// the rank. Counts and indices are whole numbers, so no order of the atomic
// additions changes the result. One workgroup per stream: the stream's weights
// are read from HBM once and from L2 afterwards.
#include "pqkv_device.h"
#include "pqkv_launch.h"

namespace pqkv {

namespace {

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / kWave;
constexpr int kBins = 2048;

// Order-preserving key: -0 as 0, NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  uint32_t u = __builtin_bit_cast(uint32_t, w);
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

struct SelectSmem {
  uint32_t hist[kBins];
  uint32_t wave_sum[kSelWaves], wave_above[kSelWaves], wave_tie[kSelWaves];
  uint32_t digit, rank;
};

// Inclusive prefix sum of v over the wave's lanes.
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v, int lane) {
#pragma unroll
  for (int s = 1; s < kWave; s <<= 1) {
    const uint32_t o = __shfl_up(v, s, kWave);
    if (lane >= s) v += o;
  }
  return v;
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const float *__restrict__ weights, int64_t stride,
                                                                   int S, int keep, int sink, int recent,
                                                                   int *__restrict__ kept) {
  __shared__ SelectSmem sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float *w = weights + blockIdx.x * stride;
  int *out = kept + (int64_t)blockIdx.x * keep;
  // each wave takes one contiguous run of whole 64-position steps
  const int steps = (S + kSelThreads - 1) / kSelThreads;
  const int begin = wave * steps * kWave, end = min(S, begin + steps * kWave);
  auto key_at = [&](int i) { return i < sink || i >= S - recent ? 0xFFFFFFFFu : weight_key(w[i]); };

  uint32_t found = 0, mask = 0, rank = (uint32_t)keep;   // rank: of the wanted key among those matching `found`
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    const uint32_t low = (1u << bits) - 1;
    for (int i = tid; i < kBins; i += kSelThreads) sm.hist[i] = 0;
    __syncthreads();
    for (int i = begin + lane; i < end; i += kWave) {
      const uint32_t key = key_at(i);
      if ((key & mask) == found) atomicAdd(&sm.hist[(key >> shift) & low], 1u);
    }
    __syncthreads();
    // thread t: bins 2047 - 2t and 2046 - 2t, counted from the top
    const int b1 = kBins - 1 - 2 * tid;
    const uint32_t c1 = sm.hist[b1], c0 = sm.hist[b1 - 1];
    const uint32_t incl = wave_prefix(c1 + c0, lane);
    if (lane == 63) sm.wave_sum[wave] = incl;
    __syncthreads();
    uint32_t before = incl - c1 - c0;
    for (int i = 0; i < wave; ++i) before += sm.wave_sum[i];
    if (before < rank && rank <= before + c1 + c0) {
      const bool first = rank <= before + c1;
      sm.digit = (uint32_t)(first ? b1 : b1 - 1);
      sm.rank = rank - before - (first ? 0u : c1);
    }
    __syncthreads();
    found |= sm.digit << shift;
    mask |= low << shift;
    rank = sm.rank;
    __syncthreads();
  }
  // `found` is the border key; of the positions on it the first `rank` stay
  uint32_t above = 0, ties = 0;
  for (int i = begin + lane; i - lane < end; i += kWave) {
    const uint32_t key = i < end ? key_at(i) : 0u;
    above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < end && key > found));
    ties += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < end && key == found));
  }
  if (lane == 0) {
    sm.wave_above[wave] = above;
    sm.wave_tie[wave] = ties;
  }
  __syncthreads();
  uint32_t n_above = 0, n_tie = 0;
  for (int i = 0; i < wave; ++i) {
    n_above += sm.wave_above[i];
    n_tie += sm.wave_tie[i];
  }
  for (int i = begin + lane; i - lane < end; i += kWave) {
    const uint32_t key = i < end ? key_at(i) : 0u;
    const uint64_t ma = __builtin_amdgcn_ballot_w64(i < end && key > found);
    const uint64_t mt = __builtin_amdgcn_ballot_w64(i < end && key == found);
    const uint32_t a = n_above + lanes_below(ma), t = n_tie + lanes_below(mt);
    const bool stays = i < end && (key > found || (key == found && t < rank));
    if (stays) out[a + min(t, rank)] = i;
    n_above += __builtin_popcountll(ma);
    n_tie += __builtin_popcountll(mt);
  }
}

// Rows of every part of the listed positions, a workgroup per kGatherRows
// result rows of one stream: their source positions are read once into LDS and
// serve all parts. A row moves in units of 8 or 4 bytes.
constexpr int kGatherRows = 256;

template <typename U>
__device__ __forceinline__ void gather_part(const GatherPart &p, const int *src, int64_t stream, int row0, int rows,
                                            int keep, FastDiv per_row) {
  const uint32_t n = per_row.d, total = (uint32_t)rows * n;
  for (uint32_t i = threadIdx.x; i < total; i += 256) {
    const uint32_t r = per_row.div(i), c = i - r * n;
    const int t = src[r], o = row0 + (int)r;
    U v = 0;
    if (t >= 0) {
      const uint8_t *from = p.src_pages ? p.src_pages[stream * p.src_max_pages + (t >> p.src_shift)] +
                                              (int64_t)(t & ((1 << p.src_shift) - 1)) * p.row_bytes
                                        : p.src + stream * p.src_stride + (int64_t)t * p.row_bytes;
      v = ((const U *)from)[c];
    }
    uint8_t *to = p.dst_pages ? p.dst_pages[stream * p.dst_max_pages + (o >> p.dst_shift)] +
                                    (int64_t)(o & ((1 << p.dst_shift) - 1)) * p.row_bytes
                              : p.dst + stream * p.dst_stride + (int64_t)o * p.row_bytes;
    if (o < keep || p.dst_pages) ((U *)to)[c] = v;
  }
}

struct GatherKernelArgs {
  GatherArgs a;
  FastDiv per_row[kMaxGather];   // units of a row
};

__global__ void __launch_bounds__(256) gather_rows_kernel(const GatherKernelArgs k) {
  __shared__ int src[kGatherRows];
  const GatherArgs &a = k.a;
  const uint32_t tiles = (uint32_t)(a.fill + kGatherRows - 1) / kGatherRows;
  const int64_t stream = blockIdx.x / tiles;
  const int row0 = (int)(blockIdx.x - (uint32_t)stream * tiles) * kGatherRows, rows = min(kGatherRows, a.fill - row0);
  if ((int)threadIdx.x < rows) {
    const int o = row0 + (int)threadIdx.x;
    const int t = o < a.keep ? a.kept[stream * a.keep + o] : -1;
    src[threadIdx.x] = t < a.S ? t : -1;   // a position outside the cache moves zeros
  }
  __syncthreads();
  for (int i = 0; i < a.n_parts; ++i) {
    const GatherPart &p = a.part[i];
    if (p.unit == 8) gather_part<uint64_t>(p, src, stream, row0, rows, a.keep, k.per_row[i]);
    else gather_part<uint32_t>(p, src, stream, row0, rows, a.keep, k.per_row[i]);
  }
}

}  // namespace

hipError_t launch_evict_select(const float *weights, int64_t stride, int64_t n_streams, int S, int keep, int sink,
                               int recent, int *kept, hipStream_t s) {
  evict_select_kernel<<<(unsigned)n_streams, kSelThreads, 0, s>>>(weights, stride, S, keep, sink, recent, kept);
  return hipGetLastError();
}

hipError_t launch_gather_rows(const GatherArgs &a, int64_t n_streams, hipStream_t s) {
  const int64_t grid = (int64_t)((a.fill + kGatherRows - 1) / kGatherRows) * n_streams;
  auto units = [&](int i) { return FastDiv(i < a.n_parts ? (uint32_t)(a.part[i].row_bytes / a.part[i].unit) : 1u); };
  const GatherKernelArgs k{a, {units(0), units(1), units(2), units(3), units(4), units(5)}};
  gather_rows_kernel<<<(unsigned)grid, 256, 0, s>>>(k);
  return hipGetLastError();
}

}  // namespace pqkv
