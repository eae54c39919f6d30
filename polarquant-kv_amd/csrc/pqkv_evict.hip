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
// additions changes the result. One workgroup per stream, its keys in registers
// up to 65536 positions (KPT per thread), so that the weights are read once and
// all their loads are in flight together; longer streams are read again in each
// pass, from L2. Weights crowd into few exponents, so the first digit's
// additions meet in few bins: there each bin has eight counters, a lane's by its
// number. Bound by the instructions of one compute unit per stream, which grow
// with KPT, empty steps included (128 streams of unequal weights: 11.6 us with 20,
// 13.0 with 24): KPT is the number of steps rounded up to a multiple of four (2 where
// that is enough) up to 32768 positions, above, where few caches are, to 48 or 64.
// 15.7 us for 128 such streams of 32768 positions, 21 where a quarter of the weights
// are zeros; 11 and 14 for 32 of 16385, 5.5 for 32 of 1025.
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

constexpr int kCopies = 8;   // counters per bin

struct SelectSmem {
  uint32_t hist[kBins * kCopies];
  uint32_t wave_sum[kSelWaves], wave_above[kSelWaves], wave_tie[kSelWaves];
  uint32_t digit, rank, count;
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

template <int KPT>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const float *__restrict__ weights, int64_t stride,
                                                                   int S, int keep, int sink, int recent,
                                                                   int *__restrict__ kept) {
  __shared__ __align__(16) SelectSmem sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float *w = weights + blockIdx.x * stride;
  int *out = kept + (int64_t)blockIdx.x * keep;
  // Each wave takes one contiguous run of whole 64-position steps. Positions
  // past the last one have the lowest key, and the highest numbers, so they are
  // never among the first `keep` and need no test of their own.
  const int steps = KPT > 0 ? KPT : (S + kSelThreads - 1) / kSelThreads;
  const int begin = wave * steps * kWave;
  auto key_of = [&](int i, float x) {
    const uint32_t key = i < sink || i >= S - recent ? 0xFFFFFFFFu : weight_key(x);
    return i < S ? key : 0u;
  };
  uint32_t keys[KPT > 0 ? KPT : 1];
  if constexpr (KPT > 0) {
#pragma unroll
    for (int j = 0; j < KPT; ++j)
      keys[j] = __builtin_bit_cast(uint32_t, w[min(begin + j * kWave + lane, S - 1)]);
#pragma unroll
    for (int j = 0; j < KPT; ++j) keys[j] = key_of(begin + j * kWave + lane, __builtin_bit_cast(float, keys[j]));
  }
  // f(key, position) for the wave's positions, step by step
  auto each = [&](auto f) {
    if constexpr (KPT > 0) {
#pragma unroll
      for (int j = 0; j < KPT; ++j) f(keys[j], begin + j * kWave + lane);
    } else {
      constexpr int U = 16;   // loads in flight
      for (int j0 = 0; j0 < steps; j0 += U) {
        const int i0 = begin + j0 * kWave + lane;
        float x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = w[min(i0 + u * kWave, S - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (j0 + u >= steps) break;
          f(key_of(i0 + u * kWave, x[u]), i0 + u * kWave);
        }
      }
    }
  };

  // rank: of the wanted key among those matching `found`; on_border: keys equal to it
  uint32_t found = 0, mask = 0, rank = (uint32_t)keep, on_border = 0;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    const int copies = pass == 0 ? kCopies : 1;
    const uint32_t low = (1u << bits) - 1;
    for (int i = tid; i < kBins * copies / 4; i += kSelThreads) ((u32x4 *)sm.hist)[i] = (u32x4){0u, 0u, 0u, 0u};
    __syncthreads();
    each([&](uint32_t key, int) {
      if ((key & mask) == found)
        atomicAdd(&sm.hist[((key >> shift) & low) * copies + (lane & (copies - 1))], 1u);
    });
    __syncthreads();
    // thread t: bins 2047 - 2t and 2046 - 2t, counted from the top
    const int b1 = kBins - 1 - 2 * tid;
    uint32_t c0, c1;
    if (pass == 0) {
      const u32x4 *h = (const u32x4 *)(sm.hist + (b1 - 1) * kCopies);
      const u32x4 x0 = h[0] + h[1], x1 = h[2] + h[3];
      c0 = x0.x + x0.y + x0.z + x0.w;
      c1 = x1.x + x1.y + x1.z + x1.w;
    } else {
      c0 = sm.hist[b1 - 1];
      c1 = sm.hist[b1];
    }
    const uint32_t incl = wave_prefix(c1 + c0, lane);
    if (lane == 63) sm.wave_sum[wave] = incl;
    __syncthreads();
    uint32_t before = incl - c1 - c0;
#pragma unroll
    for (int i = 0; i < kSelWaves; ++i) before += i < wave ? sm.wave_sum[i] : 0u;
    if (before < rank && rank <= before + c1 + c0) {
      const bool first = rank <= before + c1;
      sm.digit = (uint32_t)(first ? b1 : b1 - 1);
      sm.rank = rank - before - (first ? 0u : c1);
      sm.count = first ? c1 : c0;
    }
    __syncthreads();
    found |= sm.digit << shift;
    mask |= low << shift;
    rank = sm.rank;
    on_border = sm.count;
  }
  // `found` is the border key; of the positions on it the first `rank` stay.
  // Where all of them do (no equal weights across the border), one comparison
  // says what stays; else the ties are counted beside the keys above.
  auto lead = [&](uint32_t above, uint32_t ties, uint32_t &n_above, uint32_t &n_tie) {
    if (lane == 0) {
      sm.wave_above[wave] = above;
      sm.wave_tie[wave] = ties;
    }
    __syncthreads();
    n_above = n_tie = 0;
#pragma unroll
    for (int i = 0; i < kSelWaves; ++i) {
      n_above += i < wave ? sm.wave_above[i] : 0u;
      n_tie += i < wave ? sm.wave_tie[i] : 0u;
    }
  };
  uint32_t above = 0, ties = 0, n_above, n_tie;
  if (rank == on_border) {
    each([&](uint32_t key, int) { above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key >= found)); });
    lead(above, 0, n_above, n_tie);
    each([&](uint32_t key, int i) {
      const uint64_t m = __builtin_amdgcn_ballot_w64(key >= found);
      if (key >= found) out[n_above + lanes_below(m)] = i;
      n_above += __builtin_popcountll(m);
    });
    return;
  }
  each([&](uint32_t key, int) {
    above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key > found));
    ties += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key == found));
  });
  lead(above, ties, n_above, n_tie);
  each([&](uint32_t key, int i) {
    const uint64_t ma = __builtin_amdgcn_ballot_w64(key > found), mt = __builtin_amdgcn_ballot_w64(key == found);
    const uint32_t a = n_above + lanes_below(ma), t = n_tie + lanes_below(mt);
    if (key > found || (key == found && t < rank)) out[a + min(t, rank)] = i;
    n_above += __builtin_popcountll(ma);
    n_tie += __builtin_popcountll(mt);
  });
}

// Rows of the listed positions, a workgroup per `rows_per` result rows of one
// stream and one array: their source positions are read once into LDS. A row
// moves in units of 8 or 4 bytes, the units of a workgroup in the order of the
// result, kMoves per thread in flight. Bound by the bytes, of which the source's
// come in whole 64-byte pieces: a 72-byte row out of its neighbours costs about
// two of them. 8192 of 32768 rows (two arrays of 72 bytes, 12 bytes of weights and
// positions) of 128 streams: 100 us, 365 MB read where 155 are kept, 155 written,
// 5.2 TB/s.
constexpr int kGatherRows = 256, kMoves = 8;

struct GatherKernelArgs {
  GatherArgs a;
  FastDiv per_row[kMaxGather];   // units of a row
  int rows_per;
};

template <typename U>
__device__ __forceinline__ void gather_part(const GatherPart &p, const int *src, int64_t stream, int row0, int rows,
                                            FastDiv per_row) {
  const uint32_t n = per_row.d, total = (uint32_t)rows * n;
  for (uint32_t i0 = threadIdx.x; i0 < total; i0 += 256 * kMoves) {
    U v[kMoves];
#pragma unroll
    for (int j = 0; j < kMoves; ++j) {
      const uint32_t i = i0 + 256 * j;
      v[j] = 0;
      if (i >= total) continue;
      const uint32_t r = per_row.div(i);
      const int t = src[r];
      if (t < 0) continue;
      const uint8_t *from = p.src_pages ? p.src_pages[stream * p.src_max_pages + (t >> p.src_shift)] +
                                              (int64_t)(t & ((1 << p.src_shift) - 1)) * p.row_bytes
                                        : p.src + stream * p.src_stride + (int64_t)t * p.row_bytes;
      v[j] = ((const U *)from)[i - r * n];
    }
#pragma unroll
    for (int j = 0; j < kMoves; ++j) {
      const uint32_t i = i0 + 256 * j;
      if (i >= total) continue;
      const uint32_t r = per_row.div(i);
      const int o = row0 + (int)r;
      uint8_t *to = p.dst_pages ? p.dst_pages[stream * p.dst_max_pages + (o >> p.dst_shift)] +
                                      (int64_t)(o & ((1 << p.dst_shift) - 1)) * p.row_bytes
                                : p.dst + stream * p.dst_stride + (int64_t)o * p.row_bytes;
      ((U *)to)[i - r * n] = v[j];
    }
  }
}

__global__ void __launch_bounds__(256) gather_rows_kernel(const GatherKernelArgs k) {
  __shared__ int src[kGatherRows];
  const GatherArgs &a = k.a;
  const uint32_t tiles = (uint32_t)(a.fill + k.rows_per - 1) / (uint32_t)k.rows_per;
  const int64_t stream = blockIdx.x / tiles;
  const int row0 = (int)(blockIdx.x - (uint32_t)stream * tiles) * k.rows_per;
  const GatherPart &p = a.part[blockIdx.y];
  // contiguous results end at keep; pages are filled up with zeros
  const int rows = min(k.rows_per, (p.dst_pages || p.dst_table ? a.fill : a.keep) - row0);
  if (p.dst_table) {   // the pages that start in these rows
    const int page = 1 << p.dst_shift, first = (row0 + page - 1) >> p.dst_shift;
    const int pg = first + (int)threadIdx.x;
    if ((pg << p.dst_shift) < row0 + rows)
      p.dst_table[stream * p.dst_max_pages + pg] = p.dst + stream * p.dst_stride + (int64_t)pg * page * p.row_bytes;
  }
  if ((int)threadIdx.x < rows) {
    const int o = row0 + (int)threadIdx.x;
    const int t = o < a.keep ? a.kept[stream * a.keep + o] : -1;
    src[threadIdx.x] = t < a.S ? t : -1;   // a position outside the cache moves zeros
  }
  __syncthreads();
  if (rows <= 0) return;
  if (p.unit == 8) gather_part<uint64_t>(p, src, stream, row0, rows, k.per_row[blockIdx.y]);
  else gather_part<uint32_t>(p, src, stream, row0, rows, k.per_row[blockIdx.y]);
}

}  // namespace

hipError_t launch_evict_select(const float *weights, int64_t stride, int64_t n_streams, int S, int keep, int sink,
                               int recent, int *kept, hipStream_t s) {
  const int steps = (S + kSelThreads - 1) / kSelThreads;
#define PQKV_SELECT(K) \
  evict_select_kernel<K><<<(unsigned)n_streams, kSelThreads, 0, s>>>(weights, stride, S, keep, sink, recent, kept)
  if (steps <= 2) PQKV_SELECT(2);
  else if (steps <= 4) PQKV_SELECT(4);
  else if (steps <= 8) PQKV_SELECT(8);
  else if (steps <= 12) PQKV_SELECT(12);
  else if (steps <= 16) PQKV_SELECT(16);
  else if (steps <= 20) PQKV_SELECT(20);
  else if (steps <= 24) PQKV_SELECT(24);
  else if (steps <= 28) PQKV_SELECT(28);
  else if (steps <= 32) PQKV_SELECT(32);
  else if (steps <= 48) PQKV_SELECT(48);
  else if (steps <= 64) PQKV_SELECT(64);
  else PQKV_SELECT(0);
#undef PQKV_SELECT
  return hipGetLastError();
}

hipError_t launch_gather_rows(const GatherArgs &a, int64_t n_streams, hipStream_t s) {
  // fewer rows per workgroup where that leaves compute units without one
  const int rows_per = (int64_t)a.fill * n_streams < 1024 * kGatherRows ? 64 : kGatherRows;
  const dim3 grid((unsigned)((int64_t)((a.fill + rows_per - 1) / rows_per) * n_streams), a.n_parts);
  auto units = [&](int i) { return FastDiv(i < a.n_parts ? (uint32_t)(a.part[i].row_bytes / a.part[i].unit) : 1u); };
  const GatherKernelArgs k{a, {units(0), units(1), units(2), units(3), units(4), units(5)}, rows_per};
  gather_rows_kernel<<<grid, 256, 0, s>>>(k);
  return hipGetLastError();
}

}  // namespace pqkv
