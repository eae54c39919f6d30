// C ABI of a cache under a budget: decode with weights, the weights of a
// chunk, eviction, and rotary positions. Host code: validation, workspace
// layouts and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>

#include "../../include/pqkv.h"
#include "pqkv_launch.h"

using pqkv::fail_status;
using pqkv::kMaxGroupWeights;
using pqkv::report_hip_error;

namespace {

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }
constexpr int kMaxTokens = 1 << 24;      // 32-bit byte offsets into 8 rows of logits
constexpr int64_t kMaxGrid = INT_MAX;

// The weights' strides against the shape; returns PQKV_OK or the failure.
int check_weights(const char *what, const float *in, int64_t in_stride, const float *out, int64_t out_stride, int B,
                  int Hkv, int S) {
  if (S == 0) return PQKV_OK;
  if (!out) return fail_status(PQKV_ERR_INVALID, "%s: null weights_out", what);
  if (((uintptr_t)in | (uintptr_t)out) % 4) return fail_status(PQKV_ERR_INVALID, "%s: unaligned weights", what);
  if (out_stride < S || (in && in_stride < S))
    return fail_status(PQKV_ERR_INVALID, "%s: a weights stride is below S=%d", what, S);
  if (in) {
    // the same array, or arrays apart
    const int64_t n = (int64_t)B * Hkv;
    const uintptr_t i0 = (uintptr_t)in, i1 = i0 + 4 * (uintptr_t)((n - 1) * in_stride + S);
    const uintptr_t o0 = (uintptr_t)out, o1 = o0 + 4 * (uintptr_t)((n - 1) * out_stride + S);
    if (i0 < o1 && o0 < i1 && !(i0 == o0 && in_stride == out_stride))
      return fail_status(PQKV_ERR_INVALID, "%s: weights_out overlaps weights_in", what);
  }
  return PQKV_OK;
}

int64_t logit_stride(int S) { return ((int64_t)S + 63) / 64 * 64; }

int decode_weights_run(const void *q, int q_dtype, const float *R, const uint8_t *k_cache, const uint8_t *v_cache,
                       const float *k_cb, const float *v_cb, int n_bits, const uint8_t *qjl, const float *p_rot, int m,
                       int B, int Hq, int Hkv, int S, int S_max, int d, float scale, void *out, int out_dtype,
                       const float *in, int64_t in_stride, float *w_out, int64_t w_stride, void *ws, size_t ws_bytes,
                       void *stream, const pqkv::PagedCache *pg) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || S < 0)
    return fail_status(PQKV_ERR_INVALID, "decode_weights: B=%d Hq=%d Hkv=%d S=%d", B, Hq, Hkv, S);
  if (S >= kMaxTokens) return fail_status(PQKV_ERR_UNSUPPORTED, "decode_weights: S=%d", S);
  if (Hq / Hkv > kMaxGroupWeights) return fail_status(PQKV_ERR_UNSUPPORTED, "decode_weights: group size %d", Hq / Hkv);
  if ((int64_t)B * Hkv * (S / 1024 + 1) + (int64_t)B * Hq > kMaxGrid) return fail_status(PQKV_ERR_UNSUPPORTED, "decode_weights: size");
  const int c = check_weights("decode_weights", in, in_stride, w_out, w_stride, B, Hkv, S);
  if (c != PQKV_OK) return c;
  const size_t base = S > 0 ? align256(pqkv_decode_workspace_bytes(B, Hq, Hkv, S, d)) : 0;
  if (S > 0) {
    const size_t need = pqkv_decode_attn_weights_workspace_bytes(B, Hq, Hkv, S, d);
    if (!ws || ws_bytes < need)
      return fail_status(PQKV_ERR_WORKSPACE, "decode_weights: workspace %zu < %zu bytes", ws_bytes, need);
    if ((uintptr_t)ws % 16) return fail_status(PQKV_ERR_INVALID, "decode_weights: workspace must be 16-byte aligned");
  }
  const pqkv::DecodeWeights wt{(float *)((char *)ws + base), logit_stride(S), in, in_stride, w_out, w_stride};
  return pqkv::decode_attn_run(q, q_dtype, R, k_cache, v_cache, k_cb, v_cb, n_bits, n_bits, nullptr, nullptr, qjl,
                               p_rot, m, B, Hq, Hkv, S, S_max, d, scale, out, out_dtype, ws, base, false, nullptr,
                               stream, pg, &wt);
}

// One pass of a chunk's weights over `rows` rows of every stream, and its
// workspace: with QJL the rotated queries and their projections, the rows'
// records and factors, the token blocks' partials, the rows' statistics, the row chunks' sums.
struct WeightsPlan {
  int tokens, tblocks, rows, chunk_rows;
  size_t q, pq, records, factor, part, stat, col;
  size_t bytes() const { return q + pq + records + factor + part + stat + col; }
  int chunks(int r) const { return (r + chunk_rows - 1) / chunk_rows; }
};
// Rows of a stream up to which a workgroup takes 128 tokens, not 256: three
// waves per SIMD instead of two hide the decoding of the keys, which is then a
// larger part of the work (32 query / 8 kv heads, d = 128: 256 rows on 32768
// tokens 129 us against 156, 2048 rows on 16512 tokens 384 against 411); with
// more rows each operand read serves four tiles instead of two (32764 rows on
// 8191 tokens take 4 % more with 128).
constexpr int kFewRows = 2048;
int row_tiles(int rows) { return (rows + 63) / 64 * 4; }
// shrink: passes of 2^-shrink times the rows, for less room.
constexpr int kMaxShrink = 4;
WeightsPlan weights_plan(int B, int Hq, int Hkv, int Sq, int S, int d, bool qjl, int shrink = 0) {
  WeightsPlan p;
  const int64_t streams = (int64_t)B * Hkv, total = (int64_t)Sq * (Hq / Hkv);
  p.tokens = qjl || total <= kFewRows ? 128 : 256;
  p.tblocks = (S + p.tokens - 1) / p.tokens;
  // rows of a pass: partials within 256 MB, records within 512 MB, but 64 rows
  // at least, whose partials are 4 bytes per position
  const int64_t rec_row = (int64_t)d * (qjl ? 8 : 4);
  int64_t rows = std::min((int64_t)(256 << 20 >> shrink) / (streams * p.tblocks * (int64_t)sizeof(float2)),
                          (int64_t)(512 << 20 >> shrink) / (streams * rec_row));
  rows = std::max<int64_t>(rows / 64 * 64, 64);
  p.rows = (int)std::min(rows, total);
  // rows of a workgroup: about 1024 workgroups; at least 128 rows, under which
  // decoding the keys is most of the work, at most 1024, whose records (0.5 MB at
  // d = 128) a group of workgroups shares in L2 and which leave the last round
  // of a long chunk short (with 2048 rows 32764 rows on 8191 tokens take 2 % more)
  const int64_t want = p.rows * streams * p.tblocks / 1024;
  p.chunk_rows = (int)std::min<int64_t>(std::max<int64_t>((want + 63) / 64 * 64, 128), 1024);
  p.q = qjl ? align256((size_t)B * Hq * Sq * d * 4) : 0;
  p.pq = p.q;
  p.records = align256((size_t)streams * row_tiles(p.rows) * 16 * rec_row);
  p.factor = align256((size_t)streams * row_tiles(p.rows) * 16 * sizeof(float));
  p.part = align256((size_t)streams * p.tblocks * p.rows * sizeof(float2));
  p.stat = align256((size_t)streams * row_tiles(p.rows) * 16 * sizeof(float2));
  // (one chunk's sums are the result: no room for them)
  const int chunks = p.chunks(p.rows);
  p.col = chunks > 1 ? align256((size_t)streams * chunks * p.tblocks * p.tokens * sizeof(float)) : 0;
  return p;
}

bool weights_shape_ok(int B, int Hq, int Hkv, int Sq, int S, int d) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || S <= 0 || Hq % Hkv || (d != 64 && d != 128)) return false;
  const int G = Hq / Hkv;
  const int64_t tblocks = ((int64_t)S + 127) / 128;
  // grids, row numbers and positions within 31 bits
  return S < kMaxTokens && G <= kMaxGroupWeights && (int64_t)Sq * G < INT_MAX / 2 &&
         (int64_t)B * Hkv * tblocks <= (1 << 24) && (int64_t)B * Hq * Sq <= ((int64_t)1 << 40) / d;
}

int attn_weights_run(const void *q, int q_dtype, const float *R, const uint8_t *k_cache, const float *codebook,
                     int n_bits, const uint8_t *qjl, const float *p_rot, int m, int B, int Hq, int Hkv, int Sq,
                     int q_start, int S, int S_max, int d, float scale, int causal, const float *in, int64_t in_stride,
                     float *out, int64_t out_stride, void *ws, size_t ws_bytes, void *stream,
                     const pqkv::PagedCache *pg) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq < 0 || S < 0 || S_max < S || q_start < 0)
    return fail_status(PQKV_ERR_INVALID, "attn_weights: B=%d Hq=%d Hkv=%d Sq=%d q_start=%d S=%d S_max=%d", B, Hq, Hkv,
                       Sq, q_start, S, S_max);
  if (Hq % Hkv) return fail_status(PQKV_ERR_INVALID, "attn_weights: Hq=%d not a multiple of Hkv=%d", Hq, Hkv);
  if (d != 64 && d != 128) return fail_status(PQKV_ERR_UNSUPPORTED, "attn_weights: d=%d", d);
  if (n_bits != 2 && n_bits != 4) return fail_status(PQKV_ERR_UNSUPPORTED, "attn_weights: n_bits=%d", n_bits);
  if (q_dtype != PQKV_F32 && q_dtype != PQKV_F16) return fail_status(PQKV_ERR_UNSUPPORTED, "attn_weights: dtype");
  const bool has_qjl = qjl != nullptr || (pg && pg->s_pages != nullptr);
  if (has_qjl != (p_rot != nullptr)) return fail_status(PQKV_ERR_INVALID, "attn_weights: qjl and p_rot go together");
  if (has_qjl && m != d) return fail_status(PQKV_ERR_UNSUPPORTED, "attn_weights: QJL needs m == d");
  if (!(scale > 0.0f) || !std::isfinite(scale))
    return fail_status(PQKV_ERR_INVALID, "attn_weights: scale must be > 0");
  if (causal && (int64_t)q_start + Sq > S)
    return fail_status(PQKV_ERR_INVALID, "attn_weights: causal queries at %d..%lld are not all in the cache (S=%d)",
                       q_start, (long long)q_start + Sq - 1, S);
  const int c = check_weights("attn_weights", in, in_stride, out, out_stride, B, Hkv, S);
  if (c != PQKV_OK || S == 0) return c;
  hipStream_t st = (hipStream_t)stream;
  const int64_t streams = (int64_t)B * Hkv;
  if (!weights_shape_ok(B, Hq, Hkv, Sq > 0 ? Sq : 1, S, d))
    return fail_status(PQKV_ERR_UNSUPPORTED, "attn_weights: B=%d Hq=%d Hkv=%d Sq=%d S=%d", B, Hq, Hkv, Sq, S);
  if (Sq == 0) {
    if (in == out) return PQKV_OK;
    return report_hip_error(pqkv::launch_weights_copy(in, in_stride, out, out_stride, streams, S, st),
                            "attn_weights copy");
  }
  if (!q || !R || !codebook || (pg ? !pg->k_pages : !k_cache))
    return fail_status(PQKV_ERR_INVALID, "attn_weights: null pointer");
  if ((uintptr_t)R % 16 || (uintptr_t)p_rot % 16)
    return fail_status(PQKV_ERR_INVALID, "attn_weights: R and p_rot must be 16-byte aligned");
  WeightsPlan p = weights_plan(B, Hq, Hkv, Sq, S, d, has_qjl);
  for (int shrink = 1; shrink <= kMaxShrink && ws_bytes < p.bytes(); ++shrink)
    p = weights_plan(B, Hq, Hkv, Sq, S, d, has_qjl, shrink);
  if (!ws || ws_bytes < p.bytes())
    return fail_status(PQKV_ERR_WORKSPACE, "attn_weights: workspace %zu < %zu bytes", ws_bytes, p.bytes());
  if ((uintptr_t)ws % 16) return fail_status(PQKV_ERR_INVALID, "attn_weights: workspace must be 16-byte aligned");
  char *w = (char *)ws;
  auto take = [&](size_t bytes) {
    char *at = w;
    w += bytes;
    return at;
  };
  float *q32 = (float *)take(p.q), *pq32 = (float *)take(p.pq);
  const int64_t nvec = (int64_t)B * Hq * Sq;
  const float qs = scale * 1.4426950408889634f;
  // the queries are rotated on their way into the rows' records, or before
  // where projections need them rotated too
  if (has_qjl) {
    const int t = pqkv::prof_begin("weights_rotate", st);
    const hipError_t r = pqkv::launch_rotate2(q, q_dtype, R, p_rot, q32, pq32, nvec, d, qs, 1.0f / (float)m, st);
    pqkv::prof_end(t, st);
    if (r != hipSuccess) return report_hip_error(r, "attn_weights query rotation");
  }
  pqkv::AttnWeightsArgs a;
  memset(&a, 0, sizeof(a));
  a.q = has_qjl ? q32 : nullptr;
  a.pq = has_qjl ? pq32 : nullptr;
  a.x = q;
  a.x_dtype = q_dtype;
  a.R = R;
  a.q_scale = qs;
  a.k_cache = k_cache;
  a.qjl = qjl;
  if (pg) {
    a.k_pages = pg->k_pages;
    a.s_pages = pg->s_pages;
    a.page_shift = pg->page_shift;
    a.max_pages = pg->max_pages;
  }
  a.codebook = codebook;
  a.bits = n_bits;
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.Sq = Sq;
  a.q_start = q_start;
  a.S = S;
  a.S_max = S_max;
  a.d = d;
  a.causal = causal ? 1 : 0;
  a.tblocks = p.tblocks;
  a.tokens = p.tokens;
  a.chunk_rows = p.chunk_rows;
  a.records = (uint8_t *)take(p.records);
  a.row_factor = (float *)take(p.factor);
  a.part = (float2 *)take(p.part);
  a.stat = (float2 *)take(p.stat);
  a.col = (float *)take(p.col);
  a.out = out;
  a.out_stride = out_stride;
  const int total = Sq * a.G;
  for (int row0 = 0; row0 < total; row0 += p.rows) {
    a.row0 = row0;
    a.rows = std::min(p.rows, total - row0);
    a.row_tiles = row_tiles(a.rows);
    a.chunks = p.chunks(a.rows);
    a.in = row0 ? out : in;
    a.in_stride = row0 ? out_stride : in_stride;
    const int tok = pqkv::prof_begin("attn_weights", st);
    const hipError_t e = pqkv::launch_attn_weights(a, st);
    pqkv::prof_end(tok, st);
    if (e != hipSuccess) return report_hip_error(e, "attn_weights launch");
  }
  return PQKV_OK;
}

int rotary_run(const char *what, const void *q, const int64_t q_strides[3], void *q_out, int Hq, const void *k,
               const int64_t k_strides[3], void *k_out, int Hkv, int dtype, const int64_t *positions,
               int64_t positions_stride, const double *freqs, int B, int T, int d, int rot_dim, int interleaved,
               float amplitude, int inverse, void *stream, const pqkv::RotaryAxes *axes) {
  if (B < 0 || T < 0 || Hq < 0 || Hkv < 0)
    return fail_status(PQKV_ERR_INVALID, "%s: B=%d T=%d Hq=%d Hkv=%d", what, B, T, Hq, Hkv);
  if (d < 2 || d > 1024 || rot_dim < 2 || rot_dim > d || rot_dim % 2)
    return fail_status(PQKV_ERR_UNSUPPORTED, "%s: rot_dim=%d of d=%d", what, rot_dim, d);
  if (dtype != PQKV_F32 && dtype != PQKV_F16 && dtype != PQKV_BF16)
    return fail_status(PQKV_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  if (!std::isfinite(amplitude)) return fail_status(PQKV_ERR_INVALID, "%s: amplitude must be finite", what);
  if (B == 0 || T == 0 || (Hq == 0 && Hkv == 0)) return PQKV_OK;
  if ((Hq && (!q || !q_out || !q_strides)) || (Hkv && (!k || !k_out || !k_strides)) || !positions || !freqs)
    return fail_status(PQKV_ERR_INVALID, "%s: null pointer", what);
  const uintptr_t size = dtype == PQKV_F32 ? 4 : 2;
  if ((Hq && ((uintptr_t)q | (uintptr_t)q_out) % size) || (Hkv && ((uintptr_t)k | (uintptr_t)k_out) % size) ||
      (uintptr_t)positions % 8 || (uintptr_t)freqs % 8)
    return fail_status(PQKV_ERR_INVALID, "%s: unaligned pointer", what);
  if (positions_stride < 0) return fail_status(PQKV_ERR_INVALID, "%s: positions_stride < 0", what);
  if ((int64_t)B * T > kMaxGrid || (int64_t)Hq + Hkv > 65535)
    return fail_status(PQKV_ERR_UNSUPPORTED, "%s: B=%d T=%d heads=%lld", what, B, T, (long long)Hq + Hkv);
  pqkv::RotaryArgs a;
  memset(&a, 0, sizeof(a));
  if (Hq) {
    a.q = q;
    a.q_out = q_out;
    std::copy(q_strides, q_strides + 3, a.q_stride);
  }
  if (Hkv) {
    a.k = k;
    a.k_out = k_out;
    std::copy(k_strides, k_strides + 3, a.k_stride);
  }
  a.positions = positions;
  a.pos_batch_stride = positions_stride;
  a.freqs = freqs;
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.T = T;
  a.d = d;
  a.rot_dim = rot_dim;
  a.interleaved = interleaved ? 1 : 0;
  a.inverse = inverse ? 1 : 0;
  a.amplitude = amplitude;
  const int tok = pqkv::prof_begin("rotary", (hipStream_t)stream);
  const hipError_t e = axes ? pqkv::launch_rotary_axes(a, *axes, dtype, (hipStream_t)stream)
                            : pqkv::launch_rotary(a, dtype, (hipStream_t)stream);
  pqkv::prof_end(tok, (hipStream_t)stream);
  return report_hip_error(e, "rotary launch");
}

}  // namespace

namespace pqkv {

int rotary_axes(const char *what, const uint8_t *axes, int n_axes, int rot_dim, int64_t stride, RotaryAxes *out) {
  if (n_axes < 1 || n_axes > 256 || stride < 0 || !axes || rot_dim < 2 || rot_dim > 2 * kMaxRotaryPairs)
    return fail_status(PQKV_ERR_INVALID, "%s: n_axes=%d rot_dim=%d positions_axis_stride=%lld", what, n_axes, rot_dim,
                       (long long)stride);
  out->stride = stride;
  memset(out->of, 0, sizeof(out->of));
  for (int i = 0; i < rot_dim / 2; ++i) {
    if (axes[i] >= n_axes) return fail_status(PQKV_ERR_INVALID, "%s: pair %d has axis %d of %d", what, i, axes[i], n_axes);
    out->of[i] = axes[i];
  }
  return PQKV_OK;
}

}  // namespace pqkv

extern "C" {

size_t pqkv_decode_attn_weights_workspace_bytes(int B, int Hq, int Hkv, int S, int d) {
  const size_t base = pqkv_decode_workspace_bytes(B, Hq, Hkv, S, d);
  if (base == 0 || S <= 0) return base;
  return align256(base) + align256((size_t)B * Hq * logit_stride(S) * 4);
}

int pqkv_decode_attn_weights(const void *q, int q_dtype, const float *R, const uint8_t *k_cache,
                             const uint8_t *v_cache, const float *k_codebook, const float *v_codebook, int n_bits,
                             const uint8_t *qjl_signs, const float *p_rot, int m, int B, int Hq, int Hkv, int S,
                             int S_max, int d, float scale, void *out, int out_dtype, const float *weights_in,
                             int64_t weights_in_stride, float *weights_out, int64_t weights_out_stride,
                             void *workspace, size_t workspace_bytes, void *stream) {
  return decode_weights_run(q, q_dtype, R, k_cache, v_cache, k_codebook, v_codebook, n_bits, qjl_signs, p_rot, m, B,
                            Hq, Hkv, S, S_max, d, scale, out, out_dtype, weights_in, weights_in_stride, weights_out,
                            weights_out_stride, workspace, workspace_bytes, stream, nullptr);
}

int pqkv_decode_attn_weights_paged(const void *q, int q_dtype, const float *R, const uint8_t *const *k_pages,
                                   const uint8_t *const *v_pages, int page_tokens, int max_pages,
                                   const float *k_codebook, const float *v_codebook, int n_bits,
                                   const uint8_t *const *qjl_pages, const float *p_rot, int m, int B, int Hq, int Hkv,
                                   int S, int d, float scale, void *out, int out_dtype, const float *weights_in,
                                   int64_t weights_in_stride, float *weights_out, int64_t weights_out_stride,
                                   void *workspace, size_t workspace_bytes, void *stream) {
  const int shift = pqkv::paged_validate("decode_weights_paged", page_tokens, max_pages, S);
  if (shift < 0) return shift;
  const pqkv::PagedCache pg{k_pages, v_pages, qjl_pages, shift, max_pages};
  return decode_weights_run(q, q_dtype, R, nullptr, nullptr, k_codebook, v_codebook, n_bits, nullptr, p_rot, m, B, Hq,
                            Hkv, S, S, d, scale, out, out_dtype, weights_in, weights_in_stride, weights_out,
                            weights_out_stride, workspace, workspace_bytes, stream, &pg);
}

size_t pqkv_attn_weights_workspace_bytes(int B, int Hq, int Hkv, int Sq, int S, int d, int qjl) {
  if (!weights_shape_ok(B, Hq, Hkv, Sq, S, d)) return 0;
  return weights_plan(B, Hq, Hkv, Sq, S, d, qjl != 0).bytes();
}

size_t pqkv_attn_weights_workspace_least_bytes(int B, int Hq, int Hkv, int Sq, int S, int d, int qjl) {
  if (!weights_shape_ok(B, Hq, Hkv, Sq, S, d)) return 0;
  return weights_plan(B, Hq, Hkv, Sq, S, d, qjl != 0, kMaxShrink).bytes();
}

int pqkv_attn_weights(const void *q, int q_dtype, const float *R, const uint8_t *k_cache, const float *k_codebook,
                      int n_bits, const uint8_t *qjl_signs, const float *p_rot, int m, int B, int Hq, int Hkv, int Sq,
                      int q_start, int S, int S_max, int d, float scale, int causal, const float *weights_in,
                      int64_t weights_in_stride, float *weights_out, int64_t weights_out_stride, void *workspace,
                      size_t workspace_bytes, void *stream) {
  return attn_weights_run(q, q_dtype, R, k_cache, k_codebook, n_bits, qjl_signs, p_rot, m, B, Hq, Hkv, Sq, q_start, S,
                          S_max, d, scale, causal, weights_in, weights_in_stride, weights_out, weights_out_stride,
                          workspace, workspace_bytes, stream, nullptr);
}

int pqkv_attn_weights_paged(const void *q, int q_dtype, const float *R, const uint8_t *const *k_pages,
                            int page_tokens, int max_pages, const float *k_codebook, int n_bits,
                            const uint8_t *const *qjl_pages, const float *p_rot, int m, int B, int Hq, int Hkv,
                            int Sq, int q_start, int S, int d, float scale, int causal, const float *weights_in,
                            int64_t weights_in_stride, float *weights_out, int64_t weights_out_stride,
                            void *workspace, size_t workspace_bytes, void *stream) {
  const int shift = pqkv::paged_validate("attn_weights_paged", page_tokens, max_pages, S);
  if (shift < 0) return shift;
  const pqkv::PagedCache pg{k_pages, nullptr, qjl_pages, shift, max_pages};
  return attn_weights_run(q, q_dtype, R, nullptr, k_codebook, n_bits, nullptr, p_rot, m, B, Hq, Hkv, Sq, q_start, S, S,
                          d, scale, causal, weights_in, weights_in_stride, weights_out, weights_out_stride, workspace,
                          workspace_bytes, stream, &pg);
}

int pqkv_evict_select(const float *weights, int64_t weights_stride, int64_t n_streams, int S, int keep, int sink,
                      int recent, int32_t *kept, void *stream) {
  if (n_streams < 0 || n_streams > kMaxGrid || S < 0 || S > INT_MAX - 2048 || sink < 0 || recent < 0)
    return fail_status(PQKV_ERR_INVALID, "evict_select: n_streams=%lld S=%d sink=%d recent=%d", (long long)n_streams,
                       S, sink, recent);
  if (keep < std::min<int64_t>(S, (int64_t)sink + recent) || keep > S)
    return fail_status(PQKV_ERR_INVALID, "evict_select: keep=%d of S=%d positions with sink=%d recent=%d", keep, S, sink,
                       recent);
  if (n_streams == 0 || keep == 0) return PQKV_OK;
  if (!weights || !kept) return fail_status(PQKV_ERR_INVALID, "evict_select: null pointer");
  if ((uintptr_t)weights % 4 || (uintptr_t)kept % 4)
    return fail_status(PQKV_ERR_INVALID, "evict_select: unaligned pointer");
  if (weights_stride < S) return fail_status(PQKV_ERR_INVALID, "evict_select: weights_stride below S=%d", S);
  const int tok = pqkv::prof_begin("evict_select", (hipStream_t)stream);
  const hipError_t e = pqkv::launch_evict_select(weights, weights_stride, n_streams, S, keep, std::min(sink, S),
                                                 std::min(recent, S), kept, (hipStream_t)stream);
  pqkv::prof_end(tok, (hipStream_t)stream);
  return report_hip_error(e, "evict_select launch");
}

int pqkv_gather_rows(int n_arrays, const pqkv_row_array *src, const pqkv_row_array *dst, const int *row_bytes,
                     const int32_t *kept, int64_t n_streams, int S, int keep, int fill, void *stream) {
  if (n_arrays < 0 || n_arrays > PQKV_MAX_GATHER || n_streams < 0 || S < 0 || keep < 0 || fill < keep)
    return fail_status(PQKV_ERR_INVALID, "gather_rows: n_arrays=%d n_streams=%lld S=%d keep=%d fill=%d", n_arrays,
                       (long long)n_streams, S, keep, fill);
  if (n_arrays == 0 || n_streams == 0 || fill == 0) return PQKV_OK;
  if (!src || !dst || !row_bytes || (keep > 0 && !kept))
    return fail_status(PQKV_ERR_INVALID, "gather_rows: null pointer");
  if (n_streams > kMaxGrid || n_streams * (((int64_t)fill + 63) / 64) > kMaxGrid)
    return fail_status(PQKV_ERR_UNSUPPORTED, "gather_rows: n_streams=%lld fill=%d", (long long)n_streams, fill);
  pqkv::GatherArgs a;
  memset(&a, 0, sizeof(a));
  for (int i = 0; i < n_arrays; ++i) {
    pqkv::GatherPart &p = a.part[i];
    const int rb = row_bytes[i];
    if (rb <= 0 || rb % 4 || rb > 65536)
      return fail_status(PQKV_ERR_UNSUPPORTED, "gather_rows: row_bytes[%d]=%d", i, rb);
    uintptr_t align = (uintptr_t)rb;
    for (const pqkv_row_array *r : {&src[i], &dst[i]}) {
      const bool is_src = r == &src[i];
      const int64_t rows = is_src ? S : fill;
      if (r->pages) {
        const int shift = pqkv::paged_validate("gather_rows", r->page_tokens, r->max_pages, rows);
        if (shift < 0) return shift;
        (is_src ? p.src_shift : p.dst_shift) = shift;
        (is_src ? p.src_max_pages : p.dst_max_pages) = r->max_pages;
        if (is_src || !r->base) continue;
        if ((uintptr_t)r->base % 16 || r->stride % 16 || ((int64_t)r->page_tokens * rb) % 16)
          return fail_status(PQKV_ERR_INVALID, "gather_rows: pages of array %d are not 16-byte aligned", i);
      } else if (!r->base && rows > 0) {
        return fail_status(PQKV_ERR_INVALID, "gather_rows: null array %d", i);
      }
      if (((uintptr_t)r->base | (uintptr_t)r->stride) % 4)
        return fail_status(PQKV_ERR_INVALID, "gather_rows: array %d is not 4-byte aligned", i);
      const int64_t held = is_src ? S : r->pages ? (rows + r->page_tokens - 1) / r->page_tokens * r->page_tokens : keep;
      if (r->stride < held * rb)
        return fail_status(PQKV_ERR_INVALID, "gather_rows: array %d: stride %lld below its rows", i,
                           (long long)r->stride);
      align |= (uintptr_t)r->base | (uintptr_t)r->stride;
    }
    const bool table = dst[i].pages && dst[i].base;
    p.src = (const uint8_t *)src[i].base;
    p.src_pages = src[i].pages;
    p.src_stride = src[i].stride;
    p.dst = (uint8_t *)const_cast<void *>(dst[i].base);
    p.dst_pages = table ? nullptr : (uint8_t *const *)dst[i].pages;
    p.dst_table = table ? (uint8_t **)dst[i].pages : nullptr;
    p.dst_stride = dst[i].stride;
    p.row_bytes = rb;
    p.unit = align % 8 == 0 ? 8 : 4;
  }
  a.n_parts = n_arrays;
  a.kept = kept;
  a.S = S;
  a.keep = keep;
  a.fill = fill;
  const int tok = pqkv::prof_begin("gather_rows", (hipStream_t)stream);
  const hipError_t e = pqkv::launch_gather_rows(a, n_streams, (hipStream_t)stream);
  pqkv::prof_end(tok, (hipStream_t)stream);
  return report_hip_error(e, "gather_rows launch");
}

int pqkv_rotary(const void *q, const int64_t q_strides[3], void *q_out, int Hq, const void *k,
                const int64_t k_strides[3], void *k_out, int Hkv, int dtype, const int64_t *positions,
                int64_t positions_stride, const double *freqs, int B, int T, int d, int rot_dim, int interleaved,
                float amplitude, int inverse, void *stream) {
  return rotary_run("rotary", q, q_strides, q_out, Hq, k, k_strides, k_out, Hkv, dtype, positions, positions_stride,
                    freqs, B, T, d, rot_dim, interleaved, amplitude, inverse, stream, nullptr);
}

int pqkv_rotary_axes(const void *q, const int64_t q_strides[3], void *q_out, int Hq, const void *k,
                     const int64_t k_strides[3], void *k_out, int Hkv, int dtype, const int64_t *positions,
                     int64_t positions_axis_stride, int64_t positions_stride, int n_axes, const uint8_t *axes,
                     const double *freqs, int B, int T, int d, int rot_dim, int interleaved, float amplitude,
                     int inverse, void *stream) {
  pqkv::RotaryAxes ax;
  const int c = pqkv::rotary_axes("rotary_axes", axes, n_axes, rot_dim, positions_axis_stride, &ax);
  if (c != PQKV_OK) return c;
  return rotary_run("rotary_axes", q, q_strides, q_out, Hq, k, k_strides, k_out, Hkv, dtype, positions,
                    positions_stride, freqs, B, T, d, rot_dim, interleaved, amplitude, inverse, stream, &ax);
}

}  // extern "C"
