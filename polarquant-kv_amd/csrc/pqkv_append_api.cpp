// C ABI of appending with the rotation on the way, and of reading slots back. Host code: validation and
// launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>

#include "../../include/pqkv.h"
#include "pqkv_launch.h"

using pqkv::fail_status;
using pqkv::report_hip_error;

namespace {

struct AppendPages {
  uint8_t *const *k, *const *v, *const *s;
  int page_shift, max_pages;
};

int append_run(const char *what, const void *k, const int64_t k_strides[3], const void *v, const int64_t v_strides[3],
               const void *q, const int64_t q_strides[3], void *q_out, int Hq, int dtype, const int64_t *positions,
               int64_t axis_stride, int64_t pos_stride, int n_axes, const uint8_t *axes, const double *freqs,
               int rot_dim, int interleaved, float amplitude, const float *R, const float *k_cb, const float *v_cb,
               int n_bits, const float *p_rot, int m, int B, int Hkv, int T, int d, int64_t start,
               const int64_t *starts, const int64_t *counts, int S, uint8_t *k_blocks, uint8_t *v_blocks,
               uint8_t *signs, const AppendPages *pg, void *stream) {
  if (B < 0 || Hkv < 0 || T < 0 || Hq < 0 || S < 0)
    return fail_status(PQKV_ERR_INVALID, "%s: B=%d Hkv=%d T=%d Hq=%d S=%d", what, B, Hkv, T, Hq, S);
  if (d != 64 && d != 128) return fail_status(PQKV_ERR_UNSUPPORTED, "%s: d=%d", what, d);
  if (rot_dim < 2 || rot_dim > d || rot_dim % 2)
    return fail_status(PQKV_ERR_UNSUPPORTED, "%s: rot_dim=%d of d=%d", what, rot_dim, d);
  if (dtype != PQKV_F32 && dtype != PQKV_F16 && dtype != PQKV_BF16)
    return fail_status(PQKV_ERR_UNSUPPORTED, "%s: dtype %d", what, dtype);
  if (n_bits != 2 && n_bits != 4) return fail_status(PQKV_ERR_UNSUPPORTED, "%s: n_bits=%d", what, n_bits);
  if (!std::isfinite(amplitude)) return fail_status(PQKV_ERR_INVALID, "%s: amplitude must be finite", what);
  const bool qjl = signs != nullptr || (pg && pg->s != nullptr);
  if (qjl != (p_rot != nullptr)) return fail_status(PQKV_ERR_INVALID, "%s: qjl and p_rot go together", what);
  if (qjl && m != d) return fail_status(PQKV_ERR_UNSUPPORTED, "%s: QJL needs m == d", what);
  if (!starts && (start < 0 || start > S || T > S - start))
    return fail_status(PQKV_ERR_INVALID, "%s: %d slots from %lld on, of %d", what, T, (long long)start, S);
  pqkv::RotaryAxes ax;
  const uint8_t one[pqkv::kMaxRotaryPairs] = {};
  const int c = pqkv::rotary_axes(what, axes ? axes : one, axes ? n_axes : 1, rot_dim, axes ? axis_stride : 0, &ax);
  if (c != PQKV_OK) return c;
  if (pos_stride < 0) return fail_status(PQKV_ERR_INVALID, "%s: positions_stride < 0", what);
  if (B == 0 || T == 0) return PQKV_OK;
  if (!positions || !freqs || (Hq && (!q || !q_strides || !q_out)))
    return fail_status(PQKV_ERR_INVALID, "%s: null pointer", what);
  // rows of (sequence, token), tiles of (row, head) and the slots' numbers within 31 bits
  if ((int64_t)B * T > INT_MAX / 32 || (int64_t)B * Hkv > INT_MAX || (int64_t)Hq > 65535)
    return fail_status(PQKV_ERR_UNSUPPORTED, "%s: B=%d T=%d Hkv=%d Hq=%d", what, B, T, Hkv, Hq);
  const uintptr_t size = dtype == PQKV_F32 ? 4 : 2;
  if ((uintptr_t)positions % 8 || (uintptr_t)freqs % 8 || (uintptr_t)starts % 8 || (uintptr_t)counts % 8 ||
      (Hkv && ((uintptr_t)k | (uintptr_t)v) % size) || (Hq && ((uintptr_t)q | (uintptr_t)q_out) % size))
    return fail_status(PQKV_ERR_INVALID, "%s: unaligned pointer", what);
  hipStream_t st = (hipStream_t)stream;
  // (a cache without a slot: there is nothing to write, and no page to find)
  if (Hkv && S > 0) {
    if (!k || !v || !k_strides || !v_strides || !R || !k_cb || !v_cb)
      return fail_status(PQKV_ERR_INVALID, "%s: null pointer", what);
    if (pg ? (!pg->k || !pg->v) : (!k_blocks || !v_blocks))
      return fail_status(PQKV_ERR_INVALID, "%s: null cache", what);
    if (((uintptr_t)k_blocks | (uintptr_t)v_blocks) % 2 || (uintptr_t)signs % 4 || (uintptr_t)R % 4 ||
        (uintptr_t)p_rot % 4)
      return fail_status(PQKV_ERR_INVALID, "%s: unaligned cache or matrix", what);
    pqkv::AppendArgs a;
    memset(&a, 0, sizeof(a));
    a.k = k;
    a.v = v;
    std::copy(k_strides, k_strides + 3, a.k_stride);
    std::copy(v_strides, v_strides + 3, a.v_stride);
    a.positions = positions;
    a.pos_batch_stride = pos_stride;
    a.freqs = freqs;
    a.R = R;
    a.k_cb = k_cb;
    a.v_cb = v_cb;
    a.p_rot = p_rot;
    a.k_blocks = k_blocks;
    a.v_blocks = v_blocks;
    a.signs = signs;
    if (pg) {
      a.k_pages = pg->k;
      a.v_pages = pg->v;
      a.s_pages = pg->s;
      a.page_shift = pg->page_shift;
      a.max_pages = pg->max_pages;
    }
    a.starts = starts;
    a.counts = counts;
    a.start = start;
    a.B = B;
    a.Hkv = Hkv;
    a.T = T;
    a.d = d;
    a.S = S;
    a.rot_dim = rot_dim;
    a.interleaved = interleaved ? 1 : 0;
    a.bits = n_bits;
    a.vec_bytes = (int)pqkv_vector_bytes(d, n_bits);
    a.amplitude = amplitude;
    a.axes = ax;
    const int tok = pqkv::prof_begin("append", st);
    const hipError_t e = pqkv::launch_append(a, dtype, st);
    pqkv::prof_end(tok, st);
    if (e != hipSuccess) return report_hip_error(e, "append launch");
  }
  if (!Hq) return PQKV_OK;
  return axes ? pqkv_rotary_axes(q, q_strides, q_out, Hq, nullptr, nullptr, nullptr, 0, dtype, positions, axis_stride,
                                 pos_stride, n_axes, axes, freqs, B, T, d, rot_dim, interleaved, amplitude, 0, stream)
              : pqkv_rotary(q, q_strides, q_out, Hq, nullptr, nullptr, nullptr, 0, dtype, positions, pos_stride, freqs,
                            B, T, d, rot_dim, interleaved, amplitude, 0, stream);
}

}  // namespace

extern "C" {

int pqkv_dequantize_slots(const uint8_t *blocks, int64_t stride, const uint8_t *const *pages, int page_tokens,
                          int max_pages, const float *codebook, int n_bits, void *out, int out_dtype,
                          int64_t n_streams, int S, int d, void *stream) {
  if (n_streams < 0 || S < 0) return fail_status(PQKV_ERR_INVALID, "dequantize_slots: n_streams=%lld S=%d", (long long)n_streams, S);
  if (d != 64 && d != 128) return fail_status(PQKV_ERR_UNSUPPORTED, "dequantize_slots: d=%d", d);
  if (n_bits != 2 && n_bits != 4) return fail_status(PQKV_ERR_UNSUPPORTED, "dequantize_slots: n_bits=%d", n_bits);
  if (out_dtype != PQKV_F32 && out_dtype != PQKV_F16) return fail_status(PQKV_ERR_UNSUPPORTED, "dequantize_slots: dtype");
  int shift = 0;
  if (pages) {
    shift = pqkv::paged_validate("dequantize_slots", page_tokens, max_pages, S);
    if (shift < 0) return shift;
  }
  if (n_streams == 0 || S == 0) return PQKV_OK;
  if ((!blocks && !pages) || !codebook || !out) return fail_status(PQKV_ERR_INVALID, "dequantize_slots: null pointer");
  if ((uintptr_t)blocks % 2 || (!pages && stride % 2) || (uintptr_t)out % 16)
    return fail_status(PQKV_ERR_INVALID, "dequantize_slots: unaligned pointer");
  if (!pages && stride < S * pqkv_vector_bytes(d, n_bits))
    return fail_status(PQKV_ERR_INVALID, "dequantize_slots: stride %lld below a stream's bytes", (long long)stride);
  if (n_streams > 0xFFFFFFFFll / S) return fail_status(PQKV_ERR_UNSUPPORTED, "dequantize_slots: n_streams=%lld S=%d", (long long)n_streams, S);
  const pqkv::SlotsArgs a{blocks, stride, pages, shift, max_pages, codebook, out, n_streams * S, S};
  const int tok = pqkv::prof_begin("dequantize_slots", (hipStream_t)stream);
  const hipError_t e = pqkv::launch_slots(a, d, n_bits, out_dtype, (hipStream_t)stream);
  pqkv::prof_end(tok, (hipStream_t)stream);
  return report_hip_error(e, "dequantize_slots launch");
}

int pqkv_append_rotary(const void *k, const int64_t k_strides[3], const void *v, const int64_t v_strides[3],
                       const void *q, const int64_t q_strides[3], void *q_out, int Hq, int dtype,
                       const int64_t *positions, int64_t positions_axis_stride, int64_t positions_stride, int n_axes,
                       const uint8_t *axes, const double *freqs, int rot_dim, int interleaved, float amplitude,
                       const float *R, const float *k_codebook, const float *v_codebook, int n_bits,
                       const float *p_rot, int m, int B, int Hkv, int T, int d, int64_t start, const int64_t *starts,
                       const int64_t *counts, int S, uint8_t *k_blocks, uint8_t *v_blocks, uint8_t *qjl_signs,
                       void *stream) {
  return append_run("append_rotary", k, k_strides, v, v_strides, q, q_strides, q_out, Hq, dtype, positions,
                    positions_axis_stride, positions_stride, n_axes, axes, freqs, rot_dim, interleaved, amplitude, R,
                    k_codebook, v_codebook, n_bits, p_rot, m, B, Hkv, T, d, start, starts, counts, S, k_blocks,
                    v_blocks, qjl_signs, nullptr, stream);
}

int pqkv_append_rotary_paged(const void *k, const int64_t k_strides[3], const void *v, const int64_t v_strides[3],
                             const void *q, const int64_t q_strides[3], void *q_out, int Hq, int dtype,
                             const int64_t *positions, int64_t positions_axis_stride, int64_t positions_stride,
                             int n_axes, const uint8_t *axes, const double *freqs, int rot_dim, int interleaved,
                             float amplitude, const float *R, const float *k_codebook, const float *v_codebook,
                             int n_bits, const float *p_rot, int m, int B, int Hkv, int T, int d, int64_t start,
                             const int64_t *starts, const int64_t *counts, int S, uint8_t *const *k_pages,
                             uint8_t *const *v_pages, int page_tokens, int max_pages, uint8_t *const *qjl_pages,
                             void *stream) {
  const int shift = pqkv::paged_validate("append_rotary_paged", page_tokens, max_pages, S);
  if (shift < 0) return shift;
  const AppendPages pg{k_pages, v_pages, qjl_pages, shift, max_pages};
  return append_run("append_rotary_paged", k, k_strides, v, v_strides, q, q_strides, q_out, Hq, dtype, positions,
                    positions_axis_stride, positions_stride, n_axes, axes, freqs, rot_dim, interleaved, amplitude, R,
                    k_codebook, v_codebook, n_bits, p_rot, m, B, Hkv, T, d, start, starts, counts, S, nullptr, nullptr,
                    nullptr, &pg, stream);
}

}  // extern "C"
