// C ABI of attention behind a window. Host code: validation, workspace layouts
// and launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "../../include/pqkv.h"
#include "pqkv_launch.h"

using pqkv::fail_status;
using pqkv::report_hip_error;

namespace {

constexpr int kMaxTokens = 1 << 24;      // as for weights: positions times bytes within 31 bits
constexpr float kLog2e = 1.4426950408889634f;

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

pqkv::Window window_of(int64_t start, const int64_t *starts, const int64_t *counts, int Sq, int window, int sinks,
                       int S) {
  pqkv::Window w{};
  w.starts = starts;
  w.counts = counts;
  w.start = start;
  w.count = Sq;
  // (a window or sinks of more than the cache are those of the cache: sums of
  // positions and sizes stay within 31 bits)
  w.size = std::min(window, std::max(S, 1));
  w.sinks = std::min(sinks, S);
  return w;
}

// One split has nothing to join: its rows are normalised and rotated back on the fp32
// matrix cores. Single launches between two events (which are most of the smallest), us, against
// the merge kernel's: d = 128 6.8 and 6.6 for 256 rows, 6.8 and 7.0 for 512, 7.0 and 8.0 for
// 1024, 7.2 and 11.9 for 2048, 7.1 and 19.5 for 4096; d = 64 within 0.1 up to 768, 6.1 and
// 6.4 for 1024, 6.0 and 6.5 for 2048, 6.2 and 8.4 for 4096.
constexpr int64_t kMergeMfmaRows = 512;

// One row per sequence: the splits of a stream's tiles, as many as the decode
// kernel takes for as many tokens.
int row_splits(int B, int Hkv, int S, const pqkv::Window &w) {
  const int all = (S + 63) / 64;
  const int tiles = std::min((w.size + 126) / 64 + (w.sinks + 63) / 64, all);
  int splits = 1, tps = 0;
  pqkv::mfma_split_plan((int64_t)B * Hkv, std::max(tiles, 1) * 64, &splits, &tps);
  return splits;
}

bool window_shape_ok(int B, int Hq, int Hkv, int Sq, int S, int d, bool qjl) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq <= 0 || S < 0 || Hq % Hkv || (d != 64 && d != 128)) return false;
  if (S >= kMaxTokens || (int64_t)B * Hkv > 65535 || (int64_t)B * Hq * Sq > ((int64_t)1 << 40) / d) return false;
  if (Sq == 1) return true;
  const int rows = pqkv::prefill_rows_per_block(qjl);
  if (Hq / Hkv > rows) return false;
  const int qt = rows / (Hq / Hkv);
  // (a padded chunk's positions and row numbers within 31 bits)
  return Sq < kMaxTokens && (int64_t)((Sq - 1) / qt + 1) * B * Hkv * 64 < 0x7fffffff;
}

int window_run(const char *what, const void *q, int q_dtype, const float *R, const uint8_t *k_cache,
               const uint8_t *v_cache, const float *k_cb, const float *v_cb, int n_bits, const uint8_t *qjl_signs,
               const float *p_rot, int m, int B, int Hq, int Hkv, int Sq, int64_t start, const int64_t *starts,
               const int64_t *counts, int window, int sinks, int S, int d, float scale, void *out, int out_dtype,
               void *ws, size_t ws_bytes, void *stream, const pqkv::PagedCache *pg) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || Sq < 0 || S < 0 || window < 1 || sinks < 0)
    return fail_status(PQKV_ERR_INVALID, "%s: B=%d Hq=%d Hkv=%d Sq=%d S=%d window=%d sinks=%d", what, B, Hq, Hkv, Sq, S,
                       window, sinks);
  if (Hq % Hkv) return fail_status(PQKV_ERR_INVALID, "%s: Hq=%d not a multiple of Hkv=%d", what, Hq, Hkv);
  if (d != 64 && d != 128) return fail_status(PQKV_ERR_UNSUPPORTED, "%s: d=%d", what, d);
  if (n_bits != 2 && n_bits != 4) return fail_status(PQKV_ERR_UNSUPPORTED, "%s: n_bits=%d", what, n_bits);
  if ((q_dtype != PQKV_F32 && q_dtype != PQKV_F16) || (out_dtype != PQKV_F32 && out_dtype != PQKV_F16))
    return fail_status(PQKV_ERR_UNSUPPORTED, "%s: dtype", what);
  const bool qjl = qjl_signs != nullptr || (pg && pg->s_pages != nullptr);
  if (qjl != (p_rot != nullptr)) return fail_status(PQKV_ERR_INVALID, "%s: qjl and p_rot go together", what);
  if (qjl && m != d) return fail_status(PQKV_ERR_UNSUPPORTED, "%s: QJL needs m == d", what);
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail_status(PQKV_ERR_INVALID, "%s: scale must be > 0", what);
  if (!starts && (start < 0 || start > S || Sq > S - start))
    return fail_status(PQKV_ERR_INVALID, "%s: %d rows from %lld on are not all in the cache (S=%d)", what, Sq,
                       (long long)start, S);
  if (Sq == 0) return PQKV_OK;
  if (!window_shape_ok(B, Hq, Hkv, Sq, S, d, qjl))
    return fail_status(PQKV_ERR_UNSUPPORTED, "%s: B=%d Hq=%d Hkv=%d Sq=%d S=%d", what, B, Hq, Hkv, Sq, S);
  if (!q || !R || !out) return fail_status(PQKV_ERR_INVALID, "%s: null pointer", what);
  if ((uintptr_t)R % 16 || (uintptr_t)p_rot % 16)
    return fail_status(PQKV_ERR_INVALID, "%s: R and p_rot must be 16-byte aligned", what);
  if ((uintptr_t)starts % 8 || (uintptr_t)counts % 8)
    return fail_status(PQKV_ERR_INVALID, "%s: unaligned starts or counts", what);
  hipStream_t st = (hipStream_t)stream;
  const int64_t nvec = (int64_t)B * Hq * Sq;
  if (S == 0)
    return report_hip_error(pqkv::launch_fill_zero(out, (size_t)nvec * d * (out_dtype == PQKV_F32 ? 4 : 2), st),
                            "window zero fill");
  if ((pg ? (!pg->k_pages || !pg->v_pages) : (!k_cache || !v_cache)) || !k_cb || !v_cb)
    return fail_status(PQKV_ERR_INVALID, "%s: null cache or codebook", what);
  const size_t need = pqkv_window_attn_workspace_bytes(B, Hq, Hkv, Sq, S, d, window, sinks, qjl);
  if (!ws || ws_bytes < need)
    return fail_status(PQKV_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", what, ws_bytes, need);
  if ((uintptr_t)ws % 16) return fail_status(PQKV_ERR_INVALID, "%s: workspace must be 16-byte aligned", what);
  const pqkv::Window w = window_of(start, starts, counts, Sq, window, sinks, S);
  const int64_t vb = pqkv_vector_bytes(d, n_bits);
  char *base = (char *)ws;
  auto rotate = [&](const char *name, float *q32, float *pq32, float qs, float ps) {
    const int t = pqkv::prof_begin(name, st);
    const hipError_t e = qjl ? pqkv::launch_rotate2(q, q_dtype, R, p_rot, q32, pq32, nvec, d, qs, ps, st)
                             : pqkv::launch_rotate(q, q_dtype, R, q32, PQKV_F32, nvec, d, 0, qs, st);
    pqkv::prof_end(t, st);
    return e;
  };
  if (Sq == 1) {
    const int splits = row_splits(B, Hkv, S, w);
    size_t q_off, part_off, pq_off;
    pqkv::decode_workspace_layout(B, Hq, splits, d, &q_off, &part_off, &pq_off);
    pqkv::DecodeArgs a;
    memset(&a, 0, sizeof(a));
    a.q = (float *)(base + q_off);
    a.pq = qjl ? (float *)(base + pq_off) : nullptr;
    a.part = (float *)(base + part_off);
    hipError_t e = rotate("window_rotate", (float *)(base + q_off), (float *)(base + pq_off), scale * kLog2e,
                          1.0f / (float)m);
    if (e != hipSuccess) return report_hip_error(e, "window query rotation");
    a.k_cache = k_cache;
    a.v_cache = v_cache;
    a.k_cb = k_cb;
    a.v_cb = v_cb;
    a.cb_levels = 16;
    a.qjl = qjl_signs;
    if (pg) {
      a.k_pages = pg->k_pages;
      a.v_pages = pg->v_pages;
      a.s_pages = pg->s_pages;
      a.page_shift = pg->page_shift;
      a.max_pages = pg->max_pages;
    }
    a.B = B;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.gq = Hq / Hkv;
    a.S = a.S_max = S;
    a.d = d;
    a.splits = a.split_stride = splits;
    a.n_heads = Hkv;
    a.k_head_stride = a.v_head_stride = S * vb;
    a.k_batch_stride = a.v_batch_stride = a.k_head_stride * Hkv;
    a.win = w;
    // a group's heads in launches of at most kMaxGroup, equal parts where it divides
    const int n_sub = (a.gq + pqkv::kMaxGroup - 1) / pqkv::kMaxGroup;
    for (int i = 0; i < n_sub; ++i) {
      a.g = a.gq / n_sub + (i < a.gq % n_sub ? 1 : 0);
      const int t = pqkv::prof_begin("window_split", st);
      e = pqkv::launch_decode_mfma_window(a, n_bits, st);
      pqkv::prof_end(t, st);
      if (e != hipSuccess) return report_hip_error(e, "window split launch");
      a.q_off += a.g;
    }
    const int t = pqkv::prof_begin("window_merge", st);
    e = splits == 1 && nvec >= kMergeMfmaRows
            ? pqkv::launch_rotate_part_mfma(a.part, R, out, out_dtype, nvec, d, st)
            : pqkv::launch_decode_merge(a.part, R, out, out_dtype, B * Hq, splits, d, st);
    pqkv::prof_end(t, st);
    return report_hip_error(e, "window merge launch");
  }
  const pqkv::PrefillPlan plan = pqkv::prefill_window_plan(B, Hq, Hkv, Sq, S, qjl, w);
  pqkv::PrefillArgs a;
  memset(&a, 0, sizeof(a));
  float *o32 = (float *)base;      // rotated outputs, where splits are joined
  a.x = q;
  a.x_f16 = q_dtype == PQKV_F16;
  a.out = out;
  a.out_f16 = out_dtype == PQKV_F16;
  a.R = R;
  a.p_rot = p_rot;
  a.q_scale = scale * kLog2e * pqkv::kPrefillPlaneScale;
  a.p_scale = 1.0f / ((float)m * pqkv::kPrefillPlaneScale);
  a.o = o32;
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.k_cb = k_cb;
  a.v_cb = v_cb;
  a.qjl = qjl_signs;
  a.k_head_stride = a.v_head_stride = S * vb;
  a.k_batch_stride = a.v_batch_stride = a.k_head_stride * Hkv;
  a.k_tok_stride = a.v_tok_stride = vb;
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.Sq = Sq;
  a.S = a.S_max = S;
  a.d = d;
  a.causal = 1;
  a.qt = plan.qt;
  a.qtiles = plan.qtiles;
  a.splits = plan.splits;
  a.n_heads = Hkv;
  a.part_o = (float *)(base + align256((size_t)nvec * d * 4));
  a.part_ml = a.part_o + plan.part_rows * d;
  if (pg) {
    a.k_pages = pg->k_pages;
    a.v_pages = pg->v_pages;
    a.s_pages = pg->s_pages;
    a.page_shift = pg->page_shift;
    a.max_pages = pg->max_pages;
  }
  a.win = w;
  int t = pqkv::prof_begin("window_attn", st);
  hipError_t e = pqkv::launch_prefill_window(a, n_bits, st);
  pqkv::prof_end(t, st);
  if (e != hipSuccess || plan.splits == 1) return report_hip_error(e, "window launch");
  t = pqkv::prof_begin("window_out_rotate", st);
  e = pqkv::launch_rotate(o32, PQKV_F32, R, out, out_dtype, nvec, d, 1, 1.0f, st);
  pqkv::prof_end(t, st);
  return report_hip_error(e, "window output rotation");
}

}  // namespace

extern "C" {

size_t pqkv_window_attn_workspace_bytes(int B, int Hq, int Hkv, int Sq, int S, int d, int window, int sinks, int qjl) {
  if (!window_shape_ok(B, Hq, Hkv, Sq, S, d, qjl != 0) || window < 1 || sinks < 0) return 0;
  const pqkv::Window w = window_of(0, nullptr, nullptr, Sq, window, sinks, S);
  if (Sq == 1) return pqkv::decode_workspace_layout(B, Hq, row_splits(B, Hkv, S, w), d, nullptr, nullptr, nullptr);
  // (the outputs of one split are final; 256 bytes, so that 0 means a shape that no call takes)
  const pqkv::PrefillPlan p = pqkv::prefill_window_plan(B, Hq, Hkv, Sq, S, qjl != 0, w);
  return p.splits == 1 ? 256 : align256((size_t)B * Hq * Sq * d * 4) + p.part_bytes(d);
}

int pqkv_window_attn(const void *q, int q_dtype, const float *R, const uint8_t *k_cache, const uint8_t *v_cache,
                     const float *k_codebook, const float *v_codebook, int n_bits, const uint8_t *qjl_signs,
                     const float *p_rot, int m, int B, int Hq, int Hkv, int Sq, int64_t start, const int64_t *starts,
                     const int64_t *counts, int window, int sinks, int S, int d, float scale, void *out,
                     int out_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  return window_run("window_attn", q, q_dtype, R, k_cache, v_cache, k_codebook, v_codebook, n_bits, qjl_signs, p_rot,
                    m, B, Hq, Hkv, Sq, start, starts, counts, window, sinks, S, d, scale, out, out_dtype, workspace,
                    workspace_bytes, stream, nullptr);
}

int pqkv_window_attn_paged(const void *q, int q_dtype, const float *R, const uint8_t *const *k_pages,
                           const uint8_t *const *v_pages, int page_tokens, int max_pages, const float *k_codebook,
                           const float *v_codebook, int n_bits, const uint8_t *const *qjl_pages, const float *p_rot,
                           int m, int B, int Hq, int Hkv, int Sq, int64_t start, const int64_t *starts,
                           const int64_t *counts, int window, int sinks, int S, int d, float scale, void *out,
                           int out_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  const int shift = pqkv::paged_validate("window_attn_paged", page_tokens, max_pages, S);
  if (shift < 0) return shift;
  const pqkv::PagedCache pg{k_pages, v_pages, qjl_pages, shift, max_pages};
  return window_run("window_attn_paged", q, q_dtype, R, nullptr, nullptr, k_codebook, v_codebook, n_bits, nullptr,
                    p_rot, m, B, Hq, Hkv, Sq, start, starts, counts, window, sinks, S, d, scale, out, out_dtype,
                    workspace, workspace_bytes, stream, &pg);
}

}  // extern "C"
