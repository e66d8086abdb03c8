// api.hip - the extern "C" entry points declared in include/ttcd.h:
// argument validation (before any HIP call, so every error path is
// testable without a GPU), status/error reporting, and the host replay of
// the attention schedule used by the coverage tests.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>
#include <mutex>

#include "internal.h"
#include "kv4_sweep.h"
#include "schedule.h"
#include "ttcd.h"

namespace {

thread_local char g_err[512] = "";

ttcd_status fail(ttcd_status st, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return st;
}

ttcd_status ok() {
  g_err[0] = '\0';
  return TTCD_OK;
}

ttcd_status from_hip(hipError_t e, const char* what) {
  if (e == hipSuccess) return ok();
  return fail(TTCD_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Largest K/V token stride (elements) the tile loads' 32-bit lane offsets reach.
constexpr int64_t kMaxTokenStride = int64_t(1) << 25;

// Checks shared by both attention entry points.
ttcd_status check_attn(const void* q, const void* k, const void* v, const void* o, int B, int T,
                       int Hq, int Hkv, int D, const int64_t* qs, const int64_t* ks,
                       const int64_t* vs, const int64_t* os, ttcd_dtype dtype) {
  if (!q || !k || !v || !o) return fail(TTCD_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!qs || !ks || !vs || !os) return fail(TTCD_ERR_INVALID_ARGUMENT, "null stride array");
  if (B < 1 || T < 1 || Hq < 1 || Hkv < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "B, T, Hq, Hkv must be >= 1 (got %d, %d, %d, %d)", B,
                T, Hq, Hkv);
  if (Hq % Hkv != 0)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "Hq (%d) must be a multiple of Hkv (%d)", Hq, Hkv);
  if (D != 64 && D != 128)
    return fail(TTCD_ERR_UNSUPPORTED, "head_dim %d not supported (64 or 128)", D);
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "attention dtype must be bf16 or f16");
  if (qs[3] != 1 || ks[3] != 1 || vs[3] != 1 || os[3] != 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "head_dim must be contiguous (d-stride 1)");
  const int64_t* all[4] = {qs, ks, vs, os};
  for (int t = 0; t < 4; ++t)
    for (int i = 0; i < 3; ++i)
      if (all[t][i] % 8 != 0 || all[t][i] < 0)
        return fail(TTCD_ERR_UNSUPPORTED,
                    "strides must be non-negative multiples of 8 elements (16-byte rows)");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o))
    return fail(TTCD_ERR_UNSUPPORTED, "tensor base pointers must be 16-byte aligned");
  // The K/V tile loads address a lane's chunk with a 32-bit byte offset from the
  // tile's first key: 63 token strides of 2-byte elements plus one row must fit.
  if (ks[1] > kMaxTokenStride || vs[1] > kMaxTokenStride)
    return fail(TTCD_ERR_UNSUPPORTED, "k/v token stride above %lld elements",
                (long long)kMaxTokenStride);
  const int64_t nqb = (T + ttcd::kBlockM - 1) / ttcd::kBlockM;
  if ((int64_t)B * Hq * nqb > 0x7fffffffLL)  // bound on workgroups for either geometry
    return fail(TTCD_ERR_UNSUPPORTED, "grid too large");
  return TTCD_OK;
}

// The lazy-rescale threshold: finite, 0 (exact running max) .. 16. Every
// probability p = exp2(s*c - m*c) stays <= 2^rescale_log2 and is rounded to
// the input dtype before PV: bf16 holds any such p, but f16 rounds values
// >= 65520 to +inf, so F16 is limited to 15 (p <= 32768).
ttcd_status check_rescale(float rescale_log2, ttcd_dtype dtype) {
  const float hi = dtype == TTCD_DTYPE_F16 ? 15.f : 16.f;
  if (!(rescale_log2 >= 0.f && rescale_log2 <= hi))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "rescale_log2 must be in [0, %g] for this dtype (got %g)",
                (double)hi, (double)rescale_log2);
  return TTCD_OK;
}

ttcd::AttnArgs fill_args(const void* q, const void* k, const void* v, int B, int T, int Hq,
                         int Hkv, const int64_t* qs, const int64_t* ks, const int64_t* vs,
                         const int64_t* os, float sm_scale) {
  ttcd::AttnArgs a = {};
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_sb = qs[0];
  a.q_st = qs[1];
  a.q_sh = qs[2];
  a.k_sb = ks[0];
  a.k_st = ks[1];
  a.k_sh = ks[2];
  a.v_sb = vs[0];
  a.v_st = vs[1];
  a.v_sh = vs[2];
  a.o_sb = os[0];
  a.o_st = os[1];
  a.o_sh = os[2];
  a.B = B;
  a.T = T;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  const int span = ttcd::wg_span_tokens(a.G);
  a.q_off = 0;
  a.qb0 = 0;
  a.nqb = (T + span - 1) / span;  // query blocks per (b, slice)
  a.c = sm_scale * 1.4426950408889634f;
  return a;
}

ttcd::Elem elem(ttcd_dtype d) {
  return d == TTCD_DTYPE_BF16 ? ttcd::Elem::BF16
                              : (d == TTCD_DTYPE_F16 ? ttcd::Elem::F16 : ttcd::Elem::F32);
}

}  // namespace

extern "C" {

const char* ttcd_status_string(ttcd_status status) {
  switch (status) {
    case TTCD_OK: return "TTCD_OK";
    case TTCD_ERR_INVALID_ARGUMENT: return "TTCD_ERR_INVALID_ARGUMENT";
    case TTCD_ERR_UNSUPPORTED: return "TTCD_ERR_UNSUPPORTED";
    case TTCD_ERR_HIP: return "TTCD_ERR_HIP";
  }
  return "TTCD_ERR_UNKNOWN";
}

const char* ttcd_last_error(void) { return g_err; }

int ttcd_abi_version(void) { return TTCD_ABI_VERSION; }

// Tq query rows at absolute positions Tk - Tq .. Tk - 1 against Tk keys
// (flash-attention's bottom-right aligned causal mask); q / o are (B, Tq, ...),
// k / v (B, Tk, ...), lse (B, Hq, Tq).
static ttcd_status set_rows(ttcd::AttnArgs* a, int Tq, int Tk) {
  if (Tq < 1 || Tq > Tk)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need 1 <= Tq <= Tk (got Tq=%d, Tk=%d)", Tq, Tk);
  const int span = ttcd::wg_span_tokens(a->G);
  a->q_off = Tk - Tq;
  a->qb0 = a->q_off / span;
  a->nqb = (Tk + span - 1) / span - a->qb0;
  a->lse_sh = Tq;
  a->lse_sb = (int64_t)a->Hq * Tq;
  return TTCD_OK;
}

// ---------------------------------------------------------------------------
// Splitting a call over keys. A cached prefill of few query rows launches few
// workgroups, each sweeping thousands of keys one tile after the other while
// most CUs idle. The band of distances is then cut into parts, each swept by a
// workgroup of its own into fp32 partials in the caller's workspace, which
// one more launch adds up through their LSEs.
namespace {

struct SplitPlan {
  int near_parts = 0, far_parts = 0;  // 0: not split
  int near_step = 0, far_step = 0;
  int parts() const { return near_parts + far_parts; }
};

constexpr size_t kSplitMaxBytes = size_t(64) << 20;

size_t split_part_bytes(int B, int Tq, int Hq, int D) {
  return (size_t)B * Tq * Hq * (D + 1) * sizeof(float);
}

// Parts of the band [lo, hi), cut at mid (mid == hi: one band; else the near
// parts end there). The rule is a model of the call's time in us, its rates
// fitted to an MI355X: a slot takes `alone` with its CU to itself and `busy`
// of the CU's time when it shares it, a launch 8 to start and end, the sum 3
// and its traffic at 5 TB/s. A split has to promise 18 %: the model is up to that
// far off where the CUs hold two or three workgroups. Of 2000 split calls drawn from 1
// to 14000 queries on 100 to 32000 cached keys, 8 sets of heads and windows of 6000
// to full, the geometric mean took 0.31 of its unsplit time and none
// more than 1.08 of it. Not split: calls whose queries are the whole sequence, the
// exact running max, which is the reference kernel's own order of accumulation,
// and sweeps of up to 72 tiles (windows of up to about 4500 keys). The last is no
// matter of speed: rows of such calls keep the bits that the whole prompt's call
// gives them (tests/test_kv_attn_gpu.py). Longer sweeps give that up, unless the
// caller passes no workspace (split_keys=False in Python).
//
// Measured (us, whole -> split, on a full window of cached keys). Window 8192,
// 16/8 heads of 128: 1 query 123 -> 24, 64 127 -> 30, 300 128 -> 42, 600
// 128 -> 63, 1000 129 -> 86, 2048 183 -> 167; 15/5 heads of 64: 1 query
// 95 -> 20, 500 98 -> 42, 1000 99 -> 60, 2048 106 -> 90. Not split by this rule:
// 11186 queries on 16383 keys, 4/4 heads of 128, full causal (513; in two parts
// 600). What the line at 72 tiles leaves, 16/8 heads of 128: window 4096, 1 query
// 66 -> 18, 300 69 -> 33; 2048 35 -> 16 and 39 -> 27; 1024 20 -> 13 and 24 -> 23; 15/5
// heads of 64, window 4096: 51 -> 17 and 53 -> 31.
SplitPlan split_plan(int B, int Tq, int Tk, int Hq, int Hkv, int D, int lo, int mid, int hi,
                     float rescale_log2) {
  SplitPlan none, best;
  if (Tq >= Tk || rescale_log2 <= 0.f) return none;
  hi = hi < Tk ? hi : Tk;
  mid = mid < hi ? mid : hi;
  if (lo >= hi) return none;
  const int G = Hq / Hkv, rows = ttcd::wave_rows(G), span = ttcd::wg_span_tokens(G);
  const int sweep = (hi - lo + span - 1) / ttcd::kBlockN + 1;
  if (sweep <= 72) return none;
  const int64_t blocks = (Tk + span - 1) / span - (Tk - Tq) / span;
  const int64_t nwg = (int64_t)B * Hkv * (G / (ttcd::kWaveRows / rows)) * blocks;
  const double alone = D == 128 ? 0.95 : 0.70, busy = D == 128 ? 0.80 : 0.45;
  const int cus = ttcd::kXcd * ttcd::kXcdCus, places = D == 128 ? 2 : 3;
  // keys that the rows lack at their sequence's start, on average
  const double first = Tk - Tq + 1, last = hi - 1;  // histories shorter than hi
  const double missing =
      first > last ? 0.0 : (last - first + 1) * (hi - 0.5 * (first + last)) / Tq;
  const double mean = sweep - (missing < hi - lo ? missing : hi - lo) / ttcd::kBlockN;
  // parts of at most `step` of the band's distances
  auto model = [&](int parts, int step) {
    const double n = (double)((nwg * parts + cus - 1) / cus), ends = parts > 1 ? 1.5 : 0.0;
    const double longest = sweep * ((double)step / (hi - lo)) + ends;
    // A workgroup that waits for a place is one of the long ones; parts much longer
    // than the mean meet on a CU by chance.
    const double each = (n > places && parts > 1 ? sweep : mean) / parts + ends;
    const double chance = parts > 1 && longest > 1.5 * each ? longest - 1.5 * each : 0.0;
    const double work = n * busy * (each + chance);
    double t = 8.0 + (alone * longest > work ? alone * longest : work);
    if (parts > 1) t += 3.0 + 2.0 * parts * split_part_bytes(B, Tq, Hq, D) / 5e6;
    return t;
  };
  double least = 0.82 * model(1, hi - lo);
  for (int p = 2; p <= 16 && sweep / p >= 4; ++p) {
    if (p * split_part_bytes(B, Tq, Hq, D) > kSplitMaxBytes) break;
    SplitPlan sp;
    auto cut = [&](int width, int parts, int* n, int* step) {
      *step = ((width + parts - 1) / parts + ttcd::kBlockN - 1) / ttcd::kBlockN * ttcd::kBlockN;
      *n = (width + *step - 1) / *step;
    };
    const int far = hi - mid;
    int near_p = far > 0 ? (int)((int64_t)p * (mid - lo) / (hi - lo)) : p;
    near_p = near_p < 1 ? 1 : near_p;
    cut(mid - lo, near_p, &sp.near_parts, &sp.near_step);
    if (far > 0) cut(far, p - near_p > 1 ? p - near_p : 1, &sp.far_parts, &sp.far_step);
    const int step = sp.near_step > sp.far_step ? sp.near_step : sp.far_step;
    const double t = model(sp.parts(), step < hi - lo ? step : hi - lo);
    if (t >= least) continue;
    least = t;
    best = sp;
  }
  return best;
}

// Launch the split form of a (whose o_t, o_s, lse_t, lse_s and strides are the
// call's) in `ws`.
ttcd_status run_split(ttcd::AttnArgs a, const SplitPlan& sp, int Tq, int D, int lo, int mid,
                      int hi, ttcd_dtype dtype, void* ws, void* stream) {
  const int64_t rows = (int64_t)a.B * Tq * a.Hq;
  ttcd::CombineArgs c = {};
  c.part = static_cast<const float*>(ws);
  c.part_lse = c.part + rows * D * sp.parts();
  c.o = a.o_t;
  c.o_near = a.o_s;
  c.lse = a.lse_t;
  c.lse_near = a.lse_s;
  c.B = a.B;
  c.T = Tq;
  c.H = a.Hq;
  c.D = D;
  c.parts = sp.parts();
  c.near_parts = sp.near_parts;
  c.sb = a.o_sb;
  c.st = a.o_st;
  c.sh = a.o_sh;
  a.o_t = ws;
  a.o_s = nullptr;
  a.lse_t = const_cast<float*>(c.part_lse);
  a.lse_s = nullptr;
  a.o_sh = D;
  a.o_st = (int64_t)a.Hq * D;
  a.o_sb = (int64_t)Tq * a.o_st;
  a.o_sp = rows * D;
  a.lse_sp = rows;
  a.parts = sp.parts();
  a.near_parts = sp.near_parts;
  a.near_step = sp.near_step;
  a.far_step = sp.far_step;
  hi = hi < a.T ? hi : a.T;
  mid = mid < hi ? mid : hi;
  a.near = {lo, mid};
  a.far = {mid, hi};
  a.sched = ttcd::make_band_schedule(a.T, lo, hi, ttcd::wave_rows(a.G));
  hipStream_t hs = static_cast<hipStream_t>(stream);
  ttcd_status st = from_hip(ttcd::launch_attn(a, D, elem(dtype), hs), "split attention launch");
  if (st != TTCD_OK) return st;
  return from_hip(ttcd::launch_attn_combine(c, elem(dtype), hs), "attention combine launch");
}

bool split_fits(const SplitPlan& sp, const void* ws, size_t bytes, int B, int Tq, int Hq, int D) {
  return sp.parts() > 1 && ws != nullptr && (reinterpret_cast<uintptr_t>(ws) & 15u) == 0 &&
         bytes >= sp.parts() * split_part_bytes(B, Tq, Hq, D);
}

}  // namespace

size_t ttcd_attn_kv_workspace_bytes(int B, int Tq, int Tk, int Hq, int Hkv, int D, int band_lo,
                                    int band_mid, int band_hi, float rescale_log2) {
  if (B < 1 || Tq < 1 || Tq > Tk || Hkv < 1 || Hq < Hkv || Hq % Hkv != 0 ||
      (D != 64 && D != 128) || band_lo < 0)
    return 0;
  if (band_hi < 0) band_hi = Tk;
  if (band_mid < 0) band_mid = band_hi;
  if (band_mid <= band_lo || band_mid > band_hi) return 0;
  const SplitPlan sp =
      split_plan(B, Tq, Tk, Hq, Hkv, D, band_lo, band_mid, band_hi, rescale_log2);
  return sp.parts() > 1 ? sp.parts() * split_part_bytes(B, Tq, Hq, D) : 0;
}

ttcd_status ttcd_dual_window_attn_kv_ws_fwd(
    const void* q, const void* k, const void* v, void* o_t, void* o_s, float* lse_t, float* lse_s,
    int B, int Tq, int Tk, int Hq, int Hkv, int D, const int64_t q_stride[4],
    const int64_t k_stride[4], const int64_t v_stride[4], const int64_t o_stride[4], int window_t,
    int window_s, float sm_scale, float rescale_log2, ttcd_dtype dtype, void* workspace,
    size_t workspace_bytes, void* stream) {
  ttcd_status st =
      check_attn(q, k, v, o_t, B, Tk, Hq, Hkv, D, q_stride, k_stride, v_stride, o_stride, dtype);
  if (st == TTCD_OK) st = check_rescale(rescale_log2, dtype);
  if (st != TTCD_OK) return st;
  if (!o_s) return fail(TTCD_ERR_INVALID_ARGUMENT, "null student output pointer");
  if (!aligned16(o_s)) return fail(TTCD_ERR_UNSUPPORTED, "o_s must be 16-byte aligned");
  if (window_t < 0) window_t = Tk;
  if (window_s < 1) return fail(TTCD_ERR_INVALID_ARGUMENT, "window_s must be >= 1 (got %d)", window_s);
  if (window_s > window_t)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "window_s (%d) must be <= window_t (%d)", window_s,
                window_t);
  if (!(sm_scale > 0.f) || !isfinite(sm_scale))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "sm_scale must be finite and > 0");
  ttcd::AttnArgs a = fill_args(q, k, v, B, Tk, Hq, Hkv, q_stride, k_stride, v_stride, o_stride,
                               sm_scale);
  st = set_rows(&a, Tq, Tk);
  if (st != TTCD_OK) return st;
  a.o_t = o_t;
  a.o_s = o_s;
  a.lse_t = lse_t;
  a.lse_s = lse_s;
  a.rescale_log2 = rescale_log2;
  if (workspace_bytes > 0) {
    const SplitPlan sp =
        split_plan(B, Tq, Tk, Hq, Hkv, D, 0, window_s, window_t, rescale_log2);
    if (split_fits(sp, workspace, workspace_bytes, B, Tq, Hq, D))
      return run_split(a, sp, Tq, D, 0, window_s, window_t, dtype, workspace, stream);
  }
  a.sched = ttcd::make_dual_schedule(Tk, window_s, window_t, ttcd::wave_rows(a.G));
  return from_hip(ttcd::launch_attn(a, D, elem(dtype), static_cast<hipStream_t>(stream)),
                  "dual-window attention launch");
}

ttcd_status ttcd_dual_window_attn_kv_fwd(const void* q, const void* k, const void* v, void* o_t,
                                         void* o_s, float* lse_t, float* lse_s, int B, int Tq,
                                         int Tk, int Hq, int Hkv, int D,
                                         const int64_t q_stride[4], const int64_t k_stride[4],
                                         const int64_t v_stride[4], const int64_t o_stride[4],
                                         int window_t, int window_s, float sm_scale,
                                         float rescale_log2, ttcd_dtype dtype, void* stream) {
  return ttcd_dual_window_attn_kv_ws_fwd(q, k, v, o_t, o_s, lse_t, lse_s, B, Tq, Tk, Hq, Hkv, D,
                                         q_stride, k_stride, v_stride, o_stride, window_t,
                                         window_s, sm_scale, rescale_log2, dtype, nullptr, 0,
                                         stream);
}

ttcd_status ttcd_dual_window_attn_fwd(const void* q, const void* k, const void* v, void* o_t,
                                      void* o_s, float* lse_t, float* lse_s, int B, int T,
                                      int Hq, int Hkv, int D, const int64_t q_stride[4],
                                      const int64_t k_stride[4], const int64_t v_stride[4],
                                      const int64_t o_stride[4], int window_t, int window_s,
                                      float sm_scale, ttcd_dtype dtype, void* stream) {
  return ttcd_dual_window_attn_kv_fwd(q, k, v, o_t, o_s, lse_t, lse_s, B, T, T, Hq, Hkv, D,
                                      q_stride, k_stride, v_stride, o_stride, window_t, window_s,
                                      sm_scale, ttcd::kDefaultRescaleLog2, dtype, stream);
}

ttcd_status ttcd_band_attn_kv_ws_fwd(const void* q, const void* k, const void* v, void* o,
                                     float* lse, int B, int Tq, int Tk, int Hq, int Hkv, int D,
                                     const int64_t q_stride[4], const int64_t k_stride[4],
                                     const int64_t v_stride[4], const int64_t o_stride[4],
                                     int band_lo, int band_hi, float sm_scale,
                                     float rescale_log2, ttcd_dtype dtype, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  ttcd_status st =
      check_attn(q, k, v, o, B, Tk, Hq, Hkv, D, q_stride, k_stride, v_stride, o_stride, dtype);
  if (st == TTCD_OK) st = check_rescale(rescale_log2, dtype);
  if (st != TTCD_OK) return st;
  if (band_lo < 0 || band_hi <= band_lo)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need 0 <= band_lo < band_hi (got %d, %d)", band_lo,
                band_hi);
  if (!(sm_scale > 0.f) || !isfinite(sm_scale))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "sm_scale must be finite and > 0");
  ttcd::AttnArgs a = fill_args(q, k, v, B, Tk, Hq, Hkv, q_stride, k_stride, v_stride, o_stride,
                               sm_scale);
  st = set_rows(&a, Tq, Tk);
  if (st != TTCD_OK) return st;
  a.o_t = o;
  a.lse_t = lse;
  a.rescale_log2 = rescale_log2;
  if (workspace_bytes > 0) {
    const SplitPlan sp =
        split_plan(B, Tq, Tk, Hq, Hkv, D, band_lo, band_hi, band_hi, rescale_log2);
    if (split_fits(sp, workspace, workspace_bytes, B, Tq, Hq, D))
      return run_split(a, sp, Tq, D, band_lo, band_hi, band_hi, dtype, workspace, stream);
  }
  a.sched = ttcd::make_band_schedule(Tk, band_lo, band_hi, ttcd::wave_rows(a.G));
  return from_hip(ttcd::launch_attn(a, D, elem(dtype), static_cast<hipStream_t>(stream)),
                  "band attention launch");
}

ttcd_status ttcd_band_attn_kv_fwd(const void* q, const void* k, const void* v, void* o,
                                  float* lse, int B, int Tq, int Tk, int Hq, int Hkv, int D,
                                  const int64_t q_stride[4], const int64_t k_stride[4],
                                  const int64_t v_stride[4], const int64_t o_stride[4],
                                  int band_lo, int band_hi, float sm_scale, float rescale_log2,
                                  ttcd_dtype dtype, void* stream) {
  return ttcd_band_attn_kv_ws_fwd(q, k, v, o, lse, B, Tq, Tk, Hq, Hkv, D, q_stride, k_stride,
                                  v_stride, o_stride, band_lo, band_hi, sm_scale, rescale_log2,
                                  dtype, nullptr, 0, stream);
}

ttcd_status ttcd_band_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse,
                               int B, int T, int Hq, int Hkv, int D, const int64_t q_stride[4],
                               const int64_t k_stride[4], const int64_t v_stride[4],
                               const int64_t o_stride[4], int band_lo, int band_hi,
                               float sm_scale, ttcd_dtype dtype, void* stream) {
  return ttcd_band_attn_kv_fwd(q, k, v, o, lse, B, T, T, Hq, Hkv, D, q_stride, k_stride,
                               v_stride, o_stride, band_lo, band_hi, sm_scale,
                               ttcd::kDefaultRescaleLog2, dtype, stream);
}

// Packed sequences (flash-attention's varlen layout): q / o are (total, Hq, D),
// k / v (total, Hkv, D), LSEs (Hq, total); sequence b is rows
// cu_seqlens[b] .. cu_seqlens[b+1]-1. The kernel reads cu_seqlens on the
// device (no host sync) and clamps every sequence to [0, total) and to
// max_seqlen rows, so malformed offsets cannot move an access out of the
// tensors; rows outside every sequence are not written.
static ttcd_status varlen_args(ttcd::AttnArgs* a, const void* q, const void* k, const void* v,
                               const void* o, const int32_t* cu_seqlens, int nseq,
                               int max_seqlen, int total, int Hq, int Hkv, int D,
                               const int64_t* qs3, const int64_t* ks3, const int64_t* vs3,
                               const int64_t* os3, float sm_scale, float rescale_log2,
                               ttcd_dtype dtype) {
  if (!cu_seqlens) return fail(TTCD_ERR_INVALID_ARGUMENT, "null cu_seqlens");
  if (check_rescale(rescale_log2, dtype) != TTCD_OK) return TTCD_ERR_INVALID_ARGUMENT;
  if (!qs3 || !ks3 || !vs3 || !os3) return fail(TTCD_ERR_INVALID_ARGUMENT, "null stride array");
  if (nseq < 1 || max_seqlen < 1 || total < 0)
    return fail(TTCD_ERR_INVALID_ARGUMENT,
                "need nseq >= 1, max_seqlen >= 1, total >= 0 (got %d, %d, %d)", nseq, max_seqlen,
                total);
  if (!(sm_scale > 0.f) || !isfinite(sm_scale))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "sm_scale must be finite and > 0");
  const int64_t qs[4] = {0, qs3[0], qs3[1], qs3[2]}, ks[4] = {0, ks3[0], ks3[1], ks3[2]};
  const int64_t vs[4] = {0, vs3[0], vs3[1], vs3[2]}, os[4] = {0, os3[0], os3[1], os3[2]};
  ttcd_status st = check_attn(q, k, v, o, nseq, max_seqlen, Hq, Hkv, D, qs, ks, vs, os, dtype);
  if (st != TTCD_OK) return st;
  *a = fill_args(q, k, v, nseq, max_seqlen, Hq, Hkv, qs, ks, vs, os, sm_scale);
  a->cu_seqlens = cu_seqlens;
  a->total = total;
  a->lse_sb = 0;
  a->lse_sh = total;
  a->rescale_log2 = rescale_log2;
  return TTCD_OK;
}

ttcd_status ttcd_dual_window_attn_varlen_fwd(const void* q, const void* k, const void* v,
                                             void* o_t, void* o_s, float* lse_t, float* lse_s,
                                             const int32_t* cu_seqlens, int nseq, int max_seqlen,
                                             int total, int Hq, int Hkv, int D,
                                             const int64_t q_stride[3],
                                             const int64_t k_stride[3],
                                             const int64_t v_stride[3],
                                             const int64_t o_stride[3], int window_t,
                                             int window_s, float sm_scale, float rescale_log2,
                                             ttcd_dtype dtype, void* stream) {
  ttcd::AttnArgs a;
  ttcd_status st = varlen_args(&a, q, k, v, o_t, cu_seqlens, nseq, max_seqlen, total, Hq, Hkv,
                               D, q_stride, k_stride, v_stride, o_stride, sm_scale, rescale_log2,
                               dtype);
  if (st != TTCD_OK) return st;
  if (!o_s) return fail(TTCD_ERR_INVALID_ARGUMENT, "null student output pointer");
  if (!aligned16(o_s)) return fail(TTCD_ERR_UNSUPPORTED, "o_s must be 16-byte aligned");
  if (window_s < 1) return fail(TTCD_ERR_INVALID_ARGUMENT, "window_s must be >= 1 (got %d)", window_s);
  if (window_t >= 0 && window_s > window_t)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "window_s (%d) must be <= window_t (%d)", window_s,
                window_t);
  // full causal: a teacher window no sequence reaches (clamped to each length)
  if (window_t < 0) window_t = 0x3fffffff;
  a.o_t = o_t;
  a.o_s = o_s;
  a.lse_t = lse_t;
  a.lse_s = lse_s;
  a.win_a = window_s;
  a.win_b = window_t;
  a.sched = ttcd::make_dual_schedule(max_seqlen, window_s, window_t, ttcd::wave_rows(a.G));
  return from_hip(ttcd::launch_attn(a, D, elem(dtype), static_cast<hipStream_t>(stream)),
                  "varlen dual-window attention launch");
}

ttcd_status ttcd_band_attn_varlen_fwd(const void* q, const void* k, const void* v, void* o,
                                      float* lse, const int32_t* cu_seqlens, int nseq,
                                      int max_seqlen, int total, int Hq, int Hkv, int D,
                                      const int64_t q_stride[3], const int64_t k_stride[3],
                                      const int64_t v_stride[3], const int64_t o_stride[3],
                                      int band_lo, int band_hi, float sm_scale,
                                      float rescale_log2, ttcd_dtype dtype, void* stream) {
  ttcd::AttnArgs a;
  ttcd_status st = varlen_args(&a, q, k, v, o, cu_seqlens, nseq, max_seqlen, total, Hq, Hkv, D,
                               q_stride, k_stride, v_stride, o_stride, sm_scale, rescale_log2,
                               dtype);
  if (st != TTCD_OK) return st;
  if (band_lo < 0 || band_hi <= band_lo)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need 0 <= band_lo < band_hi (got %d, %d)", band_lo,
                band_hi);
  a.o_t = o;
  a.lse_t = lse;
  a.win_a = band_lo;
  a.win_b = band_hi;
  a.sched = ttcd::make_band_schedule(max_seqlen, band_lo, band_hi, ttcd::wave_rows(a.G));
  return from_hip(ttcd::launch_attn(a, D, elem(dtype), static_cast<hipStream_t>(stream)),
                  "varlen band attention launch");
}

ttcd_status ttcd_lse_merge_fwd(const void* o_s, const float* lse_s, const void* o_f,
                               const float* lse_f, void* o_t, int B, int T, int H, int D,
                               int row_start, const int64_t o_stride[4], ttcd_dtype dtype,
                               void* stream) {
  if (!o_s || !lse_s || !o_f || !lse_f || !o_t || !o_stride)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (B < 1 || T < 1 || H < 1 || D < 8)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "B, T, H must be >= 1 and D >= 8");
  if (D % 8 != 0) return fail(TTCD_ERR_UNSUPPORTED, "D must be a multiple of 8");
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "merge dtype must be bf16 or f16");
  if (o_stride[3] != 1) return fail(TTCD_ERR_INVALID_ARGUMENT, "D must be contiguous");
  for (int i = 0; i < 3; ++i)
    if (o_stride[i] % 8 != 0 || o_stride[i] < 0)
      return fail(TTCD_ERR_UNSUPPORTED, "strides must be non-negative multiples of 8");
  if (!aligned16(o_s) || !aligned16(o_f) || !aligned16(o_t))
    return fail(TTCD_ERR_UNSUPPORTED, "outputs must be 16-byte aligned");
  if (row_start < 0) return fail(TTCD_ERR_INVALID_ARGUMENT, "row_start must be >= 0");
  ttcd::MergeArgs m = {o_s, lse_s, o_f, lse_f, o_t, B, T, H, D, row_start,
                       o_stride[0], o_stride[1], o_stride[2],
                       o_stride[0], o_stride[1], o_stride[2]};
  return from_hip(ttcd::launch_lse_merge(m, elem(dtype), static_cast<hipStream_t>(stream)),
                  "lse merge launch");
}

// ---------------------------------------------------------------------------
// The LSE-combination variant as one call (lse_dual_window_attn_fa3_fast,
// profiling/lse_dual_attn.py:134-160, with the cached-prefill rows of the kv
// forms). Query rows whose absolute position is below window_s have an empty
// far band: they are one student call, copied to o_t. The other rows run in
// chunks that fit the scratch: per chunk a student call (o_s rows + lse_s),
// a far-band call (o_f + lse_f) and the merge into o_t. Each row's tiles,
// order and arithmetic depend only on its absolute position, so the result
// does not depend on the chunking.
namespace {

constexpr size_t kScratchAlign = 256;
size_t align_up(size_t x) { return (x + kScratchAlign - 1) & ~(kScratchAlign - 1); }

struct LseDual {
  const void *q, *k, *v;
  void *o_t, *o_s;
  int B, Tq, Tk, Hq, Hkv, D, WT, WS;
  const int64_t *qs, *ks, *vs, *os;
  float sm_scale, rescale_log2;
  ttcd_dtype dtype;
  int esize() const { return 2; }
  // first query row with a far band (absolute position >= WS)
  int n0() const {
    const int r = WS - (Tk - Tq);
    return r < 0 ? 0 : (r > Tq ? Tq : r);
  }
  // scratch of a chunk of `rows` rows: o_f (B, rows, Hq, D), lse_s and lse_f (B, Hq, rows)
  size_t chunk_bytes(int64_t rows) const {
    return align_up((size_t)B * rows * Hq * D * esize()) + 2 * align_up((size_t)B * Hq * rows * 4);
  }
  // most rows per chunk that `bytes` of scratch hold (a multiple of the
  // 128-row query block when at least one block fits); 0 if not even one row
  int64_t rows_fitting(size_t bytes) const {
    const int64_t need = Tq - n0();
    if (need <= 0) return 1;
    if (chunk_bytes(need) <= bytes) return need;
    const size_t per_row = (size_t)B * Hq * (D * esize() + 8);
    int64_t r = bytes > 3 * kScratchAlign ? (int64_t)((bytes - 3 * kScratchAlign) / per_row) : 0;
    while (r > 0 && chunk_bytes(r) > bytes) --r;
    if (r >= ttcd::kBlockM) r -= r % ttcd::kBlockM;
    return r;
  }
};

// Window and pointer checks of the LSE variant (the band calls check the rest).
ttcd_status check_lse_dual(LseDual* a, int window_t, int window_s) {
  if (!a->q || !a->k || !a->v || !a->o_t || !a->o_s)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!a->qs || !a->ks || !a->vs || !a->os)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null stride array");
  if (a->B < 1 || a->Tq < 1 || a->Tq > a->Tk || a->Hq < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need B >= 1, Hq >= 1, 1 <= Tq <= Tk (got %d, %d, %d, %d)",
                a->B, a->Hq, a->Tq, a->Tk);
  if (a->dtype != TTCD_DTYPE_BF16 && a->dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "attention dtype must be bf16 or f16");
  if (window_t < 0) window_t = a->Tk;
  if (window_s < 1) return fail(TTCD_ERR_INVALID_ARGUMENT, "window_s must be >= 1 (got %d)", window_s);
  // lse_dual_attn.py:20: the far band [WS, WT) must not be empty
  if (window_s >= window_t)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "window_s (%d) must be < window_t (%d)", window_s,
                window_t);
  if (!aligned16(a->o_t) || !aligned16(a->o_s))
    return fail(TTCD_ERR_UNSUPPORTED, "outputs must be 16-byte aligned");
  // everything the band calls check, before any HIP call
  ttcd_status st = check_attn(a->q, a->k, a->v, a->o_t, a->B, a->Tk, a->Hq, a->Hkv, a->D, a->qs,
                              a->ks, a->vs, a->os, a->dtype);
  if (st == TTCD_OK) st = check_rescale(a->rescale_log2, a->dtype);
  if (!(a->sm_scale > 0.f) || !isfinite(a->sm_scale))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "sm_scale must be finite and > 0");
  if (st != TTCD_OK) return st;
  a->WT = window_t;
  a->WS = window_s;
  return TTCD_OK;
}

// Run the variant with `ws_bytes` of device scratch at `ws` (256-byte aligned).
ttcd_status run_lse_dual(const LseDual& a, char* ws, size_t ws_bytes, void* stream) {
  const int qoff = a.Tk - a.Tq, n0 = a.n0();
  const int64_t rows = a.rows_fitting(ws_bytes);
  if (n0 < a.Tq && rows < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "scratch of %zu bytes holds no query row (need %zu)",
                ws_bytes, a.chunk_bytes(1));
  const size_t es = a.esize();
  const char* q = static_cast<const char*>(a.q);
  char* o_s = static_cast<char*>(a.o_s);
  char* o_t = static_cast<char*>(a.o_t);
  const ttcd::Elem et = elem(a.dtype);
  hipStream_t hs = static_cast<hipStream_t>(stream);
  ttcd_status st;
  if (n0 > 0) {
    // rows below WS: the student call alone; o_t = o_s
    st = ttcd_band_attn_kv_fwd(a.q, a.k, a.v, a.o_s, nullptr, a.B, n0, qoff + n0, a.Hq, a.Hkv,
                               a.D, a.qs, a.ks, a.vs, a.os, 0, a.WS, a.sm_scale, a.rescale_log2,
                               a.dtype, stream);
    if (st != TTCD_OK) return st;
    ttcd::MergeArgs m = {a.o_s, nullptr, a.o_s, nullptr, a.o_t, a.B, n0, a.Hq, a.D, n0,
                         a.os[0], a.os[1], a.os[2], a.os[0], a.os[1], a.os[2]};
    st = from_hip(ttcd::launch_lse_merge(m, et, hs), "lse variant copy launch");
    if (st != TTCD_OK) return st;
  }
  for (int64_t r0 = n0; r0 < a.Tq; r0 += rows) {
    const int r1 = (int)(r0 + rows < a.Tq ? r0 + rows : a.Tq);
    const int tc = r1 - (int)r0, tk = qoff + r1;
    char* o_f = ws;
    float* lse_s = reinterpret_cast<float*>(ws + align_up((size_t)a.B * tc * a.Hq * a.D * es));
    float* lse_f = reinterpret_cast<float*>(reinterpret_cast<char*>(lse_s) +
                                            align_up((size_t)a.B * a.Hq * tc * 4));
    const int64_t fs[4] = {(int64_t)tc * a.Hq * a.D, (int64_t)a.Hq * a.D, a.D, 1};
    const void* qc = q + (size_t)r0 * a.qs[1] * es;
    void* osc = o_s + (size_t)r0 * a.os[1] * es;
    st = ttcd_band_attn_kv_fwd(qc, a.k, a.v, osc, lse_s, a.B, tc, tk, a.Hq, a.Hkv, a.D, a.qs,
                               a.ks, a.vs, a.os, 0, a.WS, a.sm_scale, a.rescale_log2, a.dtype,
                               stream);
    if (st != TTCD_OK) return st;
    st = ttcd_band_attn_kv_fwd(qc, a.k, a.v, o_f, lse_f, a.B, tc, tk, a.Hq, a.Hkv, a.D, a.qs,
                               a.ks, a.vs, fs, a.WS, a.WT, a.sm_scale, a.rescale_log2, a.dtype,
                               stream);
    if (st != TTCD_OK) return st;
    ttcd::MergeArgs m = {osc, lse_s, o_f, lse_f, o_t + (size_t)r0 * a.os[1] * es, a.B, tc, a.Hq,
                         a.D, 0, a.os[0], a.os[1], a.os[2], fs[0], fs[1], fs[2]};
    st = from_hip(ttcd::launch_lse_merge(m, et, hs), "lse variant merge launch");
    if (st != TTCD_OK) return st;
  }
  return ok();
}

}  // namespace

size_t ttcd_lse_dual_window_attn_workspace_bytes(int B, int Tq, int Tk, int Hq, int D,
                                                 int window_s) {
  if (B < 1 || Tq < 1 || Tq > Tk || Hq < 1 || D < 1 || window_s < 1) return 0;
  LseDual a = {};
  a.B = B;
  a.Tq = Tq;
  a.Tk = Tk;
  a.Hq = Hq;
  a.D = D;
  a.WS = window_s;
  const int64_t need = Tq - a.n0();
  return need > 0 ? a.chunk_bytes(need) : 0;
}

ttcd_status ttcd_lse_dual_window_attn_fwd(const void* q, const void* k, const void* v,
                                          void* o_t, void* o_s, int B, int Tq, int Tk, int Hq,
                                          int Hkv, int D, const int64_t q_stride[4],
                                          const int64_t k_stride[4], const int64_t v_stride[4],
                                          const int64_t o_stride[4], int window_t, int window_s,
                                          float sm_scale, float rescale_log2, ttcd_dtype dtype,
                                          void* workspace, size_t workspace_bytes, void* stream) {
  LseDual a = {q, k, v, o_t, o_s, B, Tq, Tk, Hq, Hkv, D, 0, 0, q_stride, k_stride, v_stride,
               o_stride, sm_scale, rescale_log2, dtype};
  ttcd_status st = check_lse_dual(&a, window_t, window_s);
  if (st != TTCD_OK) return st;
  if (workspace_bytes > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "workspace must be non-null and 256-byte aligned");
  return run_lse_dual(a, static_cast<char*>(workspace), workspace_bytes, stream);
}

// ---------------------------------------------------------------------------
// Allocation-free LSE variant. Its scratch is a file-scope device array: one
// copy per GPU the library runs on, held until the process ends. On the host
// the array's name is only a stand-in, never a device address: the address
// is resolved once per device with hipGetSymbolAddress (that device current)
// and only that pointer is passed to kernels. Every call on one GPU shares the
// array; the variant writes each scratch element before reading it, so
// nothing needs clearing, but calls that overlap in time on one GPU (different
// streams without ordering) race on it.
namespace {
constexpr size_t kNoAllocScratchBytes = size_t(64) << 20;
}  // namespace
static __device__ __align__(256) unsigned char scratch[kNoAllocScratchBytes];

namespace {
constexpr int kMaxDevices = 64;
std::mutex g_scratch_mu;
void* g_scratch_ptr[kMaxDevices] = {};

// Device address of `scratch` on the device of `stream` (the current device
// for the null stream), resolved on first use there.
ttcd_status scratch_for(void* stream, char** out) {
  int cur = 0;
  hipError_t e = hipGetDevice(&cur);
  if (e != hipSuccess) return from_hip(e, "hipGetDevice");
  int dev = cur;
  if (stream != nullptr) {
    hipDevice_t d = 0;
    e = hipStreamGetDevice(static_cast<hipStream_t>(stream), &d);
    if (e != hipSuccess) return from_hip(e, "hipStreamGetDevice");
    dev = d;
  }
  if (dev < 0 || dev >= kMaxDevices)
    return fail(TTCD_ERR_UNSUPPORTED, "device %d beyond the %d the scratch table holds", dev,
                kMaxDevices);
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (g_scratch_ptr[dev] == nullptr) {
    if (dev != cur) {
      e = hipSetDevice(dev);
      if (e != hipSuccess) return from_hip(e, "hipSetDevice");
    }
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (dev != cur) {
      const hipError_t e2 = hipSetDevice(cur);
      if (e == hipSuccess && e2 != hipSuccess) e = e2;
    }
    if (e != hipSuccess) return from_hip(e, "hipGetSymbolAddress(scratch)");
    if (p == nullptr || (reinterpret_cast<uintptr_t>(p) & 255u) != 0)
      return fail(TTCD_ERR_HIP, "scratch symbol has no 256-byte aligned device address");
    g_scratch_ptr[dev] = p;
  }
  *out = static_cast<char*>(g_scratch_ptr[dev]);
  return TTCD_OK;
}
}  // namespace

size_t ttcd_lse_dual_window_attn_noalloc_scratch_bytes(void) { return kNoAllocScratchBytes; }

ttcd_status ttcd_lse_dual_window_attn_noalloc_fwd(
    const void* q, const void* k, const void* v, void* o_t, void* o_s, int B, int Tq, int Tk,
    int Hq, int Hkv, int D, const int64_t q_stride[4], const int64_t k_stride[4],
    const int64_t v_stride[4], const int64_t o_stride[4], int window_t, int window_s,
    float sm_scale, float rescale_log2, ttcd_dtype dtype, void* stream) {
  LseDual a = {q, k, v, o_t, o_s, B, Tq, Tk, Hq, Hkv, D, 0, 0, q_stride, k_stride, v_stride,
               o_stride, sm_scale, rescale_log2, dtype};
  ttcd_status st = check_lse_dual(&a, window_t, window_s);
  if (st != TTCD_OK) return st;
  if (a.n0() < a.Tq && a.rows_fitting(kNoAllocScratchBytes) < 1)
    return fail(TTCD_ERR_UNSUPPORTED,
                "B * Hq too large for the %zu-byte scratch: one query row needs %zu bytes",
                kNoAllocScratchBytes, a.chunk_bytes(1));
  char* ws = nullptr;
  st = scratch_for(stream, &ws);
  if (st != TTCD_OK) return st;
  return run_lse_dual(a, ws, kNoAllocScratchBytes, stream);
}

ttcd_status ttcd_causal_dwconv_chunked_fwd(const void* x, const void* w, void* y, int64_t N,
                                           int C, int D, int K, ttcd_dtype x_dtype,
                                           ttcd_dtype w_dtype, void* stream) {
  if (!x || !w || !y) return fail(TTCD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (N < 0 || C < 0 || D < 0) return fail(TTCD_ERR_INVALID_ARGUMENT, "negative extent");
  if (K < 1 || K > 64) return fail(TTCD_ERR_INVALID_ARGUMENT, "kernel size %d not in [1, 64]", K);
  if ((unsigned)x_dtype > TTCD_DTYPE_F32 || (unsigned)w_dtype > TTCD_DTYPE_F32)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "unknown dtype");
  if (N == 0 || C == 0 || D == 0) return ok();
  return from_hip(ttcd::launch_dwconv(x, w, y, N, C, D, K, elem(x_dtype), elem(w_dtype),
                                      static_cast<hipStream_t>(stream)),
                  "depthwise conv launch");
}

ttcd_status ttcd_rope_table_fwd(void* cos_table, void* sin_table, const float* inv_freq,
                                int rows, int half_dim, ttcd_dtype dtype, void* stream) {
  if (!cos_table || !sin_table || !inv_freq)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (rows < 0 || half_dim < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need rows >= 0 and half_dim >= 1 (got %d, %d)", rows,
                half_dim);
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "table dtype must be bf16 or f16");
  if (rows == 0) return ok();
  return from_hip(ttcd::launch_rope_table(cos_table, sin_table, inv_freq, rows, half_dim,
                                          elem(dtype), static_cast<hipStream_t>(stream)),
                  "rope table launch");
}

ttcd_status ttcd_rope_fwd(const void* q, const void* k, void* q_out, void* k_out,
                          const float* inv_freq, int num_freq, const void* positions,
                          int positions_64, const int64_t position_stride[2], int64_t offset,
                          int B, int T, int Hq, int Hkv, int D, const int64_t q_stride[4],
                          const int64_t k_stride[4], const int64_t q_out_stride[4],
                          const int64_t k_out_stride[4], int interleaved, int inverse,
                          float scale, ttcd_dtype dtype, void* stream) {
  if (!q || !q_out || !inv_freq) return fail(TTCD_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (Hkv < 0 || (Hkv > 0 && (!k || !k_out)))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null tensor pointer (k, Hkv = %d)", Hkv);
  if (!q_stride || !q_out_stride || (Hkv > 0 && (!k_stride || !k_out_stride)) ||
      (positions && !position_stride))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null stride array");
  if (B < 1 || T < 1 || Hq < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "B, T, Hq must be >= 1 (got %d, %d, %d)", B, T, Hq);
  if (D < 2 || D > 1024) return fail(TTCD_ERR_UNSUPPORTED, "head_dim %d not in 2 .. 1024", D);
  if (num_freq < 1 || 2 * (int64_t)num_freq > D)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need 1 <= num_freq <= head_dim / 2 (got %d of %d)",
                num_freq, D);
  if ((unsigned)dtype > TTCD_DTYPE_F32) return fail(TTCD_ERR_INVALID_ARGUMENT, "unknown dtype");
  if (!isfinite(scale)) return fail(TTCD_ERR_INVALID_ARGUMENT, "scale must be finite");
  constexpr int64_t kFar = int64_t(1) << 53;
  if (!positions && (offset < -kFar || offset > kFar - (T - 1)))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "offset %lld: positions must be within 2^53",
                (long long)offset);
  const int64_t heads = (int64_t)Hq + Hkv;
  if ((int64_t)B * T > 0x7fffffffLL || heads * D > (1 << 28))
    return fail(TTCD_ERR_UNSUPPORTED, "grid too large");
  const int64_t* all[4] = {q_stride, q_out_stride, Hkv > 0 ? k_stride : q_stride,
                           Hkv > 0 ? k_out_stride : q_out_stride};
  for (int t = 0; t < 4; ++t)
    if (all[t][3] != 1)
      return fail(TTCD_ERR_INVALID_ARGUMENT, "head_dim must be contiguous (d-stride 1)");
  ttcd::RopeArgs a = {};
  a.q = q;
  a.q_out = q_out;
  a.inv_freq = inv_freq;
  a.positions = positions;
  a.pos64 = positions_64 != 0;
  a.inverse = inverse != 0;
  if (positions) {
    a.pos_sb = position_stride[0];
    a.pos_st = position_stride[1];
  }
  a.offset = offset;
  a.scale = scale;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.D = D;
  a.n = num_freq;
  a.tokens = (int64_t)B * T;
  a.T = ttcd::make_fast_div(T);
  a.q_sb = q_stride[0];
  a.q_st = q_stride[1];
  a.q_sh = q_stride[2];
  a.qo_sb = q_out_stride[0];
  a.qo_st = q_out_stride[1];
  a.qo_sh = q_out_stride[2];
  if (Hkv > 0) {
    a.k = k;
    a.k_out = k_out;
    a.k_sb = k_stride[0];
    a.k_st = k_stride[1];
    a.k_sh = k_stride[2];
    a.ko_sb = k_out_stride[0];
    a.ko_st = k_out_stride[1];
    a.ko_sh = k_out_stride[2];
  }
  const hipError_t e = ttcd::launch_rope(a, interleaved != 0, elem(dtype),
                                         static_cast<hipStream_t>(stream));
  if (e == hipErrorInvalidConfiguration) return fail(TTCD_ERR_UNSUPPORTED, "grid too large");
  return from_hip(e, "rope launch");
}

ttcd_status ttcd_qk_norm_rope_fwd(const void* q, const void* k, void* q_out, void* k_out,
                                  const void* q_norm_w, const void* k_norm_w, ttcd_dtype w_dtype,
                                  float eps, const void* cos_table, const void* sin_table,
                                  int table_rows, int B, int T, int Hq, int Hkv, int D,
                                  const int64_t q_stride[4], const int64_t k_stride[4],
                                  const int64_t q_out_stride[4], const int64_t k_out_stride[4],
                                  int seqlen_offset, ttcd_dtype dtype, void* stream) {
  if (!q || !k || !q_out || !k_out || !cos_table || !sin_table)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!q_stride || !k_stride || !q_out_stride || !k_out_stride)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null stride array");
  if ((q_norm_w == nullptr) != (k_norm_w == nullptr))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "give both norm weights or neither");
  if (B < 1 || T < 1 || Hq < 1 || Hkv < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "B, T, Hq, Hkv must be >= 1 (got %d, %d, %d, %d)", B,
                T, Hq, Hkv);
  if (D != 64 && D != 128)
    return fail(TTCD_ERR_UNSUPPORTED, "head_dim %d not supported (64 or 128)", D);
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "q/k dtype must be bf16 or f16");
  if (q_norm_w && (unsigned)w_dtype > TTCD_DTYPE_F32)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "unknown norm weight dtype");
  if (!(eps >= 0.f) || !isfinite(eps))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0");
  if (seqlen_offset < 0) return fail(TTCD_ERR_INVALID_ARGUMENT, "seqlen_offset must be >= 0");
  if ((int64_t)seqlen_offset + T > (int64_t)table_rows)
    return fail(TTCD_ERR_INVALID_ARGUMENT,
                "rotary tables too short: seqlen_offset + T = %lld > table rows %d",
                (long long)seqlen_offset + T, table_rows);
  const int64_t* all[4] = {q_stride, k_stride, q_out_stride, k_out_stride};
  for (int t = 0; t < 4; ++t) {
    if (all[t][3] != 1)
      return fail(TTCD_ERR_INVALID_ARGUMENT, "head_dim must be contiguous (d-stride 1)");
    for (int i = 0; i < 3; ++i)
      if (all[t][i] % 8 != 0 || all[t][i] < 0)
        return fail(TTCD_ERR_UNSUPPORTED,
                    "strides must be non-negative multiples of 8 elements (16-byte rows)");
  }
  if (!aligned16(q) || !aligned16(k) || !aligned16(q_out) || !aligned16(k_out) ||
      !aligned16(cos_table) || !aligned16(sin_table))
    return fail(TTCD_ERR_UNSUPPORTED, "tensor base pointers must be 16-byte aligned");
  ttcd::PrologueArgs a = {};
  a.q = q;
  a.k = k;
  a.q_out = q_out;
  a.k_out = k_out;
  a.q_w = q_norm_w;
  a.k_w = k_norm_w;
  a.cos = cos_table;
  a.sin = sin_table;
  a.eps = eps;
  a.offset = seqlen_offset;
  a.B = B;
  a.T = T;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.D = D;
  a.q_sb = q_stride[0];
  a.q_st = q_stride[1];
  a.q_sh = q_stride[2];
  a.k_sb = k_stride[0];
  a.k_st = k_stride[1];
  a.k_sh = k_stride[2];
  a.qo_sb = q_out_stride[0];
  a.qo_st = q_out_stride[1];
  a.qo_sh = q_out_stride[2];
  a.ko_sb = k_out_stride[0];
  a.ko_st = k_out_stride[1];
  a.ko_sh = k_out_stride[2];
  return from_hip(ttcd::launch_qk_norm_rope(a, elem(dtype), elem(w_dtype),
                                            static_cast<hipStream_t>(stream)),
                  "qk norm + rope launch");
}

ttcd_status ttcd_dual_residual_rmsnorm_fwd(const void* attn_t, const void* attn_s,
                                           const void* residual, const void* norm_w,
                                           ttcd_dtype w_dtype, float eps, void* hidden_out,
                                           void* residual_out, void* student_out,
                                           int64_t rows, int hidden, ttcd_dtype dtype,
                                           void* stream) {
  if (!attn_t || !attn_s || !residual || !norm_w || !hidden_out || !residual_out ||
      !student_out)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (rows < 0 || hidden < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need rows >= 0 and hidden >= 1");
  if (hidden % 8 != 0 || hidden > 2048)
    return fail(TTCD_ERR_UNSUPPORTED, "hidden size %d not supported (a multiple of 8, <= 2048)",
                hidden);
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "activation dtype must be bf16 or f16");
  if ((unsigned)w_dtype > TTCD_DTYPE_F32)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "unknown norm weight dtype");
  if (!(eps >= 0.f) || !isfinite(eps))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0");
  const void* all[6] = {attn_t, attn_s, residual, hidden_out, residual_out, student_out};
  for (int i = 0; i < 6; ++i)
    if (!aligned16(all[i]))
      return fail(TTCD_ERR_UNSUPPORTED, "tensor base pointers must be 16-byte aligned");
  if (w_dtype != TTCD_DTYPE_F32 && !aligned16(norm_w))
    return fail(TTCD_ERR_UNSUPPORTED, "16-bit norm weights must be 16-byte aligned");
  if (rows == 0) return ok();
  return from_hip(ttcd::launch_dual_residual_rmsnorm(
                      attn_t, attn_s, residual, norm_w, elem(w_dtype), eps, hidden_out,
                      residual_out, student_out, rows, hidden, elem(dtype),
                      static_cast<hipStream_t>(stream)),
                  "dual residual rmsnorm launch");
}

ttcd_status ttcd_rmsnorm_fwd(const void* x, const void* residual, const void* norm_w,
                             ttcd_dtype w_dtype, float eps, void* y, void* residual_out,
                             int64_t rows, int hidden, ttcd_dtype dtype, void* stream) {
  if (!x || !norm_w || !y) return fail(TTCD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if ((residual == nullptr) != (residual_out == nullptr))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "pass residual and residual_out both or neither");
  if (rows < 0 || hidden < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need rows >= 0 and hidden >= 1");
  if (hidden % 8 != 0 || hidden > 2048)
    return fail(TTCD_ERR_UNSUPPORTED, "hidden size %d not supported (a multiple of 8, <= 2048)",
                hidden);
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "activation dtype must be bf16 or f16");
  if ((unsigned)w_dtype > TTCD_DTYPE_F32)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "unknown norm weight dtype");
  if (!(eps >= 0.f) || !isfinite(eps))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0");
  const void* all[4] = {x, y, residual, residual_out};
  for (int i = 0; i < 4; ++i)
    if (all[i] && !aligned16(all[i]))
      return fail(TTCD_ERR_UNSUPPORTED, "tensor base pointers must be 16-byte aligned");
  if (w_dtype != TTCD_DTYPE_F32 && !aligned16(norm_w))
    return fail(TTCD_ERR_UNSUPPORTED, "16-bit norm weights must be 16-byte aligned");
  if (rows == 0) return ok();
  return from_hip(ttcd::launch_dual_residual_rmsnorm(
                      x, nullptr, residual, norm_w, elem(w_dtype), eps, y, residual_out, nullptr,
                      rows, hidden, elem(dtype), static_cast<hipStream_t>(stream)),
                  "rmsnorm launch");
}

ttcd_status ttcd_add_rmsnorm_fwd(const void* x, const void* residual, const void* norm_w,
                                 ttcd_dtype w_dtype, float eps, void* y, void* sum_out,
                                 int64_t rows, int hidden, ttcd_dtype dtype, void* stream) {
  if (!x || !residual || !norm_w || !y || !sum_out)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (rows < 0 || hidden < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need rows >= 0 and hidden >= 1");
  if (hidden % 8 != 0 || hidden > 2048)
    return fail(TTCD_ERR_UNSUPPORTED, "hidden size %d not supported (a multiple of 8, <= 2048)",
                hidden);
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "activation dtype must be bf16 or f16");
  if ((unsigned)w_dtype > TTCD_DTYPE_F32)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "unknown norm weight dtype");
  if (!(eps >= 0.f) || !isfinite(eps))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0");
  const void* all[4] = {x, residual, y, sum_out};
  for (int i = 0; i < 4; ++i)
    if (!aligned16(all[i]))
      return fail(TTCD_ERR_UNSUPPORTED, "tensor base pointers must be 16-byte aligned");
  if (w_dtype != TTCD_DTYPE_F32 && !aligned16(norm_w))
    return fail(TTCD_ERR_UNSUPPORTED, "16-bit norm weights must be 16-byte aligned");
  if (rows == 0) return ok();
  return from_hip(ttcd::launch_dual_residual_rmsnorm(
                      x, nullptr, residual, norm_w, elem(w_dtype), eps, y, sum_out, nullptr,
                      rows, hidden, elem(dtype), static_cast<hipStream_t>(stream), true),
                  "add rmsnorm launch");
}

ttcd_status ttcd_swiglu_fwd(const void* gate, const void* up, void* out, int64_t rows, int cols,
                            int64_t gate_stride, int64_t up_stride, int64_t out_stride,
                            ttcd_dtype dtype, void* stream) {
  if (!gate || !up || !out) return fail(TTCD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (rows < 0 || cols < 1) return fail(TTCD_ERR_INVALID_ARGUMENT, "need rows >= 0, cols >= 1");
  if (gate_stride < cols || up_stride < cols || out_stride < cols)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "row strides must be >= cols");
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "dtype must be bf16 or f16");
  if (cols % 8 != 0 || gate_stride % 8 != 0 || up_stride % 8 != 0 || out_stride % 8 != 0)
    return fail(TTCD_ERR_UNSUPPORTED, "cols and row strides must be multiples of 8");
  if (!aligned16(gate) || !aligned16(up) || !aligned16(out))
    return fail(TTCD_ERR_UNSUPPORTED, "tensor base pointers must be 16-byte aligned");
  if (rows == 0) return ok();
  return from_hip(ttcd::launch_swiglu(gate, up, out, rows, cols, gate_stride, up_stride,
                                      out_stride, elem(dtype), static_cast<hipStream_t>(stream)),
                  "swiglu launch");
}

ttcd_status ttcd_linear_rows_fwd(const void* x, int64_t x_stride, const void* w, void* y, int M,
                                 int N, int K, int swiglu, ttcd_dtype dtype, void* stream) {
  if (!x || !w || !y) return fail(TTCD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (M < 1 || N < 1 || K < 1 || x_stride < K)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need M, N, K >= 1 and x_stride >= K");
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "dtype must be bf16 or f16");
  if (K % 32 != 0 || x_stride % 8 != 0)
    return fail(TTCD_ERR_UNSUPPORTED, "K must be a multiple of 32 and x_stride of 8");
  if (!aligned16(x) || !aligned16(w))
    return fail(TTCD_ERR_UNSUPPORTED, "x and w must be 16-byte aligned");
  if ((M + 15) / 16 > 65535) return fail(TTCD_ERR_UNSUPPORTED, "too many rows (grid y)");
  const ttcd::LinearArgs a{x, x_stride, w, y, M, N, K, swiglu != 0};
  return from_hip(ttcd::launch_linear_rows(a, elem(dtype), static_cast<hipStream_t>(stream)),
                  "linear launch");
}

// Both forms of the feature pass.
static ttcd_status ttt_features(const ttcd::TttFeatureArgs& a, ttcd_dtype w_dtype,
                                ttcd_dtype dtype, void* stream) {
  if (!a.gu_t || !a.z || (a.nchunk > 1 && !a.diff) ||
      ((a.nchunk > 1 || a.last_student) && (!a.gu_s || !a.z_hat)))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (a.B < 1 || a.nchunk < 1 || a.C < 1 || a.I < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need B, nchunk, chunk, inter >= 1");
  if (a.gu_st < 2 * (int64_t)a.I)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "gate|up row stride must be >= 2 * inter");
  if (a.K < 1 || ((a.w_t || a.w_s) && a.K > 8))
    return fail(TTCD_ERR_UNSUPPORTED, "conv kernel size must be in 1..8");
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "dtype must be bf16 or f16");
  if ((unsigned)w_dtype > TTCD_DTYPE_F32)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "unknown conv weight dtype");
  if (a.I % 8 != 0 || a.gu_st % 8 != 0)
    return fail(TTCD_ERR_UNSUPPORTED, "inter and the gate|up row stride must be multiples of 8");
  const void* all[5] = {a.gu_t, a.gu_s, a.z, a.z_hat, a.diff};
  for (int i = 0; i < 5; ++i)
    if (all[i] && !aligned16(all[i]))
      return fail(TTCD_ERR_UNSUPPORTED, "tensor base pointers must be 16-byte aligned");
  ttcd::TttFeatureArgs k = a;
  if (!a.w_t && !a.w_s) k.K = 1;
  return from_hip(ttcd::launch_ttt_features(k, elem(dtype), elem(w_dtype),
                                            static_cast<hipStream_t>(stream)),
                  "ttt features launch");
}

ttcd_status ttcd_ttt_features_fwd(const void* gu_t, const void* gu_s, int64_t gu_stride,
                                  const void* conv_t, const void* conv_s, ttcd_dtype w_dtype,
                                  int kernel_size, void* z, void* z_hat, void* diff, int B,
                                  int nchunk, int chunk, int inter, ttcd_dtype dtype,
                                  void* stream) {
  const int64_t rows = (int64_t)nchunk * chunk;
  return ttt_features({gu_t, gu_s, gu_stride, rows, rows, conv_t, conv_s, kernel_size, z, z_hat,
                       diff, B, nchunk, chunk, inter, rows, true},
                      w_dtype, dtype, stream);
}

ttcd_status ttcd_ttt_features_tokens_fwd(const void* gu_t, int64_t t_rows, const void* gu_s,
                                         int64_t s_rows, int64_t gu_stride, const void* conv_t,
                                         const void* conv_s, ttcd_dtype w_dtype,
                                         int kernel_size, void* z, void* z_hat, void* diff,
                                         int B, int tokens, int chunk, int inter,
                                         ttcd_dtype dtype, void* stream) {
  if (tokens < 1 || chunk < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need tokens, chunk >= 1");
  const int nchunk = (int)(((int64_t)tokens + chunk - 1) / chunk);
  if (t_rows < tokens || (nchunk > 1 && s_rows < (int64_t)(nchunk - 1) * chunk))
    return fail(TTCD_ERR_INVALID_ARGUMENT,
                "t_rows must be >= tokens and s_rows >= the updating chunks' rows");
  return ttt_features({gu_t, gu_s, gu_stride, t_rows, s_rows, conv_t, conv_s, kernel_size, z,
                       z_hat, diff, B, nchunk, chunk, inter, tokens, false},
                      w_dtype, dtype, stream);
}

ttcd_status ttcd_ttt_proj_beta_t_fwd(const void* pd, int64_t pd_stride, const void* beta,
                                    int64_t beta_batch_stride, void* pdt, int B, int nupd,
                                    int chunk, int H, ttcd_dtype dtype, void* stream) {
  if (!pd || !pdt) return fail(TTCD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (B < 1 || nupd < 1 || chunk < 1 || H < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need B, nupd, chunk, H >= 1");
  if (pd_stride < H || (beta && beta_batch_stride < (int64_t)nupd * chunk))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "pd row stride must be >= H and the beta batch "
                                           "stride >= nupd * chunk");
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "dtype must be bf16 or f16");
  if ((int64_t)B * nupd > 65535)
    return fail(TTCD_ERR_UNSUPPORTED, "B * nupd above 65535 (grid z)");
  ttcd::TttProjBetaArgs a{pd, pd_stride, beta, beta_batch_stride, pdt, B, nupd, chunk, H};
  return from_hip(ttcd::launch_ttt_proj_beta_t(a, elem(dtype), static_cast<hipStream_t>(stream)),
                  "ttt pd*beta launch");
}

ttcd_status ttcd_ttt_beta_fwd(const void* t, int64_t t_rows, const void* b_proj, void* beta,
                              int B, int rows, int H, ttcd_dtype dtype, void* stream) {
  if (!t || !b_proj || !beta) return fail(TTCD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (B < 1 || rows < 1 || H < 1 || t_rows < rows)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need B, rows, H >= 1 and t_rows >= rows");
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "dtype must be bf16 or f16");
  if (H % 8 != 0 || !aligned16(t) || !aligned16(b_proj))
    return fail(TTCD_ERR_UNSUPPORTED, "H must be a multiple of 8 and t, b_proj 16-byte aligned");
  ttcd::TttBetaArgs a{t, t_rows, b_proj, beta, B, rows, H};
  return from_hip(ttcd::launch_ttt_beta(a, elem(dtype), static_cast<hipStream_t>(stream)),
                  "ttt beta launch");
}

ttcd_status ttcd_ttt_scan_fwd(const void* dw, const void* w_cur, float lr, void* steps_t,
                              void* w_next, int nupd, int nsteps, int H, int inter,
                              ttcd_dtype dtype, void* stream) {
  if (!w_cur || !steps_t || (nupd > 0 && !dw))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (H < 1 || inter < 1 || nupd < 0 || nsteps < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need H, inter, nsteps >= 1 and nupd >= 0");
  // chunk s of the group uses cs[s - 1]: there must be one for every step but the first
  if (nsteps > nupd + 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "nsteps (%d) must be <= nupd + 1 (%d)", nsteps,
                nupd + 1);
  if (w_next && nupd < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "w_next needs at least one update");
  if (!isfinite(lr)) return fail(TTCD_ERR_INVALID_ARGUMENT, "lr must be finite");
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "dtype must be bf16 or f16");
  ttcd::TttScanArgs a{dw, w_cur, lr, steps_t, w_next, nupd, nsteps, H, inter};
  return from_hip(ttcd::launch_ttt_scan(a, elem(dtype), static_cast<hipStream_t>(stream)),
                  "ttt scan launch");
}

// ---------------------------------------------------------------------------
// The 4-bit key / value cache.
namespace {

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

ttcd_status check_kv4(const ttcd_kv4_cache* c) {
  if (!c || !c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales || !c->lengths)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null cache pointer");
  if (c->batch < 1 || c->kv_heads < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need batch, kv_heads >= 1 (got %d, %d)", c->batch,
                c->kv_heads);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(TTCD_ERR_UNSUPPORTED, "head_dim %d not supported (64 or 128)", c->head_dim);
  if (c->capacity < 32 || c->capacity % 32 != 0 || c->capacity > ttcd::kKv4MaxLength)
    return fail(TTCD_ERR_INVALID_ARGUMENT,
                "capacity must be a multiple of 32 in 32 .. 2^30 (got %d)", c->capacity);
  if (!aligned16(c->k_codes) || !aligned16(c->v_codes) || !aligned4(c->v_scales) ||
      !aligned4(c->lengths))
    return fail(TTCD_ERR_UNSUPPORTED,
                "codes must be 16-byte aligned, v_scales and lengths 4-byte aligned");
  if ((int64_t)c->batch * c->kv_heads > 65535)
    return fail(TTCD_ERR_UNSUPPORTED, "batch * kv_heads above 65535 (grid y)");
  return TTCD_OK;
}

ttcd::Kv4Cache kv4(const ttcd_kv4_cache* c) {
  return {static_cast<uint8_t*>(c->k_codes), static_cast<uint8_t*>(c->k_scales),
          static_cast<uint8_t*>(c->v_codes), static_cast<uint8_t*>(c->v_scales),
          c->lengths, c->batch, c->kv_heads, c->head_dim, c->capacity};
}

ttcd_status check_kv4_dtype(ttcd_dtype dtype) {
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "dtype must be bf16 or f16");
  return TTCD_OK;
}

ttcd_status check_kv4_strides(const void* p, const int64_t* s) {
  if (!p) return fail(TTCD_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!s) return fail(TTCD_ERR_INVALID_ARGUMENT, "null stride array");
  if (s[3] != 1) return fail(TTCD_ERR_INVALID_ARGUMENT, "head_dim must be contiguous (d-stride 1)");
  for (int i = 0; i < 3; ++i)
    if (s[i] % 8 != 0 || s[i] < 0)
      return fail(TTCD_ERR_UNSUPPORTED,
                  "strides must be non-negative multiples of 8 elements (16-byte rows)");
  if (!aligned16(p))
    return fail(TTCD_ERR_UNSUPPORTED, "tensor base pointers must be 16-byte aligned");
  return TTCD_OK;
}

// A workgroup a row of the sum over the parts. (By a division: batch * Hq * Tq may pass 64
// bits, and rows that wrapped around to none ended the process in kv4_plan.)
bool kv4_rows_fit(const ttcd_kv4_cache* c, int Tq, int Hq) {
  return (int64_t)Hq * Tq <= (0x7fffffffLL - 1024) / c->batch;
}

ttcd_status check_kv4_rows(const ttcd_kv4_cache* c, int Tq, int Hq) {
  if (Tq < 1 || Hq < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need Tq, Hq >= 1 (got %d, %d)", Tq, Hq);
  if (Hq % c->kv_heads != 0)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "Hq (%d) must be a multiple of kv_heads (%d)", Hq,
                c->kv_heads);
  if (!kv4_rows_fit(c, Tq, Hq)) return fail(TTCD_ERR_UNSUPPORTED, "grid too large");
  return TTCD_OK;
}

int kv4_window(int window) {
  return window <= 0 ? 0 : (window < ttcd::kKv4MaxLength ? window : ttcd::kKv4MaxLength);
}

struct Kv4Plan {
  int row_tiles, nrb, parts;
};

// Workgroups over rows and keys. The lengths are on the GPU: parts go by the most
// keys that a row block can see, and each takes its share of what there is.
//
// Up to 32 rows a key / value head (a token, or a few): kernels of 8 wavefronts with 16
// or 32 rows that stream the keys, bound by those: parts for 1024 workgroups, but 16
// tiles of 32 keys each at the least, two a wavefront (us, one token, 16/8 heads of
// 128: 8 sequences of 4096 keys 15.5, with 8 tiles 19.6; one of 8192 9.4, with 32 tiles
// 12.0), and none for up to 40 tiles, where the second launch costs more than it saves
// (1024 keys 7.5, split 9.0; 2048 9.0 split; 704 6.5). Parts for 512 workgroups are
// better for large batches and worse for few sequences (1024 and 512: 32 of up to 16384
// keys 58 and 55, 8 of 16384 36 and 31, 3 of 16384 21.6 and 22.0, 2 of 65001 with 15/5
// heads of 64 18.4 and 19.4; the others above the same).
//
// More: 128 rows a workgroup and tiles of 64 keys, of which a turn takes so many us
// with a CU to itself and so many for each of two that share one. What a split adds is
// its launch, its rows and its sums, written and read. Measured (us, 16/8 heads of
// 128): 300 queries on an 8192 window in 3 parts 83, 6 52, 10 48, 12 (taken) 45, 16 54;
// 1000 queries in 1 part 207, 2 127, 3 119, 4 (taken) 102; 64 queries of 32 sequences
// on a 960 window in 1 part (taken) 31, 2 61.
Kv4Plan kv4_plan(const ttcd_kv4_cache* c, int Tq, int Hq, int window) {
  const int G = Hq / c->kv_heads;
  const int64_t rows = (int64_t)Tq * G;
  Kv4Plan p;
  p.row_tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 8;
  const int rb = 16 * p.row_tiles;
  p.nrb = (int)((rows + rb - 1) / rb);
  int64_t keys = c->capacity;
  if (window > 0) {
    const int64_t span = (int64_t)window + (rb + G - 1) / G;
    keys = span < keys ? span : keys;
  }
  const int64_t groups = (int64_t)c->batch * c->kv_heads * p.nrb;
  int64_t parts = 1;
  if (p.row_tiles < 8) {
    const int64_t tiles = keys / 32 + 1;
    if (tiles > 40) parts = std::min((1024 + groups - 1) / groups, tiles / 16);
    parts = std::min(std::max(parts, (int64_t)1), (int64_t)ttcd::kKv4MaxParts);
  } else {
    const int64_t tiles = keys / 64 + 1;
    const int64_t most = std::min({512 / groups, tiles / 4, (int64_t)ttcd::kKv4MaxParts});
    const double all_rows = (double)c->batch * Hq * Tq, bytes = all_rows * (c->head_dim + 2) * 4;
    const double alone = c->head_dim == 128 ? 1.5 : 1.0, shared = c->head_dim == 128 ? 2.2 : 1.35;
    double least = 0;
    for (int64_t n = 1; n == 1 || n <= most; ++n) {
      const double turns = (double)tiles / n + 1;
      double t = turns * (groups * n <= 256 ? alone : shared);
      if (n > 1) t += 3.0 + n * bytes / 7e6 + all_rows * 5e-4;
      if (n > 1 && t >= least) continue;
      least = t;
      parts = n;
    }
  }
  p.parts = (int)parts;
  return p;
}

size_t kv4_part_bytes(const ttcd_kv4_cache* c, int Tq, int Hq) {
  return (size_t)c->batch * Tq * Hq * (c->head_dim + 2) * sizeof(float);
}

struct Span {
  const void* at;  // null: none
  int64_t bytes;
};
bool overlap(const Span& a, const Span& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
  return x && y && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes;
}
void kv4_spans(const ttcd_kv4_cache* c, Span spans[5]) {
  const int64_t n = (int64_t)c->batch * c->kv_heads * c->capacity * c->head_dim;
  spans[0] = {c->k_codes, n / 2};
  spans[1] = {c->k_scales, n / 32};
  spans[2] = {c->v_codes, n / 2};
  spans[3] = {c->v_scales, n / 32};
  spans[4] = {c->lengths, (int64_t)c->batch * 4};
}

}  // namespace

ttcd_status ttcd_kv4_append(ttcd_kv4_cache* cache, const void* k, const void* v, int T,
                            const int64_t k_stride[4], const int64_t v_stride[4],
                            const int32_t* counts, float* weights, ttcd_dtype dtype,
                            void* stream) {
  ttcd_status st = check_kv4(cache);
  if (st == TTCD_OK) st = check_kv4_dtype(dtype);
  if (st == TTCD_OK) st = check_kv4_strides(k, k_stride);
  if (st == TTCD_OK) st = check_kv4_strides(v, v_stride);
  if (st != TTCD_OK) return st;
  if (T < 1 || T > cache->capacity)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need 1 <= T <= capacity (got T=%d, capacity %d)", T,
                cache->capacity);
  ttcd::Kv4AppendArgs a = {};
  a.c = kv4(cache);
  a.k = k;
  a.v = v;
  a.k_sb = k_stride[0];
  a.k_st = k_stride[1];
  a.k_sh = k_stride[2];
  a.v_sb = v_stride[0];
  a.v_st = v_stride[1];
  a.v_sh = v_stride[2];
  a.counts = counts;
  a.weights = weights;
  a.T = T;
  return from_hip(ttcd::launch_kv4_append(a, elem(dtype), static_cast<hipStream_t>(stream)),
                  "kv4 append launch");
}

ttcd_status ttcd_kv4_read(const ttcd_kv4_cache* cache, void* k, void* v, int count,
                          ttcd_dtype dtype, void* stream) {
  ttcd_status st = check_kv4(cache);
  if (st == TTCD_OK) st = check_kv4_dtype(dtype);
  if (st != TTCD_OK) return st;
  if (!k || !v) return fail(TTCD_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!aligned16(k) || !aligned16(v))
    return fail(TTCD_ERR_UNSUPPORTED, "tensor base pointers must be 16-byte aligned");
  if (count < 1) return fail(TTCD_ERR_INVALID_ARGUMENT, "need count >= 1 (got %d)", count);
  const int64_t blocks = ((int64_t)(count + 3LL) / 4 + 1) * cache->kv_heads * (cache->head_dim / 8);
  if (blocks / 256 >= 0x7fffffffLL) return fail(TTCD_ERR_UNSUPPORTED, "grid too large");
  ttcd::Kv4ReadArgs a = {kv4(cache), k, v, count};
  return from_hip(ttcd::launch_kv4_read(a, elem(dtype), static_cast<hipStream_t>(stream)),
                  "kv4 read launch");
}

size_t ttcd_kv4_attn_workspace_bytes(const ttcd_kv4_cache* cache, int Tq, int Hq, int window) {
  if (!cache || cache->batch < 1 || cache->kv_heads < 1 || Tq < 1 || Hq < cache->kv_heads ||
      Hq % cache->kv_heads != 0 || (cache->head_dim != 64 && cache->head_dim != 128) ||
      cache->capacity < 32 || !kv4_rows_fit(cache, Tq, Hq))
    return 0;
  const Kv4Plan p = kv4_plan(cache, Tq, Hq, kv4_window(window));
  return p.parts > 1 ? p.parts * kv4_part_bytes(cache, Tq, Hq) : 0;
}

ttcd_status ttcd_kv4_attn_fwd(const ttcd_kv4_cache* cache, const void* q, void* o, float* lse,
                              int Tq, int Hq, const int64_t q_stride[4],
                              const int64_t o_stride[4], const int32_t* counts, int window,
                              float sm_scale, ttcd_dtype dtype, void* workspace,
                              size_t workspace_bytes, void* stream) {
  ttcd_status st = check_kv4(cache);
  if (st == TTCD_OK) st = check_kv4_dtype(dtype);
  if (st == TTCD_OK) st = check_kv4_strides(q, q_stride);
  if (st == TTCD_OK) st = check_kv4_strides(o, o_stride);
  if (st == TTCD_OK) st = check_kv4_rows(cache, Tq, Hq);
  if (st != TTCD_OK) return st;
  if (!(sm_scale > 0.f) || !isfinite(sm_scale))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "sm_scale must be finite and > 0");
  ttcd::Kv4AttnArgs a = {};
  a.c = kv4(cache);
  a.q = q;
  a.o = o;
  a.lse = lse;
  a.counts = counts;
  a.q_sb = q_stride[0];
  a.q_st = q_stride[1];
  a.q_sh = q_stride[2];
  a.o_sb = o_stride[0];
  a.o_st = o_stride[1];
  a.o_sh = o_stride[2];
  a.Tq = Tq;
  a.G = Hq / cache->kv_heads;
  a.window = kv4_window(window);
  a.c_log2 = sm_scale * 1.4426950408889634f;
  const Kv4Plan p = kv4_plan(cache, Tq, Hq, a.window);
  a.row_tiles = p.row_tiles;
  a.nrb = p.nrb;
  a.parts = 1;
  const size_t part = kv4_part_bytes(cache, Tq, Hq);
  if (p.parts > 1 && workspace && aligned16(workspace) && workspace_bytes >= p.parts * part) {
    a.parts = p.parts;
    a.part = static_cast<float*>(workspace);
    a.part_ml = a.part + p.parts * (part / sizeof(float) / (cache->head_dim + 2)) * cache->head_dim;
  }
  return from_hip(ttcd::launch_kv4_attn(a, elem(dtype), static_cast<hipStream_t>(stream)),
                  "kv4 attention launch");
}

ttcd_status ttcd_kv4_key_weights_fwd(const ttcd_kv4_cache* cache, const void* q,
                                     const float* lse, float* weights, int Tq, int Hq,
                                     const int64_t q_stride[4], const int32_t* counts,
                                     int window, float sm_scale, int accumulate,
                                     ttcd_dtype dtype, void* stream) {
  ttcd_status st = check_kv4(cache);
  if (st == TTCD_OK) st = check_kv4_dtype(dtype);
  if (st == TTCD_OK) st = check_kv4_strides(q, q_stride);
  if (st == TTCD_OK) st = check_kv4_rows(cache, Tq, Hq);
  if (st != TTCD_OK) return st;
  if (!lse || !weights) return fail(TTCD_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (!(sm_scale > 0.f) || !isfinite(sm_scale))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "sm_scale must be finite and > 0");
  if (!aligned16(weights))
    return fail(TTCD_ERR_UNSUPPORTED, "weights must be 16-byte aligned");
  ttcd::Kv4WeightsArgs a = {};
  a.c = kv4(cache);
  a.q = q;
  a.lse = lse;
  a.weights = weights;
  a.counts = counts;
  a.q_sb = q_stride[0];
  a.q_st = q_stride[1];
  a.q_sh = q_stride[2];
  a.Tq = Tq;
  a.G = Hq / cache->kv_heads;
  a.window = kv4_window(window);
  a.c_log2 = sm_scale * 1.4426950408889634f;
  a.accumulate = accumulate != 0;
  return from_hip(ttcd::launch_kv4_weights(a, elem(dtype), static_cast<hipStream_t>(stream)),
                  "kv4 key weights launch");
}

ttcd_status ttcd_kv4_evict(const ttcd_kv4_cache* cache, const float* weights, int keep,
                           int recent, ttcd_kv4_cache* out, float* new_weights, int32_t* index,
                           void* stream) {
  ttcd_status st = check_kv4(cache);
  if (st == TTCD_OK) st = check_kv4(out);
  if (st != TTCD_OK) return st;
  if (!weights || !index) return fail(TTCD_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (out->batch != cache->batch || out->kv_heads != cache->kv_heads ||
      out->head_dim != cache->head_dim)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "out must have the cache's batch, kv_heads and head_dim");
  if (keep < 1 || keep > out->capacity || recent < 0)
    return fail(TTCD_ERR_INVALID_ARGUMENT,
                "need 1 <= keep <= out's capacity and recent >= 0 (got %d, %d, %d)", keep,
                out->capacity, recent);
  const int64_t heads = (int64_t)cache->batch * cache->kv_heads;
  Span read[6], written[7];
  kv4_spans(cache, read);
  read[5] = {weights, heads * cache->capacity * 4};
  kv4_spans(out, written);
  written[5] = {new_weights, heads * out->capacity * 4};
  written[6] = {index, heads * keep * 4};
  for (int i = 0; i < 7; ++i) {
    for (const Span& r : read)
      if (overlap(written[i], r))
        return fail(TTCD_ERR_INVALID_ARGUMENT, "out must not share memory with the cache");
    for (int j = 0; j < i; ++j)
      if (overlap(written[i], written[j]))
        return fail(TTCD_ERR_INVALID_ARGUMENT, "out's parts must not share memory");
  }
  ttcd::Kv4EvictArgs a = {};
  a.c = kv4(cache);
  a.out = kv4(out);
  a.weights = weights;
  a.new_weights = new_weights;
  a.index = index;
  a.keep = keep;
  a.recent = recent;
  return from_hip(ttcd::launch_kv4_evict(a, static_cast<hipStream_t>(stream)),
                  "kv4 eviction launch");
}

namespace {

struct Kv4TreePlan {
  int row_tiles, nrb, units, least;
  size_t bytes;  // of the workspace; 0: no split
};

// The same for a tree, whose parts the kernels deal to the sequences by their lengths: up to
// 64 of them, a lane each, to share 512 workgroups, two a CU (us, nodes and sequences of up to
// 16000 keys, 16/8 heads of 128, with 256, 512 and 768: 16 of 8 30, 31, 36; 8 of 32 94, 59,
// 60; 64 of 8 76, 64, 70; 256 of 1 59, 54, 66). As many parts to every sequence took 50 for
// the first of these. No split up to 40 tiles of 32 keys, or 8 of 64: the sum of the parts
// costs more than it saves. None for so many rows that their sum, of 64 threads a row, passes
// the 2^32 threads that a launch stays below, nor above 64 sequences, which the dealing has no
// lanes for.
Kv4TreePlan kv4_tree_plan(const ttcd_kv4_cache* c, int N, int Hq, int window) {
  const int64_t rows = (int64_t)N * (Hq / c->kv_heads);
  Kv4TreePlan p = {};
  p.row_tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 8;
  const int rb = 16 * p.row_tiles;
  const bool block = p.row_tiles == 8;
  p.nrb = (int)((rows + rb - 1) / rb);
  int64_t keys = c->capacity;
  if (window > 0 && window < keys) keys = window;
  const int64_t tiles = (keys + N) / (block ? 64 : 32) + 2;  // of a sequence, at most
  if (tiles <= (block ? 8 : 40) || c->batch > 64 || c->batch * rows * c->kv_heads >= 1 << 26)
    return p;
  p.least = 4;
  const int64_t groups = (int64_t)c->kv_heads * p.nrb, all = (tiles + p.least - 1) / p.least;
  const int64_t units = std::min((512 + groups - 1) / groups, c->batch * all);
  p.units = (int)std::max(units, (int64_t)c->batch + 1);
  p.bytes = (size_t)p.units * c->kv_heads * rows * (c->head_dim + 2) * sizeof(float) +
            (size_t)c->batch * 2 * sizeof(int32_t);
  return p;
}

// The draft that a tree's nodes lie in, next to the cache of their sequences.
ttcd_status check_draft(const ttcd_kv4_cache* cache, const ttcd_kv4_cache* draft) {
  if (draft->batch != cache->batch || draft->kv_heads != cache->kv_heads ||
      draft->head_dim != cache->head_dim)
    return fail(TTCD_ERR_INVALID_ARGUMENT,
                "the draft must have the cache's batch, kv_heads and head_dim");
  Span ours[5], theirs[5];
  kv4_spans(cache, ours);
  kv4_spans(draft, theirs);
  for (const Span& x : ours)
    for (const Span& y : theirs)
      if (overlap(x, y))
        return fail(TTCD_ERR_INVALID_ARGUMENT, "the draft must not share memory with the cache");
  return TTCD_OK;
}

}  // namespace

size_t ttcd_kv4_tree_attn_workspace_bytes(const ttcd_kv4_cache* cache, int N, int Hq,
                                          int window) {
  if (!cache || cache->batch < 1 || cache->kv_heads < 1 || N < 1 || N > ttcd::kTreeNodes ||
      Hq < cache->kv_heads || Hq % cache->kv_heads != 0 ||
      (cache->head_dim != 64 && cache->head_dim != 128) || cache->capacity < 32 ||
      !kv4_rows_fit(cache, N, Hq))
    return 0;
  return kv4_tree_plan(cache, N, Hq, kv4_window(window)).bytes;
}

ttcd_status ttcd_kv4_tree_attn_fwd(const ttcd_kv4_cache* cache, const ttcd_kv4_cache* draft,
                                   const void* q, void* o, float* lse, int N, int Hq,
                                   const int64_t q_stride[4], const int64_t o_stride[4],
                                   const int32_t* parents, const int32_t* counts, int window,
                                   float sm_scale, ttcd_dtype dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  ttcd_status st = check_kv4(cache);
  if (st == TTCD_OK) st = check_kv4(draft);
  if (st == TTCD_OK) st = check_draft(cache, draft);
  if (st == TTCD_OK) st = check_kv4_dtype(dtype);
  if (st == TTCD_OK) st = check_kv4_strides(q, q_stride);
  if (st == TTCD_OK) st = check_kv4_strides(o, o_stride);
  if (st == TTCD_OK) st = check_kv4_rows(cache, N, Hq);
  if (st != TTCD_OK) return st;
  if (!parents) return fail(TTCD_ERR_INVALID_ARGUMENT, "null parents pointer");
  if (N > ttcd::kTreeNodes)
    return fail(TTCD_ERR_UNSUPPORTED, "%d nodes: at most %d", N, ttcd::kTreeNodes);
  if (N > draft->capacity)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "%d nodes in a draft of capacity %d", N,
                draft->capacity);
  if (!(sm_scale > 0.f) || !isfinite(sm_scale))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "sm_scale must be finite and > 0");
  ttcd::Kv4TreeArgs a = {};
  a.c = kv4(cache);
  a.d = kv4(draft);
  a.parents = parents;
  a.q = q;
  a.o = o;
  a.lse = lse;
  a.counts = counts;
  a.q_sb = q_stride[0];
  a.q_st = q_stride[1];
  a.q_sh = q_stride[2];
  a.o_sb = o_stride[0];
  a.o_st = o_stride[1];
  a.o_sh = o_stride[2];
  a.Tq = N;
  a.G = Hq / cache->kv_heads;
  a.window = kv4_window(window);
  a.c_log2 = sm_scale * 1.4426950408889634f;
  const Kv4TreePlan p = kv4_tree_plan(cache, N, Hq, a.window);
  a.row_tiles = p.row_tiles;
  a.nrb = p.nrb;
  a.parts = 1;
  if (p.bytes > 0 && workspace && aligned16(workspace) && workspace_bytes >= p.bytes) {
    a.units = p.units;
    a.least = p.least;
    a.part = static_cast<float*>(workspace);
    a.part_ml = a.part + (size_t)p.units * Hq * N * cache->head_dim;
    a.shares = reinterpret_cast<int32_t*>(a.part_ml + (size_t)p.units * Hq * N * 2);
  }
  return from_hip(ttcd::launch_kv4_tree_attn(a, elem(dtype), static_cast<hipStream_t>(stream)),
                  "kv4 tree attention launch");
}

ttcd_status ttcd_kv4_commit(ttcd_kv4_cache* cache, ttcd_kv4_cache* draft, const int32_t* path,
                            const int32_t* counts, int P, float* weights, int reset_draft,
                            void* stream) {
  ttcd_status st = check_kv4(cache);
  if (st == TTCD_OK) st = check_kv4(draft);
  if (st == TTCD_OK) st = check_draft(cache, draft);
  if (st != TTCD_OK) return st;
  if (!path) return fail(TTCD_ERR_INVALID_ARGUMENT, "null path pointer");
  if (P < 1 || P > cache->capacity || P > draft->capacity)
    return fail(TTCD_ERR_INVALID_ARGUMENT,
                "need 1 <= P <= the capacities (got P=%d, capacities %d and %d)", P,
                cache->capacity, draft->capacity);
  if ((int64_t)P * cache->kv_heads * (cache->head_dim / 8) > 0x7fffffffLL)
    return fail(TTCD_ERR_UNSUPPORTED, "grid too large");
  ttcd::Kv4CommitArgs a = {};
  a.c = kv4(cache);
  a.d = kv4(draft);
  a.path = path;
  a.counts = counts;
  a.weights = weights;
  a.P = P;
  a.reset = reset_draft != 0;
  return from_hip(ttcd::launch_kv4_commit(a, static_cast<hipStream_t>(stream)),
                  "kv4 commit launch");
}

ttcd_status ttcd_sample_fwd(const void* logits, int64_t row_stride, int R, int V,
                            const float* uniform, const float* temperatures, double temperature,
                            const int32_t* top_ks, int top_k, const float* top_ps, double top_p,
                            const float* min_ps, double min_p, int64_t* tokens, float* logprobs,
                            ttcd_dtype dtype, void* stream) {
  if (!logits || !uniform || !tokens)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (R < 1 || V < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need R, V >= 1 (got %d, %d)", R, V);
  if (V > ttcd::kSampleVocab)
    return fail(TTCD_ERR_UNSUPPORTED, "%d tokens a row: at most %d", V, ttcd::kSampleVocab);
  // a launch has fewer than 2^32 threads: 1024 a row
  if (R >= 1 << 22) return fail(TTCD_ERR_UNSUPPORTED, "grid too large (%d rows)", R);
  if (dtype != TTCD_DTYPE_BF16 && dtype != TTCD_DTYPE_F16)
    return fail(TTCD_ERR_UNSUPPORTED, "logits must be bf16 or f16");
  if (row_stride < 0) return fail(TTCD_ERR_INVALID_ARGUMENT, "row stride must be >= 0");
  if (reinterpret_cast<uintptr_t>(logits) & 1u)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "logits must be 2-byte aligned");
  if (!temperatures && !(temperature >= 0))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "temperature must be >= 0");
  if (!top_ks && top_k < 0) return fail(TTCD_ERR_INVALID_ARGUMENT, "top_k must be >= 0");
  if (!top_ps && !(top_p > 0)) return fail(TTCD_ERR_INVALID_ARGUMENT, "top_p must be > 0");
  if (!min_ps && !(min_p >= 0 && min_p <= 1))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "min_p must be in 0 .. 1");
  ttcd::SampleArgs a = {};
  a.logits = logits;
  a.st = row_stride;
  a.R = R;
  a.V = V;
  a.uniform = uniform;
  a.temperatures = temperatures;
  a.temperature = temperature;
  a.top_ks = top_ks;
  a.top_k = top_k;
  a.top_ps = top_ps;
  a.top_p = top_p;
  a.min_ps = min_ps;
  a.min_p = min_p;
  a.tokens = tokens;
  a.logprobs = logprobs;
  return from_hip(ttcd::launch_sample(a, elem(dtype), static_cast<hipStream_t>(stream)),
                  "sample launch");
}

ttcd_status ttcd_tree_accept(const int32_t* parents, const int64_t* tokens,
                             const int64_t* picked, const int32_t* counts, int32_t* path,
                             int32_t* accepted, int64_t* next, int B, int N, void* stream) {
  if (!parents || !tokens || !picked || !path || !accepted || !next)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "null tensor pointer");
  if (B < 1 || N < 1)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need B, N >= 1 (got %d, %d)", B, N);
  if (N > ttcd::kTreeNodes)
    return fail(TTCD_ERR_UNSUPPORTED, "%d nodes: at most %d", N, ttcd::kTreeNodes);
  if (B >= 1 << 26)  // 64 threads a sequence
    return fail(TTCD_ERR_UNSUPPORTED, "grid too large (%d sequences)", B);
  const ttcd::AcceptArgs a = {parents, tokens, picked, counts, path, accepted, next, B, N};
  return from_hip(ttcd::launch_tree_accept(a, static_cast<hipStream_t>(stream)),
                  "tree accept launch");
}

ttcd_status ttcd_attn_schedule_coverage(int T, int dual, int window_s, int window_t,
                                        int gqa_group, int32_t* counts_near,
                                        int32_t* counts_far) {
  using namespace ttcd;
  if (T < 1 || gqa_group < 1 || !counts_near || (dual && !counts_far))
    return fail(TTCD_ERR_INVALID_ARGUMENT, "bad coverage arguments");
  Schedule sc;
  if (dual) {
    if (window_t < 0) window_t = T;
    if (window_s < 1 || window_s > window_t)
      return fail(TTCD_ERR_INVALID_ARGUMENT, "need 1 <= window_s <= window_t");
    sc = make_dual_schedule(T, window_s, window_t, wave_rows(gqa_group));
  } else {
    if (window_s < 0 || window_t <= window_s)
      return fail(TTCD_ERR_INVALID_ARGUMENT, "need 0 <= band_lo < band_hi");
    sc = make_band_schedule(T, window_s, window_t, wave_rows(gqa_group));
  }
  // Workgroup geometry as launched (attn.hip): 4 waves over 4R consecutive
  // tokens, wave w owning rows r0 = t0 + R*w (R = 16 for an even gqa_group,
  // else 32).
  const int R = sc.rows;
  const int span = wg_span_tokens(gqa_group);
  const int nwg = (T + span - 1) / span;
  for (int qb = 0; qb < nwg; ++qb) {
    const int t0 = qb * span;
    const int t_last = (t0 + span < T ? t0 + span : T) - 1;
    int n_hi, n_lo;
    if (!sc.wg_range(t0, t_last, &n_hi, &n_lo)) continue;
    auto r0_of_wave = [&](int wv) { return t0 + wv * R; };
    const SlotPlan sp = make_slot_plan(sc, r0_of_wave, n_hi, n_lo);
    const int nslot = sp.slots();
    for (int w = 0; w < kWaves; ++w) {
      const int r0 = t0 + w * R;
      if (r0 >= T) continue;
      bool student_done = false;
      const WaveSlots ws(sc, r0);  // the kernel's closed form
      // past the last slot the kernel's words load and fold nothing
      for (int k = nslot; k < nslot + 2; ++k)
        if (slot_word(sc, sp, ws, nslot, true, T, k) != 0)
          return fail(TTCD_ERR_UNSUPPORTED, "schedule error: word of slot %d past the end", k);
      for (int k = 0; k < nslot; ++k) {
        bool repeat;
        const int n = sp.tile(k, &repeat);
        const int j0 = sc.tile_start(n);
        const int act = slot_action(sc, r0, j0, repeat);
        if (ws.act(n, repeat) != act)
          return fail(TTCD_ERR_UNSUPPORTED, "schedule error: closed-form action %d != %d (r0=%d n=%d)",
                      ws.act(n, repeat), act, r0, n);
        // The kernel reads the slot only through its word: decode it and
        // check every field against the plan and the per-tile predicates.
        const uint32_t wd = slot_word(sc, sp, ws, nslot, true, T, k);
        const bool interior = j0 >= 0 && j0 + kBlockN <= T;
        if (n < 0 || word_tile(wd) != n || word_j0(sc, wd) != j0 || !(wd & kWordLoad) ||
            ((wd & kWordInterior) != 0) != interior)
          return fail(TTCD_ERR_UNSUPPORTED, "schedule error: slot word tile/load (r0=%d k=%d)", r0, k);
        if (slot_word(sc, sp, ws, nslot, false, T, k) != (wd & ~63u) + (wd & (kWordLoad | kWordInterior)))
          return fail(TTCD_ERR_UNSUPPORTED, "schedule error: idle-wave word (r0=%d k=%d)", r0, k);
        const bool w_active = (wd & kWordActive) != 0;
        if (w_active != (act != kSkip) ||
            ((wd & kWordFar) != 0) != (act == kBand2 || act == kFar) ||
            ((wd & kWordLast) != 0) != (act == kStudentLast))
          return fail(TTCD_ERR_UNSUPPORTED, "schedule error: slot word action (r0=%d k=%d)", r0, k);
        if (act != kSkip) {
          const Band b = (act == kBand2 || act == kFar) ? sc.p2 : sc.p1;
          const Band wb = word_band(sc, wd);
          if (wb.lo != b.lo || wb.hi != b.hi)
            return fail(TTCD_ERR_UNSUPPORTED, "schedule error: slot word band (r0=%d n=%d)", r0, n);
          const bool need_mask = !wave_full(r0, R, b, j0);
          if (ws.mask(n, act) != need_mask || ((wd & kWordMask) != 0) != need_mask)
            return fail(TTCD_ERR_UNSUPPORTED, "schedule error: closed-form mask (r0=%d n=%d)", r0, n);
        } else if (wd & kWordMask) {
          return fail(TTCD_ERR_UNSUPPORTED, "schedule error: mask on a skipped slot (r0=%d n=%d)", r0, n);
        }
        // From here on the replay folds what the word says, as the kernel does.
        if (!w_active) continue;
        const bool far = (wd & kWordFar) != 0;
        if (sc.dual && !far && student_done)
          return fail(TTCD_ERR_UNSUPPORTED, "schedule error: student keys after emit (r0=%d k=%d)",
                      r0, k);
        if (sc.dual && far && !student_done)
          return fail(TTCD_ERR_UNSUPPORTED, "schedule error: far keys before emit (r0=%d k=%d)",
                      r0, k);
        const Band band = word_band(sc, wd);
        const bool full = (wd & kWordMask) == 0;
        const int wj0 = word_j0(sc, wd);
        for (int i = r0; i < r0 + R && i < T; ++i) {
          for (int j = wj0; j < wj0 + kBlockN; ++j) {
            if (!(full || visible(i, j, band, T))) continue;
            if (j < 0 || j >= T)
              return fail(TTCD_ERR_UNSUPPORTED, "schedule error: key %d out of range", j);
            int32_t* cnt = far ? counts_far : counts_near;
            cnt[(int64_t)i * T + j] += 1;
          }
        }
        if (wd & kWordLast) student_done = true;
      }
      if (sc.dual && !student_done && sc.p1.lo < sc.p1.hi)
        return fail(TTCD_ERR_UNSUPPORTED, "schedule error: student output never written (r0=%d)",
                    r0);
    }
  }
  return ok();
}

ttcd_status ttcd_attn_block_coverage(int npair, int nqb, int ngrp, int packed, int32_t* counts,
                                     int64_t xcd_work[8]) {
  if (npair < 1 || nqb < 1 || ngrp < 1 || !counts || !xcd_work)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "bad block coverage arguments");
  const ttcd::BlockMap m = 
      ttcd::make_block_map(npair, packed & 1 ? 1 : npair, nqb, ngrp, packed == 1, packed == 2);
  for (int g = 0; g < m.launched(); ++g) {
    int pair, qb, grp;
    if (!m.locate(g, &pair, &qb, &grp)) continue;
    if (pair < 0 || pair >= npair || qb < 0 || qb >= nqb || grp < 0 || grp >= ngrp)
      return fail(TTCD_ERR_UNSUPPORTED, "block map error: id %d -> (%d, %d, %d)", g, pair, qb, grp);
    counts[((int64_t)pair * nqb + qb) * ngrp + grp] += 1;
    xcd_work[g % ttcd::kXcd] += packed == 2 ? 1 : (int64_t)(qb + 1) * (packed == 3 ? pair + 1 : 1);
  }
  return ok();
}

ttcd_status ttcd_kv4_block_stages(int t0, int t1) {
  if (t0 < 0 || t1 <= t0 || t1 > ttcd::kKv4MaxLength)
    return fail(TTCD_ERR_INVALID_ARGUMENT, "need 0 <= t0 < t1 <= 2^30");
  struct Stage {
    int holds = -1, written = -1, read = -1;  // a tile; intervals between barriers
  } k[2], v[2];
  int interval = 0, folded = t0, bad = -1;
  auto load = [&](int& codes, int tile) {
    if (tile < t0 || tile >= t1) bad = tile;
    codes = tile;
  };
  auto store = [&](Stage* stages, int codes, int tile) {
    Stage& s = stages[tile & 1];
    if (s.read == interval || s.written == interval) bad = tile;
    s.holds = codes;
    s.written = interval;
  };
  auto read = [&](Stage* stages, int tile) {
    Stage& s = stages[tile & 1];
    if (s.holds != tile || s.written == interval) bad = tile;
    s.read = interval;
  };
  int s0 = -1, s1 = -1;  // whose scores these are
  ttcd::kv4_sweep<int>(
      t0, t1, s0, s1, load, load, [&](int codes, int tile) { store(k, codes, tile); },
      [&](int codes, int tile) { store(v, codes, tile); },
      [&](int& s, int tile) {
        read(k, tile);
        s = tile;
      },
      [&](int& s, int tile) {
        if (s != tile) bad = tile;
      },
      [&](int& s, int tile) {
        read(v, tile);
        if (s != tile || tile != folded++) bad = tile;
      },
      [&] { ++interval; });
  if (bad >= 0 || folded != t1)
    return fail(TTCD_ERR_UNSUPPORTED, "stage error: tile %d of %d .. %d", bad, t0, t1 - 1);
  return ok();
}

}  // extern "C"
