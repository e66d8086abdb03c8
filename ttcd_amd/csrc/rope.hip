// rope.hip - rotary embedding of queries and keys at given positions, on gfx950: half
// and interleaved pairs, the first 2 n channels of a head, any frequencies.
//
// Pair i of the first 2 n channels, (x_i, x_{n+i}) or (x_2i, x_{2i+1}), turns by the
// angle p f_i: y0 = x0 c - x1 s, y1 = x0 s + x1 c with c = scale cos, s = scale sin
// (the inverse: by -p f_i); channels from 2 n on are copied. p f_i is taken in 64 bits, its
// product's remainder beside it (from position 2^29 on it has more than 53 bits), and brought
// into a quarter turn there (a float holds the angle of position 10^6 to 0.03), cosine and
// sine of the rest in 32; the products are 32 bits, rounded to the type once.
//
// A task is a vector of 16 bytes of a head (interleaved pairs, copies) or two of them
// (halves); tasks run over heads and then tokens, 512 in a row a workgroup, two a
// thread, whose loads are issued before the angles are computed. A workgroup finds the
// cosines of its tokens (a few) once, in LDS, and all heads of both tensors read them
// there: no tables, which at position 10^6 would be 256 MB.
//
// Bound by the bytes: 65536 tokens of 16 + 8 heads of 128 channels, 805 MB in 150 us (5.4
// TB/s, a copy's rate); 512 tokens 4.6 us.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "internal.h"

namespace ttcd {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeIter = 2;
constexpr int kRopeTasks = kRopeThreads * kRopeIter;

// A position as a double, exact below 2^53.
__device__ __forceinline__ double position(const RopeArgs& a, int b, int t) {
  if (a.positions == nullptr) return (double)(a.offset + t);
  const int64_t at = b * a.pos_sb + t * a.pos_st;
  return a.pos64 ? (double)static_cast<const int64_t*>(a.positions)[at]
                 : (double)static_cast<const int32_t*>(a.positions)[at];
}

// cos and sin of p f. In a quarter turn's half at most, by their series: the next terms are
// below 2^-29 there. Exact in p f, of which `lo` is what 53 bits lack, while it is below 2^53
// in size: then k is a whole number that a double holds, though far out one that is up to 2
// off, since 2 / pi is rounded, which a second step takes from the rest.
__device__ __forceinline__ float2 cos_sin(double p, double f) {
  const double angle = p * f, lo = fma(p, f, -angle);
  const double k = rint(angle * 0.63661977236758134308);  // 2 / pi
  // pi / 2 in two doubles, the second what the first lacks
  double r = fma(-k, 1.5707963267948965580, angle);
  r = fma(-k, 6.1232339957367660359e-17, r) + lo;
  const double more = rint(r * 0.63661977236758134308);
  r = fma(-more, 1.5707963267948965580, r);
  const float x = (float)r, x2 = x * x;
  float s = 2.7557319e-6f;
  s = fmaf(s, x2, -1.9841270e-4f);
  s = fmaf(s, x2, 8.3333333e-3f);
  s = fmaf(s, x2, -1.6666667e-1f);
  s = fmaf(s * x2, x, x);
  float c = -2.7557319e-7f;
  c = fmaf(c, x2, 2.4801587e-5f);
  c = fmaf(c, x2, -1.3888889e-3f);
  c = fmaf(c, x2, 4.1666667e-2f);
  c = fmaf(c, x2, -0.5f);
  c = fmaf(c, x2, 1.0f);
  const int quarter = (int)((int64_t)k + (int64_t)more) & 3;
  const float cs = quarter & 1 ? s : c, sn = quarter & 1 ? c : s;
  return {quarter == 1 || quarter == 2 ? -cs : cs, quarter >= 2 ? -sn : sn};
}

template <typename T, int N>
struct Vec {
  T e[N];
};

// The rotation of a vector whose channels the border of what turns may cut: the halves' partners
// one by one from the head (lines that are there), interleaved ones from the vector.
template <typename T, int VE, bool PAIRS>
__device__ __forceinline__ Vec<T, VE> rotate_cut(const Vec<T, VE>& x, const T* head, int d0, int n,
                                                 const float2* turn) {
  Vec<T, VE> y = x;
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    const int d = d0 + e;
    if (d >= 2 * n) break;
    const bool second = PAIRS ? d % 2 : d >= n;
    const float2 cs = turn[PAIRS ? d / 2 : second ? d - n : d];
    const T other = PAIRS ? x.e[e ^ 1] : head[second ? d - n : d + n];
    const float v = static_cast<float>(x.e[e]), w = static_cast<float>(other);
    y.e[e] = static_cast<T>(second ? fmaf(w, cs.y, v * cs.x) : fmaf(v, cs.x, -(w * cs.y)));
  }
  return y;
}

// VE elements of 16 bytes (all strides and addresses allow it), or 1. PAIRS: interleaved. CUT:
// the border of what turns lies within a vector.
template <typename T, int VE, bool PAIRS, bool CUT>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a) {
  typedef Vec<T, VE> V __attribute__((aligned(VE * sizeof(T))));
  extern __shared__ float2 turns[];  // (tokens, n)
  const int n = a.n;
  const int64_t first = (int64_t)blockIdx.x * kRopeTasks;
  const int64_t token0 = first / a.per_token.d;
  const int at0 = (int)(first - token0 * a.per_token.d);
  constexpr int R = CUT || (PAIRS && VE > 1) ? 1 : 2;  // vectors of a task
  // tasks of a head that turn
  const int turning = CUT ? (2 * n + VE - 1) / VE : PAIRS && VE > 1 ? 2 * n / VE : n / VE;

  V x[kRopeIter][2];
  int64_t dst[kRopeIter];
  int pair[kRopeIter], step[kRopeIter], tok[kRopeIter];
  T* out[kRopeIter];
  const T* in[kRopeIter];
#pragma unroll
  for (int it = 0; it < kRopeIter; ++it) {
    const int local = at0 + it * kRopeThreads + threadIdx.x;
    tok[it] = a.per_token.quot(local);
    const int64_t token = token0 + tok[it];
    out[it] = nullptr;
    if (token >= a.tokens) continue;
    const int in_token = local - tok[it] * (int)a.per_token.d;
    const int head = a.per_head.quot(in_token), u = in_token - head * (int)a.per_head.d;
    const int b = a.T.quot((int)token), t = (int)token - b * (int)a.T.d;
    const bool is_k = head >= a.Hq;
    const int h = is_k ? head - a.Hq : head;
    const T* src = is_k ? static_cast<const T*>(a.k) + b * a.k_sb + t * a.k_st + h * a.k_sh
                        : static_cast<const T*>(a.q) + b * a.q_sb + t * a.q_st + h * a.q_sh;
    out[it] = is_k ? static_cast<T*>(a.k_out) + b * a.ko_sb + t * a.ko_st + h * a.ko_sh
                   : static_cast<T*>(a.q_out) + b * a.qo_sb + t * a.qo_st + h * a.qo_sh;
    // where the task's first vector lies, how far the second, and the first pair (-1: a copy)
    int d0;
    in[it] = src;
    if (CUT) {
      pair[it] = u < turning ? 0 : -1;
      d0 = u * VE;
      step[it] = 0;
    } else if (u < turning) {
      pair[it] = PAIRS && VE > 1 ? u * VE / 2 : u * VE;
      d0 = PAIRS ? u * VE * (VE > 1 ? 1 : 2) : u * VE;
      step[it] = PAIRS ? 1 : n;
    } else {
      pair[it] = -1;
      d0 = 2 * n + (u - turning) * VE;
      step[it] = 0;
    }
    dst[it] = d0;
    x[it][0] = *reinterpret_cast<const V*>(src + d0);
    if constexpr (R == 2) x[it][1] = *reinterpret_cast<const V*>(src + d0 + step[it]);
  }
  {
    const int last = a.per_token.quot(at0 + kRopeTasks - 1);  // of the tokens from token0 on
    const int tokens = (int)min((int64_t)last + 1, a.tokens - token0);
    for (int i = threadIdx.x; i < tokens * n; i += kRopeThreads) {
      const int j = a.div_n.quot(i), f = i - j * n;
      const int token = (int)token0 + j, b = a.T.quot(token), t = token - b * (int)a.T.d;
      float2 cs = cos_sin(position(a, b, t), (double)a.inv_freq[f]);
      cs.x *= a.scale;
      cs.y *= a.inverse ? -a.scale : a.scale;
      turns[i] = cs;
    }
  }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < kRopeIter; ++it) {
    if (out[it] == nullptr) continue;
    V y0 = x[it][0], y1 = y0;
    if constexpr (R == 2) y1 = x[it][1];
    if (CUT) {
      if (pair[it] >= 0)
        y0 = rotate_cut<T, VE, PAIRS>(x[it][0], in[it], (int)dst[it], n, turns + tok[it] * n);
    } else if (pair[it] >= 0) {
      const float2* turn = turns + tok[it] * n + pair[it];
      auto rotate = [&](float2 cs, T& e0, T& e1) __attribute__((always_inline)) {
        const float v0 = static_cast<float>(e0), v1 = static_cast<float>(e1);
        e0 = static_cast<T>(fmaf(v0, cs.x, -(v1 * cs.y)));
        e1 = static_cast<T>(fmaf(v0, cs.y, v1 * cs.x));
      };
      if constexpr (R == 1) {
#pragma unroll
        for (int e = 0; e < VE / 2; ++e) rotate(turn[e], y0.e[2 * e], y0.e[2 * e + 1]);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) rotate(turn[e], y0.e[e], y1.e[e]);
      }
    }
    *reinterpret_cast<V*>(out[it] + dst[it]) = y0;
    if constexpr (R == 2)
      if (pair[it] >= 0) *reinterpret_cast<V*>(out[it] + dst[it] + step[it]) = y1;
  }
}

template <typename T, int VE, bool CUT>
hipError_t launch_layout(const RopeArgs& args, bool pairs, hipStream_t st) {
  RopeArgs a = args;
  // tasks of a head: of the channels that turn, then copies
  const int turning = pairs && VE > 1 ? 2 * a.n / VE : a.n / VE;
  const int per_head = CUT ? a.D / VE : turning + (a.D - 2 * a.n) / VE;
  const int per_token = per_head * (a.Hq + a.Hkv);
  a.per_head = make_fast_div(per_head);
  a.per_token = make_fast_div(per_token);
  a.div_n = make_fast_div(a.n);
  const int64_t blocks = (a.tokens * per_token + kRopeTasks - 1) / kRopeTasks;
  // a launch has fewer than 2^32 threads
  if (blocks >= (int64_t(1) << 32) / kRopeThreads) return hipErrorInvalidConfiguration;
  // tokens that 512 tasks in a row can touch
  const int64_t span = std::min((int64_t)(kRopeTasks - 1 + per_token - 1) / per_token + 1, a.tokens);
  const size_t lds = (size_t)span * a.n * sizeof(float2);
  if (pairs)
    hipLaunchKernelGGL((rope_kernel<T, VE, true, CUT>), dim3((unsigned)blocks), dim3(kRopeThreads), lds,
                       st, a);
  else
    hipLaunchKernelGGL((rope_kernel<T, VE, false, CUT>), dim3((unsigned)blocks), dim3(kRopeThreads),
                       lds, st, a);
  return hipGetLastError();
}

// Vectors where heads are whole ones at multiples of 16 bytes: two of them a task where the
// border of what turns is one of theirs too, else with a partner read apart, which needs
// outputs that are not the inputs (12382 tokens of 6 heads of 64, 7 pairs each: 11.2 us, one
// element a task 17.5).
template <typename T>
hipError_t launch_typed(const RopeArgs& a, bool pairs, hipStream_t st) {
  constexpr int VE = 16 / sizeof(T);
  const int64_t strides[] = {a.q_sb,  a.q_st,  a.q_sh,  a.k_sb,  a.k_st,  a.k_sh,
                             a.qo_sb, a.qo_st, a.qo_sh, a.ko_sb, a.ko_st, a.ko_sh};
  bool wide = a.D % VE == 0;
  for (int64_t s : strides) wide = wide && s % VE == 0;
  for (const void* p : {a.q, a.k, (const void*)a.q_out, (const void*)a.k_out})
    wide = wide && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
  if (!wide) return launch_layout<T, 1, false>(a, pairs, st);
  if ((pairs ? 2 * a.n : a.n) % VE == 0) return launch_layout<T, VE, false>(a, pairs, st);
  if (a.q == a.q_out || (a.k != nullptr && a.k == a.k_out))
    return launch_layout<T, 1, false>(a, pairs, st);
  return launch_layout<T, VE, true>(a, pairs, st);
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, bool pairs, Elem dtype, hipStream_t stream) {
  switch (dtype) {
    case Elem::BF16: return launch_typed<__bf16>(a, pairs, stream);
    case Elem::F16: return launch_typed<_Float16>(a, pairs, stream);
    default: return launch_typed<float>(a, pairs, stream);
  }
}

}  // namespace ttcd
