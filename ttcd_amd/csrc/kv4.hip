// kv4.hip - a key / value cache held in 4 bits: quantising new rows into it,
// reading them back, attention over it, the attention weight of its keys and
// the eviction of those with the least, on gfx950.
//
// Format. Blocks of 32 channels of one position share a power of two 2^e
// (byte e + 127); a value is a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6
// (e2m1), rounded to nearest even. e is the least with no value over 6 2^e: the
// largest value of a block weighs most in a dot product. Clipped is only what lies
// above 6 times the largest 2^e: infinities, f16 above 49152 (65504, the largest,
// loses a quarter) and bf16 above 1.5 2^127. Scales are powers of two because every
// held value is then exact in bf16 and f16 (the range of e sees to that, below): gfx950
// converts pairs of codes to either in one instruction, products with q are exact in an
// MFMA, and no code depends on how a division rounds.
//
// Position p is in slot p % C, C a multiple of 32, so 32 positions from a
// multiple of 32 on are 32 slots in a row, wherever the ring has wrapped. A
// key is the A operand of K q^T as it lies: lane (m, quarter) of a 16-key tile
// reads a quarter of row m. A value has to be read by channel over 8 keys, so
// words of 8 channels of 4 neighbouring slots lie side by side: lane r reads
// the words of channels 8 r .. of 4 keys in 16 bytes, and a transposed pair of
// conversions is one permute.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "internal.h"
#include "kv4_sweep.h"
#include "wave.h"

namespace ttcd {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLog2e = 1.44269504088896341f;

// The exponents of a scale keep 0.5 2^e .. 6 2^e normal numbers of bf16, and
// numbers (normal or not) of f16.
template <typename T>
struct Fmt;
template <>
struct Fmt<__bf16> {
  typedef bf16x2 v2;
  typedef bf16x8 v8;
  static constexpr int kLoExp = -125, kHiExp = 125;
  static constexpr float kBias = 0.f;
  template <int J>
  static __device__ __forceinline__ uint32_t cvt(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, J));
  }
  template <int J>
  static __device__ __forceinline__ uint32_t pack(uint32_t old, uint32_t pair, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(bf16x2, pair), s, J);
  }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float lo(uint32_t p) { return __uint_as_float(p << 16); }
  static __device__ __forceinline__ float hi(uint32_t p) {
    return __uint_as_float(p & 0xffff0000u);
  }
};
template <>
struct Fmt<_Float16> {
  typedef f16x2 v2;
  typedef f16x8 v8;
  static constexpr int kLoExp = -23, kHiExp = 13;
  static constexpr float kBias = 7.f;
  template <int J>
  static __device__ __forceinline__ uint32_t cvt(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, J));
  }
  template <int J>
  static __device__ __forceinline__ uint32_t pack(uint32_t old, uint32_t pair, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(f16x2, pair), s, J);
  }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float lo(uint32_t p) {
    return static_cast<float>(__builtin_bit_cast(f16x2, p)[0]);
  }
  static __device__ __forceinline__ float hi(uint32_t p) {
    return static_cast<float>(__builtin_bit_cast(f16x2, p)[1]);
  }
};

__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __uint_as_float(byte << 23);
}

// scale_of byte J of w, in one instruction.
template <int J>
__device__ __forceinline__ float scale_byte(uint32_t w, uint32_t shift23) {
  uint32_t r;
  if constexpr (J == 0)
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_0" : "=v"(r) : "v"(shift23), "v"(w));
  else if constexpr (J == 1)
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_1" : "=v"(r) : "v"(shift23), "v"(w));
  else if constexpr (J == 2)
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_2" : "=v"(r) : "v"(shift23), "v"(w));
  else
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_3" : "=v"(r) : "v"(shift23), "v"(w));
  return __uint_as_float(r);
}
__device__ __forceinline__ void scales4(uint32_t w, float* s) {
  const uint32_t shift = 23;
  s[0] = scale_byte<0>(w, shift);
  s[1] = scale_byte<1>(w, shift);
  s[2] = scale_byte<2>(w, shift);
  s[3] = scale_byte<3>(w, shift);
}

// 8 codes as 8 values, channel 0 in the low half of the first register.
template <typename T>
__device__ __forceinline__ u32x4 values8(uint32_t w, float s) {
  return u32x4{Fmt<T>::template cvt<0>(w, s), Fmt<T>::template cvt<1>(w, s),
               Fmt<T>::template cvt<2>(w, s), Fmt<T>::template cvt<3>(w, s)};
}

template <typename T>
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
  typename Fmt<T>::v2 v;
  v[0] = static_cast<T>(a);
  v[1] = static_cast<T>(b);
  return __builtin_bit_cast(uint32_t, v);
}

// Positions of a sequence, as its lengths entry says (a malformed one is
// brought into range: no access depends on its value).
__device__ __forceinline__ int length_of(const int32_t* lengths, int b) {
  const int n = lengths[b];
  return n < 0 ? 0 : (n > kKv4MaxLength ? kKv4MaxLength : n);
}

__device__ __forceinline__ int count_of(const int32_t* counts, int b, int T) {
  if (counts == nullptr) return T;
  const int n = counts[b];
  return n < 0 ? 0 : (n > T ? T : n);
}

// The length of a sequence after n more positions. One that passes the limit drops by a
// multiple of the capacity to no less than the capacity: what is held, in which slot and
// how far before what else stays as it is, and a ring may go on for ever. (Of a capacity
// above half the limit there is no such length; it stays at the limit.)
__device__ __forceinline__ int length_after(int len, int n, int C) {
  const uint32_t total = (uint32_t)len + (uint32_t)n;
  if (total <= (uint32_t)kKv4MaxLength) return (int)total;
  if (C > kKv4MaxLength / 2) return kKv4MaxLength;
  return C + (int)(total % (uint32_t)C);
}

// ---------------------------------------------------------------------------
// Append. 4 slots in a row (a word group of the values) of one head are D / 2
// threads, each with 8 channels of one of them: 16 bytes in, 4 out, of a key and
// of a value. Threads go by channel first for the keys and by slot first for the
// values, as either lies in the cache, so a wavefront's stores are whole lines.
// The 4 threads of a block find its largest magnitude by two shuffles. Bound by its
// traffic and by its launch: 4096 positions of 8 heads of 128 take 7.0 us (21 MB, 3.0
// TB/s, of which some 3 us are any launch's); a token of 32 sequences 3.5.
template <typename T>
__device__ __forceinline__ uint32_t quantise8(u32x4 x, int d1, int d2, uint32_t* scale) {
  // NaN counts as 0: the format holds none
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float lo = Fmt<T>::lo(x[j]), hi = Fmt<T>::hi(x[j]);
    if (!(lo == lo)) x[j] &= 0xffff0000u;
    if (!(hi == hi)) x[j] &= 0x0000ffffu;
    top = fmaxf(top, fmaxf(fabsf(lo), fabsf(hi)));  // fmaxf passes NaN over
  }
  top = fmaxf(top, __shfl_xor(top, d1));
  top = fmaxf(top, __shfl_xor(top, d2));
  // top = 1.f 2^E <= 1.5 2^(e + 2)
  const uint32_t bits = __float_as_uint(top);
  int exp = (int)(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x400000u ? 2 : 1);
  exp = min(max(exp, Fmt<T>::kLoExp), Fmt<T>::kHiExp);
  *scale = (uint32_t)(exp + 127);
  const float s = scale_of(*scale);
  uint32_t w = Fmt<T>::template pack<0>(0u, x[0], s);
  w = Fmt<T>::template pack<1>(w, x[1], s);
  w = Fmt<T>::template pack<2>(w, x[2], s);
  return Fmt<T>::template pack<3>(w, x[3], s);
}

// Thread i of D / 2 of the group-th group of slots from the sequence's end on.
template <typename T, int D>
__device__ __forceinline__ void append_words(const Kv4AppendArgs& a, int b, int h, int len,
                                             int n_new, int group, int i) {
  constexpr int R = D / 8;
  const int ek = i / R, rk = i % R, ev = i & 3, rv = i >> 2;
  const int p = ((len >> 2) + group) * 4;
  const int tk = p + ek - len, tv = p + ev - len;
  const bool on_k = tk >= 0 && tk < n_new, on_v = tv >= 0 && tv < n_new;
  u32x4 xk = {0u, 0u, 0u, 0u}, xv = xk;
  if (on_k)
    xk = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.k) + b * a.k_sb + tk * a.k_st +
                                         h * a.k_sh + rk * 8);
  if (on_v)
    xv = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.v) + b * a.v_sb + tv * a.v_st +
                                         h * a.v_sh + rv * 8);
  uint32_t sk, sv;
  const uint32_t wk = quantise8<T>(xk, 1, 2, &sk), wv = quantise8<T>(xv, 4, 8, &sv);
  const int64_t row = ((int64_t)b * a.c.H + h) * a.c.C + (uint32_t)p % (uint32_t)a.c.C;
  if (on_k) {
    *reinterpret_cast<uint32_t*>(a.c.kc + ((row + ek) * R + rk) * 4) = wk;
    if ((rk & 3) == 0) a.c.ks[(row + ek) * (D / 32) + (rk >> 2)] = (uint8_t)sk;
    if (a.weights != nullptr && rk == 0) a.weights[row + ek] = 0.f;
  }
  if (on_v) {
    const int64_t g = row >> 2;
    *reinterpret_cast<uint32_t*>(a.c.vc + ((g * R + rv) * 4 + ev) * 4) = wv;
    if ((rv & 3) == 0) a.c.vs[(g * (D / 32) + (rv >> 2)) * 4 + ev] = (uint8_t)sv;
  }
}

// SMALL: one workgroup writes all of a sequence's rows and then its length;
// else the lengths are another launch's.
template <typename T, int D, bool SMALL>
__global__ __launch_bounds__(SMALL ? 1024 : 256) void append_kernel(Kv4AppendArgs a) {
  constexpr int PER = D / 2;  // threads per group of 4 slots
  const int b = SMALL ? blockIdx.x : blockIdx.y;
  const int len = length_of(a.c.len, b), n_new = count_of(a.counts, b, a.T);
  const int groups = ((len + n_new + 3) >> 2) - (len >> 2);
  if constexpr (SMALL) {
    const int items = groups * a.c.H * PER;
    for (int i = threadIdx.x; i < items; i += 1024) {
      const int g = i / PER;
      append_words<T, D>(a, b, g % a.c.H, len, n_new, g / a.c.H, i % PER);
    }
    __syncthreads();  // every thread has read the length
    if (threadIdx.x == 0) a.c.len[b] = length_after(len, n_new, a.c.C);
  } else {
    const int g = (int)(((int64_t)blockIdx.x * 256 + threadIdx.x) / PER);
    if (g < groups * a.c.H)
      append_words<T, D>(a, b, g % a.c.H, len, n_new, g / a.c.H, threadIdx.x % PER);
  }
}

__global__ void advance_kernel(Kv4AppendArgs a) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < a.c.B)
    a.c.len[b] = length_after(length_of(a.c.len, b), count_of(a.counts, b, a.T), a.c.C);
}

template <typename T, int D>
hipError_t launch_append(const Kv4AppendArgs& a, hipStream_t st) {
  const int64_t items = ((int64_t)(a.T + 3) / 4 + 1) * a.c.H * (D / 2);
  if (items <= 8 * 1024) {
    hipLaunchKernelGGL((append_kernel<T, D, true>), dim3(a.c.B), dim3(1024), 0, st, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((append_kernel<T, D, false>), dim3((unsigned)((items + 255) / 256), a.c.B),
                     dim3(256), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(advance_kernel, dim3((a.c.B + 255) / 256), dim3(256), 0, st, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Read back the last `count` positions. A thread takes 8 channels of the 4
// slots of a group: 16 bytes of value codes in one load, 4 rows of 16 bytes out
// for keys and for values each. Bound by its traffic: 16384 positions of 2 x 8 heads of
// 128, 170 MB, in 27.0 us (6.3 TB/s).
template <typename T, int D>
__global__ __launch_bounds__(256) void read_kernel(Kv4ReadArgs a) {
  constexpr int R = D / 8, BL = D / 32;
  const int b = blockIdx.y;
  const int len = length_of(a.c.len, b);
  const int p0 = len - a.count;  // may be below 0
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int r = (int)(i % R), h = (int)(i / R % a.c.H);
  const int64_t gi = i / ((int64_t)R * a.c.H);
  const int p = (int)((int64_t)(p0 >> 2) + gi) * 4;  // floor: aligned below 0 too
  if (p >= len) return;
  const int first = len > a.c.C ? len - a.c.C : 0;
  const bool any = p + 3 >= first;  // then p >= 0: first is one of the 4 at the least
  u32x4 vw = {0u, 0u, 0u, 0u};
  uint32_t vsw = 0u, kw[4], ksb[4];
  if (any) {
    const int64_t row = ((int64_t)b * a.c.H + h) * a.c.C + p % a.c.C, g = row >> 2;
    vw = *reinterpret_cast<const u32x4*>(a.c.vc + (g * R + r) * 16);
    vsw = *reinterpret_cast<const uint32_t*>(a.c.vs + (g * BL + (r >> 2)) * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      kw[e] = *reinterpret_cast<const uint32_t*>(a.c.kc + ((row + e) * R + r) * 4);
      ksb[e] = a.c.ks[(row + e) * BL + (r >> 2)];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int t = p + e - p0;
    if (t < 0 || t >= a.count) continue;
    const int64_t at = ((((int64_t)b * a.count + t) * a.c.H + h) * R + r) * 8;
    u32x4 k = {0u, 0u, 0u, 0u}, v = k;
    if (any && p + e >= first) {
      k = values8<T>(kw[e], scale_of(ksb[e]));
      v = values8<T>(vw[e], scale_of((vsw >> (8 * e)) & 255u));
    }
    *reinterpret_cast<u32x4*>(static_cast<T*>(a.k) + at) = k;
    *reinterpret_cast<u32x4*>(static_cast<T*>(a.v) + at) = v;
  }
}

template <typename T, int D>
hipError_t launch_read(const Kv4ReadArgs& a, hipStream_t st) {
  const int64_t items = ((int64_t)(a.count + 3) / 4 + 1) * a.c.H * (D / 8);
  hipLaunchKernelGGL((read_kernel<T, D>), dim3((unsigned)((items + 255) / 256), a.c.B), dim3(256),
                     0, st, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Attention. The rows of a key / value head are its group's query heads times
// the new positions; a wavefront holds NT tiles of 16 of them and sweeps tiles
// of 32 keys: S^T = K Q^T (16x16x32: keys x rows), online softmax over the
// registers, O^T = V^T P^T with P as it lies after the first product (the keys
// of a lane's quarter are the 8 that the second product wants from it, in the
// order in which it then reads V). The 8 wavefronts of a workgroup take every
// eighth tile of its part of the keys and are added through LDS; the parts of a
// row are added by a second launch (by the last workgroup to end, it cost 7 us more
// of 63 with write-through stores, and fences between the XCDs' caches 400).
//
// The reference maximum of a row moves only where a score exceeds it by more
// than 8 (log2): up to then probabilities stay under 2^8, and the four
// quarters of a row need not agree on a maximum at every tile. P is rounded to
// the inputs' type for the product, as the prefill kernels round it; sums and
// statistics are fp32. In f16 the reference is 7 lower (probabilities up to
// 2^15), so that small ones keep 7 bits more above f16's least step.
//
// Bound by the codes it reads: a token of 32 sequences of up to 16384 keys, 16/8 heads
// of 128, 294 MB in 53 us (5.6 TB/s), and 4.8 for the sum of its 4 parts. Loads are 16
// bytes a lane straight into operands, a tile ahead; nothing is staged, as nothing is
// shared. With 4 wavefronts a workgroup the parts and their sums double (64.9 against
// 63.5 us in all; one token of 257 keys 5.2 against 4.8).
//
// FAR: a cache that the last-level cache cannot hold beside anything else is read past
// the caches (us, two of them in turn: the token of 32 sequences 63 -> 58, of 8 of 16384
// keys, 143 MB, 39 -> 37), a smaller one through them. Of 44 MB that pays where it is
// there from the call before (18.4 us, past them 18.9) and not where 350 MB of others
// have passed by (20.5, past them 19.7), as a model's other layers do; 9 MB the same (9.4
// and 9.8; 10.2 and 9.7). By the capacity: the lengths are on the GPU.
//
// Over a tree (kv4_tree_attn) the rows are its nodes, and the draft's tiles come behind the
// cache's. 16 nodes of 8 sequences of up to 16000 keys, 77 MB: 24.5 us and 5.2 for the sum of
// the parts; 8 nodes of 32, 294 MB: 59 in all (5.0 TB/s). Workgroups of 4 wavefronts, two of
// them on a CU, parts dealt by the lengths and two tiles on their way brought the first from
// 50.6 in all to 30.4.
constexpr int kRowWaves = 8;
constexpr int kTreeWaves = 4;  // of a workgroup over a tree's rows

template <typename Args>
constexpr bool is_tree = false;
template <>
constexpr bool is_tree<Kv4TreeArgs> = true;

template <bool FAR, typename V>
__device__ __forceinline__ V codes(const V* p) {
  if constexpr (FAR)
    return __builtin_nontemporal_load(p);
  else
    return *p;
}

template <int D>
struct KvTile {
  u32x4 v[2];
  uint32_t vs[2];
  u32x4 k[2];  // D = 64: the first two words
  uint32_t ks[2];
};

template <typename T, int D, int NT>
struct RowState {
  f32x4 o[NT][D / 16];
  float m[NT], l[NT];
};

// 8 keys' values of channels (2 j, 2 j + 1) of the words w0, w1 as the two A
// operands of those channels.
template <typename T, int J>
__device__ __forceinline__ void transpose_pair(const uint32_t (&w)[8], const float (&s)[8],
                                               u32x4* even, u32x4* odd) {
  uint32_t c[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = Fmt<T>::template cvt<J>(w[e], s[e]);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    (*even)[e] = __builtin_amdgcn_perm(c[2 * e + 1], c[2 * e], 0x05040100u);
    (*odd)[e] = __builtin_amdgcn_perm(c[2 * e + 1], c[2 * e], 0x07060302u);
  }
}

// What a tile's rows see of it: keys lo .. hi of each row's, any_lo .. any_hi of anyone's.
template <int NT>
struct RangeMask {
  const int (&lo)[NT], (&hi)[NT];
  int p0, any_lo, any_hi;
  __device__ __forceinline__ bool row(int nt, int key) const {
    return p0 + key >= lo[nt] && p0 + key <= hi[nt];
  }
  __device__ __forceinline__ bool any(int key) const {
    return p0 + key >= any_lo && p0 + key <= any_hi;
  }
};
// The same as a bit a key.
template <int NT>
struct BitMask {
  uint32_t rows[NT], all;
  __device__ __forceinline__ bool row(int nt, int key) const { return (rows[nt] >> key) & 1; }
  __device__ __forceinline__ bool any(int key) const { return (all >> key) & 1; }
};

template <typename T, int D, int NT, typename Mask>
__device__ __forceinline__ void fold_tile(RowState<T, D, NT>& st, const KvTile<D>& kv,
                                          const u32x4 (&q)[NT][D / 32], float c, bool masked,
                                          const Mask& mask, int lane) {
  constexpr int STEPS = D / 32, NM = D / 16;
  const int quarter = lane >> 4;
  f32x4 s[NT][2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const float sc = scale_of(kv.ks[g]);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const u32x4 kf = values8<T>(kv.k[g][i], sc);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        s[nt][g] = Fmt<T>::mfma(kf, q[nt][i], i == 0 ? f32x4{} : s[nt][g]);
    }
  }
  uint32_t vs0 = kv.vs[0], vs1 = kv.vs[1];
  if (masked) {
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = 16 * g + 4 * quarter + e;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          if (!mask.row(nt, key)) s[nt][g][e] = -INFINITY;
        // what no row sees may be anything, and a slot without a position is: make it
        // finite, for 0 times it to be 0
        if (!mask.any(key)) {
          if (g == 0)
            vs0 &= ~(255u << (8 * e));
          else
            vs1 &= ~(255u << (8 * e));
        }
      }
  }
  u32x4 pf[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float top = -INFINITY;
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, s[nt][g][e]);
    top *= c;
    if (__any(top > st.m[nt] + 8.0f)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float m = fmaxf(st.m[nt], top);
      const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st.m[nt] - m);
      st.m[nt] = m;
      st.l[nt] *= f;
#pragma unroll
      for (int i = 0; i < NM; ++i) st.o[nt][i] *= f;
    }
    const float ref = st.m[nt] == -INFINITY ? 0.f : st.m[nt] - Fmt<T>::kBias;
    float pr[8];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pr[4 * g + e] = __builtin_amdgcn_exp2f(fmaf(s[nt][g][e], c, -ref));
        st.l[nt] += pr[4 * g + e];
      }
#pragma unroll
    for (int e = 0; e < 4; ++e) pf[nt][e] = pair_of<T>(pr[2 * e], pr[2 * e + 1]);
  }
  uint32_t w[8];
  float sc[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = kv.v[0][e];
    w[4 + e] = kv.v[1][e];
  }
  scales4(vs0, sc);
  scales4(vs1, sc + 4);
  if constexpr (D == 64) {  // the lane's 4 channels of the word
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] >>= (lane & 1) * 16;
  }
  auto product = [&](int i, u32x4 even, u32x4 odd) __attribute__((always_inline)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      st.o[nt][2 * i] = Fmt<T>::mfma(even, pf[nt], st.o[nt][2 * i]);
      st.o[nt][2 * i + 1] = Fmt<T>::mfma(odd, pf[nt], st.o[nt][2 * i + 1]);
    }
  };
  u32x4 even, odd;
  transpose_pair<T, 0>(w, sc, &even, &odd);
  product(0, even, odd);
  transpose_pair<T, 1>(w, sc, &even, &odd);
  product(1, even, odd);
  if constexpr (D == 128) {
    transpose_pair<T, 2>(w, sc, &even, &odd);
    product(2, even, odd);
    transpose_pair<T, 3>(w, sc, &even, &odd);
    product(3, even, odd);
  }
}

// The keys [lo, hi] that a row sees; none of a row that the sequence lacks.
struct RowRange {
  int lo, hi;
};
__device__ __forceinline__ RowRange row_range(int t, int n_new, int len, int C, int W) {
  if (t >= n_new) return {1, 0};
  const int pos = len - n_new + t;
  int lo = max(0, len - C);
  if (W > 0) lo = max(lo, pos - W + 1);
  return {lo, pos};
}

// A tree's nodes (kv4_tree_attn): node i of a sequence is at position length + depth(i), and
// sees the cache up to the window before that, itself and its ancestors, keys of the draft,
// those of them that the window reaches. They are bits: after s steps a node has those of
// 2^s, itself among them, and knows the one after the last, so 8 steps are enough for 256
// nodes, and the depth's logarithm is what it takes (walking up one by one would wait for LDS
// at every node of a chain). Nodes behind the last see nothing.
struct TreeBits {
  uint32_t up[kTreeNodes][kTreeNodes / 32];
  int depth[kTreeNodes], next[kTreeNodes];
};
template <int THREADS>
__device__ __forceinline__ void tree_bits(TreeBits& tree, const int32_t* parents, int n,
                                          int window) {
  static_assert(THREADS >= kTreeNodes, "a thread a node");
  constexpr int WORDS = kTreeNodes / 32;
  const int i = threadIdx.x;
  int next = -1;
  if (i < n) {
    next = parents[i];
    if (next >= i || next < 0) next = -1;  // a parent comes before its node
  }
  if (i < kTreeNodes) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) tree.up[i][w] = w == i / 32 && i < n ? 1u << (i % 32) : 0u;
    tree.depth[i] = next >= 0;
    tree.next[i] = next;
  }
  while (__syncthreads_or(next >= 0)) {  // a node's next falls by half its distance at least
    uint32_t up[WORDS];
    int depth = 0, after = -1;
    if (next >= 0) {
#pragma unroll
      for (int w = 0; w < WORDS; ++w) up[w] = tree.up[next][w];
      depth = tree.depth[next];
      after = tree.next[next];
    }
    __syncthreads();
    if (next >= 0) {
#pragma unroll
      for (int w = 0; w < WORDS; ++w) tree.up[i][w] |= up[w];
      tree.depth[i] += depth;
      tree.next[i] = next = after;
    }
  }
  if (window > 0 && window < n) {
    if (i < n && tree.depth[i] >= window) {
      const int least = tree.depth[i] - window + 1;
      for (int w = 0; w <= i / 32; ++w) {
        uint32_t left = tree.up[i][w];
        while (left != 0) {
          const int e = __builtin_ctz(left);
          left &= left - 1;
          if (tree.depth[32 * w + e] < least) tree.up[i][w] &= ~(1u << e);
        }
      }
    }
    __syncthreads();
  }
}

// Bits lo .. hi of a word, those of them that there are.
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
  if (lo > hi || hi < 0 || lo > 31) return 0u;
  return (0xffffffffu << max(lo, 0)) & (0xffffffffu >> (31 - min(hi, 31)));
}

__device__ __forceinline__ RowRange node_range(int i, int n, int depth, int len, int C, int W) {
  if (i >= n) return {1, 0};
  int lo = max(0, len - C);
  if (W > 0) lo = max(lo, len + depth - W + 1);
  return {lo, len - 1};
}

// A workgroup's share: part `part` of sequence b's tiles, those from `part * tiles` on, and
// where its sums go, row 0's place among the parts' rows.
struct Share {
  int b, h, rb, part, parts;
  int tiles;      // of a part; 0: those there are, dealt evenly
  int64_t sums;
};
template <int KEYS>
__device__ __forceinline__ Share share_of(const Kv4AttnArgs& a, int id, int) {
  const int part = id % a.parts, rest = id / a.parts;
  const int rb = rest % a.nrb, bh = rest / a.nrb;
  const int b = bh / a.c.H;
  return {b, bh - b * a.c.H, rb, part, a.parts, 0,
          ((int64_t)part * a.c.B * a.c.H + bh) * ((int64_t)a.Tq * a.G)};
}

// How a tree's sequences share their parts: as many tiles of KEYS keys to each part, whatever
// the sequence, so that a batch of mixed lengths ends at once. A lane a sequence.
struct TreeShares {
  uint32_t first, parts;  // of the lane's sequence
  int tiles;              // of a part
};
template <int KEYS>
__device__ __forceinline__ TreeShares tree_shares(const Kv4TreeArgs& a, int lane) {
  uint32_t tiles = 0;
  if (lane < a.c.B) {
    const int len = length_of(a.c.len, lane);
    const int n = min(count_of(a.counts, lane, a.Tq), length_of(a.d.len, lane));
    if (n > 0) {
      const RowRange keys = node_range(0, n, 0, len, a.c.C, a.window);
      tiles = (n + KEYS - 1) / KEYS;
      if (keys.lo <= keys.hi) tiles += keys.hi / KEYS - keys.lo / KEYS + 1;
    }
  }
  // The least tiles a part with which there are no more parts than units: between all of
  // them full, and every sequence's last one short.
  const uint32_t all = sum_of(tiles), most = max_of(tiles), units = a.units, B = a.c.B;
  uint32_t lo = max(max((all + units - 1) / units, (most + kKv4MaxParts - 1) / kKv4MaxParts),
                    (uint32_t)a.least);
  uint32_t hi = max(lo, (all + units - B - 1) / (units - B));
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if (sum_of((tiles + mid - 1) / mid) <= units)
      hi = mid;
    else
      lo = mid + 1;
  }
  TreeShares s;
  s.tiles = lo;
  s.parts = (tiles + s.tiles - 1) / s.tiles;
  s.first = scan_before<uint32_t>(s.parts, lane);
  return s;
}
template <int KEYS>
__device__ __forceinline__ Share share_of(const Kv4TreeArgs& a, int id, int lane) {
  if (a.units == 0) return share_of<KEYS>(static_cast<const Kv4AttnArgs&>(a), id, lane);
  const TreeShares s = tree_shares<KEYS>(a, lane);
  if (id == 0 && threadIdx.x < a.c.B) {  // for the sums of the parts
    a.shares[2 * lane] = s.first;
    a.shares[2 * lane + 1] = s.parts;
  }
  const uint32_t unit = id % a.units;
  const int rest = id / a.units, rb = rest % a.nrb, h = rest / a.nrb;
  const uint64_t mine = __ballot(unit - s.first < s.parts);
  if (mine == 0) return {-1, h, rb, 0, 0, 0, 0};
  const int b = __builtin_ctzll(mine);
  return {b, h, rb, (int)(unit - lane_of(s.first, b)), (int)lane_of(s.parts, b), s.tiles,
          ((int64_t)unit * a.c.H + h) * ((int64_t)a.Tq * a.G)};
}

template <typename T, int D, int NT, bool FAR, typename Args>
__global__ __launch_bounds__(64 * (is_tree<Args> ? kTreeWaves : kRowWaves),
                             is_tree<Args> ? 4 - NT : 1) void kv4_rows_kernel(Args a) {
  constexpr bool TREE = is_tree<Args>;
  constexpr int WAVES = TREE ? kTreeWaves : kRowWaves;
  constexpr int STEPS = D / 32, NM = D / 16, RB = 16 * NT, R = D / 8;
  __shared__ __attribute__((aligned(16))) float so[WAVES][16][D + 4];
  __shared__ float sml[WAVES][RB][2];
  static_assert(sizeof(TreeBits) <= sizeof(so), "the tree lies where the sums come later");
  TreeBits& tree = *reinterpret_cast<TreeBits*>(&so);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int quarter = lane >> 4, n = lane & 15;
  const Share mine = share_of<32>(a, blockIdx.x, lane);
  const int part = mine.part, parts = mine.parts, b = mine.b, h = mine.h, bh = b * a.c.H + h;
  const int rb = mine.rb;
  if (TREE && b < 0) return;
  const int len = length_of(a.c.len, b);
  int n_new = count_of(a.counts, b, a.Tq);
  if constexpr (TREE) n_new = min(n_new, length_of(a.d.len, b));
  const int row0 = rb * RB, C = a.c.C;

  u32x4 q[NT][STEPS];
  int lo[NT], hi[NT];
  RowState<T, D, NT> st;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = row0 + 16 * nt + n, t = min(row / a.G, a.Tq - 1);
    const T* src = static_cast<const T*>(a.q) + b * a.q_sb + t * a.q_st +
                   (int64_t)(h * a.G + row % a.G) * a.q_sh + quarter * (D / 4);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) q[nt][i] = *reinterpret_cast<const u32x4*>(src + 8 * i);
    if constexpr (!TREE) {
      const RowRange rr = row_range(row / a.G, n_new, len, C, a.window);
      lo[nt] = rr.lo;
      hi[nt] = rr.hi;
    }
    st.m[nt] = -INFINITY;
    st.l[nt] = 0.f;
#pragma unroll
    for (int i = 0; i < NM; ++i) st.o[nt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // the block's keys, and those that all its rows see
  const int t_lo = row0 / a.G, t_hi = min((row0 + RB - 1) / a.G, n_new - 1);
  if (t_lo <= t_hi) {
    // (of a tree: bounds of all its rows' ranges, from a root to the deepest that there could be)
    const RowRange first = TREE ? node_range(0, n_new, 0, len, C, a.window)
                                : row_range(t_lo, n_new, len, C, a.window);
    const RowRange last = TREE ? node_range(0, n_new, n_new - 1, len, C, a.window)
                               : row_range(t_hi, n_new, len, C, a.window);
    if constexpr (TREE) {  // of rows whose tiles nothing cuts
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        lo[nt] = 0;
        hi[nt] = len - 1;
      }
    }
    if (TREE || first.lo <= last.hi) {
      const int tile_lo = first.lo >> 5;
      // of the cache; a tree's draft follows
      const int held = first.lo <= last.hi ? (last.hi >> 5) - tile_lo + 1 : 0;
      const int tiles = TREE ? held + ((n_new + 31) >> 5) : held;
      const int per = TREE && mine.tiles > 0 ? mine.tiles : (tiles + parts - 1) / parts;
      const int t0 = tile_lo + part * per, t1 = min(t0 + per, tile_lo + tiles);
      // a lane's place in 16 keys' rows; the rest of an address is the wavefront's
      const int word = D == 128 ? n : n >> 1;
      const uint32_t k_at = n * (D / 2) + quarter * (D / 8), ks_at = n * (D / 32) + quarter * (D / 4) / 32;
      const uint32_t v_at = (quarter * R + word) * 16, vs_at = (quarter * (D / 32) + word / 4) * 4;
      const int64_t row = (int64_t)bh * C;
      const uint8_t* const kc = a.c.kc + row * (D / 2);
      const uint8_t* const ks = a.c.ks + row * (D / 32);
      const uint8_t* const vc = a.c.vc + row * (D / 2);
      const uint8_t* const vs = a.c.vs + row * (D / 32);
      auto load = [&](KvTile<D>& kv, int at, int slot) __attribute__((always_inline)) {
        const uint8_t* k0 = kc + (int64_t)slot * (D / 2);
        const uint8_t* s0 = ks + (int64_t)slot * (D / 32);
        const uint8_t* v0 = vc + (int64_t)slot * (D / 2);
        const uint8_t* t0 = vs + (int64_t)slot * (D / 32);
        if constexpr (TREE) {
          if (at >= tile_lo + held) {
            const int64_t node = (int64_t)bh * a.d.C + (at - tile_lo - held) * 32;
            k0 = a.d.kc + node * (D / 2);
            s0 = a.d.ks + node * (D / 32);
            v0 = a.d.vc + node * (D / 2);
            t0 = a.d.vs + node * (D / 32);
          }
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if constexpr (D == 128) {
            kv.k[g] = codes<FAR>(reinterpret_cast<const u32x4*>(k0 + (k_at + 16 * g * (D / 2))));
          } else {
            const u32x2 half =
                codes<FAR>(reinterpret_cast<const u32x2*>(k0 + (k_at + 16 * g * (D / 2))));
            kv.k[g][0] = half[0];
            kv.k[g][1] = half[1];
          }
          kv.ks[g] = s0[ks_at + 16 * g * (D / 32)];
          kv.v[g] = codes<FAR>(reinterpret_cast<const u32x4*>(v0 + (v_at + 16 * g * (D / 2))));
          kv.vs[g] = *reinterpret_cast<const uint32_t*>(t0 + (vs_at + 16 * g * (D / 32)));
        }
      };
      const int step = WAVES * 32 % C;
      int tile = t0 + wave;
      int slot = (int)((uint32_t)(tile * 32) % (uint32_t)C);
      auto fold = [&](const KvTile<D>& kv) __attribute__((always_inline)) {
        if constexpr (TREE) {
          const int node = (tile - tile_lo - held) * 32;  // the draft's first, from 0 on
          const bool masked = node >= 0 || tile * 32 < last.lo || tile * 32 + 31 > first.hi;
          BitMask<NT> mask = {};
          if (masked) {
            const int p0 = tile * 32;
            mask.all = node >= 0 ? bits_between(0, n_new - 1 - node)
                                 : bits_between(first.lo - p0, last.hi - p0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mask.rows[nt] = node >= 0 ? tree.up[(row0 + 16 * nt + n) / a.G][node >> 5]
                                        : bits_between(lo[nt] - p0, hi[nt] - p0);
          }
          fold_tile<T, D, NT>(st, kv, q, a.c_log2, masked, mask, lane);
        } else {
          const bool masked = tile * 32 < last.lo || tile * 32 + 31 > first.hi;
          const RangeMask<NT> mask = {lo, hi, tile * 32, first.lo, last.hi};
          fold_tile<T, D, NT>(st, kv, q, a.c_log2, masked, mask, lane);
        }
        tile += WAVES;
      };
      // AHEAD tiles are on their way while one is folded
      constexpr int AHEAD = TREE ? 2 : 1;
      auto next = [&](KvTile<D>& kv) __attribute__((always_inline)) {
        if (tile + AHEAD * WAVES >= t1) return;
        slot += step;
        if (slot >= C) slot -= C;
        load(kv, tile + AHEAD * WAVES, slot);
      };
      KvTile<D> kv[AHEAD + 1];
      if (tile < t1) load(kv[0], tile, slot);
      if constexpr (TREE) {
        if (tile + WAVES < t1) {
          slot += step;
          if (slot >= C) slot -= C;
          load(kv[1], tile + WAVES, slot);
        }
        // the tree where a tile of the part needs it: the draft's, and those that the window cuts
        if (t0 < t1 && (t1 > tile_lo + held || t0 * 32 < last.lo)) {
          tree_bits<64 * WAVES>(tree, a.parents + (int64_t)b * a.Tq, n_new, a.window);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int node = (row0 + 16 * nt + n) / a.G;
            const RowRange rr = node_range(node, n_new, tree.depth[node], len, C, a.window);
            lo[nt] = rr.lo;
            hi[nt] = rr.hi;
          }
        }
      }
      while (tile < t1) {
#pragma unroll
        for (int i = 0; i <= AHEAD; ++i) {
          next(kv[(i + AHEAD) % (AHEAD + 1)]);
          fold(kv[i]);
          if (tile >= t1) break;
        }
      }
    }
  }
  if constexpr (TREE) __syncthreads();  // the tree is read
  // add the wavefronts
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float l = st.l[nt];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    // a row that the sequence lacks saw the tiles that nobody's mask cuts
    const bool none = TREE ? (row0 + 16 * nt + n) / a.G >= n_new : lo[nt] > hi[nt];
    if (quarter == 0) {
      sml[wave][16 * nt + n][0] = none ? -INFINITY : st.m[nt] - Fmt<T>::kBias;
      sml[wave][16 * nt + n][1] = none ? 0.f : l;
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (nt > 0) __syncthreads();  // the tile before is read
    // accumulator element e of product i: channel NM (4 quarter + e) + i
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < NM; ++i)
        so[wave][n][NM * (4 * quarter + e) + i] = st.o[nt][i][e];
    __syncthreads();
    constexpr int PER = D * 16 / (64 * WAVES);  // channels a thread
    constexpr int TPR = D / PER;                    // threads a row
    const int r = threadIdx.x / TPR, d0 = (threadIdx.x % TPR) * PER;
    const int row = row0 + 16 * nt + r;
    if (row < a.Tq * a.G) {
      float m = -INFINITY, l = 0.f, o[PER];
#pragma unroll
      for (int w = 0; w < WAVES; ++w) m = fmaxf(m, sml[w][16 * nt + r][0]);
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = __builtin_amdgcn_exp2f(sml[w][16 * nt + r][0] - ref);
        l = fmaf(sml[w][16 * nt + r][1], f, l);
#pragma unroll
        for (int i = 0; i < PER; ++i) o[i] = fmaf(so[w][r][d0 + i], f, o[i]);
      }
      if (parts > 1) {
        const int64_t at = mine.sums + row;
        if (threadIdx.x % TPR == 0) {
          a.part_ml[2 * at] = m;
          a.part_ml[2 * at + 1] = l;
        }
        if (l != 0.f) {  // an empty part is not read
#pragma unroll
          for (int i = 0; i < PER; ++i) a.part[at * D + d0 + i] = o[i];
        }
      } else {
        const int t = row / a.G, head = h * a.G + row % a.G;
        const float inv = 1.f / l;
        T* dst = static_cast<T*>(a.o) + b * a.o_sb + t * a.o_st + head * a.o_sh + d0;
        uint32_t w[PER / 2];
#pragma unroll
        for (int i = 0; i < PER / 2; ++i)
          w[i] = l == 0.f ? 0u : pair_of<T>(o[2 * i] * inv, o[2 * i + 1] * inv);
        if constexpr (PER == 8)
          *reinterpret_cast<u32x4*>(dst) = u32x4{w[0], w[1], w[2], w[3]};
        else if constexpr (PER == 4)
          *reinterpret_cast<u32x2*>(dst) = u32x2{w[0], w[1]};
        else
          *reinterpret_cast<uint32_t*>(dst) = w[0];
        if (a.lse != nullptr && threadIdx.x % TPR == 0)
          a.lse[((int64_t)b * a.G * a.c.H + head) * a.Tq + t] =
              l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Attention of many rows. A workgroup's 4 wavefronts hold 32 rows each and sweep
// the same tiles of 64 keys; a tile is converted once, a quarter of it by
// each wavefront, into LDS, where K and V lie as the operands of 32x32x16 MFMAs
// (every read and write is 16 bytes a lane and 512 in a row). S^T = K Q^T, then
// O^T = V^T P^T with P as it lies after the first product.
//
// The order of loads, conversions, products and barriers is kv4_sweep.h's; two stages of
// each in LDS and one barrier a turn. (With a branch for the last turn 279 us, as code of
// its own 272.)
//
// Bound by the matrix pipe and the exponentials, which take about as long: 4096
// queries on an 8192 window, 16/8 heads of 128, 256 us, 1074 TFLOP/s (a large library
// product reaches 1226 on the same card). Two workgroups a CU, 64 KiB of LDS and 256
// registers each. 64 rows a wavefront, which would halve the operand reads, spill
// (1169 us); every wavefront converting for itself, without LDS, took 476; scheduling
// groups of a product, a read and 6 VALU operations 277 to 289.
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c);
template <>
__device__ __forceinline__ f32x16 mfma32<__bf16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 mfma32<_Float16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// A tree's nodes in more than 32 rows a kv head take this kernel too: 64 nodes of 4 sequences
// over a window of 8192 keys, 128 rows a head, 32 us (530 TFLOP/s: parts of 8 or 9 tiles,
// whose start and end take as long) and 8.4 for the sum of the parts.
constexpr int kBlockKeys = 64;

template <typename T, int D, typename Args>
__global__ __launch_bounds__(256, 2) void kv4_block_kernel(Args a) {
  constexpr bool TREE = is_tree<Args>;
  constexpr int KS = D / 16;  // steps of 16 channels
  constexpr int MB = D / 32;  // blocks of 32 channels
  constexpr int W = D / 8;    // words of 8 channels
  constexpr int TILE = kBlockKeys * D * 2;  // bytes of a converted K or V tile
  constexpr int RB = 128;
  __shared__ __attribute__((aligned(1024))) char smem[4 * TILE];  // K, K, V, V
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, n = lane & 31;
  const Share mine = share_of<kBlockKeys>(a, blockIdx.x, lane);
  const int part = mine.part, parts = mine.parts, b = mine.b, h = mine.h, bh = b * a.c.H + h;
  const int rb = mine.rb;
  if (TREE && b < 0) return;
  const int len = length_of(a.c.len, b);
  int n_new = count_of(a.counts, b, a.Tq);
  if constexpr (TREE) n_new = min(n_new, length_of(a.d.len, b));
  const int row0 = rb * RB, C = a.c.C;

  const int row = row0 + wave * 32 + n, t = min(row / a.G, a.Tq - 1), head = h * a.G + row % a.G;
  u32x4 q[KS];
  {
    const T* src = static_cast<const T*>(a.q) + b * a.q_sb + t * a.q_st + (int64_t)head * a.q_sh +
                   half * 8;
#pragma unroll
    for (int i = 0; i < KS; ++i) q[i] = *reinterpret_cast<const u32x4*>(src + 16 * i);
  }
  RowRange rr;
  __shared__ std::conditional_t<TREE, TreeBits, char> tree[1];
  if constexpr (TREE)
    rr = {0, len - 1};  // of rows whose tiles no window cuts
  else
    rr = row_range(row / a.G, n_new, len, C, a.window);
  float m = -INFINITY, l = 0.f;
  f32x16 o[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) o[i] = f32x16{};
  // tiles [t0, t1) of 64 keys that the workgroup folds, and the keys that any row sees
  int t0 = 0, t1 = 0, any_lo = 0, any_hi = -1;
  int draft = 0;  // the first tile of a tree's draft, behind the cache's
  const int t_lo = row0 / a.G, t_hi = min((row0 + RB - 1) / a.G, n_new - 1);
  if (t_lo <= t_hi) {
    const RowRange first = TREE ? node_range(0, n_new, 0, len, C, a.window)
                                : row_range(t_lo, n_new, len, C, a.window);
    const RowRange last = TREE ? node_range(0, n_new, n_new - 1, len, C, a.window)
                               : row_range(t_hi, n_new, len, C, a.window);
    if (TREE || first.lo <= last.hi) {
      const int tile_lo = first.lo / kBlockKeys;
      const int held = first.lo <= last.hi ? last.hi / kBlockKeys - tile_lo + 1 : 0;
      const int tiles = TREE ? held + (n_new + kBlockKeys - 1) / kBlockKeys : held;
      draft = tile_lo + held;
      const int per = TREE && mine.tiles > 0 ? mine.tiles : (tiles + parts - 1) / parts;
      t0 = tile_lo + part * per;
      t1 = min(t0 + per, tile_lo + tiles);
      any_lo = first.lo;
      any_hi = last.hi;
      if constexpr (TREE) {
        // the tree where a tile of the part needs it: the draft's, and those that the window cuts
        if (t0 < t1 && (t1 > draft || t0 * kBlockKeys < last.lo)) {
          tree_bits<256>(tree[0], a.parents + (int64_t)b * a.Tq, n_new, a.window);
          const int node = row / a.G;
          rr = node_range(node, n_new, tree[0].depth[node], len, C, a.window);
        }
      }
    }
  }
  // the keys that all rows of this wavefront see
  int in_lo = 0, in_hi = -1;
  {
    const int w0 = (row0 + wave * 32) / a.G;
    const int w1 = min((row0 + wave * 32 + 31) / a.G, n_new - 1);
    if (w0 <= w1) {
      in_lo = (TREE ? node_range(0, n_new, n_new - 1, len, C, a.window)
                    : row_range(w1, n_new, len, C, a.window)).lo;
      in_hi = (TREE ? node_range(0, n_new, 0, len, C, a.window)
                    : row_range(w0, n_new, len, C, a.window)).hi;
    }
  }

  // Conversion. Keys: lane (key 16 wave + lane % 16, quarter of its channels).
  // Values: the 16 keys of step `wave`, lane = channels (w, k) of its half's 8.
  const int kq = lane >> 4, km = wave * 16 + (lane & 15);
  const int vw = n % W, vk = n / W;
  struct Codes {
    u32x4 c[2];
    uint32_t s[2];
  };
  // the slot of a tile's 16 keys of this wavefront: its halves may lie apart where
  // the ring ends, a multiple of 32 slots from anything
  auto slot_of = [&](int tile) __attribute__((always_inline)) {
    return (int)((uint32_t)(tile * kBlockKeys + wave * 16) % (uint32_t)C);
  };
  // the cache that a tile lies in, and its 16 keys' row there
  auto cache_of = [&](int tile) __attribute__((always_inline)) {
    if constexpr (TREE) return tile >= draft ? a.d : a.c;
    return a.c;
  };
  auto row_of = [&](int tile) __attribute__((always_inline)) {
    if constexpr (TREE) {
      // what lies behind the draft's end wraps: memory that is there, and no row sees it
      if (tile >= draft)
        return (int64_t)bh * a.d.C + (int)((uint32_t)((tile - draft) * kBlockKeys + wave * 16) %
                                           (uint32_t)a.d.C);
    }
    return (int64_t)bh * C + slot_of(tile);
  };
  auto load_k = [&](Codes& kc, int tile) __attribute__((always_inline)) {
    const Kv4Cache from = cache_of(tile);
    const int64_t row = row_of(tile) + (lane & 15);
    const uint8_t* src = from.kc + row * (D / 2) + kq * (D / 8);
    if constexpr (D == 128) {
      kc.c[0] = *reinterpret_cast<const u32x4*>(src);
    } else {
      const u32x2 x = *reinterpret_cast<const u32x2*>(src);
      kc.c[0][0] = x[0];
      kc.c[0][1] = x[1];
    }
    kc.s[0] = from.ks[row * (D / 32) + kq * (D / 4) / 32];
  };
  auto load_v = [&](Codes& vc, int tile) __attribute__((always_inline)) {
    const Kv4Cache from = cache_of(tile);
    const int64_t g = (row_of(tile) >> 2) + half;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      vc.c[i] = *reinterpret_cast<const u32x4*>(from.vc + ((g + 2 * i) * W + vw) * 16);
      vc.s[i] = *reinterpret_cast<const uint32_t*>(from.vs + ((g + 2 * i) * (D / 32) + vw / 4) * 4);
    }
  };
  auto store_k = [&](const Codes& kc, int tile) __attribute__((always_inline)) {
    char* dst = smem + (tile & 1) * TILE + (km >> 5) * (32 * D * 2) + (km & 31) * 16;
    const float s = scale_of(kc.s[0]);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {  // chunk c of 8 channels: step c / 2, half c % 2
      const int c = kq * (D / 32) + i;
      *reinterpret_cast<u32x4*>(dst + c * 512) = values8<T>(kc.c[0][i], s);
    }
  };
  auto store_v = [&](const Codes& vc, int tile) __attribute__((always_inline)) {
    char* dst = smem + (2 + (tile & 1)) * TILE + wave * (16 * D * 2) + lane * 16;
    uint32_t w[8];
    float s[8];
    const int p = tile * kBlockKeys + wave * 16 + 4 * half;  // the lane's first key
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = vc.c[0][e] >> (vk * 4 * MB);
      w[4 + e] = vc.c[1][e] >> (vk * 4 * MB);
    }
    scales4(vc.s[0], s);
    scales4(vc.s[1], s + 4);
    // what no row sees may be anything, and a slot without a position is: make it
    // finite, for 0 times it to be 0
    if (TREE && tile >= draft) {
      const int i = p - draft * kBlockKeys;  // the lane's first node
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e] = i + e < n_new ? s[e] : 0.f;
        s[4 + e] = i + 8 + e < n_new ? s[4 + e] : 0.f;
      }
    } else if (tile * kBlockKeys < any_lo || tile * kBlockKeys + kBlockKeys - 1 > any_hi) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e] = p + e >= any_lo && p + e <= any_hi ? s[e] : 0.f;
        s[4 + e] = p + 8 + e >= any_lo && p + 8 + e <= any_hi ? s[4 + e] : 0.f;
      }
    }
    u32x4 even, odd;
    transpose_pair<T, 0>(w, s, &even, &odd);
    *reinterpret_cast<u32x4*>(dst) = even;
    *reinterpret_cast<u32x4*>(dst + 1024) = odd;
    if constexpr (MB == 4) {
      transpose_pair<T, 1>(w, s, &even, &odd);
      *reinterpret_cast<u32x4*>(dst + 2 * 1024) = even;
      *reinterpret_cast<u32x4*>(dst + 3 * 1024) = odd;
    }
  };

  f32x16 sa[2], sb[2];
  auto scores = [&](f32x16 (&s)[2], int tile) __attribute__((always_inline)) {
    const char* src = smem + (tile & 1) * TILE + lane * 16;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(src + kb * (32 * D * 2) + i * 1024);
        s[kb] = mfma32<T>(kf, q[i], i == 0 ? f32x16{} : s[kb]);
      }
  };
  // masks tile's scores and moves the reference where they exceed it by 2^8
  auto settle = [&](f32x16 (&s)[2], int tile) __attribute__((always_inline)) {
    const int p0 = tile * kBlockKeys;
    if constexpr (TREE) {
      if (tile >= draft || p0 < in_lo || p0 + kBlockKeys - 1 > in_hi) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const uint32_t seen =
              (tile >= draft ? tree[0].up[row / a.G][2 * (tile - draft) + kb]
                             : bits_between(rr.lo - p0 - 32 * kb, rr.hi - p0 - 32 * kb)) >>
              (4 * half);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (!(seen & (1u << (8 * (e >> 2) + (e & 3))))) s[kb][e] = -INFINITY;
        }
      }
    } else if (p0 < in_lo || p0 + kBlockKeys - 1 > in_hi) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int p = p0 + 32 * kb + 8 * (e >> 2) + 4 * half + (e & 3);
          if (p < rr.lo || p > rr.hi) s[kb][e] = -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int e = 1; e < 16; ++e) top = fmaxf(top, s[0][e]);
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, s[1][e]);
    top *= a.c_log2;
    if (__any(top > m + 8.0f)) {
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m, top);
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int i = 0; i < MB; ++i) o[i] *= f;
    }
  };
  // adds a tile's probabilities times its values
  auto fold = [&](f32x16 (&s)[2], int tile) __attribute__((always_inline)) {
    u32x4 p[4];
    const float ref = m == -INFINITY ? 0.f : m - Fmt<T>::kBias;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x0 =
            __builtin_amdgcn_exp2f(fmaf(s[j >> 1][8 * (j & 1) + 2 * e], a.c_log2, -ref));
        const float x1 =
            __builtin_amdgcn_exp2f(fmaf(s[j >> 1][8 * (j & 1) + 2 * e + 1], a.c_log2, -ref));
        l += x0 + x1;
        p[j][e] = pair_of<T>(x0, x1);
      }
    const char* src = smem + (2 + (tile & 1)) * TILE + lane * 16;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const u32x4 vf = *reinterpret_cast<const u32x4*>(src + j * (16 * D * 2) + i * 1024);
        o[i] = mfma32<T>(vf, p[j], o[i]);
      }
  };
  if (t0 < t1)
    kv4_sweep<Codes>(t0, t1, sa, sb, load_k, load_v, store_k, store_v, scores, settle, fold,
                     [] { __syncthreads(); });

  // saw the tiles that nobody's mask cuts
  const bool none = TREE ? row / a.G >= n_new : rr.lo > rr.hi;
  l = none ? 0.f : l + __shfl_xor(l, 32);
  m = none ? -INFINITY : m - Fmt<T>::kBias;
  const int rows = a.Tq * a.G, wrow0 = row0 + wave * 32;
  const int64_t at0 = mine.sums;
  if (half == 0 && row < rows) {
    if (parts > 1) {
      a.part_ml[2 * (at0 + row)] = m;
      a.part_ml[2 * (at0 + row) + 1] = l;
    } else if (a.lse != nullptr) {
      a.lse[((int64_t)b * a.G * a.c.H + head) * a.Tq + t] =
          l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
    }
  }
  // The wavefront's 32 rows through its quarter of the stages, chunk c of 16 bytes at
  // c ^ (row % chunks): a lane has pieces of one row, a line is written by as many
  // lanes as it has chunks.
  __syncthreads();  // every stage is read
  char* const rows_at = smem + wave * TILE;
  const float inv = 1.f / l;
  // Accumulator element e of block i: row rho = 8 (e / 4) + 4 half + e % 4, that is
  // channel 8 (rho % W) + MB (rho / W) + i: 8 in a row a word.
#pragma unroll
  for (int wi = 0; wi < W / 2; ++wi) {  // the lane's words: those with bit 2 as its half
    const int w = 8 * (wi >> 2) + 4 * half + (wi & 3);
    float x[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      // rho = w + W (c / MB): element 4 (rho / 8) + wi % 4
      const int e = 4 * ((8 * (wi >> 2) + W * (c / MB)) >> 3) + (wi & 3);
      x[c] = o[c % MB][e];
    }
    if (parts > 1) {
      char* const dst = rows_at + n * (D * 4);
      *reinterpret_cast<f32x4*>(dst + ((2 * w) ^ (n & (2 * W - 1))) * 16) =
          f32x4{x[0], x[1], x[2], x[3]};
      *reinterpret_cast<f32x4*>(dst + ((2 * w + 1) ^ (n & (2 * W - 1))) * 16) =
          f32x4{x[4], x[5], x[6], x[7]};
    } else {
      u32x4 y;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        y[c] = l == 0.f ? 0u : pair_of<T>(x[2 * c] * inv, x[2 * c + 1] * inv);
      *reinterpret_cast<u32x4*>(rows_at + n * (D * 2) + (w ^ (n & (W - 1))) * 16) = y;
    }
  }
  __syncthreads();
  if (parts > 1) {
    constexpr int CH = 2 * W;
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) {
      const int r = i * (64 / CH) + lane / CH, c = lane % CH;
      if (wrow0 + r < rows)  // of a part without keys too, which is not read
        *reinterpret_cast<u32x4*>(a.part + (at0 + wrow0 + r) * D + 4 * c) =
            *reinterpret_cast<const u32x4*>(rows_at + r * (D * 4) + (c ^ (r & (CH - 1))) * 16);
    }
  } else {
    constexpr int CH = W;
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) {
      const int r = i * (64 / CH) + lane / CH, c = lane % CH;
      const int to = (wrow0 + r) / a.G, ho = h * a.G + (wrow0 + r) - to * a.G;
      if (wrow0 + r < rows)
        *reinterpret_cast<u32x4*>(static_cast<T*>(a.o) + b * a.o_sb + to * a.o_st + ho * a.o_sh +
                                  8 * c) =
            *reinterpret_cast<const u32x4*>(rows_at + r * (D * 2) + (c ^ (r & (CH - 1))) * 16);
    }
  }
}

// The parts of a row, at most 64: every wavefront finds their weights, a part a
// lane; D / 4 threads with 4 channels each in every one of the 256 / (D / 4) groups
// share the sums between them. (One thread after the other over the parts took 29
// us for 103 of them; 64 of 30 rows take 3.9.)
//
// Where they are: `parts` rows `all` apart, the first `id`.
struct Parts {
  int parts;
  int64_t id, all;
};
__device__ __forceinline__ Parts parts_of(const Kv4AttnArgs& a, int bh, int row) {
  const int64_t rows = (int64_t)a.Tq * a.G;
  return {a.parts, bh * rows + row, a.c.B * a.c.H * rows};
}
__device__ __forceinline__ Parts parts_of(const Kv4TreeArgs& a, int bh, int row) {
  const int64_t rows = (int64_t)a.Tq * a.G;
  const int b = bh / a.c.H, h = bh - b * a.c.H;
  return {a.shares[2 * b + 1], ((int64_t)a.shares[2 * b] * a.c.H + h) * rows + row,
          a.c.H * rows};
}

template <typename T, int D, typename Args>
__global__ __launch_bounds__(256) void kv4_combine_kernel(Args a) {
  constexpr int TH = D / 4, GR = 256 / TH;
  __shared__ f32x4 so[GR][TH];
  const int rows = a.Tq * a.G;
  const int bh = blockIdx.x / rows, row = blockIdx.x - bh * rows;
  const int b = bh / a.c.H, h = bh - b * a.c.H;
  const int d4 = threadIdx.x % TH, g = threadIdx.x / TH, lane = threadIdx.x & 63;
  const Parts in = parts_of(a, bh, row);
  if (is_tree<Args> && in.parts == 1) return;  // written by the part
  const int64_t id = in.id, all = in.all;
  float m = -INFINITY, l = 0.f;
  if (lane < in.parts) {
    const float* ml = a.part_ml + 2 * (lane * all + id);
    m = ml[0];
    l = ml[1];
  }
  float top = m;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  float f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
  const bool empty = l == 0.f;  // such a part's sums are not there
  l = empty ? 0.f : l * f;
  f = empty ? -1.f : f;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) l += __shfl_xor(l, d);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  const float* src = a.part + id * D + 4 * d4;
  for (int p0 = 0; p0 < in.parts; p0 += GR) {
    const int p = p0 + g;
    const float w = __shfl(f, p & 63);
    if (p < in.parts && !(w < 0.f)) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(src + p * all * D);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(v[e], w, o[e]);
    }
  }
  so[g][d4] = o;
  __syncthreads();
  if (g != 0) return;
#pragma unroll
  for (int i = 1; i < GR; ++i) o += so[i][d4];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int t = row / a.G, head = h * a.G + row % a.G;
  T* dst = static_cast<T*>(a.o) + b * a.o_sb + t * a.o_st + head * a.o_sh + 4 * d4;
  *reinterpret_cast<u32x2*>(dst) =
      u32x2{pair_of<T>(o[0] * inv, o[1] * inv), pair_of<T>(o[2] * inv, o[3] * inv)};
  if (a.lse != nullptr && d4 == 0)
    a.lse[((int64_t)b * a.G * a.c.H + head) * a.Tq + t] =
        l == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(l)) * kLn2;
}

// The same with few parts (up to 16) of many rows (1024 and more): a wavefront has a
// row to itself, D / 64 channels a lane, and no other to wait for (us, the sum's share
// of all: 4 parts of 16000 rows 104 -> 99; fewer rows leave too few wavefronts: 16 of
// 16 rows 9.5 -> 10.8).
template <typename T, int D, typename Args>
__global__ __launch_bounds__(256) void kv4_combine_rows_kernel(Args a) {
  constexpr int CL = D / 64, LANES = is_tree<Args> ? 64 : 16;  // of parts, at most
  const int rows = a.Tq * a.G;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t out = (int64_t)blockIdx.x * 4 + wave;
  if (out >= (int64_t)a.c.B * a.c.H * rows) return;
  const int bh = (int)(out / rows), row = (int)(out - (int64_t)bh * rows);
  const int b = bh / a.c.H, h = bh - b * a.c.H;
  const Parts in = parts_of(a, bh, row);
  if (is_tree<Args> && in.parts == 1) return;  // written by the part
  const int64_t id = in.id, all = in.all;
  float m = -INFINITY, l = 0.f;
  if (lane < in.parts) {
    const float* ml = a.part_ml + 2 * (lane * all + id);
    m = ml[0];
    l = ml[1];
  }
  float top = m;
#pragma unroll
  for (int d = 1; d < LANES; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  float f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
  const bool empty = l == 0.f;  // such a part's sums are not there
  l = empty ? 0.f : l * f;
  f = empty ? -1.f : f;
#pragma unroll
  for (int d = 1; d < LANES; d *= 2) l += __shfl_xor(l, d);
  l = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(l)));
  float o[CL];
#pragma unroll
  for (int i = 0; i < CL; ++i) o[i] = 0.f;
  const float* src = a.part + id * D + CL * lane;
  for (int p0 = 0; p0 < in.parts; p0 += 4) {
    float x[4][CL];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < CL; ++i) x[j][i] = src[min(p0 + j, in.parts - 1) * all * D + i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // an empty part, or one past the last, holds anything
      const float w = __shfl(f, p0 + j);
      if (p0 + j < in.parts && !(w < 0.f))
#pragma unroll
        for (int i = 0; i < CL; ++i) o[i] = fmaf(x[j][i], w, o[i]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int t = row / a.G, head = h * a.G + row - t * a.G;
  T* dst = static_cast<T*>(a.o) + b * a.o_sb + t * a.o_st + head * a.o_sh + CL * lane;
  if constexpr (CL == 2)
    *reinterpret_cast<uint32_t*>(dst) = pair_of<T>(o[0] * inv, o[1] * inv);
  else
    *dst = static_cast<T>(o[0] * inv);
  if (a.lse != nullptr && lane == 0)
    a.lse[((int64_t)b * a.G * a.c.H + head) * a.Tq + t] =
        l == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(l)) * kLn2;
}

template <typename T, int D, typename Args>
hipError_t launch_attn_typed(const Args& a, hipStream_t st) {
  int64_t groups = (int64_t)a.parts * a.nrb * a.c.B * a.c.H;
  int parts = a.parts;  // of a row
  if constexpr (is_tree<Args>) {
    if (a.units > 0) {
      groups = (int64_t)a.units * a.nrb * a.c.H;
      parts = (a.units + a.c.B - 1) / a.c.B;  // on average (more than 1)
    }
  }
  const dim3 grid((unsigned)groups);
  // codes and scales, against half of the 256 MiB of last-level cache
  const bool far = (int64_t)a.c.B * a.c.H * a.c.C * (D + D / 16) > (int64_t(128) << 20);
  const dim3 few(64 * (is_tree<Args> ? kTreeWaves : kRowWaves));
  if (a.row_tiles == 1 && far)
    hipLaunchKernelGGL((kv4_rows_kernel<T, D, 1, true, Args>), grid, few, 0, st, a);
  else if (a.row_tiles == 1)
    hipLaunchKernelGGL((kv4_rows_kernel<T, D, 1, false, Args>), grid, few, 0, st, a);
  else if (a.row_tiles == 2 && far)
    hipLaunchKernelGGL((kv4_rows_kernel<T, D, 2, true, Args>), grid, few, 0, st, a);
  else if (a.row_tiles == 2)
    hipLaunchKernelGGL((kv4_rows_kernel<T, D, 2, false, Args>), grid, few, 0, st, a);
  else
    hipLaunchKernelGGL((kv4_block_kernel<T, D, Args>), grid, dim3(256), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || parts == 1) return e;
  const int64_t rows = (int64_t)a.c.B * a.c.H * a.G * a.Tq;
  if (parts <= 16 && rows >= 1024)
    hipLaunchKernelGGL((kv4_combine_rows_kernel<T, D, Args>), dim3((unsigned)((rows + 3) / 4)),
                       dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((kv4_combine_kernel<T, D, Args>), dim3((unsigned)rows), dim3(256), 0, st,
                       a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Key weights: w_j = sum over the rows of exp(s_ij - lse_i). A lane adds up its
// 4 keys of each 16 over the rows of its column, and the 16 columns at the end, so
// no sum depends on the order of anything else. Every slot is written (added to): 0
// in those that hold nothing.

// The positions in `slots` slots from slot0 on: the newest there, len - 1 - (len - 1 -
// slot) mod C, in a row from p0 on but for a step back by C at the wrap-th, and
// negative where there is none. most: the newest of them, least: no later than any.
struct Held {
  int p0, slots, wrap, least, most;
};
__device__ __forceinline__ Held held_at(int slot0, int group, int len, int C) {
  Held x;
  x.p0 = len - 1 - (int)((uint32_t)(len - 1 - slot0 + C) % (uint32_t)C);
  x.slots = min(group, C - slot0);
  x.wrap = min(x.slots, len - x.p0);
  x.most = x.p0 + x.wrap - 1 >= 0 ? x.p0 + x.wrap - 1 : -1;
  x.least = x.wrap < x.slots && x.p0 + x.slots - 1 - C >= 0 ? max(0, x.p0 + x.wrap - C)
                                                           : max(0, x.p0);
  return x;
}

// Codes of 16 NK keys from slot0 on, those past the last slot of a head unused.
template <int D, int NK>
struct KeyCodes {
  u32x4 w[NK];  // D = 64: the first two words
  uint32_t s[NK];
};
template <int D, int NK>
__device__ __forceinline__ void load_keys(KeyCodes<D, NK>& x, const Kv4Cache& c, int bh, int slot0,
                                          int lane) {
  const int quarter = lane >> 4, n = lane & 15;
  const uint32_t at = n * (D / 2) + quarter * (D / 8), s_at = n * (D / 32) + quarter * (D / 4) / 32;
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int64_t row = (int64_t)bh * c.C + min(slot0 + 16 * i, c.C - 16);
    const uint8_t* src = c.kc + row * (D / 2);
    if constexpr (D == 128) {
      x.w[i] = *reinterpret_cast<const u32x4*>(src + at);
    } else {
      const u32x2 half = *reinterpret_cast<const u32x2*>(src + at);
      x.w[i][0] = half[0];
      x.w[i][1] = half[1];
    }
    x.s[i] = (c.ks + row * (D / 32))[s_at];
  }
}

// The sum over a row of 16 lanes, in every one of them.
template <int CTRL>
__device__ __forceinline__ float add_ror(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float row_sum(float x) {
  x = add_ror<0x121>(x);  // row_ror:1
  x = add_ror<0x122>(x);
  x = add_ror<0x124>(x);
  return add_ror<0x128>(x);
}

template <int NK>
__device__ __forceinline__ void store_weights(const Kv4WeightsArgs& a, float (&w)[NK][4], int bh,
                                              int slot0, int lane) {
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    if (slot0 + 16 * i >= a.c.C) break;
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = row_sum(w[i][e]);
    if ((lane & 15) == 0) {
      f32x4* at = reinterpret_cast<f32x4*>(a.weights + (int64_t)bh * a.c.C + slot0 + 16 * i +
                                           4 * (lane >> 4));
      if (a.accumulate) x += *at;
      *at = x;
    }
  }
}

// Up to 16 rows (a token's, or a few tokens'): they stay in registers and the keys
// stream by, the next ones loaded ahead. Bound by its traffic: a token of 8 sequences
// of up to 16000 keys, 43 MB, 13.0 us (a workgroup for every 256 keys: 22).
template <typename T, int D>
__global__ __launch_bounds__(256, 4) void kv4_weights_rows_kernel(Kv4WeightsArgs a) {
  constexpr int STEPS = D / 32, NK = 4, GROUP = 16 * NK;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int quarter = lane >> 4, n = lane & 15;
  const int C = a.c.C;
  const int bh = blockIdx.y, b = bh / a.c.H, h = bh - b * a.c.H;
  const int t = min(n / a.G, a.Tq - 1), head = h * a.G + n % a.G;
  u32x4 q[STEPS];
  {
    const T* src = static_cast<const T*>(a.q) + b * a.q_sb + t * a.q_st + (int64_t)head * a.q_sh +
                   quarter * (D / 4);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) q[i] = *reinterpret_cast<const u32x4*>(src + 8 * i);
  }
  float lse = a.lse[((int64_t)b * a.G * a.c.H + head) * a.Tq + t] * kLog2e;
  const int len = length_of(a.c.len, b), n_new = count_of(a.counts, b, a.Tq);
  const RowRange rr = row_range(n / a.G, n_new, len, C, a.window);
  // a row that does not count, or sees nothing: every exponential is 0, whatever it holds
  if (rr.lo > rr.hi || lse == -INFINITY) {
    lse = INFINITY;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) q[i] = u32x4{0u, 0u, 0u, 0u};
  }
  // what all, and any, of the rows see
  const int rows = min(16, n_new * a.G);
  const RowRange first = row_range(0, n_new, len, C, a.window);
  const RowRange last = row_range((rows - 1) / a.G, n_new, len, C, a.window);
  const int stride = gridDim.x * 4 * GROUP;
  int slot0 = (blockIdx.x * 4 + wave) * GROUP;
  if (slot0 >= C) return;
  Held at = held_at(slot0, GROUP, len, C);
  auto seen = [&](const Held& x) { return rows > 0 && x.most >= first.lo && x.least <= last.hi; };
  KeyCodes<D, NK> x = {}, next = {};
  if (seen(at)) load_keys<D, NK>(x, a.c, bh, slot0, lane);
  for (;;) {
    const int slot_n = slot0 + stride;
    const bool more = stride < C - slot0;
    const Held at_n = more ? held_at(slot_n, GROUP, len, C) : at;
    if (more && seen(at_n)) load_keys<D, NK>(next, a.c, bh, slot_n, lane);
    if (seen(at)) {
      const bool full = at.p0 >= last.lo && at.wrap == GROUP && at.p0 + GROUP - 1 <= first.hi;
      float w[NK][4];
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        f32x4 s;
        const float sc = scale_of(x.s[i]);
#pragma unroll
        for (int j = 0; j < STEPS; ++j)
          s = Fmt<T>::mfma(values8<T>(x.w[i][j], sc), q[j], j == 0 ? f32x4{} : s);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[i][e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.c_log2, -lse));
      }
      if (!full) {
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int y = 16 * i + 4 * quarter + e;
            const int p = y < at.wrap ? at.p0 + y : y < at.slots ? at.p0 + y - C : -1;
            if (p < rr.lo || p > rr.hi) w[i][e] = 0.f;
          }
      }
      store_weights<NK>(a, w, bh, slot0, lane);
    } else if (!a.accumulate && lane < at.slots) {
      a.weights[(int64_t)bh * C + slot0 + lane] = 0.f;
    }
    if (!more) return;
    slot0 = slot_n;
    at = at_n;
    x = next;
  }
}

// Many rows: a wavefront holds 64 keys and sweeps the rows; 64 rows at a time go
// through LDS, for the workgroup's 4 wavefronts, the next ones loaded a turn ahead
// (each wavefront loading 16 rows for itself, a turn ahead too, waited for them: 66
// us for 512 queries on 16384 keys, 16/8 heads of 128, against 53). Rows of 2 D
// bytes, chunk c of 16 at c ^ (row % 16), so that 16 rows' reads spread over the banks.
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void kv4_weights_kernel(Kv4WeightsArgs a) {
  constexpr int STEPS = D / 32, NK = 4, GROUP = 16 * NK, ROWS = 64;
  constexpr int CH = D / 8;            // chunks of a row
  constexpr int PASS = ROWS * CH / 256;  // a thread loads one chunk of so many rows
  constexpr int PROWS = ROWS / PASS;
  __shared__ __attribute__((aligned(16))) char sq[2][ROWS * D * 2];
  __shared__ float sl[2][ROWS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int quarter = lane >> 4, n = lane & 15;
  const int C = a.c.C;
  const int bh = blockIdx.y, b = bh / a.c.H, h = bh - b * a.c.H;
  const int slot_wg = blockIdx.x * 4 * GROUP, slot0 = slot_wg + wave * GROUP;
  const int len = length_of(a.c.len, b), n_new = count_of(a.counts, b, a.Tq);
  // rows that can see one of the workgroup's keys: pos >= least, pos - W < most
  const Held all = held_at(slot_wg, 4 * GROUP, len, C);
  const int base = len - n_new;
  int64_t t0 = 0, t1 = 0;
  if (all.most >= 0) {
    t1 = n_new;
    if (a.window > 0) t1 = min(t1, (int64_t)all.most + a.window - base);
    t1 = max(t1, (int64_t)0);
    t0 = min(max((int64_t)all.least - base, (int64_t)0), t1);
  }
  const int row_end = (int)t1 * a.G;  // at most Tq G
  int row0 = (int)t0 * a.G;
  const bool own = slot0 < C;  // a wavefront without slots loads rows for the others
  const Held at = held_at(own ? slot0 : 0, GROUP, len, C);

  uint32_t kw[NK][STEPS], ks[NK];
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int64_t row = (int64_t)bh * C + min(slot0 + 16 * i, C - 16) + n;  // past C: unused
#pragma unroll
    for (int j = 0; j < STEPS; ++j)
      kw[i][j] = *reinterpret_cast<const uint32_t*>(a.c.kc + row * (D / 2) + (4 * j + quarter) * 4);
    ks[i] = 0;
#pragma unroll
    for (int j = 0; j < STEPS; ++j) ks[i] |= (uint32_t)a.c.ks[row * STEPS + j] << (8 * j);
  }
  // The thread's rows: where they lie, moved on by 64 a turn without a division; past
  // the end they stay where they are, and do not count.
  const int dt = ROWS / a.G, dg = ROWS % a.G;
  const int64_t q_step = dt * a.q_st + dg * a.q_sh, q_wrap = a.q_st - a.G * a.q_sh;
  int row_l[PASS], g_l[PASS];
  const T* q_l[PASS];
  u32x4 qn[PASS];
#pragma unroll
  for (int i = 0; i < PASS; ++i) {
    row_l[i] = row0 + i * PROWS + tid / CH;
    const int row = max(min(row_l[i], row_end - 1), 0), t = row / a.G;
    g_l[i] = row - t * a.G;
    q_l[i] = static_cast<const T*>(a.q) + b * a.q_sb + t * a.q_st +
             (int64_t)(h * a.G + g_l[i]) * a.q_sh + tid % CH * 8;
  }
  float lse_n = 0.f;  // of row row0 + tid, threads 0 .. 63
  auto fetch = [&](int row0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      qn[i] = *reinterpret_cast<const u32x4*>(q_l[i]);
      if (row_l[i] >= row_end) qn[i] = u32x4{0u, 0u, 0u, 0u};  // whatever the row before holds
    }
    if (wave == 0) {
      const int row = min(row0 + lane, row_end - 1), t = row / a.G;
      lse_n = a.lse[((int64_t)bh * a.G + row - t * a.G) * a.Tq + t] * kLog2e;
      // a row that is not there, or sees nothing: every exponential is 0
      if (row0 + lane >= row_end || lse_n == -INFINITY) lse_n = INFINITY;
    }
  };
  auto put = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      const int row = i * PROWS + tid / CH;
      *reinterpret_cast<u32x4*>(sq[buf] + row * (D * 2) + (((tid % CH) ^ row) & (CH - 1)) * 16) =
          qn[i];
    }
    if (wave == 0) sl[buf][lane] = lse_n;
  };
  auto move_on = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      row_l[i] += ROWS;
      if (row_l[i] < row_end) {
        const bool wrap = g_l[i] + dg >= a.G;
        g_l[i] += wrap ? dg - a.G : dg;
        q_l[i] += wrap ? q_step + q_wrap : q_step;
      }
    }
  };
  float w[NK][4];
  u32x4 k[NK][STEPS];
#pragma unroll
  for (int i = 0; i < NK; ++i) {
#pragma unroll
    for (int j = 0; j < STEPS; ++j)
      k[i][j] = values8<T>(kw[i][j], scale_of((ks[i] >> (8 * j)) & 255u));
#pragma unroll
    for (int e = 0; e < 4; ++e) w[i][e] = 0.f;
  }
  const bool whole = at.p0 >= 0 && at.wrap == GROUP;  // every slot holds p0 + its number
  if (row0 < row_end) {
    fetch(row0);
    put(0);
    move_on();
  }
  int buf = 0;
  for (; row0 < row_end; row0 += ROWS, buf ^= 1) {
    __syncthreads();  // this turn's rows are written, the last turn's read
    const bool more = row0 + ROWS < row_end;
    if (more) fetch(row0 + ROWS);
    // what all of the 64 rows see
    const int t_lo = row0 / a.G, t_hi = (min(row0 + ROWS, row_end) - 1) / a.G;
    const bool full = whole && at.p0 >= row_range(t_hi, n_new, len, C, a.window).lo &&
                      at.p0 + GROUP - 1 <= row_range(t_lo, n_new, len, C, a.window).hi;
    // the scores of 16 rows are issued against the exponentials of the 16 before
    auto scores = [&](f32x4 (&s)[NK], int r) __attribute__((always_inline)) {
      const int row = 16 * r + n;
      u32x4 q[STEPS];
#pragma unroll
      for (int j = 0; j < STEPS; ++j)
        q[j] = *reinterpret_cast<const u32x4*>(sq[buf] + row * (D * 2) +
                                               (((4 * j + quarter) ^ row) & (CH - 1)) * 16);
#pragma unroll
      for (int j = 0; j < STEPS; ++j)
#pragma unroll
        for (int i = 0; i < NK; ++i)
          s[i] = Fmt<T>::mfma(k[i][j], q[j], j == 0 ? f32x4{} : s[i]);
    };
    auto add = [&](auto masked) __attribute__((always_inline)) {
      f32x4 s[2][NK];
      scores(s[0], 0);
#pragma unroll
      for (int r = 0; r < ROWS / 16; ++r) {
        if (r + 1 < ROWS / 16) scores(s[(r + 1) & 1], r + 1);
        const float lse = sl[buf][16 * r + n];
        RowRange rr = {0, 0};
        if constexpr (decltype(masked)::value)
          rr = row_range((row0 + 16 * r + n) / a.G, n_new, len, C, a.window);
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = __builtin_amdgcn_exp2f(fmaf(s[r & 1][i][e], a.c_log2, -lse));
            if constexpr (decltype(masked)::value) {
              const int y = 16 * i + 4 * quarter + e;
              const int p = y < at.wrap ? at.p0 + y : y < at.slots ? at.p0 + y - C : -1;
              w[i][e] += p >= rr.lo && p <= rr.hi ? x : 0.f;
            } else {
              w[i][e] += x;
            }
          }
      }
    };
    if (full)
      add(Bool<false>());
    else
      add(Bool<true>());
    if (more) {
      put(buf ^ 1);
      move_on();
    }
  }
  if (own) store_weights<NK>(a, w, bh, slot0, lane);
}

template <typename T, int D>
hipError_t launch_weights_typed(const Kv4WeightsArgs& a, hipStream_t st) {
  constexpr int NK = 4;
  const int groups = (a.c.C + 64 * NK - 1) / (64 * NK), heads = a.c.B * a.c.H;  // of 4 wavefronts
  if ((int64_t)a.Tq * a.G <= 16) {
    const int64_t each = ((int64_t)groups * heads + 1023) / 1024;  // groups a workgroup
    const dim3 grid((unsigned)((groups + each - 1) / each), heads);
    hipLaunchKernelGGL((kv4_weights_rows_kernel<T, D>), grid, dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((kv4_weights_kernel<T, D>), dim3(groups, heads), dim3(256), 0, st, a);
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Eviction. One workgroup per head finds the weight of the last key to keep by
// its digits, most significant first (11, 11 and 10 bits), and writes the
// positions that stay, in order. Wavefronts own runs of keys, so a key's place
// is the count of kept ones before it: in the wavefront by ballot, over the
// wavefronts by one sum. A capacity of up to 64 keys a thread is read once, into
// registers (REGS of them); a longer one at every pass (REGS = 0). Bound by a CU's
// latencies and VALU, as there are few heads: 16 of 32768 keys 19 to 22 us, of which 6 are
// the loads (read at every pass 38); 8 of 131072, at every pass, 132. The loads of 8
// keys are asked for together, also those of keys that are not there (each waited for by
// itself, behind its condition: 33 and 174). Keys past a wavefront's run are skipped by
// 8: with the copies of the rows 40 us, one by one 49; with none skipped 40, but 1001
// keys in room for 32768 21 instead of 15.5.
constexpr int kSelThreads = 1024;
constexpr int kSelStep = 8;  // loads at once

// Weights in the order of unsigned numbers between 0 and 2^32 - 1, NaN before all
// of them; -0 is 0.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (!(w == w)) return 1u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Of the lanes in m, how many come before this one.
__device__ __forceinline__ int lanes_below(uint64_t m) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

template <int REGS>
__global__ __launch_bounds__(kSelThreads) void kv4_select_kernel(Kv4EvictArgs a) {
  constexpr int WAVES = kSelThreads / 64;
  __shared__ uint32_t hist[2048];
  __shared__ uint32_t wsum[WAVES];
  __shared__ uint32_t found[3];  // digit, how many of its keys stay, and how many there are
  __shared__ int above[WAVES], equal[WAVES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bh = blockIdx.x, b = bh / a.c.H, C = a.c.C;
  const int len = length_of(a.c.len, b);
  const int n = min(len, C), first = len - n;
  const int kept = min(n, a.keep), must = min(a.recent, kept);
  const int cand = n - must;          // the older keys, of which
  const uint32_t want = kept - must;  // so many stay
  const float* wt = a.weights + (int64_t)bh * C;
  const int slot0 = (int)((uint32_t)first % (uint32_t)C);
  const int run = (n + WAVES * 64 - 1) / (WAVES * 64) * 64;  // keys of a wavefront
  const int j0 = wave * run + lane;
  // of the j-th oldest: an older key's weight, the most for a new one, 0 for none
  auto slot_of = [&](int j) __attribute__((always_inline)) {
    const int s = slot0 + j;
    return s >= C ? s - C : s;
  };
  auto order = [&](int j, float w) __attribute__((always_inline)) {
    return j < cand ? order_of(w) : j < n ? 0xffffffffu : 0u;
  };
  constexpr int STEP = REGS > 0 && REGS < kSelStep ? REGS : kSelStep;
  auto load = [&](float* w, int i0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < STEP; ++i) {  // in bounds: slot 0 for what is none of the older keys
      const int j = j0 + (i0 + i) * 64;
      w[i] = wt[j < cand ? slot_of(j) : 0];
    }
  };
  // from the run's end on the keys are the next wavefront's: none here
  auto value = [&](int i, float w) __attribute__((always_inline)) {
    return i * 64 < run ? order(j0 + i * 64, w) : 0u;
  };
  uint32_t u[REGS > 0 ? REGS : 1];
  if constexpr (REGS > 0) {
    float w[REGS];
#pragma unroll
    for (int i0 = 0; i0 < REGS; i0 += STEP)
      if (i0 * 64 < run) load(w + i0, i0);
#pragma unroll
    for (int i = 0; i < REGS; ++i) u[i] = value(i, w[i]);
  }
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (REGS > 0) {
#pragma unroll
      for (int i0 = 0; i0 < REGS; i0 += STEP) {
        if (i0 * 64 >= run) break;
#pragma unroll
        for (int i = i0; i < i0 + STEP; ++i) f(j0 + i * 64, u[i]);
      }
    } else {
      for (int i0 = 0; i0 * 64 < run; i0 += STEP) {
        float w[STEP];
        load(w, i0);
#pragma unroll
        for (int i = 0; i < STEP; ++i) f(j0 + (i0 + i) * 64, value(i0 + i, w[i]));
      }
    }
  };

  uint32_t prefix = 0, need = want;  // of the keys with this prefix, so many stay
  if (want > 0 && (int)want < cand) {
    int shift = 21, bits = 11;
    for (int pass = 0; pass < 3; ++pass) {
      for (int i = tid; i < 2048; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      const uint32_t mask = pass == 0 ? 0u : 0xffffffffu << (shift + bits);
      each([&](int j, uint32_t x) __attribute__((always_inline)) {
        if (x - 1 < 0xfffffffeu && (x & mask) == prefix)  // an older key's
          atomicAdd(&hist[(x >> shift) & ((1u << bits) - 1)], 1u);
      });
      __syncthreads();
      // bins from the top: thread t has bins 2047 - 2 t and the one below
      const uint32_t hi = hist[2047 - 2 * tid], lo = hist[2046 - 2 * tid];
      uint32_t sum = hi + lo;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const uint32_t o = __shfl_up(sum, d);
        if (lane >= d) sum += o;
      }
      if (lane == 63) wsum[wave] = sum;
      __syncthreads();
      uint32_t others = lane < wave ? wsum[lane] : 0u;  // wave < 16
#pragma unroll
      for (int d = 1; d < WAVES; d *= 2) others += __shfl_xor(others, d);
      sum += __builtin_amdgcn_readfirstlane(others);
      const uint32_t before = sum - hi - lo;
      if (before < need && need <= before + hi) {
        found[0] = 2047 - 2 * tid;
        found[1] = need - before;
        found[2] = hi;
      } else if (before + hi < need && need <= sum) {
        found[0] = 2046 - 2 * tid;
        found[1] = need - before - hi;
        found[2] = lo;
      }
      __syncthreads();
      prefix |= found[0] << shift;
      need = found[1];
      if (need == found[2]) {  // all of the digit's keys: what is above the number before it
        prefix -= 1;           // (it is not 0: then every older key would stay)
        need = 0;
        break;
      }
      bits = pass == 1 ? 10 : 11;
      shift -= bits;
      __syncthreads();
    }
  } else {  // all of the older keys, or none
    need = 0;
    prefix = want == 0 ? 0xfffffffeu : 0u;
  }
  // need of the keys equal to prefix stay, the oldest, and all above it
  int up = 0, eq = 0;
  each([&](int j, uint32_t x) __attribute__((always_inline)) {
    up += x > prefix;
    eq += x == prefix;
  });
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    up += __shfl_xor(up, d);
    eq += __shfl_xor(eq, d);
  }
  if (lane == 0) {
    above[wave] = up;
    equal[wave] = eq;
  }
  __syncthreads();
  // keys before this wavefront's run, of lanes 0 .. 15 one run each
  int eq_at = lane < wave ? equal[lane] : 0, at = lane < wave ? above[lane] : 0;
#pragma unroll
  for (int d = 1; d < WAVES; d *= 2) {
    eq_at += __shfl_xor(eq_at, d);
    at += __shfl_xor(at, d);
  }
  eq_at = __builtin_amdgcn_readfirstlane(eq_at);
  at = __builtin_amdgcn_readfirstlane(at) + min(eq_at, (int)need);
  int32_t* index = a.index + (int64_t)bh * a.keep;
  each([&](int j, uint32_t x) __attribute__((always_inline)) {
    bool stays = x > prefix;
    if (need > 0) {
      const uint64_t eqs = __ballot(x == prefix);
      stays = stays || (x == prefix && eq_at + lanes_below(eqs) < (int)need);
      eq_at += __popcll(eqs);
    }
    const uint64_t all = __ballot(stays);
    if (stays) index[at + lanes_below(all)] = first + j;
    at += __popcll(all);
  });
  for (int j = kept + tid; j < a.keep; j += kSelThreads) index[j] = -1;
  if (tid == 0 && bh % a.c.H == 0) a.out.len[b] = kept;
}

// The kept rows, 4 new slots to D / 8 threads: a thread takes 32 channels of one
// of the keys, 8 channels of the 4 values. Bound by its traffic: half of 32768 keys of
// 2 x 8 heads, 36 MB in (and as much again beside it in the same lines) and 36 out, 24
// us (4 bytes a lane of the keys: 37).
template <int D>
__global__ __launch_bounds__(256) void kv4_gather_kernel(Kv4EvictArgs a) {
  constexpr int R = D / 8, BL = D / 32;
  const int bh = blockIdx.y, C = a.c.C, CN = a.out.C;
  const int g = (int)(((int64_t)blockIdx.x * 256 + threadIdx.x) / R), r = threadIdx.x % R;
  if (4 * g >= CN) return;
  const int32_t* index = a.index + (int64_t)bh * a.keep;
  const int64_t base = (int64_t)bh * C, row_n = (int64_t)bh * CN + 4 * g, gn = row_n >> 2;
  int slot[4];  // -1: none
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int j = 4 * g + e, p = j < a.keep ? index[j] : -1;
    slot[e] = p < 0 ? -1 : (int)((uint32_t)p % (uint32_t)C);
  }
  const int ek = r / BL, ck = r % BL;
  const int sk = ek == 0 ? slot[0] : ek == 1 ? slot[1] : ek == 2 ? slot[2] : slot[3];
  u32x4 kw = {0u, 0u, 0u, 0u}, vw = kw;
  uint8_t ks = 0;
  if (sk >= 0) {
    kw = *reinterpret_cast<const u32x4*>(a.c.kc + ((base + sk) * BL + ck) * 16);
    ks = a.c.ks[(base + sk) * BL + ck];
  }
  uint32_t vsw = 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (slot[e] < 0) continue;
    const int64_t go = (base + slot[e]) >> 2;
    const int eo = slot[e] & 3;
    vw[e] = *reinterpret_cast<const uint32_t*>(a.c.vc + ((go * R + r) * 4 + eo) * 4);
    if (r < BL) vsw |= (uint32_t)a.c.vs[(go * BL + r) * 4 + eo] << (8 * e);
  }
  if (a.new_weights != nullptr && r < 4) {
    const int s = r == 0 ? slot[0] : r == 1 ? slot[1] : r == 2 ? slot[2] : slot[3];
    a.new_weights[row_n + r] = s >= 0 ? a.weights[base + s] : 0.f;
  }
  if (slot[0] < 0) return;  // kept ones come first
  if (sk >= 0) {
    *reinterpret_cast<u32x4*>(a.out.kc + ((row_n + ek) * BL + ck) * 16) = kw;
    a.out.ks[(row_n + ek) * BL + ck] = ks;
  }
  *reinterpret_cast<u32x4*>(a.out.vc + (gn * R + r) * 16) = vw;
  if (r < BL) *reinterpret_cast<uint32_t*>(a.out.vs + (gn * BL + r) * 4) = vsw;
}

// ---------------------------------------------------------------------------
// Commit: nodes of a draft become the next positions of their sequences, bit by bit.
// D / 8 threads a node and head: a word of its value each, and D / 32 of them 16 bytes of
// its key and the scales. A node of 8 heads of 128 is 1088 bytes: bound by the launch.
template <int D>
__device__ __forceinline__ void commit_words(const Kv4CommitArgs& a, int b, int h, int len, int i,
                                             int r) {
  constexpr int R = D / 8, BL = D / 32;
  const int node = min(max(a.path[(int64_t)b * a.P + i], 0), a.d.C - 1);
  const int64_t bh = (int64_t)b * a.c.H + h;
  const int64_t src = bh * a.d.C + node;
  const int64_t dst = bh * a.c.C + ((uint32_t)len + (uint32_t)i) % (uint32_t)a.c.C;
  const int es = src & 3, ed = dst & 3;
  *reinterpret_cast<uint32_t*>(a.c.vc + (((dst >> 2) * R + r) * 4 + ed) * 4) =
      *reinterpret_cast<const uint32_t*>(a.d.vc + (((src >> 2) * R + r) * 4 + es) * 4);
  if (r < BL) {
    *reinterpret_cast<u32x4*>(a.c.kc + (dst * BL + r) * 16) =
        *reinterpret_cast<const u32x4*>(a.d.kc + (src * BL + r) * 16);
    a.c.ks[dst * BL + r] = a.d.ks[src * BL + r];
    a.c.vs[((dst >> 2) * BL + r) * 4 + ed] = a.d.vs[((src >> 2) * BL + r) * 4 + es];
  }
  if (a.weights != nullptr && r == 0) a.weights[dst] = 0.f;
}

// A sequence's lengths are written by the workgroup that has read its length, so with SMALL
// it has all of the sequence's nodes; else they are another launch's. Bound by the launch and
// two loads that wait for each other, a node's number and its words: 4 nodes of one sequence
// 2.3 us, 16 of 64 sequences 3.5.
template <int D, bool SMALL>
__global__ __launch_bounds__(SMALL ? 1024 : 256) void commit_kernel(Kv4CommitArgs a) {
  constexpr int R = D / 8;
  const int b = SMALL ? blockIdx.x : blockIdx.y;
  const int len = length_of(a.c.len, b), n = count_of(a.counts, b, a.P);
  const int items = n * a.c.H * R;
  for (int64_t i = (SMALL ? 0 : (int64_t)blockIdx.x * 256) + threadIdx.x; i < items;
       i += SMALL ? 1024 : (int64_t)gridDim.x * 256) {
    const int node = (int)i / R;
    commit_words<D>(a, b, node % a.c.H, len, node / a.c.H, (int)i % R);
  }
  if constexpr (SMALL) {
    __syncthreads();  // every thread has read the length
    if (threadIdx.x == 0) {
      a.c.len[b] = length_after(len, n, a.c.C);
      if (a.reset) a.d.len[b] = 0;
    }
  }
}

__global__ void commit_lengths_kernel(Kv4CommitArgs a) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < a.c.B) {
    a.c.len[b] = length_after(length_of(a.c.len, b), count_of(a.counts, b, a.P), a.c.C);
    if (a.reset) a.d.len[b] = 0;
  }
}

template <int D>
hipError_t launch_commit_typed(const Kv4CommitArgs& a, hipStream_t st) {
  const int64_t items = (int64_t)a.P * a.c.H * (D / 8);
  if (items <= 8 * 1024) {
    hipLaunchKernelGGL((commit_kernel<D, true>), dim3(a.c.B), dim3(1024), 0, st, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((commit_kernel<D, false>), dim3((unsigned)((items + 255) / 256), a.c.B),
                     dim3(256), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(commit_lengths_kernel, dim3((a.c.B + 255) / 256), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv4_commit(const Kv4CommitArgs& a, hipStream_t st) {
  return a.c.D == 128 ? launch_commit_typed<128>(a, st) : launch_commit_typed<64>(a, st);
}

hipError_t launch_kv4_tree_attn(const Kv4TreeArgs& a, Elem dtype, hipStream_t st) {
  if (dtype == Elem::BF16)
    return a.c.D == 128 ? launch_attn_typed<__bf16, 128>(a, st)
                        : launch_attn_typed<__bf16, 64>(a, st);
  return a.c.D == 128 ? launch_attn_typed<_Float16, 128>(a, st)
                      : launch_attn_typed<_Float16, 64>(a, st);
}

hipError_t launch_kv4_append(const Kv4AppendArgs& a, Elem dtype, hipStream_t st) {
  if (dtype == Elem::BF16)
    return a.c.D == 128 ? launch_append<__bf16, 128>(a, st) : launch_append<__bf16, 64>(a, st);
  return a.c.D == 128 ? launch_append<_Float16, 128>(a, st) : launch_append<_Float16, 64>(a, st);
}

hipError_t launch_kv4_read(const Kv4ReadArgs& a, Elem dtype, hipStream_t st) {
  if (dtype == Elem::BF16)
    return a.c.D == 128 ? launch_read<__bf16, 128>(a, st) : launch_read<__bf16, 64>(a, st);
  return a.c.D == 128 ? launch_read<_Float16, 128>(a, st) : launch_read<_Float16, 64>(a, st);
}

hipError_t launch_kv4_attn(const Kv4AttnArgs& a, Elem dtype, hipStream_t st) {
  if (dtype == Elem::BF16)
    return a.c.D == 128 ? launch_attn_typed<__bf16, 128>(a, st)
                        : launch_attn_typed<__bf16, 64>(a, st);
  return a.c.D == 128 ? launch_attn_typed<_Float16, 128>(a, st)
                      : launch_attn_typed<_Float16, 64>(a, st);
}

hipError_t launch_kv4_weights(const Kv4WeightsArgs& a, Elem dtype, hipStream_t st) {
  if (dtype == Elem::BF16)
    return a.c.D == 128 ? launch_weights_typed<__bf16, 128>(a, st)
                        : launch_weights_typed<__bf16, 64>(a, st);
  return a.c.D == 128 ? launch_weights_typed<_Float16, 128>(a, st)
                      : launch_weights_typed<_Float16, 64>(a, st);
}

hipError_t launch_kv4_evict(const Kv4EvictArgs& a, hipStream_t st) {
  const int heads = a.c.B * a.c.H;
  // registers by the keys a thread may have: 1001 in room for 1024 take 6.2 us with one,
  // 7.8 with 8, 11.2 read at every pass
  const int per = (a.c.C + kSelThreads - 1) / kSelThreads;
  if (per <= 1)
    hipLaunchKernelGGL((kv4_select_kernel<1>), dim3(heads), dim3(kSelThreads), 0, st, a);
  else if (per <= 8)
    hipLaunchKernelGGL((kv4_select_kernel<8>), dim3(heads), dim3(kSelThreads), 0, st, a);
  else if (per <= 32)
    hipLaunchKernelGGL((kv4_select_kernel<32>), dim3(heads), dim3(kSelThreads), 0, st, a);
  else if (per <= 64)
    hipLaunchKernelGGL((kv4_select_kernel<64>), dim3(heads), dim3(kSelThreads), 0, st, a);
  else
    hipLaunchKernelGGL((kv4_select_kernel<0>), dim3(heads), dim3(kSelThreads), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t items = (int64_t)(a.out.C / 4) * (a.c.D / 8);
  const dim3 grid((unsigned)((items + 255) / 256), heads);
  if (a.c.D == 128)
    hipLaunchKernelGGL((kv4_gather_kernel<128>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((kv4_gather_kernel<64>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace ttcd
