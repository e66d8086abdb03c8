// sample.hip - a token from every row of logits, and the walk over a tree of drafted
// tokens that keeps those which agree, on gfx950.
//
// Sampling. Tokens rank by logit, of equal ones the lower index first, and weigh
// w = exp((x - max) / temperature). Kept are the first top_k, of those the shortest run
// with at least top_p of their sum, of those the ones with w >= min_p; the token is the
// first whose running sum exceeds uniform times the sum of all kept.
//
// A 16-bit logit has one of 65536 values, and everything above depends on a row only
// through how often each value comes: no sort, and no exponential of a token, but one for 8
// values in a row, which are a step apart, with a product for each of the others, in 64 bits,
// as are all sums. Counting is exact in any order, so a row's token does not depend on how
// its sums are laid out. A workgroup takes a row: it counts the values in LDS (16 bits a
// count, 128 KiB), finds the last kept value and the drawn one with how many of its tokens
// come before the drawn token, and looks for that one in the row, most of which is still in
// registers.
//
// Of a row of 151936 bf16 logits alone (25.7 us on a CU): zeroing 0.8 us, counting 12.2 (LDS
// atomics: 11 cycles for 64 tokens), sums of the values' weights 3.5 (f16, whose rows have
// 8 times the values, 7; 64 lanes a block with an exponential for every two values 4.9 and
// 14.7), cuts and draw 3.7 (one wavefront's latencies), the token 2.6. 256 rows, 78 MB: 35
// us, of which counting, at the rate of the memory (4.4 TB/s), is 17.6. Reading the row again
// for the token took 9.3 of 256 rows and 3.5 of one; the order of a value taken while
// counting, instead of its bits, 4 more. Not counting what a bound under the first top_k
// leaves out (20 of 151936: one row 25.9 to 25.1 us, 64 29.0 to 28.1, 256 34.3 to 34.6) was
// not worth its code.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "internal.h"
#include "wave.h"

namespace ttcd {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int16_t s16x2 __attribute__((ext_vector_type(2)));

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kBlocks = 512;     // of 128 values, 64 words of 2 counts
constexpr uint32_t kHeavy = 8192;  // a count of this and more moves to the list
constexpr uint32_t kHeavyBits = (0x10000u - kHeavy) * 0x10001u;  // that such a count has some of
constexpr int kHeavyMost = kSampleVocab / kHeavy + 1;
// Vectors of a thread between two looks at the counts: 7 turns of 1024 of them, with what a
// count may have by then, are below 65536.
constexpr int kStretch = 7;
constexpr int kHeld = 2 * kStretch;  // that stay in registers
constexpr int kGroup = 3;  // turns that are streamed at once; two groups make a stretch
constexpr int kTurnsMost = kSampleVocab / 8 / kSampleThreads + 1;

// The order of a 16-bit value is 0x7fff less its bits, of a negative one its bits: the
// largest come first. Infinity is kFirst, the last number above -infinity kLast; outside of
// those lie -infinity and NaN.
constexpr uint32_t kZero = 0x7fff;  // the order of +0; that of -0 is the next
template <typename T>
struct Order;
template <>
struct Order<__bf16> {
  static constexpr uint32_t kFirst = 0x7fff - 0x7f80, kLast = 0x7fff + 0x7f80;
};
template <>
struct Order<_Float16> {
  static constexpr uint32_t kFirst = 0x7fff - 0x7c00, kLast = 0x7fff + 0x7c00;
};
__device__ __forceinline__ uint32_t bits_of(uint32_t order) {
  return order <= kZero ? kZero - order : order;
}
template <typename T>
__device__ __forceinline__ double value_of(uint32_t order) {
  return (double)static_cast<float>(__builtin_bit_cast(T, (uint16_t)bits_of(order)));
}

struct Row {
  uint32_t* hist;       // [32768] counts of the values of bits 2 i and 2 i + 1
  double* sums;         // [kBlocks] of weights up to and with a block of 128 orders
  uint32_t* counts;     // the same of tokens
  uint32_t* tokens;     // of the block alone
  uint32_t* heavy;      // [2 kHeavyMost] order, count
  uint32_t nheavy, first, last;  // kFirst, kLast
  const double* powers; // [64] of 2^(i / 64)
  double top, per_t;    // the highest logit, and 1 / temperature

  // exp(y), y <= 0: 2^(k / 64) times the exponential of what is left, at most ln 2 / 128, by
  // its series up to the fifth power (the sixth is below 2^-54; what ln 2 / 64 lacks in 53
  // bits is worth 2^-55 |y|).
  __device__ __forceinline__ double weight_at(double x) const {
    if (top > 1e300) return x == top ? 1.0 : 0.0;  // infinity
    const double y = fmax((x - top) * per_t, -800.0);  // 0 from there on
    const double k = rint(y * 92.332482616893656877);  // 64 / ln 2
    const double r = fma(-k, 0.010830424696249145, y);
    double e = fma(r, 1.0 / 120, 1.0 / 24);
    e = fma(e, r, 1.0 / 6);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    const int n = (int)k;
    const double p = powers[n & 63];
    return ldexp(fma(p * r, e, p), n >> 6);
  }
  template <typename T>
  __device__ __forceinline__ double weight(uint32_t order) const {
    return weight_at(value_of<T>(order));
  }
  // The word of the counts of orders 2 i (in the low half) and 2 i + 1.
  __device__ __forceinline__ uint32_t word(int i) const {
    const uint32_t w = hist[i <= (int)kZero / 2 ? kZero / 2 - i : i];
    return i <= (int)kZero / 2 ? w << 16 | w >> 16 : w;
  }
  // Four of them, of orders 8 i and on.
  __device__ __forceinline__ u32x4 words(int i) const {
    const bool up = 8 * i <= (int)kZero;
    const u32x4 w = *reinterpret_cast<const u32x4*>(hist + (up ? (kZero - 7) / 2 - 4 * i : 4 * i));
    auto turned = [](uint32_t v) __attribute__((always_inline)) { return v << 16 | v >> 16; };
    return up ? u32x4{turned(w[3]), turned(w[2]), turned(w[1]), turned(w[0])} : w;
  }
  // Those counts, 0 for what is no number.
  __device__ __forceinline__ void count(uint32_t w, uint32_t order, uint32_t* c0,
                                        uint32_t* c1) const {
    uint32_t a = w & 0xffffu, b = w >> 16;
#pragma unroll 1
    for (uint32_t j = 0; j < nheavy; ++j) {
      if (heavy[2 * j] == order) a += heavy[2 * j + 1];
      if (heavy[2 * j] == order + 1) b += heavy[2 * j + 1];
    }
    *c0 = order >= first && order <= last ? a : 0;
    *c1 = order + 1 >= first && order + 1 <= last ? b : 0;
  }
};

// A value of a row, and how much comes before it.
struct Place {
  uint32_t order;
  uint32_t count;   // of its tokens
  double before;    // sum of weights
  uint32_t rank;    // tokens
  double weight;    // of one
};

// The first value that comes and, with its own tokens, reaches what is asked for (the last
// up to `limit` if none does): by tokens, by the sum of weights, or by more than the sum.
// One wavefront. first, last: blocks, of which limit's is the last or comes after it.
enum class By { Tokens, Sum, More };
template <typename T>
__device__ __forceinline__ Place find(const Row& row, By by, uint32_t rank, double sum,
                                      uint32_t limit, int first, int last, int lane) {
  auto reached = [&](uint32_t r, double s) __attribute__((always_inline)) {
    return by == By::Tokens ? r >= rank : by == By::Sum ? s >= sum : s > sum;
  };
  last = min(last, (int)(limit >> 7));
  int blk = last;
  for (int b0 = first; b0 < last; b0 += 64) {
    const int b = min(b0 + lane, kBlocks - 1);
    const bool hit = b0 + lane < last && row.tokens[b] > 0 && reached(row.counts[b], row.sums[b]);
    const uint64_t hits = __ballot(hit);
    if (hits != 0) {
      blk = b0 + __builtin_ctzll(hits);
      break;
    }
  }
  uint32_t c0, c1;
  const uint32_t o0 = blk * 128 + 2 * lane;
  row.count(row.word(blk * 64 + lane), o0, &c0, &c1);
  if (o0 > limit) c0 = 0;
  if (o0 + 1 > limit) c1 = 0;
  const double w0 = row.weight<T>(o0), w1 = row.weight<T>(o0 + 1);
  const uint32_t r0 = (blk == 0 ? 0 : row.counts[blk - 1]) + scan_before<uint32_t>(c0 + c1, lane);
  const double s0 =
      (blk == 0 ? 0.0 : row.sums[blk - 1]) +
      scan_before<double>((c0 ? c0 * w0 : 0.0) + (c1 ? c1 * w1 : 0.0), lane);
  const uint32_t r1 = r0 + c0;
  const double s1 = s0 + (c0 ? c0 * w0 : 0.0);
  const bool hit0 = c0 && reached(r1, s1), hit1 = c1 && reached(r1 + c1, s1 + c1 * w1);
  const uint64_t hits = __ballot(hit0 || hit1), there = __ballot(c0 || c1);
  const int at = hits != 0 ? __builtin_ctzll(hits) : there != 0 ? 63 - __builtin_clzll(there) : 0;
  const bool second = hits != 0 ? !hit0 : c1 != 0;  // in the lane that counts
  Place p;
  p.order = lane_of(second ? o0 + 1 : o0, at);
  p.count = lane_of(second ? c1 : c0, at);
  p.before = lane_of(second ? s1 : s0, at);
  p.rank = lane_of(second ? r1 : r0, at);
  p.weight = lane_of(second ? w1 : w0, at);
  return p;
}

// The row's elements that lie in whole aligned 16 bytes, [head, head + 8 vectors), and the rest.
struct Span {
  int head, vectors;
  __device__ __forceinline__ Span(const void* row, int V) {
    const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15u) / 2;
    head = min(off == 0 ? 0 : 8 - off, V);
    vectors = (V - head) / 8;
  }
};

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t hist[32768];
  __shared__ double sums[kBlocks], powers[64];
  __shared__ uint32_t counts[kBlocks], ntok[kBlocks];
  __shared__ uint32_t heavy[2 * kHeavyMost], nheavy, least;
  __shared__ int most;
  __shared__ uint32_t drawn, skip, many, seen[kTurnsMost * kSampleWaves];
  constexpr uint32_t kFirst = Order<T>::kFirst, kLast = Order<T>::kLast;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = blockIdx.x, V = a.V;
  const uint16_t* row = static_cast<const uint16_t*>(a.logits) + r * a.st;
  const Span span(row, V);
  // the i-th vector
  const char* const body_at = reinterpret_cast<const char*>(row + span.head);
  auto body = [&](int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const u32x4*>(body_at + (uint32_t)i * 16u);
  };
  const int rest = V - 8 * span.vectors;  // elements outside of the vectors
  // the i-th of those
  auto loose = [&](int i) __attribute__((always_inline)) {
    return i < span.head ? i : i + 8 * span.vectors;
  };

  double t = a.temperatures != nullptr ? (double)a.temperatures[r] : a.temperature;
  const double top_p = a.top_ps != nullptr ? (double)a.top_ps[r] : a.top_p;
  const double min_p = a.min_ps != nullptr ? (double)a.min_ps[r] : a.min_p;
  int top_k = a.top_ks != nullptr ? a.top_ks[r] : a.top_k;
  if (!(t > 0.0)) {  // the first
    t = 1.0;
    top_k = 1;
  }

#pragma unroll
  for (int i = 0; i < 8; ++i)
    *reinterpret_cast<u32x4*>(hist + 4 * (i * kSampleThreads + tid)) = u32x4{0u, 0u, 0u, 0u};
  if (tid < 64) powers[tid] = exp2(tid / 64.0);
  if (tid == 0) {
    nheavy = 0;
    least = 0xffffu;
    most = -0x8000;
  }
  __syncthreads();

  // Count, by bits. No count passes 65535: a stretch ends before one can, and those of
  // kHeavy and more then move to the list. The highest number is the highest of the bits as
  // signed 16-bit numbers, or the lowest without a sign if all are negative.
  u16x2 lowest = {0xffff, 0xffff};
  s16x2 highest = {-0x8000, -0x8000};
  auto add = [&](uint32_t at, uint32_t odd) __attribute__((always_inline)) {
    atomicAdd(reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(hist) + at), odd * 0xffffu + 1u);
  };
  auto add_pair = [&](uint32_t x) __attribute__((always_inline)) {
    add((x << 1) & 0x1fffcu, x & 1u);
    add((x >> 15) & 0x1fffcu, (x >> 16) & 1u);
    lowest = __builtin_elementwise_min(lowest, __builtin_bit_cast(u16x2, x));
    highest = __builtin_elementwise_max(highest, __builtin_bit_cast(s16x2, x));
  };
  auto add_vector = [&](const u32x4& v) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) add_pair(v[e]);
  };
  auto look = [&]() {
    __syncthreads();
    uint32_t any[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {  // all on their way before the first is looked at
      const u32x4 w = *reinterpret_cast<const u32x4*>(hist + 4 * (k * kSampleThreads + tid));
      any[k] = (w[0] | w[1] | w[2] | w[3]) & kHeavyBits;
    }
    uint32_t where = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) where |= (any[k] != 0 ? 1u : 0u) << k;
    while (where != 0) {
      const int at = 4 * (__builtin_ctz(where) * kSampleThreads + tid);
      where &= where - 1;
      for (int i = 0; i < 8; ++i) {  // the counts of 8 values
        const uint32_t word = hist[at + i / 2], n = i % 2 ? word >> 16 : word & 0xffffu;
        if (n < kHeavy) continue;
        const uint32_t bits = 2 * at + i, j = atomicAdd(&nheavy, 1u);
        heavy[2 * j] = bits < 0x8000u ? kZero - bits : bits;
        heavy[2 * j + 1] = n;
        hist[at + i / 2] = i % 2 ? word & 0xffffu : word & 0xffff0000u;
      }
    }
    __syncthreads();
  };
  if (tid < rest) {
    const uint32_t x = row[loose(tid)];
    add((x << 1) & 0x1fffcu, x & 1u);
    const uint32_t both = x | x << 16;
    lowest = __builtin_elementwise_min(lowest, __builtin_bit_cast(u16x2, both));
    highest = __builtin_elementwise_max(highest, __builtin_bit_cast(s16x2, both));
  }
  // the row's first vectors (a turn that the row does not reach: the first)
  const int turns = (span.vectors + kSampleThreads - 1) / kSampleThreads;
  u32x4 held[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const int i = j * kSampleThreads + tid;
    held[j] = span.vectors > 0 ? body(i < span.vectors ? i : 0) : u32x4{};
  }
  // f(turn, number, vector) for the turns from `from` up to `end` (numbers past the last: the
  // last vector), before(turn) ahead of each group of them; the next group is on its way.
  auto stream = [&](int from, int end, auto before, auto f) __attribute__((always_inline)) {
    if (from >= end) return;
    u32x4 next[kGroup];
    auto load = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < kGroup; ++j)
        next[j] = body(min((j0 + j) * kSampleThreads + tid, span.vectors - 1));
    };
    load(from);
#pragma unroll 1
    for (int j0 = from; j0 < end; j0 += kGroup) {
      u32x4 now[kGroup];
#pragma unroll
      for (int j = 0; j < kGroup; ++j) now[j] = next[j];
      if (j0 + kGroup < end) load(j0 + kGroup);
      before(j0);
#pragma unroll
      for (int j = 0; j < kGroup; ++j)
        if (j0 + j < end) f(j0 + j, (j0 + j) * kSampleThreads + tid, now[j]);
    }
  };
  auto count = [&](int, int i, const u32x4& v) __attribute__((always_inline)) {
    if (i < span.vectors) add_vector(v);
  };
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    if (j == kStretch && turns > j) look();
    count(j, j * kSampleThreads + tid, held[j]);
  }
  stream(kHeld, turns,
         [&](int j) __attribute__((always_inline)) {
           if ((j - kHeld) % (2 * kGroup) == 0) look();
         },
         count);
  {
    uint32_t lo = min((uint32_t)lowest[0], (uint32_t)lowest[1]);
    int hi = max((int)highest[0], (int)highest[1]);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      lo = min(lo, (uint32_t)__shfl_xor((int)lo, d));
      hi = max(hi, __shfl_xor(hi, d));
    }
    if (lane == 0) {
      atomicMin(&least, lo);
      atomicMax(&most, hi);
    }
  }
  __syncthreads();
  // -0 counts as 0: its count, to that of 0, or to the list where that could pass 65535
  if (tid == 0) {
    for (uint32_t j = 0; j < nheavy; ++j)
      if (heavy[2 * j] == kZero + 1) heavy[2 * j] = kZero;
    const uint32_t w = hist[0x4000], z = hist[0], n = w & 0xffffu;
    if (n > 0) {
      hist[0x4000] = w & 0xffff0000u;
      if (n + (z & 0xffffu) <= 0xffffu) {
        hist[0] = z + n;
      } else {
        heavy[2 * nheavy] = kZero;
        heavy[2 * nheavy + 1] = n;
        ++nheavy;
      }
    }
  }
  __syncthreads();

  Row x = {hist, sums, counts, ntok, heavy, 0, kFirst, kLast, powers, 0.0, 0.0};
  x.nheavy = __builtin_amdgcn_readfirstlane(nheavy);
  uint32_t best = most >= 0 ? kZero - most : least;
  if (best < kFirst) {  // a NaN: the first number there is
    uint32_t first = 0xffffu;
    for (int i = lane; i < 32768; i += 64) {
      uint32_t c0, c1;
      x.count(x.word(i), 2 * i, &c0, &c1);
      first = min(first, c0 ? 2u * i : c1 ? 2u * i + 1 : 0xffffu);
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) first = min(first, (uint32_t)__shfl_xor((int)first, d));
    best = first;
  }
  if (best == kZero + 1) best = kZero;
  best = __builtin_amdgcn_readfirstlane(best);
  if (best > kLast) {  // no number above -infinity
    if (tid == 0) {
      a.tokens[r] = -1;
      if (a.logprobs != nullptr) a.logprobs[r] = -INFINITY;
    }
    return;
  }

  x.top = value_of<T>(best);
  x.per_t = fmin(1.0 / t, 1e300);  // finite: what is 0 stays 0
  const int first = best >> 7;
  // Sums of blocks, 4 at a time in turns of the wavefronts: 16 lanes a block, 8 values a lane,
  // one exponential for all 8, since a block's values are a step apart and a weight's quotient
  // to the next is the block's. Lane j of a wavefront has that of its j-th block. (No other
  // number shares infinity's block.)
  constexpr int kTurns = kBlocks / 4 / kSampleWaves;
  auto block_of = [&](int turn, int j) __attribute__((always_inline)) {
    return 4 * (turn * kSampleWaves + wave) + j;
  };
  const uint32_t begin = block_of(lane / 4 % kTurns, lane % 4) * 128;
  double step = exp((value_of<T>(begin + 1) - value_of<T>(begin)) * x.per_t);
  if (!(step <= 1.0)) step = 0.0;  // where no numbers are
  u32x4 words = x.words(block_of(0, 0) * 16 + lane);
#pragma unroll 1
  for (int turn = 0; turn < kTurns; ++turn) {
    const u32x4 w = words;
    const int b = block_of(turn, lane / 16);
    words = x.words(block_of(min(turn + 1, kTurns - 1), 0) * 16 + lane);
    uint32_t n = 0;
    double s = 0.0;
    if (x.nheavy > 0 || __ballot((w[0] | w[1] | w[2] | w[3]) != 0) != 0) {
      const double q = __shfl(step, 4 * turn + lane / 16);
      const uint32_t o = b * 128 + 8 * (lane % 16);
      double weight = x.weight<T>(max(o, best));  // 1 for best itself, exactly
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t c0, c1;
        x.count(w[i], o + 2 * i, &c0, &c1);
        n += c0 + c1;
        s = fma((double)c0, weight, s);
        if (o + 2 * i >= best) weight *= q;
        s = fma((double)c1, weight, s);
        if (o + 2 * i + 1 >= best) weight *= q;
      }
      n = sum_of_row(n);
      s = sum_of_row(s);
    }
    if (lane % 16 == 0) {
      ntok[b] = n;
      sums[b] = s;
    }
  }
  __syncthreads();
  if (wave == 0) {
    // running sums over the blocks, 8 a lane
    constexpr int PER = kBlocks / 64;
    uint32_t n[PER], all = 0, bits = 0;
    double s[PER], total = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      n[i] = ntok[PER * lane + i];
      s[i] = sums[PER * lane + i];
      bits |= (n[i] > 0 ? 1u : 0u) << i;
      all = n[i] += all;
      total = s[i] += total;
    }
    const uint32_t before_n = scan_before<uint32_t>(all, lane, &all);
    const double before_s = scan_before<double>(total, lane, &total);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      counts[PER * lane + i] = n[i] + before_n;
      sums[PER * lane + i] = s[i] + before_s;
    }
    const int end = 63 - __builtin_clzll(__ballot(bits != 0));  // the last lane with tokens
    const int final = PER * end + 31 - __builtin_clz(lane_of(bits, end));  // and block
    // The kept tokens end in the value `last`, with `ends` of its own; their sum is total.
    // One cut after the other, then the draw (a loop, for find to be there once).
    uint32_t last = kLast, ends = 0xffffffffu;
    Place p = {};
    double want = 0.0;
    enum { kTopK, kTopP, kMinP, kDraw, kStages };
#pragma unroll 1
    for (int stage = kTopK; stage < kStages; ++stage) {
      By by = By::Tokens;
      uint32_t rank = all;
      if (stage == kTopK) {
        if (top_k <= 0 || (uint32_t)top_k >= all) continue;
        rank = top_k;
      } else if (stage == kTopP) {
        if (!(top_p < 1.0)) continue;
        by = By::Sum;
        want = top_p * total;
      } else if (stage == kMinP) {
        if (!(min_p > 0.0)) continue;
        // the last order whose weight is at least min_p (no less than the first)
        uint32_t lo = best;
        for (uint32_t step = 1024; step > 0; step = step == 1024 ? 16 : step == 16 ? 1 : 0) {
          const uint32_t o = lo + step * (lane + 1);
          const bool in = o <= kLast && x.weight<T>(min(o, kLast)) >= min_p;
          lo += step * (uint32_t)__popcll(__ballot(in));
        }
        if (lo >= last) continue;
        uint32_t c0, c1;
        const uint32_t o0 = (lo & ~127u) + 2 * lane;
        x.count(x.word(o0 / 2), o0, &c0, &c1);
        rank = sum_of((o0 <= lo ? c0 : 0) + (o0 + 1 <= lo ? c1 : 0));
        if (lo >= 128) rank += counts[(lo >> 7) - 1];
      } else if (stage == kDraw) {
        by = By::More;
        want = (double)a.uniform[r] * total;
      }
      p = find<T>(x, by, rank, want, last, first, final, lane);
      uint32_t m = rank - p.rank;
      if (stage == kTopP) {
        const uint32_t most = p.order == last ? min(ends, p.count) : p.count;
        const double need = ceil((want - p.before) / p.weight);
        m = need < 1.0 ? 1u : need < (double)most ? (uint32_t)need : most;
        // the quotient is rounded: the least m by the sums themselves
        if (m > 1 && p.before + (m - 1) * p.weight >= want) --m;
        if (m < most && p.before + m * p.weight < want) ++m;
      }
      if (stage != kDraw) {
        last = p.order;
        ends = m;
        total = p.before + m * p.weight;
      }
    }
    const uint32_t mine = p.order == last ? min(ends, p.count) : p.count;
    const double j = floor((want - p.before) / p.weight);
    uint32_t at = j < 1.0 ? 0u : j < (double)mine ? (uint32_t)j : mine - 1;
    if (at > 0 && p.before + at * p.weight > want) --at;
    if (at + 1 < mine && p.before + (at + 1) * p.weight <= want) ++at;
    if (lane == 0) {
      drawn = p.order;
      skip = at;
      many = p.count;
      if (a.logprobs != nullptr) a.logprobs[r] = (float)log(p.weight / total);
    }
  }
  __syncthreads();

  // The skip-th token of the drawn value, of either zero for 0.
  const uint32_t pattern = drawn == kZero ? 0u : bits_of(drawn);
  const uint32_t keep = drawn == kZero ? 0x7fffu : 0xffffu;
  const uint32_t pattern2 = pattern * 0x10001u, keep2 = keep * 0x10001u;
  auto is = [&](uint32_t bits) __attribute__((always_inline)) { return (bits & keep) == pattern; };
  // bits 15 and 31: whether the halves are the pattern
  auto equal = [&](uint32_t w) __attribute__((always_inline)) {
    const uint32_t z = (w & keep2) ^ pattern2;
    return ~(((z & 0x7fff7fffu) + 0x7fff7fffu) | z | 0x7fff7fffu);
  };
  // which elements of a vector, a bit each
  auto matches = [&](const u32x4& v) __attribute__((always_inline)) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t e = equal(v[j]);
      m |= ((e >> 15) & 1u) << (2 * j) | (e >> 31) << (2 * j + 1);
    }
    return m;
  };
  // The one there is, or, in their order, the loose ones before the vectors, the vectors by
  // turns and wavefronts, the loose ones behind.
  const bool one = many == 1;
  if (one && tid < rest && is(row[loose(tid)])) a.tokens[r] = loose(tid);
  auto seek = [&](int j, int i, const u32x4& v) __attribute__((always_inline)) {
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) n += __popc(equal(v[e]));
    if (i >= span.vectors) n = 0;
    if (one) {
      if (n) a.tokens[r] = span.head + 8 * i + __builtin_ctz(matches(v));
    } else {
      n = sum_of(n);
      if (lane == 0) seen[j * kSampleWaves + wave] = n;
    }
  };
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
    if (j < turns) seek(j, j * kSampleThreads + tid, held[j]);
  stream(kHeld, turns, [](int) {}, seek);
  if (one) return;
  __syncthreads();
  if (wave != 0) return;
  const bool mine = lane < rest && is(row[loose(lane)]);
  const uint64_t heads = __ballot(mine && lane < span.head);
  const uint64_t tails = __ballot(mine && lane >= span.head);
  const uint64_t below = (1ull << lane) - 1;
  uint32_t left = skip;
  if (left < (uint32_t)__popcll(heads)) {
    if (((heads >> lane) & 1) && (uint32_t)__popcll(heads & below) == left)
      a.tokens[r] = loose(lane);
    return;
  }
  left -= __popcll(heads);
  for (int e0 = 0; e0 < turns * kSampleWaves; e0 += 64) {
    const uint32_t n = e0 + lane < turns * kSampleWaves ? seen[e0 + lane] : 0;
    uint32_t all;
    const uint32_t before = scan_before<uint32_t>(n, lane, &all);
    if (left >= all) {
      left -= all;
      continue;
    }
    const int at = __builtin_ctzll(__ballot(left >= before && left < before + n));
    left -= lane_of(before, at);
    const int i = (e0 + at) * 64 + lane;  // the 64 vectors of that turn and wavefront
    const uint32_t m = i < span.vectors ? matches(body(i)) : 0;
    const uint32_t prior = scan_before<uint32_t>(__popc(m), lane);
    if (left >= prior && left < prior + __popc(m)) {
      uint32_t bits = m;
      for (uint32_t k = left - prior; k > 0; --k) bits &= bits - 1;
      a.tokens[r] = span.head + 8 * i + __builtin_ctz(bits);
    }
    return;
  }
  if (((tails >> lane) & 1) && left == (uint32_t)__popcll(tails & below)) a.tokens[r] = loose(lane);
}

// The walk over a tree: from node 0 to its first child whose token was picked at it, and on.
// A wavefront a sequence, 4 nodes a lane; children come after their parents, so a step looks
// at the nodes behind the last. A parent that does not come before its node is none. Bound by
// the launch, the loads and a step's 4 ballots: 16 nodes 2.2 us, 256 sequences of 256 4.0.
__global__ __launch_bounds__(64) void tree_accept_kernel(AcceptArgs a) {
  constexpr int PER = kTreeNodes / 64;
  __shared__ int64_t picked[kTreeNodes];
  const int lane = threadIdx.x, b = blockIdx.x, N = a.N;
  int count = a.counts != nullptr ? a.counts[b] : N;
  count = min(max(count, 0), N);
  int parent[PER];
  int64_t token[PER];
  int32_t path[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = 64 * j + lane;
    const int64_t at = (int64_t)b * N + i;
    parent[j] = -1;
    token[j] = 0;
    path[j] = -1;
    if (i < count) {
      parent[j] = a.parents[at];
      if (parent[j] >= i) parent[j] = -1;
      token[j] = a.tokens[at];
      picked[i] = a.picked[at];
    }
  }
  __syncthreads();
  int cur = count > 0 ? 0 : -1, m = 0;
  int64_t next = -1;
  while (cur >= 0) {  // cur rises: at most N turns
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (64 * j + lane == m) path[j] = cur;
    ++m;
    next = picked[cur];
    int child = -1;
#pragma unroll
    for (int j = PER - 1; j >= 0; --j) {
      const uint64_t hits = __ballot(parent[j] == cur && token[j] == next);
      if (hits != 0) child = 64 * j + __builtin_ctzll(hits);
    }
    cur = child;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (64 * j + lane < N) a.path[(int64_t)b * N + 64 * j + lane] = path[j];
  if (lane == 0) {
    a.accepted[b] = m;
    a.next[b] = next;
  }
}

}  // namespace

template <typename T>
hipError_t launch_sample_typed(const SampleArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(sample_kernel<T>, dim3(a.R), dim3(kSampleThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_sample(const SampleArgs& a, Elem dtype, hipStream_t stream) {
  return dtype == Elem::BF16 ? launch_sample_typed<__bf16>(a, stream)
                             : launch_sample_typed<_Float16>(a, stream);
}

hipError_t launch_tree_accept(const AcceptArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(tree_accept_kernel, dim3(a.B), dim3(64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace ttcd
