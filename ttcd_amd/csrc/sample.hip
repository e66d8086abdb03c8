// sample.hip - a token from every row of logits, and the walk over a tree of drafted
// tokens that keeps those which agree, on gfx950.
//
// Sampling. Tokens rank by logit, of equal ones the lower index first, and weigh
// w = exp((x - max) / temperature). Kept are the first top_k, of those the shortest run
// with at least top_p of their sum, of those the ones with w >= min_p; the token is the
// first whose running sum exceeds uniform times the sum of all kept.
//
// A 16-bit logit has one of 65536 values, and everything above depends on a row only
// through how often each value comes: no sort, and no exponential of a token, but one of
// every value that occurs, in 64 bits, as are all sums. Counting is exact in any order, so
// a row's token does not depend on how its sums are laid out. A workgroup takes a row: it
// counts the values in LDS (16 bits a count, 128 KiB), finds the last kept value and the
// drawn one with how many of its tokens come before the drawn token, and reads the row
// again for the token itself.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "internal.h"

namespace ttcd {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kBlocks = 512;     // of 128 values, 64 words of 2 counts
constexpr int kHeavy = 8192;     // a count above this moves to the list
constexpr int kHeavyMost = kSampleVocab / kHeavy;

// The order of a 16-bit value, the largest (infinity) 0, those up to kLast numbers above
// -infinity, then -infinity and NaN.
template <typename T>
struct Order;
template <>
struct Order<__bf16> {
  static constexpr uint32_t kInf = 0x7f80;
};
template <>
struct Order<_Float16> {
  static constexpr uint32_t kInf = 0x7c00;
};
template <typename T>
constexpr uint32_t first_of() { return 0x7fffu - Order<T>::kInf; }  // before the shift
template <typename T>
constexpr uint32_t last_of() { return 0x7fffu + Order<T>::kInf - first_of<T>(); }
template <typename T>
constexpr uint32_t zero_of() { return 0x7fffu - first_of<T>(); }  // of +0; -0 is the next

// Both halves of a word. A positive value's bits turn around below 0x7fff, a negative one's
// are in order as they are.
template <typename T>
__device__ __forceinline__ uint32_t order_pair(uint32_t x) {
  const uint32_t sign = (x >> 15) & 0x00010001u;
  const uint32_t o = x ^ ((sign << 15) - sign) ^ 0x7fff7fffu;
  constexpr uint32_t f = first_of<T>();
  // halves apart: the lower one's borrow stays its own
  return ((o - (f << 16)) & 0xffff0000u) | ((o - f) & 0xffffu);
}

// The value of an order.
template <typename T>
__device__ __forceinline__ double value_of(uint32_t order) {
  const uint32_t o = order + first_of<T>();
  const uint16_t bits = (uint16_t)(o < 0x8000u ? o ^ 0x7fffu : o);
  return (double)static_cast<float>(__builtin_bit_cast(T, bits));
}

// Sums over the lanes before this one (all: over all of them).
template <typename V>
__device__ __forceinline__ V scan_before(V x, int lane, V* all = nullptr) {
  V sum = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const V o = __shfl_up(sum, d);
    if (lane >= d) sum += o;
  }
  if (all != nullptr) *all = __shfl(sum, 63);
  const V before = __shfl_up(sum, 1);
  return lane == 0 ? V(0) : before;
}

template <typename T>
struct Row {
  uint32_t* hist;       // [32768] counts of orders 2 i and 2 i + 1
  double* sums;         // [kBlocks] of weights before a block of 128 orders, ..
  double* block;        // .. and of its own
  uint32_t* counts;     // the same of tokens
  uint32_t* tokens;
  uint32_t* heavy;      // [2 kHeavyMost] order, count
  uint32_t nheavy;
  double top, t;        // the highest logit, and the temperature

  __device__ __forceinline__ double weight(uint32_t order) const {
    const double x = value_of<T>(order);
    return x == top ? 1.0 : exp((x - top) / t);
  }
  // The counts of the orders 2 i and 2 i + 1, 0 for what is no number.
  __device__ __forceinline__ void count(int i, uint32_t* c0, uint32_t* c1) const {
    const uint32_t w = hist[i];
    uint32_t a = w & 0xffffu, b = w >> 16;
    for (uint32_t j = 0; j < nheavy; ++j) {
      if (heavy[2 * j] == 2u * i) a += heavy[2 * j + 1];
      if (heavy[2 * j] == 2u * i + 1) b += heavy[2 * j + 1];
    }
    if (2 * i == (int)zero_of<T>()) {  // -0 is 0
      a += b;
      b = 0;
    }
    *c0 = 2u * i <= last_of<T>() ? a : 0;
    *c1 = 2u * i + 1 <= last_of<T>() ? b : 0;
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

// The first value that comes and, with its own tokens, reaches what is asked for, of those
// up to `limit`, which comes itself (limit if none does): by tokens, by the sum of weights,
// or by more than the sum. One wavefront.
enum class By { Tokens, Sum, More };
template <typename T>
__device__ __forceinline__ Place find(const Row<T>& row, By by, uint32_t rank, double sum,
                                      uint32_t limit, int lane) {
  auto reached = [&](uint32_t r, double s) __attribute__((always_inline)) {
    return by == By::Tokens ? r >= rank : by == By::Sum ? s >= sum : s > sum;
  };
  int blk = limit >> 7;
  for (int b0 = 0; b0 < (int)(limit >> 7); b0 += 64) {
    const int b = b0 + lane;
    const uint32_t n = row.tokens[b];
    const bool hit = b < (int)(limit >> 7) && n > 0 &&
                     reached(row.counts[b] + n, row.sums[b] + row.block[b]);
    const uint64_t hits = __ballot(hit);
    if (hits != 0) {
      blk = b0 + __builtin_ctzll(hits);
      break;
    }
  }
  uint32_t c0, c1;
  row.count(blk * 64 + lane, &c0, &c1);
  const uint32_t o0 = blk * 128 + 2 * lane;
  if (o0 > limit) c0 = 0;
  if (o0 + 1 > limit) c1 = 0;
  const double w0 = c0 ? row.weight(o0) : 0.0, w1 = c1 ? row.weight(o0 + 1) : 0.0;
  const uint32_t r0 = row.counts[blk] + scan_before<uint32_t>(c0 + c1, lane);
  const double s0 = row.sums[blk] + scan_before<double>(c0 * w0 + c1 * w1, lane);
  const uint32_t r1 = r0 + c0;
  const double s1 = s0 + c0 * w0;
  const bool hit0 = c0 && reached(r1, s1), hit1 = c1 && reached(r1 + c1, s1 + c1 * w1);
  const uint64_t hits = __ballot(hit0 || hit1), there = __ballot(c0 || c1);
  const int at = hits != 0 ? __builtin_ctzll(hits) : 63 - __builtin_clzll(there);
  const bool second = hits != 0 ? !hit0 : c1 != 0;  // in the lane that counts
  Place p;
  p.order = __shfl(second ? o0 + 1 : o0, at);
  p.count = __shfl(second ? c1 : c0, at);
  p.before = __shfl(second ? s1 : s0, at);
  p.rank = __shfl(second ? r1 : r0, at);
  p.weight = __shfl(second ? w1 : w0, at);
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
  __shared__ double sums[kBlocks], block[kBlocks];
  __shared__ uint32_t counts[kBlocks], ntok[kBlocks];
  __shared__ uint32_t heavy[2 * kHeavyMost], nheavy, best;
  __shared__ uint32_t drawn, skip, many, seen[kSampleWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = blockIdx.x, V = a.V;
  const uint16_t* row = static_cast<const uint16_t*>(a.logits) + r * a.st;
  const Span span(row, V);
  const u32x4* body = reinterpret_cast<const u32x4*>(row + span.head);
  const int rest = V - 8 * span.vectors;  // elements outside of the vectors
  // the i-th of those
  auto loose = [&](int i) __attribute__((always_inline)) {
    return i < span.head ? i : i + 8 * span.vectors;
  };

#pragma unroll
  for (int i = 0; i < 8; ++i)
    *reinterpret_cast<u32x4*>(hist + 4 * (i * kSampleThreads + tid)) = u32x4{0u, 0u, 0u, 0u};
  if (tid == 0) {
    nheavy = 0;
    best = 0xffffu;
  }
  __syncthreads();

  // Count. No count passes 65535: a stretch ends before one can, and those above kHeavy
  // then move to the list.
  uint32_t least = 0xffffu;
  auto add = [&](uint32_t o) __attribute__((always_inline)) {
    atomicAdd(hist + (o >> 1), 1u + (o & 1u) * 0xffffu);
    least = min(least, o);
  };
  auto add_pair = [&](uint32_t x) __attribute__((always_inline)) {
    const uint32_t o = order_pair<T>(x);
    add(o & 0xffffu);
    add(o >> 16);
  };
  if (tid < rest) add(order_pair<T>(row[loose(tid)]) & 0xffffu);
  int done = rest, from = 0;  // elements since the last look, and vectors
  while (from < span.vectors) {
    const int to = min(span.vectors, from + (65535 - done) / 8);
    for (int i = from + tid; i < to; i += kSampleThreads) {
      const u32x4 x = body[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) add_pair(x[j]);
    }
    from = to;
    done = kHeavy;
    if (from < span.vectors) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = 4 * (i * kSampleThreads + tid);
        const u32x4 w = *reinterpret_cast<const u32x4*>(hist + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t lo = w[e] & 0xffffu, hi = w[e] >> 16;
          if (lo <= kHeavy && hi <= kHeavy) continue;
          if (lo > kHeavy) {
            const uint32_t j = atomicAdd(&nheavy, 1u);
            heavy[2 * j] = 2 * (at + e);
            heavy[2 * j + 1] = lo;
          }
          if (hi > kHeavy) {
            const uint32_t j = atomicAdd(&nheavy, 1u);
            heavy[2 * j] = 2 * (at + e) + 1;
            heavy[2 * j + 1] = hi;
          }
          hist[at + e] = (lo > kHeavy ? 0u : lo) | (hi > kHeavy ? 0u : hi << 16);
        }
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) least = min(least, (uint32_t)__shfl_xor((int)least, d));
  if (lane == 0) atomicMin(&best, least);
  __syncthreads();
  if (best > last_of<T>()) {  // no number above -infinity
    if (tid == 0) {
      a.tokens[r] = -1;
      if (a.logprobs != nullptr) a.logprobs[r] = -INFINITY;
    }
    return;
  }

  double t = a.temperatures != nullptr ? (double)a.temperatures[r] : a.temperature;
  const double top_p = a.top_ps != nullptr ? (double)a.top_ps[r] : a.top_p;
  const double min_p = a.min_ps != nullptr ? (double)a.min_ps[r] : a.min_p;
  int top_k = a.top_ks != nullptr ? a.top_ks[r] : a.top_k;
  if (!(t > 0.0)) {  // the first
    t = 1.0;
    top_k = 1;
  }
  Row<T> x = {hist, sums, block, counts, ntok, heavy, nheavy, value_of<T>(best), t};
  for (int b = wave; b < kBlocks; b += kSampleWaves) {
    uint32_t c0, c1;
    x.count(b * 64 + lane, &c0, &c1);
    uint32_t n = 0;
    double s = 0.0;
    if (__any(c0 + c1 > 0)) {
      n = c0 + c1;
      if (c0) s = c0 * x.weight(b * 128 + 2 * lane);
      if (c1) s += c1 * x.weight(b * 128 + 2 * lane + 1);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        n += __shfl_xor(n, d);
        s += __shfl_xor(s, d);
      }
    }
    if (lane == 0) {
      ntok[b] = n;
      block[b] = s;
    }
  }
  __syncthreads();
  if (wave == 0) {
    uint32_t all = 0;
    double total = 0.0;
    for (int b0 = 0; b0 < kBlocks; b0 += 64) {
      uint32_t n;
      double s;
      const uint32_t nb = all + scan_before<uint32_t>(ntok[b0 + lane], lane, &n);
      const double sb = total + scan_before<double>(block[b0 + lane], lane, &s);
      counts[b0 + lane] = nb;
      sums[b0 + lane] = sb;
      all += n;
      total += s;
    }
    // The kept tokens end in the value `last`, with `ends` of its own; their sum is total.
    // One cut after the other, then the draw (a loop, for find to be there once).
    uint32_t last = last_of<T>(), ends = 0;
    Place p = {};
    double want = 0.0;
    enum { kAll, kTopK, kTopP, kMinP, kDraw, kStages };
#pragma unroll 1
    for (int stage = kAll; stage < kStages; ++stage) {
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
          lo += step * (uint32_t)__popcll(__ballot(o <= last_of<T>() && x.weight(o) >= min_p));
        }
        if (lo >= last) continue;
        uint32_t c0, c1;
        x.count((lo >> 7) * 64 + lane, &c0, &c1);
        const uint32_t o0 = (lo & ~127u) + 2 * lane;
        rank = (o0 <= lo ? c0 : 0) + (o0 + 1 <= lo ? c1 : 0);
#pragma unroll
        for (int d = 1; d < 64; d *= 2) rank += __shfl_xor(rank, d);
        rank += counts[lo >> 7];
      } else if (stage == kDraw) {
        by = By::More;
        want = (double)a.uniform[r] * total;
      }
      p = find<T>(x, by, rank, want, last, lane);
      uint32_t m = rank - p.rank;
      if (stage == kTopP) {
        const uint32_t most = p.order == last ? ends : p.count;
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
    const uint32_t mine = p.order == last ? ends : p.count;
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

  // The skip-th token of the drawn value. -0 counts as 0.
  const uint32_t want = drawn;
  uint32_t left = skip;
  const bool zero = want == zero_of<T>();
  auto is = [&](uint32_t o) __attribute__((always_inline)) {
    return o == want || (zero && o == want + 1);
  };
  // bit i: element i of a vector
  auto matches = [&](const u32x4& v) __attribute__((always_inline)) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t o = order_pair<T>(v[j]);
      m |= (is(o & 0xffffu) ? 1u : 0u) << (2 * j) | (is(o >> 16) ? 2u : 0u) << (2 * j);
    }
    return m;
  };
  if (many == 1) {
    if (tid < rest && is(order_pair<T>(row[loose(tid)]) & 0xffffu)) a.tokens[r] = loose(tid);
    for (int i = tid; i < span.vectors; i += kSampleThreads) {
      const uint32_t m = matches(body[i]);
      if (m) a.tokens[r] = span.head + 8 * i + __builtin_ctz(m);
    }
    return;
  }
  // In their order: the loose ones before the vectors, a run of vectors a wavefront, the
  // loose ones behind. The wavefront whose run it is in reads it once more.
  const int run = (span.vectors + kSampleWaves - 1) / kSampleWaves;
  const int lo = min(wave * run, span.vectors), hi = min(lo + run, span.vectors);
  uint32_t n = 0;
  for (int i = lo + lane; i < hi; i += 64) n += __popc(matches(body[i]));
#pragma unroll
  for (int d = 1; d < 64; d *= 2) n += __shfl_xor(n, d);
  if (lane == 0) seen[wave] = n;
  __syncthreads();
  const bool mine = lane < rest && is(order_pair<T>(row[loose(lane)]) & 0xffffu);
  const uint64_t heads = __ballot(mine && lane < span.head), tails = __ballot(mine && lane >= span.head);
  const uint64_t below = (1ull << lane) - 1;
  uint32_t before = __popcll(heads);
  if (wave == 0 && ((heads >> lane) & 1) && (uint32_t)__popcll(heads & below) == left)
    a.tokens[r] = loose(lane);
  for (int w = 0; w < wave; ++w) before += seen[w];
  if (left >= before && left < before + n) {
    left -= before;
    for (int i0 = lo; i0 < hi; i0 += 64) {
      const uint32_t m = i0 + lane < hi ? matches(body[i0 + lane]) : 0;
      uint32_t all;
      const uint32_t prior = scan_before<uint32_t>(__popc(m), lane, &all);
      if (left < all) {
        if (left >= prior && left < prior + __popc(m)) {
          uint32_t bits = m;
          for (uint32_t k = left - prior; k > 0; --k) bits &= bits - 1;
          a.tokens[r] = span.head + 8 * (i0 + lane) + __builtin_ctz(bits);
        }
        break;
      }
      left -= all;
    }
  }
  if (wave == kSampleWaves - 1) {
    before += n;
    if (((tails >> lane) & 1) && left == before + (uint32_t)__popcll(tails & below))
      a.tokens[r] = loose(lane);
  }
}

// The walk over a tree: from node 0 to its first child whose token was picked at it, and on.
// A wavefront a sequence, 4 nodes a lane; children come after their parents, so a step looks
// at the nodes behind the last. A parent that does not come before its node is none.
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

hipError_t launch_sample(const SampleArgs& a, Elem dtype, hipStream_t stream) {
  if (dtype == Elem::BF16)
    hipLaunchKernelGGL(sample_kernel<__bf16>, dim3(a.R), dim3(kSampleThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(sample_kernel<_Float16>, dim3(a.R), dim3(kSampleThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_tree_accept(const AcceptArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(tree_accept_kernel, dim3(a.B), dim3(64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace ttcd
