// Log probabilities of given tokens, the entropy of their distributions and the most likely alternatives, in one pass
// over the logits x [rows, vocab], and the gradient of all three.
//
//   m = max x,  s = sum e^(x - m),  t = sum (x - m) e^(x - m)
//   lse = m + log s,  logprob = x[target] - lse,  entropy = log s - t / s  (no difference of large numbers)
//   dx = g_logprob (1[target] - p) - g_entropy p (log p + entropy) + sum_j g_top[j] (1[top j] - p)
//
// Forward: a thread keeps (m, s, t) of its own elements in fp32 and the maximum of every step of 16-byte loads.
// Alternatives: a bound that at least k elements reach and few others do comes from the threads' maxima; only steps
// whose maximum reaches it are read again (from L1 or L2), and the candidates are ranked against each other by
// (value, lower index).  Rows in which too many elements reach the bound find the k-th value by bisection and take its
// first holders in order: constant ones, and masked ones with so few finite logits that some warp holds fewer than the
// bound asks of each, which makes it -inf (30 finite logits of 128256 with 20 alternatives: one row 74 us, others 11;
// 1024 rows 4.2 ms, others 0.11).
// Rows of up to 4096 logits are a warp's each, longer ones a block's, or a cluster's where there are few of them.
// Bounded by memory: one read of the logits.  Backward: one read and one write, from the last row on, which the forward
// has read last (L2).  bf16, 4096 rows of 128256: 177 us, 5.9 TB/s of 6.5 that a copy reaches; with 5 alternatives 222;
// 4095 rows of 50257: 80 us, 5.2 TB/s (5.7 a wave of blocks, and 8 us to start and end), the gradient 122 us, 6.8 TB/s.
#include <cooperative_groups.h>

#include "dependent.cuh"
#include "tc_util.cuh"
#include "token_logprobs.cuh"
#include "tree.cuh"

namespace tsa {

namespace {

constexpr int kBlock = 256, kWarps = kBlock / 32;
constexpr int kUnroll = 4;  // vectors in flight a thread
constexpr int kCandidates = 256;
constexpr int kPeakBytes = 64 * 1024;
constexpr int kWarpRow = 4096;  // longest row of a warp
constexpr int kMaxCluster = 8;
constexpr int kBlocksPerSm = 5;  // of the row kernel (launch bounds)
// Warps' rows and the gradient, whose parts are independent, run in smaller blocks (4095 rows of 50257 with gradients:
// 219 against 226 us; 4756 of 182: 10.8 against 11.8); a row's block or cluster in larger ones (one row of 260000 with
// 20 alternatives: 14.7 against 18.8 us, 300 of 128256 30.6 against 40.6).
constexpr int kSmallBlock = 128, kSmallWarps = kSmallBlock / 32, kSmallPerSm = 10;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1.0e6f;  // stands for differences below it: e^kFar is 0, and 0 * kFar is too
constexpr float kLowest = -3.402823466e38f;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The order of floats as that of unsigned integers above 0: -0 equals 0, NaN comes last.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0xffffffffu) return __int_as_float(0x7fc00000);
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// 16 bytes of logits: their maximum (NaN where one is), and pairs of them in fp32.
template <typename T> struct Vec {
  static constexpr int kN = 16 / sizeof(T);
};
template <typename T>
__device__ __forceinline__ uint64_t pair_of(const uint4& v, int i);
template <>
__device__ __forceinline__ uint64_t pair_of<float>(const uint4& v, int i) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  return ptx::f2pack(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
}
template <>
__device__ __forceinline__ uint64_t pair_of<__nv_bfloat16>(const uint4& v, int i) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  return ptx::f2pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
template <>
__device__ __forceinline__ uint64_t pair_of<__half>(const uint4& v, int i) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  return ptx::f2pack(f.x, f.y);
}
__device__ __forceinline__ float peak_of(const uint4& v, float) {
  return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
}
template <typename P>
__device__ __forceinline__ P as_pair(uint32_t w) {
  return *reinterpret_cast<const P*>(&w);
}
__device__ __forceinline__ float peak_of(const uint4& v, __nv_bfloat16) {
  using P = __nv_bfloat162;
  const P p = __hmax2_nan(__hmax2_nan(as_pair<P>(v.x), as_pair<P>(v.y)), __hmax2_nan(as_pair<P>(v.z), as_pair<P>(v.w)));
  return __bfloat162float(__hmax_nan(__low2bfloat16(p), __high2bfloat16(p)));
}
__device__ __forceinline__ float peak_of(const uint4& v, __half) {
  const __half2 p = __hmax2_nan(__hmax2_nan(as_pair<__half2>(v.x), as_pair<__half2>(v.y)),
                                __hmax2_nan(as_pair<__half2>(v.z), as_pair<__half2>(v.w)));
  return __half2float(__hmax_nan(__low2half(p), __high2half(p)));
}

// Elements [begin, begin + count) of a row: those before the first 16-byte boundary, whole vectors, and those behind.
template <typename T> struct Span {
  const T* x;  // the row's element `begin`
  int begin, count, head, vectors;
  __device__ __forceinline__ Span(const T* row, int from, int n) : x(row + from), begin(from), count(n) {
    const int off = (int)(reinterpret_cast<uintptr_t>(x) & 15);
    head = min(n, off ? (16 - off) / (int)sizeof(T) : 0);
    vectors = (n - head) / Vec<T>::kN;
  }
  __device__ __forceinline__ int edges() const { return count - vectors * Vec<T>::kN; }
  __device__ __forceinline__ int edge_index(int i) const { return i < head ? i : i + vectors * Vec<T>::kN; }
  __device__ __forceinline__ float at(int i) const { return Elem<T>::to_acc(x[i]); }
};

struct Sums {
  float m, s, t;  // reference (not below any element), sum of e^(x - m), sum of (x - m) e^(x - m)
};

// To another, not lower, reference.
__device__ __forceinline__ void rebase(Sums& a, float m) {
  const float d = max_nan(a.m - m, kFar);
  const float f = ex2(d * kLog2e);
  a.t = (a.t + d * a.s) * f;
  a.s *= f;
  a.m = m;
}
__device__ __forceinline__ void add(Sums& a, float x) {
  const float d = max_nan(x - a.m, kFar);
  const float e = ex2(d * kLog2e);
  a.s += e;
  a.t = fmaf(d, e, a.t);
}
__device__ __forceinline__ void join(Sums& a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  rebase(a, m);
  rebase(b, m);
  a.s += b.s;
  a.t += b.t;
}
__device__ __forceinline__ void join_warp(Sums& a) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    join(a, Sums{__shfl_xor_sync(0xffffffffu, a.m, off), __shfl_xor_sync(0xffffffffu, a.s, off),
                 __shfl_xor_sync(0xffffffffu, a.t, off)});
}

// One thread's pass over its part of a span: thread `id` of `threads`, one peak for every 2^shift steps (kTop).
template <typename T, bool kTop>
__device__ __forceinline__ void scan(const Span<T>& span, int id, int threads, int shift, float* peaks, Sums& a,
                                     float& peak) {
  constexpr int N = Vec<T>::kN;
  const uint4* body = reinterpret_cast<const uint4*>(span.x + span.head);
  const uint64_t log2e2 = ptx::f2pack(kLog2e, kLog2e);
  uint64_t s2 = 0, t2 = 0;  // pairs of zeros
  auto fold = [&] {         // the pairs' sums into a
    float s0, s1, t0, t1;
    ptx::f2unpack(s2, s0, s1);
    ptx::f2unpack(t2, t0, t1);
    a.s += s0 + s1;
    a.t += t0 + t1;
    s2 = t2 = 0;
  };
  // At most 2 (N - 1) elements outside vectors, one a thread at most.  Under way during the pass, but for alternatives,
  // whose kernel the register costs more (4096 rows of 128256: 226 against 222 us without, 180 against 177 with none).
  const bool edge = id < span.edges();
  float edge_x = !kTop && edge ? span.at(span.edge_index(id)) : -INFINITY;
  uint4 raw[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    if (id + u * threads < span.vectors) raw[u] = body[id + u * threads];
  for (int v0 = id, step = 0; v0 < span.vectors; v0 += threads * kUnroll, ++step) {
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v0 + u * threads < span.vectors) top = max_nan(top, peak_of(raw[u], T()));
    if (kTop) {
      float* slot = peaks + (step >> shift) * threads;  // this thread's own
      *slot = (step & ((1 << shift) - 1)) ? max_nan(*slot, top) : top;
      peak = max_nan(peak, top);
    }
    if (top > a.m) {
      fold();
      rebase(a, top);
    }
    const uint64_t minus = ptx::f2pack(-a.m, -a.m);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (v0 + u * threads >= span.vectors) break;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        float d0, d1;
        ptx::f2unpack(ptx::add2(pair_of<T>(raw[u], i), minus), d0, d1);
        const uint64_t d = ptx::f2pack(max_nan(d0, kFar), max_nan(d1, kFar));
        ptx::f2unpack(ptx::fma2(d, log2e2, 0ull), d0, d1);
        const uint64_t e = ptx::f2pack(ex2(d0), ex2(d1));
        s2 = ptx::add2(s2, e);
        t2 = ptx::fma2(d, e, t2);
      }
      const int next = v0 + (kUnroll + u) * threads;  // under way while the others are added
      if (next < span.vectors) raw[u] = body[next];
    }
  }
  fold();
  if (edge) {
    if (kTop) edge_x = span.at(span.edge_index(id));
    if (edge_x > a.m) rebase(a, edge_x);
    add(a, edge_x);
    if (kTop) peak = max_nan(peak, edge_x);
  }
}

// A row's target: its logit, and whether it has one.
struct Target {
  float logit, instead;  // log probability without a logit: 0 of an ignored one, NaN of one outside the vocabulary
  bool inside;
  template <typename T>
  __device__ __forceinline__ void read(const ts_token_logprobs& p, int64_t row, const T* x) {
    if (!p.logprob) return;
    const int64_t target = p.targets[row];
    inside = target >= 0 && target < p.vocab && target != p.ignore_index;
    instead = target == p.ignore_index ? 0.f : __int_as_float(0x7fc00000);
    logit = inside ? Elem<T>::to_acc(x[target]) : 0.f;
  }
};

// What a row's sums give, by one thread.  A row of -inf has no distribution: log probabilities of -inf, no entropy.
__device__ __forceinline__ float finish(const ts_token_logprobs& p, int64_t row, const Target& target, const Sums& a) {
  const bool none = a.s == 0.f;
  const float log_s = none ? -INFINITY : logf(a.s);
  if (p.norm) {
    p.norm[2 * row] = a.m;
    p.norm[2 * row + 1] = log_s;
  }
  if (p.entropy) p.entropy[row] = none ? 0.f : log_s - a.t / a.s;
  if (p.logprob) p.logprob[row] = !target.inside ? target.instead : none ? -INFINITY : (target.logit - a.m) - log_s;
  return log_s;
}

__device__ __forceinline__ void write_top(const ts_token_logprobs& p, int64_t row, int place, uint64_t found, float m,
                                          float log_s) {
  p.top_indices[row * p.top + place] = (int64_t)(int)~(uint32_t)found;
  p.top_logprobs[row * p.top + place] =
      log_s == -INFINITY ? -INFINITY : (value_of((uint32_t)(found >> 32)) - m) - log_s;
}

// The largest k of a span's elements, ranked in front of all others, by a warp (kGroup = 32) or a block.
template <typename T, int kGroup> struct Select {
  uint64_t* found;       // [kCandidates] (value's order, ~index of the row)
  uint32_t *count, *tmp;  // tmp: a word a warp
  int* list;              // [kCandidates]
  uint32_t* listed;
  int id;

  __device__ __forceinline__ void sync() const {
    if (kGroup == 32)
      __syncwarp();
    else
      __syncthreads();
  }
  __device__ __forceinline__ uint32_t sum(uint32_t n) const {
    n = __reduce_add_sync(0xffffffffu, n);
    if (kGroup == 32) return n;
    __syncthreads();
    if (id % 32 == 0) tmp[id / 32] = n;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < kGroup / 32; ++w) all += tmp[w];
    return all;
  }
  // A bound that at least k elements reach, from every thread's largest (0: it has none).  Block: of the r-th largest
  // of every warp, r = ceil(k / warps), the smallest.  Warp: the k-th largest.
  __device__ __forceinline__ uint32_t bound(uint32_t mine, int k) const {
    const int rounds = kGroup == 32 ? k : (k + kGroup / 32 - 1) / (kGroup / 32);
    uint32_t top = 0;
    for (int r = 0; r < rounds; ++r) {
      top = __reduce_max_sync(0xffffffffu, mine);
      const uint32_t holders = __ballot_sync(0xffffffffu, mine == top);
      if (id % 32 == __ffs(holders) - 1) mine = 0;
    }
    if (kGroup == 32) return top;
    if (id % 32 == 0) tmp[id / 32] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kGroup / 32; ++w) top = min(top, tmp[w]);
    return top;
  }
  __device__ __forceinline__ void offer(const Span<T>& span, float x, int i, uint32_t least) const {
    const uint32_t key = order_of(x);
    if (key < least) return;
    const uint32_t at = atomicAdd(count, 1u);
    if (at < kCandidates) found[at] = (uint64_t)key << 32 | (uint32_t)~(span.begin + i);
  }
  __device__ uint32_t count_from(const Span<T>& span, uint32_t key) const {
    uint32_t n = 0;
    for (int i = id; i < span.count; i += kGroup) n += order_of(span.at(i)) >= key;
    return sum(n);
  }
  // Too many reach the bound: the k-th value by bisection; all above it, and its first holders in order.
  __device__ void by_bisection(const Span<T>& span, int k) const {
    uint32_t low = 1, high = 0xffffffffu;  // at least k elements reach low
    while (low < high) {
      const uint32_t mid = high - (high - low) / 2;
      if (count_from(span, mid) >= (uint32_t)k)
        low = mid;
      else
        high = mid - 1;
    }
    const uint32_t want = k - (low == 0xffffffffu ? 0 : count_from(span, low + 1));
    sync();
    if (id == 0) *count = 0;
    sync();
    uint32_t had = 0;  // holders before this step's
    for (int i0 = 0; i0 < span.count; i0 += kGroup) {
      const int i = i0 + id;
      const uint32_t key = i < span.count ? order_of(span.at(i)) : 0;
      const uint32_t votes = __ballot_sync(0xffffffffu, key == low);
      uint32_t before = had + __popc(votes & ((1u << (id % 32)) - 1u));
      if (kGroup == 32) {
        had += __popc(votes);
      } else {
        __syncthreads();
        if (id % 32 == 0) tmp[id / 32] = __popc(votes);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kGroup / 32; ++w) {
          if (w < id / 32) before += tmp[w];
          had += tmp[w];
        }
      }
      if (key > low || (key == low && before < want))
        found[atomicAdd(count, 1u)] = (uint64_t)key << 32 | (uint32_t)~(span.begin + i);
    }
    sync();
  }
  // Candidates into `found`; their number.  `count` is 0, and all threads' peaks are visible to themselves.
  __device__ __forceinline__ uint32_t run(const Span<T>& span, int k, uint32_t mine, const float* peaks, int shift) const {
    const uint32_t least = bound(mine, k);
    if (id == 0) *listed = 0;
    sync();
    // The steps that hold candidates, and the few elements outside vectors.
    if (mine >= least) {
      const int stride = (kGroup * kUnroll) << shift;
      for (int v0 = id, slot = 0; v0 < span.vectors; v0 += stride, ++slot)
        if (order_of(peaks[slot * kGroup]) >= least) {
          const uint32_t at = atomicAdd(listed, 1u);
          if (at < kCandidates) list[at] = v0;
        }
      for (int i = id; i < span.edges(); i += kGroup) offer(span, span.at(span.edge_index(i)), span.edge_index(i), least);
    }
    sync();
    // Their vectors, one a thread.
    const uint32_t steps = *listed;
    const int per = kUnroll << shift;
    if (steps <= kCandidates)
      for (int x = id; x < (int)steps * per; x += kGroup) {
        const int v = list[x / per] + x % per * kGroup;
        if (v >= span.vectors) continue;
        const uint4 raw = reinterpret_cast<const uint4*>(span.x + span.head)[v];
        if (order_of(peak_of(raw, T())) < least) continue;
        for (int i = 0; i < Vec<T>::kN; ++i)
          offer(span, span.at(span.head + v * Vec<T>::kN + i), span.head + v * Vec<T>::kN + i, least);
      }
    else if (id == 0)
      *count = kCandidates + 1;
    sync();
    uint32_t n = *count;
    sync();
    if (n > kCandidates) {
      by_bisection(span, k);
      n = *count;
    }
    return n;
  }
};

}  // namespace

// Rows of up to kWarpRow logits: a warp each.
template <typename T, bool kTop>
__global__ void __launch_bounds__(kSmallBlock) token_logprobs_warp_kernel(const __grid_constant__ ts_token_logprobs p) {
  constexpr int kPeaks = kTop ? (kWarpRow / Vec<T>::kN + 32 * kUnroll - 1) / (32 * kUnroll) * 32 : 1;
  __shared__ float s_peaks[kSmallWarps][kPeaks];
  __shared__ uint64_t s_found[kSmallWarps][kTop ? kCandidates : 1];
  __shared__ int s_list[kSmallWarps][kTop ? kCandidates : 1];
  __shared__ uint32_t s_count[kSmallWarps], s_listed[kSmallWarps];
  wait_for_previous();
  let_next_start();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t row = (int64_t)blockIdx.x * kSmallWarps + warp;
  if (row >= p.rows) return;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.stride;
  const Span<T> span(x, 0, p.vocab);
  Target target;
  if (lane == 0) target.read(p, row, x);  // under way during the pass
  Sums a = {kLowest, 0.f, 0.f};
  float peak = -INFINITY;
  scan<T, kTop>(span, lane, 32, 0, s_peaks[warp] + (kTop ? lane : 0), a, peak);
  join_warp(a);
  float log_s = 0.f;
  if (lane == 0) log_s = finish(p, row, target, a);
  if constexpr (kTop) {
    log_s = __shfl_sync(0xffffffffu, log_s, 0);
    if (lane == 0) s_count[warp] = 0;
    __syncwarp();
    const Select<T, 32> select = {s_found[warp], &s_count[warp], nullptr, s_list[warp], &s_listed[warp], lane};
    const uint32_t mine = lane < max(span.vectors, span.edges()) ? order_of(peak) : 0u;
    const uint32_t n = select.run(span, p.top, mine, s_peaks[warp] + lane, 0);
    for (uint32_t i = lane; i < n; i += 32) {
      const uint64_t me = s_found[warp][i];
      int place = 0;
      for (uint32_t j = 0; j < n; ++j) place += s_found[warp][j] > me;
      if (place < p.top) write_top(p, row, place, me, a.m, log_s);
    }
  }
}

// Longer rows: a block each, or a cluster whose blocks take a part each and hand what they found to the first.
template <typename T, bool kTop>
__global__ void __launch_bounds__(kBlock, kBlocksPerSm)
    token_logprobs_kernel(const __grid_constant__ ts_token_logprobs p, int shift, int parts) {
  extern __shared__ float s_peaks[];
  __shared__ Sums s_sums[kWarps], s_all;
  __shared__ uint64_t s_found[kCandidates];
  __shared__ uint64_t s_best[kMaxTopTokens];  // of this block's part, in order
  __shared__ int s_list[kCandidates];
  __shared__ uint32_t s_count, s_listed, s_tmp[kWarps];
  __shared__ float s_log;
  namespace cg = cooperative_groups;
  wait_for_previous();
  let_next_start();
  const int part = blockIdx.x % parts, id = threadIdx.x;
  // Parts of whole vectors' length (the first vector of a part may start anywhere).
  const int size = ((p.vocab + parts - 1) / parts + Vec<T>::kN - 1) / Vec<T>::kN * Vec<T>::kN;
  const int begin = min(p.vocab, part * size);
  const int64_t row = blockIdx.x / parts;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.stride;
  const Span<T> span(x, begin, min(p.vocab - begin, size));
  Target target;
  if (id == 0 && part == 0) target.read(p, row, x);  // under way during the pass
  Sums a = {kLowest, 0.f, 0.f};
  float peak = -INFINITY;
  scan<T, kTop>(span, id, kBlock, shift, s_peaks + (kTop ? id : 0), a, peak);
  join_warp(a);
  if (id % 32 == 0) s_sums[id / 32] = a;
  if (id == 0) s_count = 0;
  __syncthreads();
  if (id < 32) {
    a = id < kWarps ? s_sums[id] : Sums{kLowest, 0.f, 0.f};
    join_warp(a);
    if (id == 0) s_all = a;
    if (parts == 1 && id == 0) s_log = finish(p, row, target, a);
  }
  uint32_t n = 0;
  const int k = min(p.top, span.count);  // of a part
  if constexpr (kTop) {
    const Select<T, kBlock> select = {s_found, &s_count, s_tmp, s_list, &s_listed, id};
    const uint32_t mine = id < max(span.vectors, span.edges()) ? order_of(peak) : 0u;
    if (k > 0) n = select.run(span, k, mine, s_peaks + id, shift);
  }
  if (parts > 1) {
    const cg::cluster_group cluster = cg::this_cluster();
    if constexpr (kTop) {
      if (id < kMaxTopTokens) s_best[id] = 0;
      __syncthreads();
      for (uint32_t i = id; i < n; i += kBlock) {
        const uint64_t me = s_found[i];
        int place = 0;
        for (uint32_t j = 0; j < n; ++j) place += s_found[j] > me;
        if (place < k) s_best[place] = me;
      }
    }
    cluster.sync();
    if (part == 0) {
      if (id < 32) {
        a = id < parts ? *cluster.map_shared_rank(&s_all, id) : Sums{kLowest, 0.f, 0.f};
        join_warp(a);
        if (id == 0) {
          s_all = a;
          s_log = finish(p, row, target, a);
        }
      }
      if constexpr (kTop) {
        n = parts * p.top;  // at most kMaxCluster * kMaxTopTokens
        for (int i = id; i < (int)n; i += kBlock) s_found[i] = cluster.map_shared_rank(s_best, i / p.top)[i % p.top];
      }
    }
    cluster.sync();  // the other blocks' memory has been read
    if (part != 0) return;
  }
  __syncthreads();
  if constexpr (kTop)
    for (uint32_t i = id; i < n; i += kBlock) {
      const uint64_t me = s_found[i];
      int place = 0;
      for (uint32_t j = 0; j < n; ++j) place += s_found[j] > me;
      if (me && place < p.top) write_top(p, row, place, me, s_all.m, s_log);
    }
}

// ---------------------------------------------------------------------------
// Gradient: kGroup threads a (part of a row, row).
// ---------------------------------------------------------------------------
namespace {

struct BwdArgs {
  ts_token_logprobs p;
  const float *grad_logprob, *grad_entropy, *grad_top;
  void* grad;
  int64_t grad_stride;
  int parts, part;  // of a row: their number, vectors of each
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  return ptx::pack_bf16(a, b);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  return ptx::pack_f16(a, b);
}

}  // namespace

template <typename T, int kGroup>
__global__ void __launch_bounds__(kSmallBlock, kSmallPerSm) token_logprobs_bwd_kernel(const __grid_constant__ BwdArgs a) {
  constexpr int N = Vec<T>::kN;
  const ts_token_logprobs& p = a.p;
  wait_for_previous();
  let_next_start();
  const int64_t group = (int64_t)blockIdx.x * (kSmallBlock / kGroup) + threadIdx.x / kGroup;
  const int id = threadIdx.x % kGroup;
  if (group >= p.rows * a.parts) return;
  // From the last row on: those that a forward has just read are still in L2.
  const int64_t row = p.rows - 1 - group / a.parts;
  const int part = (int)(group % a.parts);
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.stride;
  T* out = reinterpret_cast<T*>(a.grad) + row * a.grad_stride;
  const Span<T> span(x, 0, p.vocab);
  const int v_first = part * a.part, v_last = min(span.vectors, v_first + a.part);
  const uint4* body = reinterpret_cast<const uint4*>(x + span.head);
  uint4 raw[kUnroll];
  auto load = [&](int v0) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v0 + u * kGroup < v_last) raw[u] = __ldcs(body + v0 + u * kGroup);
  };
  load(v_first + id);  // under way while the row's numbers are read
  float m = p.norm[2 * row], log_s = p.norm[2 * row + 1];
  const float entropy = p.entropy[row];
  const int64_t target = p.targets[row];
  const bool real = target != p.ignore_index;
  const float g_target = real && a.grad_logprob ? a.grad_logprob[row] : 0.f;
  float g_entropy = a.grad_entropy ? a.grad_entropy[row] : 0.f;
  float g_all = g_target;
  bool idle = !real && g_entropy == 0.f;
  if (a.grad_top)
    for (int j = 0; j < p.top; ++j) {
      const float g = a.grad_top[row * p.top + j];
      g_all += g;
      idle = idle && g == 0.f;
    }
  // Where the gradient's rows lie otherwise than the logits', elements are stored one by one.
  const bool aligned = (reinterpret_cast<uintptr_t>(out + span.head) & 15) == 0;
  const bool last = part == a.parts - 1;
  if (idle) {  // an ignored row that counts in nothing else has no gradient, whatever its logits are
    for (int v = v_first + id; v < v_last; v += kGroup) {
      T* to = out + span.head + (int64_t)v * N;
      if (aligned)
        *reinterpret_cast<uint4*>(to) = make_uint4(0u, 0u, 0u, 0u);
      else
        for (int i = 0; i < N; ++i) to[i] = Elem<T>::from_acc(0.f);
    }
    if (last)
      for (int i = id; i < span.edges(); i += kGroup) out[span.edge_index(i)] = Elem<T>::from_acc(0.f);
    return;
  }
  // A target outside the vocabulary has no log probability: its row's gradient is NaN, as that is.
  if (real && a.grad_logprob && (target < 0 || target >= p.vocab)) g_all = __int_as_float(0x7fc00000);
  const bool none = log_s == -INFINITY;  // a row without a distribution (every logit -inf) has no gradient
  if (none) m = log_s = g_entropy = g_all = 0.f;
  const uint64_t minus_m = ptx::f2pack(-m, -m), minus_s = ptx::f2pack(-log_s, -log_s);
  const uint64_t log2e2 = ptx::f2pack(kLog2e, kLog2e), entropy2 = ptx::f2pack(entropy, entropy);
  const uint64_t g_entropy2 = ptx::f2pack(-g_entropy, -g_entropy), g_all2 = ptx::f2pack(-g_all, -g_all);
  auto grads_of = [&](uint64_t v, float& g0, float& g1) {
    float d0, d1, e0, e1;
    ptx::f2unpack(ptx::add2(ptx::add2(v, minus_m), minus_s), d0, d1);
    const uint64_t d = ptx::f2pack(max_nan(d0, kFar), max_nan(d1, kFar));
    ptx::f2unpack(ptx::fma2(d, log2e2, 0ull), e0, e1);
    const uint64_t g = ptx::fma2(g_entropy2, ptx::add2(d, entropy2), g_all2);
    ptx::f2unpack(ptx::fma2(ptx::f2pack(ex2(e0), ex2(e1)), g, 0ull), g0, g1);
  };
  auto grad_of = [&](float v) {
    float g0, g1;
    grads_of(ptx::f2pack(v, v), g0, g1);
    return g0;
  };
  for (int v0 = v_first + id; v0 < v_last;) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = v0 + u * kGroup;
      if (v >= v_last) break;
      float g[N];
#pragma unroll
      for (int i = 0; i < N / 2; ++i) grads_of(pair_of<T>(raw[u], i), g[2 * i], g[2 * i + 1]);
      T* to = out + span.head + (int64_t)v * N;
      if (aligned) {
        uint4 w;
        if constexpr (N == 4)
          w = make_uint4(__float_as_uint(g[0]), __float_as_uint(g[1]), __float_as_uint(g[2]), __float_as_uint(g[3]));
        else
          w = make_uint4(pack2<T>(g[0], g[1]), pack2<T>(g[2], g[3]), pack2<T>(g[4], g[5]), pack2<T>(g[6], g[7]));
        __stcs(reinterpret_cast<uint4*>(to), w);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = Elem<T>::from_acc(g[i]);
      }
    }
    v0 += kGroup * kUnroll;
    load(v0);
  }
  if (last)
    for (int i = id; i < span.edges(); i += kGroup) out[span.edge_index(i)] = Elem<T>::from_acc(grad_of(span.at(span.edge_index(i))));
  // The target and the alternatives: their elements once more, with what they receive themselves.
  if (kGroup == 32)
    __syncwarp();
  else
    __syncthreads();
  if (none) return;
  const int special = a.grad_top ? p.top : 0;
  for (int s = id; s <= special; s += kGroup) {
    const int64_t i = s == 0 ? (real ? target : -1) : p.top_indices[row * p.top + s - 1];
    if (i < 0 || i >= p.vocab) continue;
    const int64_t v = (i - span.head) / N;
    const bool edge = i < span.head || v >= span.vectors;
    if (edge ? !last : v < v_first || v >= v_last) continue;
    float g = grad_of(span.at((int)i));
    if (real && i == target) g += g_target;
    for (int j = 0; j < special; ++j)
      if (p.top_indices[row * p.top + j] == i) g += a.grad_top[row * p.top + j];
    out[i] = Elem<T>::from_acc(g);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
template <typename T, bool kTop>
static cudaError_t forward_t(const ts_token_logprobs& p, cudaStream_t st) {
  if (p.vocab <= kWarpRow)
    return launch_dependent(token_logprobs_warp_kernel<T, kTop>, dim3((unsigned)ceil_div(p.rows, kSmallWarps)),
                            dim3(kSmallBlock), 0, st, p);
  // A cluster a row while there are fewer rows than blocks that the SMs hold, in parts of 4096 logits at least.
  int parts = 1;
  while (parts < kMaxCluster && (int64_t)p.rows * parts <= 2 * device_sms() && p.vocab / (2 * parts) >= 4096) parts *= 2;
  auto kern = token_logprobs_kernel<T, kTop>;
  int shift = 0;
  size_t peaks = 0;
  if (kTop) {
    const int steps = ceil_div(ceil_div(ceil_div(p.vocab, parts), Vec<T>::kN) + 1, kBlock * kUnroll);
    auto slots = [&] { return ((steps + (1 << shift) - 1) >> shift) * kBlock * sizeof(float); };
    while (slots() > kPeakBytes) ++shift;
    peaks = slots();
    const cudaError_t e = ensure_max_smem(reinterpret_cast<const void*>(kern), kPeakBytes);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(p.rows * (int64_t)parts));
  config.blockDim = dim3(kBlock);
  config.dynamicSmemBytes = peaks;
  config.stream = st;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = parts;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  config.attrs = attrs;
  config.numAttrs = parts > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&config, kern, p, shift, parts);
}

cudaError_t token_logprobs(const ts_token_logprobs& p, cudaStream_t st) {
  switch (p.dtype) {
    case TS_F32: return p.top ? forward_t<float, true>(p, st) : forward_t<float, false>(p, st);
    case TS_F16: return p.top ? forward_t<__half, true>(p, st) : forward_t<__half, false>(p, st);
    case TS_BF16: return p.top ? forward_t<__nv_bfloat16, true>(p, st) : forward_t<__nv_bfloat16, false>(p, st);
  }
  return cudaErrorInvalidValue;
}

template <typename T>
static cudaError_t backward_t(BwdArgs a, cudaStream_t st) {
  const int vectors = ceil_div(a.p.vocab, Vec<T>::kN);
  if (vectors <= 32 * kUnroll * 2) {  // a warp a row
    a.parts = 1;
    a.part = vectors;
    return launch_dependent(token_logprobs_bwd_kernel<T, 32>, dim3((unsigned)ceil_div(a.p.rows, kSmallWarps)),
                            dim3(kSmallBlock), 0, st, a);
  }
  a.part = kSmallBlock * kUnroll * 2;
  a.parts = ceil_div(vectors, a.part);
  a.part = ceil_div(vectors, a.parts);
  return launch_dependent(token_logprobs_bwd_kernel<T, kSmallBlock>, dim3((unsigned)(a.p.rows * (int64_t)a.parts)),
                          dim3(kSmallBlock), 0, st, a);
}

cudaError_t token_logprobs_bwd(const ts_token_logprobs& p, const float* grad_logprob, const float* grad_entropy,
                               const float* grad_top, void* grad_logits, int64_t grad_stride, cudaStream_t st) {
  BwdArgs a = {p, grad_logprob, grad_entropy, p.top ? grad_top : nullptr, grad_logits, grad_stride, 1, 0};
  switch (p.dtype) {
    case TS_F32: return backward_t<float>(a, st);
    case TS_F16: return backward_t<__half>(a, st);
    case TS_BF16: return backward_t<__nv_bfloat16>(a, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tsa
