// Log probabilities of given tokens, the entropy of their distributions and the most likely alternatives, in one pass
// over the logits x [rows, vocab], and the gradient of all three.
//
//   m = max x,  s = sum e^(x - m),  t = sum (x - m) e^(x - m)
//   lse = m + log s,  logprob = x[target] - lse,  entropy = log s - t / s  (no difference of large numbers)
//   dx = g_logprob (1[target] - p) - g_entropy p (log p + entropy) + sum_j g_top[j] (1[top j] - p)
//
// Forward: one block a row; a thread keeps (m, s, t) of its own elements in fp32, 16-byte loads, and every vector of
// loads also leaves its maximum in shared memory.  Alternatives: the k-th largest of the threads' maxima is a bound
// that at least k elements reach and few others do; only vectors whose maximum reaches it are read again (from L2),
// and the candidates are ranked against each other by (value, lower index).  Rows built so that too many elements
// reach the bound (constant ones, say) find the k-th value by bisection and take its first holders in order.
// Bounded by memory: one read of the logits.  Backward: one read and one write.
#include "dependent.cuh"
#include "tc_util.cuh"
#include "token_logprobs.cuh"

namespace tsa {

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kUnroll = 4;           // vectors in flight a thread
constexpr int kCandidates = 256;
constexpr int kPeakBytes = 64 * 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1.0e6f;      // stands for differences below it: e^kFar is 0, and 0 * kFar is too

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

// The order of floats as that of unsigned integers: -0 equals 0, NaN comes last.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <typename T> struct Vec {
  static constexpr int kN = 16 / sizeof(T);
  static __device__ __forceinline__ void load(const T* p, float (&x)[kN]) { unpack(*reinterpret_cast<const uint4*>(p), x); }
  static __device__ __forceinline__ void unpack(const uint4& raw, float (&x)[kN]) {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < kN; ++i) x[i] = Elem<T>::to_acc(e[i]);
  }
};

// A row as elements before the first 16-byte boundary, whole vectors, and elements behind them.
template <typename T> struct RowSpan {
  const T* x;
  int vocab, head, vectors;
  __device__ __forceinline__ RowSpan(const T* row, int n) : x(row), vocab(n) {
    const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15);
    head = min(n, off ? (16 - off) / (int)sizeof(T) : 0);
    vectors = (n - head) / Vec<T>::kN;
  }
  __device__ __forceinline__ int edges() const { return vocab - vectors * Vec<T>::kN; }
  __device__ __forceinline__ int edge_index(int i) const { return i < head ? i : i + vectors * Vec<T>::kN; }
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

struct Shared {
  Sums sums[kWarps];
  float max, log_sum;  // of the row
  uint32_t best[kThreads];  // order of every thread's maximum
  uint64_t found[kCandidates];
  uint32_t bound, count, warp_count[kWarps];
};

// Block-wide sum of one integer a thread, the same for all.
__device__ __forceinline__ uint32_t block_count(Shared& sh, uint32_t n) {
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();
  if (threadIdx.x % 32 == 0) sh.warp_count[threadIdx.x / 32] = n;
  __syncthreads();
  uint32_t all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all += sh.warp_count[w];
  return all;
}

// The row's first `want` elements equal to `key`, and all above it, into sh.found (together no more than kMaxTopTokens).
template <typename T>
__device__ void collect_in_order(Shared& sh, const RowSpan<T>& span, uint32_t key, uint32_t want) {
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  uint32_t had = 0;  // elements equal to key before this step's
  for (int i0 = 0; i0 < span.vocab; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    const uint32_t k = i < span.vocab ? order_of(Elem<T>::to_acc(span.x[i])) : 0;
    const bool above = i < span.vocab && k > key, same = i < span.vocab && k == key;
    const uint32_t votes = __ballot_sync(0xffffffffu, same);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sh.warp_count[threadIdx.x / 32] = __popc(votes);
    __syncthreads();
    uint32_t before = had;
    for (int w = 0; w < kWarps; ++w) {
      if (w < (int)threadIdx.x / 32) before += sh.warp_count[w];
      had += sh.warp_count[w];
    }
    before += __popc(votes & ((1u << (threadIdx.x % 32)) - 1u));
    if (above || (same && before < want))
      sh.found[atomicAdd(&sh.count, 1u)] = (uint64_t)k << 32 | (uint32_t)~i;
  }
  __syncthreads();
}

// Elements of the row that are at least `key`.
template <typename T>
__device__ uint32_t count_from(Shared& sh, const RowSpan<T>& span, uint32_t key) {
  uint32_t n = 0;
  for (int i = threadIdx.x; i < span.vocab; i += kThreads) n += order_of(Elem<T>::to_acc(span.x[i])) >= key;
  return block_count(sh, n);
}

}  // namespace

// kTop: s_peak holds the maxima of the threads' vectors, one for every 2^shift steps of kUnroll of them.
template <typename T, bool kTop>
__global__ void __launch_bounds__(kThreads)
    token_logprobs_kernel(const __grid_constant__ ts_token_logprobs p, int shift) {
  constexpr int N = Vec<T>::kN;
  extern __shared__ float s_peak[];
  __shared__ Shared sh;
  wait_for_previous();
  let_next_start();
  const int64_t row = blockIdx.x;
  const RowSpan<T> span(reinterpret_cast<const T*>(p.logits) + row * p.stride, p.vocab);
  const T* body = span.x + span.head;

  Sums a = {-3.402823466e38f, 0.f, 0.f};
  float peak = -INFINITY;  // of this thread's elements, NaN where one is
  for (int v0 = threadIdx.x, step = 0; v0 < span.vectors; v0 += kThreads * kUnroll, ++step) {
    uint4 raw[kUnroll];
    float step_peak = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v0 + u * kThreads < span.vectors) raw[u] = *reinterpret_cast<const uint4*>(body + (int64_t)(v0 + u * kThreads) * N);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (v0 + u * kThreads >= span.vectors) break;
      float x[N];
      Vec<T>::unpack(raw[u], x);
      float top = x[0];
#pragma unroll
      for (int i = 1; i < N; ++i) top = kTop ? max_nan(top, x[i]) : fmaxf(top, x[i]);
      if (kTop) step_peak = max_nan(step_peak, top);
      if (top > a.m) rebase(a, top);
#pragma unroll
      for (int i = 0; i < N; ++i) add(a, x[i]);
    }
    if (kTop) {
      float* slot = s_peak + (step >> shift) * kThreads + threadIdx.x;  // this thread's own
      *slot = (step & ((1 << shift) - 1)) ? max_nan(*slot, step_peak) : step_peak;
      peak = max_nan(peak, step_peak);
    }
  }
  for (int i = threadIdx.x; i < span.edges(); i += kThreads) {
    const float x = Elem<T>::to_acc(span.x[span.edge_index(i)]);
    if (x > a.m) rebase(a, x);
    add(a, x);
    if (kTop) peak = max_nan(peak, x);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    join(a, Sums{__shfl_xor_sync(0xffffffffu, a.m, off), __shfl_xor_sync(0xffffffffu, a.s, off),
                 __shfl_xor_sync(0xffffffffu, a.t, off)});
  if (threadIdx.x % 32 == 0) sh.sums[threadIdx.x / 32] = a;
  if (kTop) {
    sh.best[threadIdx.x] = threadIdx.x < max(span.vectors, span.edges()) ? order_of(peak) : 0u;  // 0: no element
    if (threadIdx.x == 0) sh.count = 0;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    a = threadIdx.x < kWarps ? sh.sums[threadIdx.x] : Sums{-3.402823466e38f, 0.f, 0.f};
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
      join(a, Sums{__shfl_xor_sync(0xffffffffu, a.m, off), __shfl_xor_sync(0xffffffffu, a.s, off),
                   __shfl_xor_sync(0xffffffffu, a.t, off)});
    if (threadIdx.x == 0) {
      // A row of -inf has no distribution: log probabilities of -inf, no entropy.
      const bool none = a.s == 0.f;
      const float log_s = none ? -INFINITY : logf(a.s);
      sh.max = a.m;
      sh.log_sum = log_s;
      if (p.norm) {
        p.norm[2 * row] = a.m;
        p.norm[2 * row + 1] = log_s;
      }
      if (p.entropy) p.entropy[row] = none ? 0.f : log_s - a.t / a.s;
      if (p.logprob) {
        const int64_t target = p.targets[row];
        float lp = __int_as_float(0x7fc00000);  // a target outside the vocabulary
        if (target == p.ignore_index)
          lp = 0.f;
        else if (target >= 0 && target < p.vocab)
          lp = none ? -INFINITY : (Elem<T>::to_acc(span.x[target]) - a.m) - log_s;
        p.logprob[row] = lp;
      }
    }
  }
  if constexpr (kTop) {
    const int k = p.top;
    // The k-th largest of the threads' maxima, equal ones by thread.
    const uint32_t mine = sh.best[threadIdx.x];
    int rank = 0;
    for (int i = 0; i < kThreads; ++i) {
      const uint32_t other = sh.best[i];
      rank += other > mine || (other == mine && i < (int)threadIdx.x);
    }
    if (rank == k - 1) sh.bound = mine;
    __syncthreads();
    const uint32_t bound = sh.bound;
    auto offer = [&](int i) {
      const uint32_t key = order_of(Elem<T>::to_acc(span.x[i]));
      if (key < bound) return;
      const uint32_t at = atomicAdd(&sh.count, 1u);
      if (at < kCandidates) sh.found[at] = (uint64_t)key << 32 | (uint32_t)~i;
    };
    if (mine >= bound) {
      const int stride = (kThreads * kUnroll) << shift;
      for (int v0 = threadIdx.x, slot = 0; v0 < span.vectors; v0 += stride, ++slot)
        if (order_of(s_peak[slot * kThreads + threadIdx.x]) >= bound && sh.count <= kCandidates)
          for (int v = v0; v < min(v0 + stride, span.vectors); v += kThreads)
            for (int i = 0; i < N; ++i) offer(span.head + v * N + i);
      for (int i = threadIdx.x; i < span.edges(); i += kThreads) offer(span.edge_index(i));
    }
    __syncthreads();
    uint32_t count = sh.count;
    if (count > kCandidates) {
      uint32_t low = 0, high = 0xffffffffu;  // at least k elements reach low
      while (low < high) {
        const uint32_t mid = high - (high - low) / 2;
        if (count_from(sh, span, mid) >= (uint32_t)k)
          low = mid;
        else
          high = mid - 1;
      }
      const uint32_t above = low == 0xffffffffu ? 0 : count_from(sh, span, low + 1);
      collect_in_order(sh, span, low, k - above);
      count = sh.count;
    }
    const float m = sh.max, log_s = sh.log_sum;
    if (threadIdx.x < count) {
      const uint64_t me = sh.found[threadIdx.x];
      int place = 0;
      for (uint32_t i = 0; i < count; ++i) place += sh.found[i] > me;
      if (place < k) {
        const int i = (int)~(uint32_t)me;
        p.top_indices[row * k + place] = i;
        p.top_logprobs[row * k + place] =
            log_s == -INFINITY ? -INFINITY : (Elem<T>::to_acc(span.x[i]) - m) - log_s;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Gradient: a block a (part of a row, row), kThreads * kUnroll vectors at most.
// ---------------------------------------------------------------------------
namespace {

struct BwdArgs {
  ts_token_logprobs p;
  const float *grad_logprob, *grad_entropy, *grad_top;
  void* grad;
  int64_t grad_stride;
  int parts, part;  // of a row: their number, elements of each (a multiple of a vector)
};

template <typename T>
__device__ __forceinline__ void store_vec(T* out, const float (&x)[Vec<T>::kN]) {
  uint4 raw;
  T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int i = 0; i < Vec<T>::kN; ++i) e[i] = Elem<T>::from_acc(x[i]);
  *reinterpret_cast<uint4*>(out) = raw;
}

}  // namespace

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(const __grid_constant__ BwdArgs a) {
  constexpr int N = Vec<T>::kN;
  const ts_token_logprobs& p = a.p;
  wait_for_previous();
  let_next_start();
  const int64_t row = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.stride;
  T* out = reinterpret_cast<T*>(a.grad) + row * a.grad_stride;
  const float m = p.norm[2 * row], log_s = p.norm[2 * row + 1], entropy = p.entropy[row];
  const int64_t target = p.targets[row];
  const bool real = target != p.ignore_index;
  const float g_target = real && a.grad_logprob ? a.grad_logprob[row] : 0.f;
  const float g_entropy = a.grad_entropy ? a.grad_entropy[row] : 0.f;
  float g_all = g_target;
  if (a.grad_top)
    for (int j = 0; j < p.top; ++j) g_all += a.grad_top[row * p.top + j];
  // A target outside the vocabulary has no log probability: its row's gradient is NaN, as that is.
  if (real && a.grad_logprob && (target < 0 || target >= p.vocab)) g_all = __int_as_float(0x7fc00000);
  const bool none = log_s == -INFINITY;  // a row without a distribution has no gradient
  auto grad_of = [&](float v) {
    if (none) return 0.f;
    const float d = max_nan((v - m) - log_s, kFar);
    return -ex2(d * kLog2e) * fmaf(g_entropy, d + entropy, g_all);
  };
  // Parts begin at vectors of the logits; where the gradient's rows lie otherwise, elements are stored one by one.
  const int off = (int)(reinterpret_cast<uintptr_t>(x) & 15);
  const int head = min(p.vocab, off ? (16 - off) / (int)sizeof(T) : 0);
  const int vectors = (p.vocab - head) / N;
  const bool aligned = (reinterpret_cast<uintptr_t>(out + head) & 15) == 0;
  const int v_first = part * (a.part / N), v_last = min(vectors, v_first + a.part / N);
  for (int v0 = v_first + threadIdx.x; v0 < v_last; v0 += kThreads * kUnroll) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v0 + u * kThreads < v_last)
        raw[u] = *reinterpret_cast<const uint4*>(x + head + (int64_t)(v0 + u * kThreads) * N);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (v0 + u * kThreads >= v_last) break;
      float v[N];
      Vec<T>::unpack(raw[u], v);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = grad_of(v[i]);
      T* to = out + head + (int64_t)(v0 + u * kThreads) * N;
      if (aligned) {
        store_vec<T>(to, v);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = Elem<T>::from_acc(v[i]);
      }
    }
  }
  const int edges = p.vocab - vectors * N;
  const bool last = part == a.parts - 1;
  if (last && (int)threadIdx.x < edges) {
    const int i = (int)threadIdx.x < head ? threadIdx.x : threadIdx.x + vectors * N;
    out[i] = Elem<T>::from_acc(grad_of(Elem<T>::to_acc(x[i])));
  }
  // The target and the alternatives: their elements once more, with what they receive themselves.
  __syncthreads();
  const int special = a.grad_top ? p.top : 0;
  if ((int)threadIdx.x <= special && !none) {
    const int64_t i = threadIdx.x == 0 ? (real ? target : -1) : p.top_indices[row * p.top + threadIdx.x - 1];
    if (i >= 0 && i < p.vocab) {
      const int64_t v = (i - head) / N;
      const bool edge = i < head || v >= vectors;
      if (edge ? last : v >= v_first && v < v_last) {
        float g = grad_of(Elem<T>::to_acc(x[i]));
        if (real && i == target) g += g_target;
        for (int j = 0; j < special; ++j)
          if (p.top_indices[row * p.top + j] == i) g += a.grad_top[row * p.top + j];
        out[i] = Elem<T>::from_acc(g);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
template <typename T>
static cudaError_t forward_t(const ts_token_logprobs& p, cudaStream_t st) {
  const dim3 grid((unsigned)p.rows), block(kThreads);
  if (!p.top) return launch_dependent(token_logprobs_kernel<T, false>, grid, block, 0, st, p, 0);
  auto kern = token_logprobs_kernel<T, true>;
  const int steps = ceil_div(ceil_div(p.vocab, Vec<T>::kN), kThreads * kUnroll);
  int shift = 0;
  while (((steps + (1 << shift) - 1) >> shift) * kThreads * (int)sizeof(float) > kPeakBytes) ++shift;
  const cudaError_t e = ensure_max_smem(reinterpret_cast<const void*>(kern), kPeakBytes);
  if (e != cudaSuccess) return e;
  return launch_dependent(kern, grid, block, ((steps + (1 << shift) - 1) >> shift) * kThreads * sizeof(float), st, p, shift);
}

cudaError_t token_logprobs(const ts_token_logprobs& p, cudaStream_t st) {
  switch (p.dtype) {
    case TS_F32: return forward_t<float>(p, st);
    case TS_F16: return forward_t<__half>(p, st);
    case TS_BF16: return forward_t<__nv_bfloat16>(p, st);
  }
  return cudaErrorInvalidValue;
}

template <typename T>
static cudaError_t backward_t(BwdArgs a, cudaStream_t st) {
  a.part = kThreads * kUnroll * 2 * Vec<T>::kN;
  a.parts = ceil_div(a.p.vocab, a.part);
  return launch_dependent(token_logprobs_bwd_kernel<T>, dim3((unsigned)(a.p.rows * a.parts)), dim3(kThreads), 0, st, a);
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
