// CUDA-core attention for the sliding window with sinks (forward and backward) and for drafted tokens over a
// cache: fp32 and fp64, and the half-type problems that the tensor-core kernels leave (head dimensions above 128 or
// not a multiple of 8, Dv != D, strides that TMA cannot address, a scale that is not positive).
//
// A block of 128 threads holds R = 16 RT rows and walks over tiles of 8 NC columns, both in shared memory.  Thread
// (ty, tx) owns rows ty + 16 r and columns tx + 8 k of the products, and channels 4 (tx + 8 c) of the accumulators, so
// that RT + NC (products) and RT + 4 DC (accumulators, four columns) 16-byte reads feed 4 RT NC and 16 RT DC
// multiply-adds.  In fp32 the next operand is on its way (cp.async) while this one is multiplied.  The arithmetic is
// exact in the accumulation type (fp32, or fp64 for fp64), exponentials in base 2.
// Which columns a row sees is a 32-bit word a row and 32 columns (tree.cuh, window.cuh).
//
// Bound by fixed latencies at two warps a scheduler, which registers and shared memory leave (half of the issue slots and
// of the multiply-add pipe in use; with half the rows a block and three or four warps the reads cost more: gradients of
// 2 x 2000 queries 1170 us against 940), and by a block's chain of tiles in small calls.  fp32, D 64, counting the pairs
// that are seen: 2 x 2000 queries, 8 heads, forward 428 us (19 TFLOP/s of 74), with a window of 500 195 us; forward and
// backward, on 4 KV heads, 1396 and 710 us; 2 x 511 queries, 4 heads on 2, a window of 128, 3 sinks, both 101 us.
// bf16 of 256 channels, 4096 queries, 16 heads on 8, a window of 1024: forward 2.86 ms (21 TFLOP/s), backward 18.8 (8).
#pragma once
#include "dependent.cuh"
#include "simt_kernels.cuh"
#include "tc_util.cuh"
#include "rows.cuh"

namespace tsa {

constexpr int kRowsThreads = 128, kRowsPad = 4;
constexpr double kLog2eD = 1.4426950408889634, kLn2D = 0.6931471805599453;

__device__ __forceinline__ float acc_exp2(float x) { return exp2f(x); }
__device__ __forceinline__ double acc_exp2(double x) { return exp2(x); }
__device__ __forceinline__ float acc_log2(float x) { return log2f(x); }
__device__ __forceinline__ double acc_log2(double x) { return log2(x); }

template <typename A> struct Quad {
  A v[4];
};
template <typename A>
__device__ __forceinline__ Quad<A> quad(const A* p) {
  Quad<A> q;
  if constexpr (sizeof(A) == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    q.v[0] = f.x, q.v[1] = f.y, q.v[2] = f.z, q.v[3] = f.w;
  } else {
    const double2 a = reinterpret_cast<const double2*>(p)[0], b = reinterpret_cast<const double2*>(p)[1];
    q.v[0] = a.x, q.v[1] = a.y, q.v[2] = b.x, q.v[3] = b.y;
  }
  return q;
}

__device__ __forceinline__ void copy_row16(void* dst, const void* src, bool live) {  // zeros where it is not live
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(dst)), "l"(src), "r"(live ? 16 : 0)
               : "memory");
}

// Which rows of a tile are zeros whatever memory holds: none, or those of a word's bits.
struct NoneGone {
  __device__ __forceinline__ bool operator()(int) const { return false; }
};
struct BitsGone {
  uint64_t bits;
  __device__ __forceinline__ bool operator()(int r) const { return bits >> r & 1u; }
};

// Rows [t0, t0 + rows) of (b, h) into shared memory, a row every `stride` elements; zeros in rows that are gone, at
// and behind row `end`, and from channel C on (to a whole quad, which is what the products read: vectors alone serve
// where C ends with one, as a double's two channels need not).  fp32 rows on 16-byte boundaries are under way when it returns (ptx::copies_done).
template <typename T, typename A, typename Gone = NoneGone>
__device__ __forceinline__ void stage_tile(A* dst, int stride, const ts_view4& src, int b, int h, int64_t t0, int rows,
                                           int64_t end, int C, Gone gone = Gone()) {
  constexpr int kVec = 16 / sizeof(T);
  const T* base = reinterpret_cast<const T*>(src.data) + (int64_t)b * src.stride[0] + (int64_t)h * src.stride[1];
  const bool vec = src.stride[3] == 1 && C % kVec == 0 && C % 4 == 0 && (src.stride[2] * sizeof(T)) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(base) % 16 == 0;
  if (vec) {
    const int per = C / kVec, n = rows * per;
    if constexpr (sizeof(T) == 4) {
      for (int x = threadIdx.x; x < n; x += kRowsThreads) {
        const int r = x / per, c = x - r * per;
        const bool live = t0 + r < end && !gone(r);
        copy_row16(dst + r * stride + c * kVec, live ? base + (t0 + r) * src.stride[2] + c * kVec : base, live);
      }
      return;
    }
    constexpr int kBatch = 4;
    for (int x0 = threadIdx.x; x0 < n; x0 += kRowsThreads * kBatch) {
      uint4 raw[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int x = x0 + u * kRowsThreads, r = x / per, c = x % per;
        raw[u] = make_uint4(0u, 0u, 0u, 0u);
        if (x < n && t0 + r < end && !gone(r))
          raw[u] = *reinterpret_cast<const uint4*>(base + (t0 + r) * src.stride[2] + c * kVec);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int x = x0 + u * kRowsThreads, r = x / per, c = x % per;
        if (x >= n) break;
        const T* e = reinterpret_cast<const T*>(&raw[u]);
        A* out = dst + r * stride + c * kVec;
#pragma unroll
        for (int i = 0; i < kVec; ++i) out[i] = Elem<T>::to_acc(e[i]);
      }
    }
    return;
  }
  const int wide = ceil_div(C, 4) * 4, n = rows * wide;
  constexpr int kBatch = 8;
  for (int x0 = threadIdx.x; x0 < n; x0 += kRowsThreads * kBatch) {
    T raw[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int x = x0 + u * kRowsThreads, r = x / wide, c = x % wide;
      raw[u] = x < n && c < C && t0 + r < end && !gone(r) ? base[(t0 + r) * src.stride[2] + c * src.stride[3]]
                                                          : Elem<T>::from_acc(A(0));
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int x = x0 + u * kRowsThreads;
      if (x < n) dst[x / wide * stride + x % wide] = Elem<T>::to_acc(raw[u]);
    }
  }
}

// Rows [r0, r0 + rows) of the packed rows (head h0 + r / tokens, token r % tokens), r < end.
template <typename T, typename A>
__device__ __forceinline__ void stage_packed(A* dst, int stride, const ts_view4& src, int b, int h0, int r0, int rows,
                                             int end, int tokens, int C) {
  constexpr int kVec = 16 / sizeof(T), kBatch = 4;
  const T* base = reinterpret_cast<const T*>(src.data) + (int64_t)b * src.stride[0];
  auto row_at = [&](int r) { return base + (int64_t)(h0 + r / tokens) * src.stride[1] + (int64_t)(r % tokens) * src.stride[2]; };
  const bool vec = src.stride[3] == 1 && C % kVec == 0 && C % 4 == 0 && (src.stride[2] * sizeof(T)) % 16 == 0 &&
                   (src.stride[1] * sizeof(T)) % 16 == 0 && reinterpret_cast<uintptr_t>(base) % 16 == 0;
  const int wide = ceil_div(C, 4) * 4, per = vec ? C / kVec : wide, n = rows * per;
  for (int x0 = threadIdx.x; x0 < n; x0 += kRowsThreads * kBatch) {
    if (vec) {
      uint4 raw[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int x = x0 + u * kRowsThreads, r = x / per, c = x % per;
        raw[u] = make_uint4(0u, 0u, 0u, 0u);
        if (x < n && r0 + r < end) raw[u] = *reinterpret_cast<const uint4*>(row_at(r0 + r) + c * kVec);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int x = x0 + u * kRowsThreads, r = x / per, c = x % per;
        if (x >= n) break;
        const T* e = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
        for (int i = 0; i < kVec; ++i) dst[r * stride + c * kVec + i] = Elem<T>::to_acc(e[i]);
      }
    } else {
      T raw[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int x = x0 + u * kRowsThreads, r = x / per, c = x % per;
        raw[u] = x < n && r0 + r < end && c < C ? row_at(r0 + r)[c * src.stride[3]] : Elem<T>::from_acc(A(0));
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int x = x0 + u * kRowsThreads;
        if (x < n) dst[x / per * stride + x % per] = Elem<T>::to_acc(raw[u]);
      }
    }
  }
}

// acc[r][k] = sum_c rows[ty + 16 r][c] cols[tx + 8 k][c].
template <int RT, int NC, typename A>
__device__ __forceinline__ void dots(A (&acc)[RT][NC], const A* rows, const A* cols, int stride, int C, int ty, int tx) {
  if constexpr (sizeof(A) == 4) {  // sums of even and of odd channels, two products an instruction
    uint64_t two[RT][NC];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int k = 0; k < NC; ++k) two[r][k] = 0;
#pragma unroll 2
    for (int c = 0; c < C; c += 4) {
      ulonglong2 a[RT], b[NC];
#pragma unroll
      for (int r = 0; r < RT; ++r) a[r] = *reinterpret_cast<const ulonglong2*>(rows + (ty + 16 * r) * stride + c);
#pragma unroll
      for (int k = 0; k < NC; ++k) b[k] = *reinterpret_cast<const ulonglong2*>(cols + (tx + 8 * k) * stride + c);
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int k = 0; k < NC; ++k) two[r][k] = ptx::fma2(a[r].x, b[k].x, two[r][k]);
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int k = 0; k < NC; ++k) two[r][k] = ptx::fma2(a[r].y, b[k].y, two[r][k]);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        float x, y;
        ptx::f2unpack(two[r][k], x, y);
        acc[r][k] = x + y;
      }
    return;
  }
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int k = 0; k < NC; ++k) acc[r][k] = A(0);
#pragma unroll 2
  for (int c = 0; c < C; c += 4) {
    Quad<A> a[RT], b[NC];
#pragma unroll
    for (int r = 0; r < RT; ++r) a[r] = quad(rows + (ty + 16 * r) * stride + c);
#pragma unroll
    for (int k = 0; k < NC; ++k) b[k] = quad(cols + (tx + 8 * k) * stride + c);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int k = 0; k < NC; ++k) acc[r][k] += a[r].v[e] * b[k].v[e];
  }
}

// acc[r][c] += sum_j w[ty + 16 r][j] cols[j][4 (tx + 8 c) ..]; w has 8 NC + kRowsPad elements a row.
template <int RT, int NC, int DC, typename A>
__device__ __forceinline__ void accumulate(A (&acc)[RT][DC][4], const A* w, const A* cols, int stride, int ty, int tx) {
  if constexpr (sizeof(A) == 4) {
    uint64_t two[RT][DC][2];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        two[r][c][0] = ptx::f2pack(acc[r][c][0], acc[r][c][1]);
        two[r][c][1] = ptx::f2pack(acc[r][c][2], acc[r][c][3]);
      }
#pragma unroll 2
    for (int j = 0; j < 8 * NC; j += 4) {
      Quad<A> p[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) p[r] = quad(w + (ty + 16 * r) * (8 * NC + kRowsPad) + j);
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        uint64_t both[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) both[r] = ptx::f2pack(p[r].v[jj], p[r].v[jj]);
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(cols + (j + jj) * stride + 4 * (tx + 8 * c));
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            two[r][c][0] = ptx::fma2(both[r], v.x, two[r][c][0]);
            two[r][c][1] = ptx::fma2(both[r], v.y, two[r][c][1]);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        ptx::f2unpack(two[r][c][0], acc[r][c][0], acc[r][c][1]);
        ptx::f2unpack(two[r][c][1], acc[r][c][2], acc[r][c][3]);
      }
    return;
  }
#pragma unroll 2
  for (int j = 0; j < 8 * NC; j += 4) {
    Quad<A> p[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) p[r] = quad(w + (ty + 16 * r) * (8 * NC + kRowsPad) + j);
#pragma unroll
    for (int jj = 0; jj < 4; ++jj)
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        const Quad<A> v = quad(cols + (j + jj) * stride + 4 * (tx + 8 * c));
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r][c][e] += p[r].v[jj] * v.v[e];
      }
  }
}

template <int RT, int DC, typename A>
__device__ __forceinline__ void clear(A (&acc)[RT][DC][4]) {
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[r][c][e] = A(0);
}

template <typename A>
__device__ __forceinline__ A lanes8_sum(A x) {
#pragma unroll
  for (int off = 4; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}
template <typename A>
__device__ __forceinline__ A lanes8_max(A x) {
#pragma unroll
  for (int off = 4; off > 0; off >>= 1) {
    const A y = __shfl_xor_sync(0xffffffffu, x, off);
    x = y > x ? y : x;
  }
  return x;
}

template <typename A, int RT, int DC> struct RowsCfg {
  static constexpr int kRows = 16 * RT;
  static constexpr int kStride = 32 * DC + kRowsPad;
  // Columns of a thread: 8 feed more multiply-adds a read, 4 leave room for a second block where rows are long.
  static constexpr int kFwdNC = sizeof(A) == 4 && DC == 2 ? 8 : 4, kBwdNC = 4;
  static constexpr int kFwdCols = 8 * kFwdNC, kBwdCols = 8 * kBwdNC;
  static constexpr size_t kFwdSmem = sizeof(A) * ((kRows + 2 * kFwdCols) * kStride + kRows * (kFwdCols + kRowsPad));
  // rows' two operands, the tile's two (twice in fp32, where the next ones are under way), P and dS
  static constexpr int kBufs = sizeof(A) == 4 ? 2 : 1;
  static constexpr size_t kBwdSmem = sizeof(A) * ((2 * kRows + 2 * kBufs * kBwdCols) * kStride +
                                                  2 * kRows * (kBwdCols + kRowsPad));
};

// The running softmax of R rows over tiles of keys.
template <typename T, int RT, int DC> struct RowsForward {
  using A = typename Elem<T>::acc;
  using C = RowsCfg<A, RT, DC>;
  static constexpr int kNC = C::kFwdNC, kCols = C::kFwdCols;
  A acc[RT][DC][4], m[RT], l[RT];
  A *q, *k, *v, *w;
  int ty, tx;

  __device__ __forceinline__ RowsForward(A* smem) {
    q = smem;
    k = q + C::kRows * C::kStride;
    v = k + kCols * C::kStride;
    w = v + kCols * C::kStride;
    ty = threadIdx.x / 8;
    tx = threadIdx.x % 8;
  }
  __device__ __forceinline__ void start() {
    clear(acc);
#pragma unroll
    for (int r = 0; r < RT; ++r) m[r] = neg_inf<A>(), l[r] = A(0);
  }
  // n tiles, tile j at key key_of(j), of head hk; bits(r, slot): what row ty + 16 r sees of the 32 keys from `slot` on.
  // Keys at and behind `end` are not read, nor the values of those of tile k0 that gone_of(k0) names.  K of the next tile
  // is under way during P.V, V during Q.K.
  template <typename Key, typename Bits, typename GoneOf>
  __device__ __forceinline__ void run(const ts_attn_params& p, int b, int hk, int n, int end, A scale2, Key key_of,
                                      Bits bits, GoneOf gone_of) {
    if (n > 0) stage_tile<T, A>(k, C::kStride, p.k, b, hk, key_of(0), kCols, end, p.head_dim);
    for (int j = 0; j < n; ++j) {
      const int k0 = key_of(j);
      ptx::copies_done();
      __syncthreads();  // K(j) is there, V(j - 1) is used up
      stage_tile<T, A>(v, C::kStride, p.v, b, hk, k0, kCols, end, p.value_dim, gone_of(k0));
      A s[RT][kNC];
      dots<RT, kNC>(s, q, k, C::kStride, p.head_dim, ty, tx);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        uint32_t see[kNC / 4];
#pragma unroll
        for (int x = 0; x < kNC / 4; ++x) see[x] = bits(r, k0 + 32 * x);
        A top = neg_inf<A>();
#pragma unroll
        for (int c = 0; c < kNC; ++c) {
          s[r][c] = (see[c / 4] >> (tx + 8 * (c % 4))) & 1u ? s[r][c] * scale2 : neg_inf<A>();
          top = s[r][c] > top ? s[r][c] : top;
        }
        top = lanes8_max(top);
        const A next = top > m[r] ? top : m[r];
        const A safe = next == neg_inf<A>() ? A(0) : next;
        const A factor = acc_exp2(m[r] - safe);
        A sum = A(0);
#pragma unroll
        for (int c = 0; c < kNC; ++c) {
          const A e = acc_exp2(s[r][c] - safe);
          w[(ty + 16 * r) * (kCols + kRowsPad) + tx + 8 * c] = e;
          sum += e;
        }
        l[r] = l[r] * factor + lanes8_sum(sum);
        m[r] = next;
#pragma unroll
        for (int c = 0; c < DC; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r][c][e] *= factor;
      }
      ptx::copies_done();
      __syncthreads();  // V(j) is there, K(j) is used up
      if (j + 1 < n) stage_tile<T, A>(k, C::kStride, p.k, b, hk, key_of(j + 1), kCols, end, p.head_dim);
      accumulate<RT, kNC, DC>(acc, w, v, C::kStride, ty, tx);
    }
  }
};

// ---------------------------------------------------------------------------
// Forward under a window: rows are consecutive queries of one head.
// ---------------------------------------------------------------------------
template <typename T, int RT, int DC>
__global__ void __launch_bounds__(kRowsThreads) rows_window_fwd_kernel(const __grid_constant__ RowsWindow a) {
  using F = RowsForward<T, RT, DC>;
  using A = typename F::A;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const ts_attn_params& p = a.p;
  wait_for_previous();
  let_next_start();
  F f(reinterpret_cast<A*>(smem_raw));
  const int h = blockIdx.y, b = blockIdx.z, hk = h / (p.q_heads / p.kv_heads);
  const int i0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * F::C::kRows;  // the longest rows first
  const int kv_end = a.kv_end(b);
  const int64_t offset = a.offset(b);
  stage_tile<T, A>(f.q, F::C::kStride, p.q, b, h, i0, F::C::kRows, p.q_len, p.head_dim);
  f.start();
  const int64_t last = (int64_t)min(i0 + F::C::kRows, p.q_len) - 1 + offset;
  const int end = (int)i64max(0, i64min(kv_end, last + 1));
  const WindowTiles wt(a.win, i0 + offset, kv_end, F::kCols);
  const A scale2 = (A)(p.scale * kLog2eD);
  f.run(p, b, hk, wt.count(ceil_div(end, F::kCols)), kv_end, scale2, [&](int j) { return wt.tile(j) * F::kCols; },
        [&](int r, int slot) {
          const int i = i0 + f.ty + 16 * r;
          if (i >= p.q_len) return 0u;
          const int64_t stop = i64min(kv_end, i + offset + 1);
          return range_bits(i + offset + 1 - a.win.window, stop, slot) |
                 range_bits(0, i64min(stop, a.win.sinks), slot);
        },
        [](int) { return NoneGone(); });
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int i = i0 + f.ty + 16 * r;
    if (i >= p.q_len) continue;
    const A inv = f.l[r] == A(0) ? A(0) : A(1) / f.l[r];  // a sum that is NaN stays one
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int ch = 4 * (f.tx + 8 * c) + e;
        if (ch < p.value_dim) *at4w<T>(p.o, b, h, i, ch) = Elem<T>::from_acc(f.acc[r][c][e] * inv);
      }
    if (p.lse && f.tx == 0)
      reinterpret_cast<A*>(p.lse)[(int64_t)b * p.lse_stride[0] + (int64_t)h * p.lse_stride[1] +
                                  (int64_t)i * p.lse_stride[2]] =
          f.l[r] == A(0) ? neg_inf<A>() : (f.m[r] + acc_log2(f.l[r])) * (A)kLn2D;
  }
}

// ---------------------------------------------------------------------------
// Drafted tokens over a cache: rows are the packed (head, node) pairs of a KV head.  Float: the line of work is
// shared equally and joined by tree_merge; double: one block a unit, which writes the result itself.
// ---------------------------------------------------------------------------
template <typename T, int RT, int DC>
__global__ void __launch_bounds__(kRowsThreads) rows_tree_kernel(const __grid_constant__ TreeArgs a) {
  using F = RowsForward<T, RT, DC>;
  using A = typename F::A;
  constexpr bool kSplit = sizeof(A) == 4;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ LinePlace s_ends[2];
  __shared__ int s_parents[kTreeNodes];
  __shared__ uint64_t s_hidden;
  const ts_attn_params& p = a.p;
  wait_for_previous();
  let_next_start();
  F f(reinterpret_cast<A*>(smem_raw));
  const TreeLine line(a, F::kCols, 0);
  const int group = p.q_heads / p.kv_heads;
  const A scale2 = (A)(p.scale * kLog2eD);
  LineWalk walk;
  if constexpr (kSplit) {
    if (threadIdx.x < 32) {
      LinePlace ends[2];
      line_share(line, threadIdx.x, blockIdx.x, a.ctas, ends);
      if (threadIdx.x == 0) s_ends[0] = ends[0], s_ends[1] = ends[1];
    }
    __syncthreads();
    walk.start(s_ends[0], s_ends[1].tiles - s_ends[0].tiles, line);
  } else {
    walk.b = blockIdx.x / line.units;
    walk.unit = blockIdx.x % line.units;
    walk.first = 0;
    walk.list = line.list(walk.b, walk.unit % line.row_tiles);
    walk.count = walk.list.count;
  }
  while (!kSplit || walk.next(line)) {
    const int b = walk.b, hk = walk.unit / a.row_tiles, r0 = walk.unit % a.row_tiles * F::C::kRows;
    const int len = tree_len(p, b);
    const int64_t base = (int64_t)len - p.q_len;
    const WindowTiles& wt = walk.list.tiles;
    __syncthreads();  // the unit before is used up
    if (a.parents && (int)threadIdx.x < p.q_len) s_parents[threadIdx.x] = a.parents[b * a.parents_stride + threadIdx.x];
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x, n = a.parents ? p.q_len : 0;  // a chain's slots are all seen
      const int32_t* parents = a.parents + b * a.parents_stride;
      const uint64_t hidden =
          n ? hidden_nodes(n, base, lane < n ? parents[lane] : -1, lane + 32 < n ? parents[lane + 32] : -1, lane) : 0;
      if (lane == 0) s_hidden = hidden;
    }
    stage_packed<T, A>(f.q, F::C::kStride, p.q, b, hk * group, r0, F::C::kRows, a.rows, p.q_len, p.head_dim);
    __syncthreads();
    NodeView view[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int i = r0 + f.ty + 16 * r;
      view[r] = tree_node(i % p.q_len, base, !a.parents, a.win, [&](int node) { return s_parents[node]; });
      if (i >= a.rows) view[r].end = 0, view[r].drafted = 0;
    }
    f.start();
    f.run(p, b, hk, walk.count, len, scale2, [&](int j) { return wt.tile(walk.first + j) * F::kCols; },
          [&](int r, int slot) { return view_bits(view[r], base, a.win.sinks, slot); },
          [&](int k0) { return BitsGone{gone_bits(s_hidden, base, len, k0)}; });
    const int64_t part = (int64_t)b * line.units + walk.unit + blockIdx.x;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = f.ty + 16 * r, i = r0 + row;
      if (i >= a.rows) continue;
      if constexpr (kSplit) {
        const int quads = part_quads(p);
        if (f.tx == 0) a.ml[part * a.part_rows + row] = make_float2(f.m[r], f.l[r]);
        float4* out = reinterpret_cast<float4*>(a.part) + part * a.part_rows * quads;
#pragma unroll
        for (int c = 0; c < DC; ++c)
          if (f.tx + 8 * c < quads)
            out[(f.tx + 8 * c) * a.part_rows + row] =
                make_float4(f.acc[r][c][0], f.acc[r][c][1], f.acc[r][c][2], f.acc[r][c][3]);
      } else {
        const int h = hk * group + i / p.q_len, node = i % p.q_len;
        const A inv = f.l[r] == A(0) ? A(0) : A(1) / f.l[r];  // a sum that is NaN stays one
#pragma unroll
        for (int c = 0; c < DC; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int ch = 4 * (f.tx + 8 * c) + e;
            if (ch < p.value_dim) *at4w<T>(p.o, b, h, node, ch) = Elem<T>::from_acc(f.acc[r][c][e] * inv);
          }
        if (p.lse && f.tx == 0)
          reinterpret_cast<A*>(p.lse)[(int64_t)b * p.lse_stride[0] + (int64_t)h * p.lse_stride[1] +
                                      (int64_t)node * p.lse_stride[2]] =
              f.l[r] == A(0) ? neg_inf<A>() : (f.m[r] + acc_log2(f.l[r])) * (A)kLn2D;
      }
    }
    if constexpr (!kSplit) break;
  }
}

// ---------------------------------------------------------------------------
// Backward under a window.  dQ: rows are queries, tiles of keys; dK and dV: rows are keys, tiles of queries of every
// head of the group.  p = 2^(s - lse), ds = p (dO.v - delta) scale.
// ---------------------------------------------------------------------------
struct RowsWindowBwd {
  ts_attn_bwd_params bp;
  WindowArgs win;
  const void* delta;  // [batch, q_heads, q_len] in the accumulation type
};

// delta = sum_c dO O, one warp a row.
template <typename T>
__global__ void __launch_bounds__(256)
    rows_delta_kernel(const __grid_constant__ ts_attn_bwd_params bp, typename Elem<T>::acc* delta) {
  using A = typename Elem<T>::acc;
  const ts_attn_params& p = bp.fwd;
  wait_for_previous();
  let_next_start();
  const int64_t row = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  if (row >= (int64_t)p.batch * p.q_heads * p.q_len) return;
  const int lane = threadIdx.x & 31, i = (int)(row % p.q_len);
  const int h = (int)(row / p.q_len % p.q_heads), b = (int)(row / p.q_len / p.q_heads);
  A sum = A(0);
  for (int c = lane; c < p.value_dim; c += 32)
    sum += Elem<T>::to_acc(*at4<T>(bp.dout, b, h, i, c)) * Elem<T>::to_acc(*at4<T>(p.o, b, h, i, c));
  sum = group_sum<32>(sum);
  if (lane == 0) delta[row] = sum;
}

// Key blocks [first, first + count) whose tiles of queries, of all heads of the group, are divided into parts.
struct RowsKeySet {
  int first, count, parts;
  void* part;
};
struct RowsKeyBlocks {
  RowsKeySet with_sinks, others;  // the former have the longest parts and come first
};

template <typename A>
__device__ __forceinline__ A row_lse2(const ts_attn_params& p, int b, int h, int i) {
  const A v = reinterpret_cast<const A*>(p.lse)[(int64_t)b * p.lse_stride[0] + (int64_t)h * p.lse_stride[1] +
                                                (int64_t)i * p.lse_stride[2]];
  return v == neg_inf<A>() ? -neg_inf<A>() : v * (A)kLog2eD;  // a row that sees nothing: every p is 0
}

// dQ of a query block of a row and head.
template <typename T, int RT, int DC>
__device__ __forceinline__ void rows_window_dq(const RowsWindowBwd& a, unsigned char* smem_raw, int index) {
  using A = typename Elem<T>::acc;
  using C = RowsCfg<A, RT, DC>;
  constexpr int kNC = C::kBwdNC, kCols = C::kBwdCols, kBufs = C::kBufs;
  const ts_attn_params& p = a.bp.fwd;
  A* q = reinterpret_cast<A*>(smem_raw);
  A* g = q + C::kRows * C::kStride;
  A* tiles = g + C::kRows * C::kStride;  // K and V, kBufs times
  A* w = tiles + 2 * kBufs * kCols * C::kStride;
  const RowsWindow rule{p, a.win};
  const int ty = threadIdx.x / 8, tx = threadIdx.x % 8;
  const int heads = p.q_heads * p.batch, bh = index % heads;
  const int h = bh % p.q_heads, b = bh / p.q_heads, hk = h / (p.q_heads / p.kv_heads);
  const int i0 = (ceil_div(p.q_len, C::kRows) - 1 - index / heads) * C::kRows;  // the longest rows first
  const int kv_end = rule.kv_end(b);
  const int64_t offset = rule.offset(b);
  stage_tile<T, A>(q, C::kStride, p.q, b, h, i0, C::kRows, p.q_len, p.head_dim);
  stage_tile<T, A>(g, C::kStride, a.bp.dout, b, h, i0, C::kRows, p.q_len, p.value_dim);
  A lse2[RT], delta[RT], acc[RT][DC][4];
  clear(acc);
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int i = i0 + ty + 16 * r;
    lse2[r] = i < p.q_len ? row_lse2<A>(p, b, h, i) : -neg_inf<A>();
    delta[r] = i < p.q_len ? reinterpret_cast<const A*>(a.delta)[((int64_t)b * p.q_heads + h) * p.q_len + i] : A(0);
  }
  const int64_t last = (int64_t)min(i0 + C::kRows, p.q_len) - 1 + offset;
  const int end = (int)i64max(0, i64min(kv_end, last + 1));
  const WindowTiles wt(a.win, i0 + offset, kv_end, kCols);
  const int n = wt.count(ceil_div(end, kCols));
  const A scale = (A)p.scale, scale2 = (A)(p.scale * kLog2eD);
  auto stage = [&](int j) {
    A* k = tiles + j % kBufs * 2 * kCols * C::kStride;
    stage_tile<T, A>(k, C::kStride, p.k, b, hk, wt.tile(j) * kCols, kCols, kv_end, p.head_dim);
    stage_tile<T, A>(k + kCols * C::kStride, C::kStride, p.v, b, hk, wt.tile(j) * kCols, kCols, kv_end, p.value_dim);
  };
  if (n > 0) stage(0);
  for (int j = 0; j < n; ++j) {
    const int k0 = wt.tile(j) * kCols;
    const A* k = tiles + j % kBufs * 2 * kCols * C::kStride;
    ptx::copies_done();
    __syncthreads();  // this tile is there, the one before is used up
    if (kBufs > 1 && j + 1 < n) stage(j + 1);
    A s[RT][kNC], d[RT][kNC];
    dots<RT, kNC>(s, q, k, C::kStride, p.head_dim, ty, tx);
    dots<RT, kNC>(d, g, k + kCols * C::kStride, C::kStride, p.value_dim, ty, tx);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int64_t stop = i64min(kv_end, i0 + ty + 16 * r + offset + 1);
      const uint32_t see = range_bits(i0 + ty + 16 * r + offset + 1 - a.win.window, stop, k0) |
                           range_bits(0, i64min(stop, a.win.sinks), k0);
#pragma unroll
      for (int c = 0; c < kNC; ++c) {
        const A pr = (see >> (tx + 8 * c)) & 1u ? acc_exp2(s[r][c] * scale2 - lse2[r]) : A(0);
        w[(ty + 16 * r) * (kCols + kRowsPad) + tx + 8 * c] = pr * (d[r][c] - delta[r]) * scale;
      }
    }
    __syncwarp();  // a row's weights are written and read by one warp
    accumulate<RT, kNC, DC>(acc, w, k, C::kStride, ty, tx);
    if (kBufs == 1 && j + 1 < n) {
      __syncthreads();
      stage(j + 1);
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int i = i0 + ty + 16 * r;
    if (i >= p.q_len) continue;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int ch = 4 * (tx + 8 * c) + e;
        if (ch < p.head_dim) *at4w<T>(a.bp.dq, b, h, i, ch) = Elem<T>::from_acc(acc[r][c][e]);
      }
  }
}

// dK and dV of (KV head and row, key block, part of its tiles of queries).  With one part they are written at once; with more,
// each part leaves its sums in `part` and rows_dkv_sum_kernel adds them in order.
template <typename T, int RT, int DC>
__device__ __forceinline__ void rows_window_dkv(const RowsWindowBwd& a, const RowsKeyBlocks& blocks, unsigned char* smem_raw,
                                                int index) {
  using A = typename Elem<T>::acc;
  using C = RowsCfg<A, RT, DC>;
  constexpr int kNC = C::kBwdNC, kCols = C::kBwdCols, kBufs = C::kBufs;
  __shared__ A s_lse2[kBufs][kCols], s_delta[kBufs][kCols];
  const ts_attn_params& p = a.bp.fwd;
  A* k = reinterpret_cast<A*>(smem_raw);
  A* v = k + C::kRows * C::kStride;
  A* tiles = v + C::kRows * C::kStride;  // Q and dO, kBufs times
  A* wp = tiles + 2 * kBufs * kCols * C::kStride;
  A* ws = wp + C::kRows * (kCols + kRowsPad);
  const RowsWindow rule{p, a.win};
  const int ty = threadIdx.x / 8, tx = threadIdx.x % 8;
  const int heads = p.kv_heads * p.batch, bh = index % heads, hk = bh % p.kv_heads, b = bh / p.kv_heads;
  const int first_others = blocks.with_sinks.count * blocks.with_sinks.parts;
  int local = index / heads;
  const RowsKeySet& set = local < first_others ? blocks.with_sinks : blocks.others;
  if (local >= first_others) local -= first_others;
  const int part = local / set.count, block = local % set.count, j0 = (set.first + block) * C::kRows;
  const int kv_end = rule.kv_end(b), rep = p.q_heads / p.kv_heads;
  const int64_t offset = rule.offset(b);
  stage_tile<T, A>(k, C::kStride, p.k, b, hk, j0, C::kRows, kv_end, p.head_dim);
  stage_tile<T, A>(v, C::kStride, p.v, b, hk, j0, C::kRows, kv_end, p.value_dim);
  A dk[RT][DC][4], dv[RT][DC][4];
  clear(dk);
  clear(dv);
  const A scale = (A)p.scale, scale2 = (A)(p.scale * kLog2eD);
  // Queries that see some of the block's keys, and this part's of them.
  const int64_t first = i64min(p.q_len, i64max(0, j0 - offset) / kCols * kCols);
  int64_t stop = p.q_len;
  if (j0 >= a.win.sinks) stop = i64min(stop, (int64_t)min(j0 + C::kRows, kv_end) - 1 - offset + a.win.window);
  if (j0 >= kv_end) stop = 0;
  const int tiles_a_head = first < stop ? (int)((stop - first + kCols - 1) / kCols) : 0;
  const int64_t all = (int64_t)rep * tiles_a_head, it0 = part * all / set.parts;
  const int n = (int)((part + 1) * all / set.parts - it0);
  auto stage = [&](int it) {
    const int h = hk * rep + (int)((it0 + it) / tiles_a_head), i0 = (int)(first + (it0 + it) % tiles_a_head * kCols);
    A* q = tiles + it % kBufs * 2 * kCols * C::kStride;
    stage_tile<T, A>(q, C::kStride, p.q, b, h, i0, kCols, p.q_len, p.head_dim);
    stage_tile<T, A>(q + kCols * C::kStride, C::kStride, a.bp.dout, b, h, i0, kCols, p.q_len, p.value_dim);
    if (threadIdx.x < kCols) {
      const int i = i0 + threadIdx.x;
      s_lse2[it % kBufs][threadIdx.x] = i < p.q_len ? row_lse2<A>(p, b, h, i) : -neg_inf<A>();
      s_delta[it % kBufs][threadIdx.x] =
          i < p.q_len ? reinterpret_cast<const A*>(a.delta)[((int64_t)b * p.q_heads + h) * p.q_len + i] : A(0);
    }
  };
  if (n > 0) stage(0);
  for (int it = 0; it < n; ++it) {
    const int i0 = (int)(first + (it0 + it) % tiles_a_head * kCols);
    const A *q = tiles + it % kBufs * 2 * kCols * C::kStride, *g = q + kCols * C::kStride;
    const A *lse2 = s_lse2[it % kBufs], *delta = s_delta[it % kBufs];
    ptx::copies_done();
    __syncthreads();  // this tile is there, the one before is used up
    if (kBufs > 1 && it + 1 < n) stage(it + 1);
    A s[RT][kNC], d[RT][kNC];
    dots<RT, kNC>(s, k, q, C::kStride, p.head_dim, ty, tx);
    dots<RT, kNC>(d, v, g, C::kStride, p.value_dim, ty, tx);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int key = j0 + ty + 16 * r;
      const int64_t from = key - offset;  // the first query that sees it
      const uint32_t see =
          key >= kv_end ? 0u
                        : range_bits(from, key < a.win.sinks ? p.q_len : i64min(p.q_len, from + a.win.window), i0);
#pragma unroll
      for (int c = 0; c < kNC; ++c) {
        const int col = tx + 8 * c;
        const A pr = (see >> col) & 1u ? acc_exp2(s[r][c] * scale2 - lse2[col]) : A(0);
        wp[(ty + 16 * r) * (kCols + kRowsPad) + col] = pr;
        ws[(ty + 16 * r) * (kCols + kRowsPad) + col] = pr * (d[r][c] - delta[col]) * scale;
      }
    }
    __syncwarp();  // a row's weights are written and read by one warp
    accumulate<RT, kNC, DC>(dv, wp, g, C::kStride, ty, tx);
    accumulate<RT, kNC, DC>(dk, ws, q, C::kStride, ty, tx);
    if (kBufs == 1 && it + 1 < n) {
      __syncthreads();
      stage(it + 1);
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int key = j0 + ty + 16 * r;
    if (key >= p.kv_len) continue;
    if (set.parts > 1) {
      // [part][row and head][row of the blocks][channels of K, of V]
      A* out = reinterpret_cast<A*>(set.part) +
               (((int64_t)part * heads + bh) * set.count * C::kRows + block * C::kRows + ty + 16 * r) *
                   (p.head_dim + p.value_dim);
#pragma unroll
      for (int c = 0; c < DC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int ch = 4 * (tx + 8 * c) + e;
          if (ch < p.head_dim) out[ch] = dk[r][c][e];
          if (ch < p.value_dim) out[p.head_dim + ch] = dv[r][c][e];
        }
      continue;
    }
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int ch = 4 * (tx + 8 * c) + e;
        if (ch < p.head_dim) *at4w<T>(a.bp.dk, b, hk, key, ch) = Elem<T>::from_acc(dk[r][c][e]);
        if (ch < p.value_dim) *at4w<T>(a.bp.dv, b, hk, key, ch) = Elem<T>::from_acc(dv[r][c][e]);
      }
  }
}

// Both in one launch, dK and dV first (a pair costs them four products, dQ three): small calls keep the SMs busy with
// either, and larger ones have one tail.  In launches one behind the other (dQ, blocks with sinks, other blocks) the
// last example above took 156 us with its forward, then 107; 2 x 2000 queries 1829, then 1402.
template <typename T, int RTQ, int RTK, int DC>
__global__ void __launch_bounds__(kRowsThreads)
    rows_window_bwd_kernel(const __grid_constant__ RowsWindowBwd a, const __grid_constant__ RowsKeyBlocks blocks, int dkv_blocks) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  wait_for_previous();
  let_next_start();
  if ((int)blockIdx.x < dkv_blocks)
    rows_window_dkv<T, RTK, DC>(a, blocks, smem_raw, blockIdx.x);
  else
    rows_window_dq<T, RTQ, DC>(a, smem_raw, blockIdx.x - dkv_blocks);
}

// dK and dV of the divided blocks' keys from their parts, one thread a channel of a key.
template <typename T>
__global__ void __launch_bounds__(256)
    rows_dkv_sum_kernel(const __grid_constant__ RowsWindowBwd a, const __grid_constant__ RowsKeyBlocks blocks, int rows) {
  using A = typename Elem<T>::acc;
  const ts_attn_params& p = a.bp.fwd;
  wait_for_previous();
  let_next_start();
  const int wide = p.head_dim + p.value_dim;
  const int64_t heads = (int64_t)p.kv_heads * p.batch;
  const int64_t first_others = blocks.with_sinks.parts > 1 ? heads * blocks.with_sinks.count * rows * wide : 0;
  int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const RowsKeySet& set = x < first_others ? blocks.with_sinks : blocks.others;
  if (x >= first_others) x -= first_others;
  const int keys = set.count * rows;
  if (set.parts <= 1 || x >= heads * keys * wide) return;
  const int ch = (int)(x % wide), local = (int)(x / wide % keys), bh = (int)(x / wide / keys);
  const int key = set.first * rows + local;
  if (key >= p.kv_len) return;
  const A* part = reinterpret_cast<const A*>(set.part) + x;
  A sum = A(0);
#pragma unroll 8
  for (int z = 0; z < set.parts; ++z) sum += part[z * heads * keys * wide];
  const ts_view4& out = ch < p.head_dim ? a.bp.dk : a.bp.dv;
  *at4w<T>(out, bh / p.kv_heads, bh % p.kv_heads, key, ch < p.head_dim ? ch : ch - p.head_dim) = Elem<T>::from_acc(sum);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
template <typename K, typename... Args>
cudaError_t launch_rows(K kernel, dim3 grid, size_t smem, cudaStream_t st, const Args&... a) {
  const cudaError_t e = ensure_max_smem(reinterpret_cast<const void*>(kernel), (int)smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(kernel, grid, dim3(kRowsThreads), smem, st, a...);
}

template <typename T, int RT, int DC>
cudaError_t rows_window_fwd_t(const RowsWindow& a, cudaStream_t st) {
  using C = RowsCfg<typename Elem<T>::acc, RT, DC>;
  const dim3 grid(ceil_div(a.p.q_len, C::kRows), a.p.q_heads, a.p.batch);
  return launch_rows(rows_window_fwd_kernel<T, RT, DC>, grid, C::kFwdSmem, st, a);
}

// The key blocks with sinks, which all the queries behind them see, and the others, each divided into as many blocks as
// the SMs hold at a time (and at most 64 parts): more of them cost more in copies of K and V and in sums that are written
// and read once more than they even out (1000 queries, 4 heads of 128, a window of 300, 100 sinks, gradients: 295 us,
// 342 with twice as many; 202 queries of 24 heads on 3 behind 501 keys 124 against 113).  Under a window of half the
// queries or more the blocks' lengths differ, and three times as many even them out (2 x 2000 queries, 8 heads on 4 of
// 64, no narrower window: 1396 us, 1511 undivided).
template <typename A>
RowsKeyBlocks rows_key_blocks(const ts_attn_params& p, const WindowArgs& win, int rows, int cols, unsigned char* ws,
                              size_t* bytes) {
  const int blocks = ceil_div(p.kv_len, rows), with_sinks = ceil_div(min(win.sinks, p.kv_len), rows);
  const int64_t heads = (int64_t)p.kv_heads * p.batch;
  const int64_t want = (win.window < p.q_len / 2 ? 2 : 6) * (int64_t)device_sms();
  *bytes = 0;
  auto divide = [&](int first, int count, int64_t seen) {
    RowsKeySet s{first, count, 0, nullptr};
    if (count == 0) return s;
    const int64_t tiles = p.q_heads / p.kv_heads * ((seen + cols - 1) / cols);
    s.parts = (int)i64max(1, i64min(i64min(64, tiles), want / i64max(1, heads * count)));
    s.part = ws ? ws + *bytes : nullptr;
    if (s.parts > 1) *bytes += sizeof(A) * (size_t)s.parts * heads * count * rows * (p.head_dim + p.value_dim);
    return s;
  };
  RowsKeyBlocks made;
  made.with_sinks = divide(0, with_sinks, p.q_len);
  made.others = divide(with_sinks, blocks - with_sinks, i64min(p.q_len, (int64_t)win.window + rows + cols));
  return made;
}

// ws null: the workspace's bytes alone.  It holds the deltas, then the parts of dK and dV.
template <typename T, int RTQ, int RTK, int DC>
cudaError_t rows_window_bwd_t(const ts_attn_bwd_params& bp, const WindowArgs& win, size_t* bytes, void* ws, cudaStream_t st) {
  using A = typename Elem<T>::acc;
  using CQ = RowsCfg<A, RTQ, DC>;
  using CK = RowsCfg<A, RTK, DC>;
  const ts_attn_params& p = bp.fwd;
  const int64_t heads = (int64_t)p.kv_heads * p.batch, q_rows = (int64_t)p.batch * p.q_heads * p.q_len;
  const size_t delta = (sizeof(A) * (size_t)q_rows + 255) / 256 * 256;
  const RowsKeyBlocks blocks =
      rows_key_blocks<A>(p, win, CK::kRows, CK::kBwdCols, ws ? reinterpret_cast<unsigned char*>(ws) + delta : nullptr, bytes);
  *bytes += delta;
  if (!ws) return cudaSuccess;
  const RowsWindowBwd a{bp, win, ws};
  cudaError_t e = launch_dependent(rows_delta_kernel<T>, dim3((unsigned)((q_rows * 32 + 255) / 256)), dim3(256), 0, st, bp,
                                   reinterpret_cast<A*>(ws));
  if (e != cudaSuccess) return e;
  const RowsKeySet &s = blocks.with_sinks, &o = blocks.others;
  const int64_t dkv = heads * ((int64_t)s.count * s.parts + (int64_t)o.count * o.parts);
  const int64_t dq = (int64_t)p.batch * p.q_heads * ceil_div(p.q_len, CQ::kRows);
  if (dkv + dq > 0x7fffffff) return cudaErrorInvalidConfiguration;
  e = launch_rows(rows_window_bwd_kernel<T, RTQ, RTK, DC>, dim3((unsigned)(dkv + dq)), std::max(CQ::kBwdSmem, CK::kBwdSmem),
                  st, a, blocks, (int)dkv);
  const int64_t divided = (s.parts > 1 ? s.count : 0) + (o.parts > 1 ? o.count : 0);
  if (e != cudaSuccess || divided == 0) return e;
  return launch_dependent(rows_dkv_sum_kernel<T>,
                          dim3((unsigned)((heads * divided * CK::kRows * (p.head_dim + p.value_dim) + 255) / 256)),
                          dim3(256), 0, st, a, blocks, (int)CK::kRows);
}

template <typename T, int RT, int DC>
cudaError_t rows_tree_t(TreeArgs& a, cudaStream_t st) {
  using A = typename Elem<T>::acc;
  using C = RowsCfg<A, RT, DC>;
  const unsigned grid = sizeof(A) == 4 ? (unsigned)a.ctas : (unsigned)(a.p.batch * a.p.kv_heads * a.row_tiles);
  const cudaError_t e = launch_rows(rows_tree_kernel<T, RT, DC>, dim3(grid), C::kFwdSmem, st, a);
  if (e != cudaSuccess || sizeof(A) == 8) return e;
  return tree_merge(a, C::kFwdCols, 0, st);
}

template <typename T, int DC>
cudaError_t rows_window_fwd_d(const RowsWindow& a, cudaStream_t st) {
  using A = typename Elem<T>::acc;
  const int rt = rows_rt(a.p.q_len, (int64_t)a.p.q_heads * a.p.batch, sizeof(A) == 8 ? (DC <= 4 ? 2 : 1) : rows_widest(32 * DC));
  if constexpr (sizeof(A) == 4 && DC == 2)
    if (rt == 4) return rows_window_fwd_t<T, 4, DC>(a, st);
  if constexpr (sizeof(A) == 4 || DC <= 4)
    if (rt == 2) return rows_window_fwd_t<T, 2, DC>(a, st);
  return rows_window_fwd_t<T, 1, DC>(a, st);
}

// Key blocks are divided along the queries, so they may be wide whatever their number.
template <typename T, int DC>
cudaError_t rows_window_bwd_d(const ts_attn_bwd_params& bp, const WindowArgs& win, size_t* bytes, void* ws, cudaStream_t st) {
  using A = typename Elem<T>::acc;
  const ts_attn_params& p = bp.fwd;
  constexpr int kMost = sizeof(A) == 8 ? 1 : DC == 2 ? 4 : DC == 4 ? 2 : 1;  // row tiles that the registers hold
  if constexpr (kMost > 1) {
    if (p.kv_len <= 16) return rows_window_bwd_t<T, 1, 1, DC>(bp, win, bytes, ws, st);
    const int rt = rows_rt(p.q_len, (int64_t)p.q_heads * p.batch, kMost);
    if constexpr (kMost == 4)
      if (rt == 4) return rows_window_bwd_t<T, 4, kMost, DC>(bp, win, bytes, ws, st);
    if (rt == 2) return rows_window_bwd_t<T, 2, kMost, DC>(bp, win, bytes, ws, st);
  }
  return rows_window_bwd_t<T, 1, kMost, DC>(bp, win, bytes, ws, st);
}

template <typename T, int DC>
int rows_tree_rt(const ts_attn_params& p) {
  using A = typename Elem<T>::acc;
  const int rows = p.q_heads / p.kv_heads * p.q_len;
  int rt = sizeof(A) == 8 ? 1 : (DC <= 4 ? 4 : 2);
  while (rt > 1 && rows <= 8 * rt) rt >>= 1;
  return rt;
}

inline int rows_tree_dc(const ts_attn_params& p) {
  const int d = max(p.head_dim, p.value_dim);
  return d <= 64 ? 2 : d <= 128 ? 4 : 8;
}

template <typename T, int DC>
cudaError_t rows_tree_d(const ts_attn_params& p, TreeArgs* a, size_t* bytes, void* workspace, cudaStream_t st) {
  const int rt = rows_tree_rt<T, DC>(p);
  TreeArgs made = tree_args(p, 16 * rt, 2 * device_sms(), bytes);
  if (!a) return cudaSuccess;  // the workspace's size alone
  made.parents = a->parents;
  made.parents_stride = a->parents_stride;
  made.win = a->win;
  tree_place(&made, workspace);
  if constexpr (sizeof(typename Elem<T>::acc) == 4) {
    if constexpr (DC <= 4)
      if (rt == 4) return rows_tree_t<T, 4, DC>(made, st);
    if (rt == 2) return rows_tree_t<T, 2, DC>(made, st);
  }
  return rows_tree_t<T, 1, DC>(made, st);
}

template <typename T>
cudaError_t rows_window_fwd_dispatch(const RowsWindow& a, cudaStream_t st) {
  switch (rows_tree_dc(a.p)) {
    case 2: return rows_window_fwd_d<T, 2>(a, st);
    case 4: return rows_window_fwd_d<T, 4>(a, st);
  }
  return rows_window_fwd_d<T, 8>(a, st);
}

template <typename T>
cudaError_t rows_window_bwd_dispatch(const ts_attn_bwd_params& bp, const WindowArgs& win, size_t* bytes, void* ws,
                                     cudaStream_t st) {
  switch (rows_tree_dc(bp.fwd)) {
    case 2: return rows_window_bwd_d<T, 2>(bp, win, bytes, ws, st);
    case 4: return rows_window_bwd_d<T, 4>(bp, win, bytes, ws, st);
  }
  return rows_window_bwd_d<T, 8>(bp, win, bytes, ws, st);
}

template <typename T>
cudaError_t rows_tree_dispatch(const ts_attn_params& p, TreeArgs* a, size_t* bytes, void* ws, cudaStream_t st) {
  switch (rows_tree_dc(p)) {
    case 2: return rows_tree_d<T, 2>(p, a, bytes, ws, st);
    case 4: return rows_tree_d<T, 4>(p, a, bytes, ws, st);
  }
  return rows_tree_d<T, 8>(p, a, bytes, ws, st);
}

#define TS_ROWS_INSTANTIATE(suffix, T)                                                                           \
  cudaError_t rows_window_fwd_##suffix(const RowsWindow& a, cudaStream_t st) {                                   \
    return rows_window_fwd_dispatch<T>(a, st);                                                                   \
  }                                                                                                              \
  cudaError_t rows_window_bwd_##suffix(const ts_attn_bwd_params& bp, const WindowArgs& win, size_t* bytes,       \
                                       void* ws, cudaStream_t st) {                                              \
    return rows_window_bwd_dispatch<T>(bp, win, bytes, ws, st);                                                  \
  }                                                                                                              \
  cudaError_t rows_tree_##suffix(const ts_attn_params& p, TreeArgs* a, size_t* bytes, void* ws, cudaStream_t st) { \
    return rows_tree_dispatch<T>(p, a, bytes, ws, st);                                                           \
  }

}  // namespace tsa
