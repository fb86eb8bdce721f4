// CUDA-core attention for the sliding window with sinks (forward and backward) and for drafted tokens over a
// cache: fp32 and fp64, and the half-type problems that the tensor-core kernels leave (head dimensions above 128 or
// not a multiple of 8, Dv != D, strides that TMA cannot address, a scale that is not positive).
//
// A block of 128 threads holds R = 16 RT rows and walks over tiles of 32 columns, both in shared memory.  Thread
// (ty, tx) owns rows ty + 16 r and columns tx + 8 k of the products, and channels 4 (tx + 8 c) of the accumulators, so
// that RT + 4 (products) and RT + DC (accumulators) 16-byte reads feed 16 RT and 4 RT DC multiply-adds.  The arithmetic
// is exact in the accumulation type (fp32, or fp64 for fp64), exponentials in base 2.
// Which columns a row sees is one 32-bit word a row and tile (tree.cuh, window.cuh).
#pragma once
#include "dependent.cuh"
#include "simt_kernels.cuh"
#include "tc_util.cuh"
#include "rows.cuh"

namespace tsa {

constexpr int kRowsThreads = 128, kRowsCols = 32, kRowsPad = 4;
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

// Rows [t0, t0 + rows) of (b, h) into shared memory, a row every `stride` elements; zeros at and behind row `end` and
// channel C (to a whole quad).
template <typename T, typename A>
__device__ __forceinline__ void stage_tile(A* dst, int stride, const ts_view4& src, int b, int h, int64_t t0, int rows,
                                           int64_t end, int C) {
  constexpr int kVec = 16 / sizeof(T);
  const T* base = reinterpret_cast<const T*>(src.data) + (int64_t)b * src.stride[0] + (int64_t)h * src.stride[1];
  const bool vec = src.stride[3] == 1 && C % kVec == 0 && (src.stride[2] * sizeof(T)) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(base) % 16 == 0;
  if (vec) {
    const int per = C / kVec, n = rows * per;
    constexpr int kBatch = 4;
    for (int x0 = threadIdx.x; x0 < n; x0 += kRowsThreads * kBatch) {
      uint4 raw[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int x = x0 + u * kRowsThreads, r = x / per, c = x % per;
        raw[u] = make_uint4(0u, 0u, 0u, 0u);
        if (x < n && t0 + r < end) raw[u] = *reinterpret_cast<const uint4*>(base + (t0 + r) * src.stride[2] + c * kVec);
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
  const int wide = ceil_div(C, 4) * 4;
  for (int x = threadIdx.x; x < rows * wide; x += kRowsThreads) {
    const int r = x / wide, c = x % wide;
    dst[r * stride + c] = c < C && t0 + r < end ? Elem<T>::to_acc(base[(t0 + r) * src.stride[2] + c * src.stride[3]])
                                                : A(0);
  }
}

// Rows [r0, r0 + rows) of the packed rows (head h0 + r / tokens, token r % tokens), r < end.
template <typename T, typename A>
__device__ __forceinline__ void stage_packed(A* dst, int stride, const ts_view4& src, int b, int h0, int r0, int rows,
                                             int end, int tokens, int C) {
  constexpr int kVec = 16 / sizeof(T), kBatch = 4;
  const T* base = reinterpret_cast<const T*>(src.data) + (int64_t)b * src.stride[0];
  auto row_at = [&](int r) { return base + (int64_t)(h0 + r / tokens) * src.stride[1] + (int64_t)(r % tokens) * src.stride[2]; };
  const bool vec = src.stride[3] == 1 && C % kVec == 0 && (src.stride[2] * sizeof(T)) % 16 == 0 &&
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
template <int RT, typename A>
__device__ __forceinline__ void dots(A (&acc)[RT][4], const A* rows, const A* cols, int stride, int C, int ty, int tx) {
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[r][k] = A(0);
#pragma unroll 2
  for (int c = 0; c < C; c += 4) {
    Quad<A> a[RT], b[4];
#pragma unroll
    for (int r = 0; r < RT; ++r) a[r] = quad(rows + (ty + 16 * r) * stride + c);
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = quad(cols + (tx + 8 * k) * stride + c);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][k] += a[r].v[e] * b[k].v[e];
  }
}

// acc[r][c] += sum_j w[ty + 16 r][j] cols[j][4 (tx + 8 c) ..]; w has kRowsCols + kRowsPad elements a row.
template <int RT, int DC, typename A>
__device__ __forceinline__ void accumulate(A (&acc)[RT][DC][4], const A* w, const A* cols, int stride, int ty, int tx) {
#pragma unroll 2
  for (int j = 0; j < kRowsCols; j += 4) {
    Quad<A> p[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) p[r] = quad(w + (ty + 16 * r) * (kRowsCols + kRowsPad) + j);
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
  static constexpr size_t kFwdSmem = sizeof(A) * ((kRows + 2 * kRowsCols) * kStride + kRows * (kRowsCols + kRowsPad));
  // rows' two operands, the tile's two, P and dS
  static constexpr size_t kBwdSmem =
      sizeof(A) * ((2 * kRows + 2 * kRowsCols) * kStride + 2 * kRows * (kRowsCols + kRowsPad));
};

// The running softmax of R rows over tiles of keys.
template <typename T, int RT, int DC> struct RowsForward {
  using A = typename Elem<T>::acc;
  using C = RowsCfg<A, RT, DC>;
  A acc[RT][DC][4], m[RT], l[RT];
  A *q, *k, *v, *w;
  int ty, tx;

  __device__ __forceinline__ RowsForward(A* smem) {
    q = smem;
    k = q + C::kRows * C::kStride;
    v = k + kRowsCols * C::kStride;
    w = v + kRowsCols * C::kStride;
    ty = threadIdx.x / 8;
    tx = threadIdx.x % 8;
  }
  __device__ __forceinline__ void start() {
    clear(acc);
#pragma unroll
    for (int r = 0; r < RT; ++r) m[r] = neg_inf<A>(), l[r] = A(0);
  }
  // Keys [k0, k0 + 32) of head hk; bits[r]: what row ty + 16 r sees of them.  Keys at and behind `end` are not read.
  template <typename Bits>
  __device__ __forceinline__ void tile(const ts_attn_params& p, int b, int hk, int k0, int end, A scale2, Bits bits) {
    __syncthreads();  // the tile before is used up
    stage_tile<T, A>(k, C::kStride, p.k, b, hk, k0, kRowsCols, end, p.head_dim);
    stage_tile<T, A>(v, C::kStride, p.v, b, hk, k0, kRowsCols, end, p.value_dim);
    __syncthreads();
    A s[RT][4];
    dots<RT>(s, q, k, C::kStride, p.head_dim, ty, tx);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const uint32_t see = bits(r);
      A top = neg_inf<A>();
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[r][c] = (see >> (tx + 8 * c)) & 1u ? s[r][c] * scale2 : neg_inf<A>();
        top = s[r][c] > top ? s[r][c] : top;
      }
      top = lanes8_max(top);
      const A next = top > m[r] ? top : m[r];
      const A safe = next == neg_inf<A>() ? A(0) : next;
      const A factor = acc_exp2(m[r] - safe);
      A sum = A(0);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const A e = acc_exp2(s[r][c] - safe);
        w[(ty + 16 * r) * (kRowsCols + kRowsPad) + tx + 8 * c] = e;
        sum += e;
      }
      l[r] = l[r] * factor + lanes8_sum(sum);
      m[r] = next;
#pragma unroll
      for (int c = 0; c < DC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][c][e] *= factor;
    }
    __syncwarp();  // a row's weights are written and read by one warp
    accumulate<RT, DC>(acc, w, v, C::kStride, ty, tx);
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
  const int i0 = blockIdx.x * F::C::kRows;
  const int kv_end = a.kv_end(b);
  const int64_t offset = a.offset(b);
  stage_tile<T, A>(f.q, F::C::kStride, p.q, b, h, i0, F::C::kRows, p.q_len, p.head_dim);
  f.start();
  const int64_t last = (int64_t)min(i0 + F::C::kRows, p.q_len) - 1 + offset;
  const int end = (int)i64max(0, i64min(kv_end, last + 1));
  const WindowTiles wt(a.win, i0 + offset, kv_end, kRowsCols);
  const int n = wt.count(ceil_div(end, kRowsCols));
  const A scale2 = (A)(p.scale * kLog2eD);
  for (int j = 0; j < n; ++j) {
    const int k0 = wt.tile(j) * kRowsCols;
    f.tile(p, b, hk, k0, kv_end, scale2, [&](int r) {
      const int i = i0 + f.ty + 16 * r;
      if (i >= p.q_len) return 0u;
      const int64_t stop = i64min(kv_end, i + offset + 1);
      return range_bits(i + offset + 1 - a.win.window, stop, k0) | range_bits(0, i64min(stop, a.win.sinks), k0);
    });
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int i = i0 + f.ty + 16 * r;
    if (i >= p.q_len) continue;
    const A inv = f.l[r] > A(0) ? A(1) / f.l[r] : A(0);
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
          f.l[r] > A(0) ? (f.m[r] + acc_log2(f.l[r])) * (A)kLn2D : neg_inf<A>();
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
  const ts_attn_params& p = a.p;
  wait_for_previous();
  let_next_start();
  F f(reinterpret_cast<A*>(smem_raw));
  const TreeLine line(a, kRowsCols, 0);
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
    walk.count = line.tiles(walk.b);
  }
  while (!kSplit || walk.next(line)) {
    const int b = walk.b, hk = walk.unit / a.row_tiles, r0 = walk.unit % a.row_tiles * F::C::kRows;
    const int len = tree_len(p, b);
    const int64_t base = (int64_t)len - p.q_len;
    const WindowTiles wt(a.win, base, len, kRowsCols);
    __syncthreads();  // the unit before is used up
    if (a.parents && (int)threadIdx.x < p.q_len) s_parents[threadIdx.x] = a.parents[b * a.parents_stride + threadIdx.x];
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
    for (int j = 0; j < walk.count; ++j) {
      const int k0 = wt.tile(walk.first + j) * kRowsCols;
      f.tile(p, b, hk, k0, len, scale2, [&](int r) { return view_bits(view[r], base, a.win.sinks, k0); });
    }
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
        const A inv = f.l[r] > A(0) ? A(1) / f.l[r] : A(0);
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
              f.l[r] > A(0) ? (f.m[r] + acc_log2(f.l[r])) * (A)kLn2D : neg_inf<A>();
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

template <typename A>
__device__ __forceinline__ A row_lse2(const ts_attn_params& p, int b, int h, int i) {
  const A v = reinterpret_cast<const A*>(p.lse)[(int64_t)b * p.lse_stride[0] + (int64_t)h * p.lse_stride[1] +
                                                (int64_t)i * p.lse_stride[2]];
  return v == neg_inf<A>() ? -neg_inf<A>() : v * (A)kLog2eD;  // a row that sees nothing: every p is 0
}

template <typename T, int RT, int DC>
__global__ void __launch_bounds__(kRowsThreads) rows_window_dq_kernel(const __grid_constant__ RowsWindowBwd a) {
  using A = typename Elem<T>::acc;
  using C = RowsCfg<A, RT, DC>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const ts_attn_params& p = a.bp.fwd;
  A* q = reinterpret_cast<A*>(smem_raw);
  A* g = q + C::kRows * C::kStride;
  A* k = g + C::kRows * C::kStride;
  A* v = k + kRowsCols * C::kStride;
  A* w = v + kRowsCols * C::kStride;
  wait_for_previous();
  let_next_start();
  const RowsWindow rule{p, a.win};
  const int ty = threadIdx.x / 8, tx = threadIdx.x % 8;
  const int h = blockIdx.y, b = blockIdx.z, hk = h / (p.q_heads / p.kv_heads);
  const int i0 = blockIdx.x * C::kRows;
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
  const WindowTiles wt(a.win, i0 + offset, kv_end, kRowsCols);
  const int n = wt.count(ceil_div(end, kRowsCols));
  const A scale = (A)p.scale, scale2 = (A)(p.scale * kLog2eD);
  for (int j = 0; j < n; ++j) {
    const int k0 = wt.tile(j) * kRowsCols;
    __syncthreads();
    stage_tile<T, A>(k, C::kStride, p.k, b, hk, k0, kRowsCols, kv_end, p.head_dim);
    stage_tile<T, A>(v, C::kStride, p.v, b, hk, k0, kRowsCols, kv_end, p.value_dim);
    __syncthreads();
    A s[RT][4], d[RT][4];
    dots<RT>(s, q, k, C::kStride, p.head_dim, ty, tx);
    dots<RT>(d, g, v, C::kStride, p.value_dim, ty, tx);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int64_t stop = i64min(kv_end, i0 + ty + 16 * r + offset + 1);
      const uint32_t see = range_bits(i0 + ty + 16 * r + offset + 1 - a.win.window, stop, k0) |
                           range_bits(0, i64min(stop, a.win.sinks), k0);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const A pr = (see >> (tx + 8 * c)) & 1u ? acc_exp2(s[r][c] * scale2 - lse2[r]) : A(0);
        w[(ty + 16 * r) * (kRowsCols + kRowsPad) + tx + 8 * c] = pr * (d[r][c] - delta[r]) * scale;
      }
    }
    __syncwarp();
    accumulate<RT, DC>(acc, w, k, C::kStride, ty, tx);
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

template <typename T, int RT, int DC>
__global__ void __launch_bounds__(kRowsThreads) rows_window_dkv_kernel(const __grid_constant__ RowsWindowBwd a) {
  using A = typename Elem<T>::acc;
  using C = RowsCfg<A, RT, DC>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ A s_lse2[kRowsCols], s_delta[kRowsCols];
  const ts_attn_params& p = a.bp.fwd;
  A* k = reinterpret_cast<A*>(smem_raw);
  A* v = k + C::kRows * C::kStride;
  A* q = v + C::kRows * C::kStride;
  A* g = q + kRowsCols * C::kStride;
  A* wp = g + kRowsCols * C::kStride;
  A* ws = wp + C::kRows * (kRowsCols + kRowsPad);
  wait_for_previous();
  let_next_start();
  const RowsWindow rule{p, a.win};
  const int ty = threadIdx.x / 8, tx = threadIdx.x % 8;
  // Blocks of the first keys first: all the queries see the sinks.
  const int hk = blockIdx.x % p.kv_heads, b = blockIdx.x / p.kv_heads, j0 = blockIdx.y * C::kRows;
  const int kv_end = rule.kv_end(b), rep = p.q_heads / p.kv_heads;
  const int64_t offset = rule.offset(b);
  stage_tile<T, A>(k, C::kStride, p.k, b, hk, j0, C::kRows, kv_end, p.head_dim);
  stage_tile<T, A>(v, C::kStride, p.v, b, hk, j0, C::kRows, kv_end, p.value_dim);
  A dk[RT][DC][4], dv[RT][DC][4];
  clear(dk);
  clear(dv);
  const A scale = (A)p.scale, scale2 = (A)(p.scale * kLog2eD);
  // Queries that see some of the block's keys.
  const int first = (int)i64min(p.q_len, i64max(0, j0 - offset) / kRowsCols * kRowsCols);
  int64_t stop = p.q_len;
  if (j0 >= a.win.sinks) stop = i64min(stop, (int64_t)min(j0 + C::kRows, kv_end) - 1 - offset + a.win.window);
  if (j0 >= kv_end) stop = 0;
  for (int h = hk * rep; h < (hk + 1) * rep; ++h)
    for (int i0 = first; i0 < stop; i0 += kRowsCols) {
      __syncthreads();
      stage_tile<T, A>(q, C::kStride, p.q, b, h, i0, kRowsCols, p.q_len, p.head_dim);
      stage_tile<T, A>(g, C::kStride, a.bp.dout, b, h, i0, kRowsCols, p.q_len, p.value_dim);
      if (threadIdx.x < kRowsCols) {
        const int i = i0 + threadIdx.x;
        s_lse2[threadIdx.x] = i < p.q_len ? row_lse2<A>(p, b, h, i) : -neg_inf<A>();
        s_delta[threadIdx.x] =
            i < p.q_len ? reinterpret_cast<const A*>(a.delta)[((int64_t)b * p.q_heads + h) * p.q_len + i] : A(0);
      }
      __syncthreads();
      A s[RT][4], d[RT][4];
      dots<RT>(s, k, q, C::kStride, p.head_dim, ty, tx);
      dots<RT>(d, v, g, C::kStride, p.value_dim, ty, tx);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int key = j0 + ty + 16 * r;
        const int64_t from = key - offset;  // the first query that sees it
        const uint32_t see = key >= kv_end ? 0u
                                           : range_bits(from, key < a.win.sinks ? p.q_len
                                                                                : i64min(p.q_len, from + a.win.window), i0);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int col = tx + 8 * c;
          const A pr = (see >> col) & 1u ? acc_exp2(s[r][c] * scale2 - s_lse2[col]) : A(0);
          wp[(ty + 16 * r) * (kRowsCols + kRowsPad) + col] = pr;
          ws[(ty + 16 * r) * (kRowsCols + kRowsPad) + col] = pr * (d[r][c] - s_delta[col]) * scale;
        }
      }
      __syncwarp();
      accumulate<RT, DC>(dv, wp, g, C::kStride, ty, tx);
      accumulate<RT, DC>(dk, ws, q, C::kStride, ty, tx);
    }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int key = j0 + ty + 16 * r;
    if (key >= p.kv_len) continue;
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

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
template <typename K, typename Args>
cudaError_t launch_rows(K kernel, dim3 grid, size_t smem, cudaStream_t st, const Args& a) {
  const cudaError_t e = ensure_max_smem(reinterpret_cast<const void*>(kernel), (int)smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(kernel, grid, dim3(kRowsThreads), smem, st, a);
}

// Row tiles of a block: the widest that the registers and shared memory hold, narrower while `rows` rows in `slices`
// grids leave SMs without two blocks.
template <typename A, int DC> int rows_rt(int rows, int64_t slices, int widest) {
  int rt = sizeof(A) == 8 ? (DC <= 4 ? 2 : 1) : (DC <= 4 ? 4 : 2);
  rt = min(rt, widest);
  while (rt > 1 && (rows <= 8 * rt || ceil_div(rows, 16 * rt) * slices < 2 * device_sms())) rt >>= 1;
  return rt;
}

template <typename T, int RT, int DC>
cudaError_t rows_window_fwd_t(const RowsWindow& a, cudaStream_t st) {
  using C = RowsCfg<typename Elem<T>::acc, RT, DC>;
  const dim3 grid(ceil_div(a.p.q_len, C::kRows), a.p.q_heads, a.p.batch);
  return launch_rows(rows_window_fwd_kernel<T, RT, DC>, grid, C::kFwdSmem, st, a);
}

template <typename T, int RT, int DC>
cudaError_t rows_window_bwd_t(const RowsWindowBwd& a, cudaStream_t st) {
  using C = RowsCfg<typename Elem<T>::acc, RT, DC>;
  const ts_attn_params& p = a.bp.fwd;
  const dim3 dq(ceil_div(p.q_len, C::kRows), p.q_heads, p.batch), dkv(p.kv_heads * p.batch, ceil_div(p.kv_len, C::kRows));
  const cudaError_t e = launch_rows(rows_window_dq_kernel<T, RT, DC>, dq, C::kBwdSmem, st, a);
  if (e != cudaSuccess) return e;
  return launch_rows(rows_window_dkv_kernel<T, RT, DC>, dkv, C::kBwdSmem, st, a);
}

template <typename T, int RT, int DC>
cudaError_t rows_tree_t(TreeArgs& a, cudaStream_t st) {
  using A = typename Elem<T>::acc;
  using C = RowsCfg<A, RT, DC>;
  const unsigned grid = sizeof(A) == 4 ? (unsigned)a.ctas : (unsigned)(a.p.batch * a.p.kv_heads * a.row_tiles);
  const cudaError_t e = launch_rows(rows_tree_kernel<T, RT, DC>, dim3(grid), C::kFwdSmem, st, a);
  if (e != cudaSuccess || sizeof(A) == 8) return e;
  return tree_merge(a, kRowsCols, 0, st);
}

template <typename T, int DC>
cudaError_t rows_window_fwd_d(const RowsWindow& a, cudaStream_t st) {
  using A = typename Elem<T>::acc;
  const int rt = rows_rt<A, DC>(a.p.q_len, (int64_t)a.p.q_heads * a.p.batch, 4);
  if constexpr (sizeof(A) == 4 && DC <= 4)
    if (rt == 4) return rows_window_fwd_t<T, 4, DC>(a, st);
  if constexpr (sizeof(A) == 4 || DC <= 4)
    if (rt == 2) return rows_window_fwd_t<T, 2, DC>(a, st);
  return rows_window_fwd_t<T, 1, DC>(a, st);
}

template <typename T, int DC>
cudaError_t rows_window_bwd_d(const RowsWindowBwd& a, cudaStream_t st) {
  using A = typename Elem<T>::acc;
  const ts_attn_params& p = a.bp.fwd;
  const int rt = rows_rt<A, DC>(min(p.q_len, p.kv_len), (int64_t)p.kv_heads * p.batch, DC <= 4 && sizeof(A) == 4 ? 2 : 1);
  if constexpr (sizeof(A) == 4 && DC <= 4)
    if (rt == 2) return rows_window_bwd_t<T, 2, DC>(a, st);
  return rows_window_bwd_t<T, 1, DC>(a, st);
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
cudaError_t rows_window_bwd_dispatch(const ts_attn_bwd_params& bp, const WindowArgs& win, void* ws, cudaStream_t st) {
  using A = typename Elem<T>::acc;
  const ts_attn_params& p = bp.fwd;
  const int64_t rows = (int64_t)p.batch * p.q_heads * p.q_len;
  const cudaError_t e = launch_dependent(rows_delta_kernel<T>, dim3((unsigned)((rows * 32 + 255) / 256)), dim3(256), 0,
                                         st, bp, reinterpret_cast<A*>(ws));
  if (e != cudaSuccess) return e;
  const RowsWindowBwd a{bp, win, ws};
  switch (rows_tree_dc(p)) {
    case 2: return rows_window_bwd_d<T, 2>(a, st);
    case 4: return rows_window_bwd_d<T, 4>(a, st);
  }
  return rows_window_bwd_d<T, 8>(a, st);
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
  cudaError_t rows_window_bwd_##suffix(const ts_attn_bwd_params& bp, const WindowArgs& win, void* ws,            \
                                       cudaStream_t st) {                                                        \
    return rows_window_bwd_dispatch<T>(bp, win, ws, st);                                                         \
  }                                                                                                              \
  cudaError_t rows_tree_##suffix(const ts_attn_params& p, TreeArgs* a, size_t* bytes, void* ws, cudaStream_t st) { \
    return rows_tree_dispatch<T>(p, a, bytes, ws, st);                                                           \
  }

}  // namespace tsa
