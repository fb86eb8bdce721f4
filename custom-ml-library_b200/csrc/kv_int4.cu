// Quantising append into the pages of a 4-bit KV cache, and the read-back of its values.
// Both move each value once: 16 bits in and 4.5 out (the append), 4.5 in and 16 out (the gather),
// so HBM should bound them: 8 rows x 2047 tokens, 8 heads, D = 128, bf16, move 86 MB each, 13 us.  Instructions do: the
// append takes 27 us there (131 a stored word, 63 % of the issue slots; fp16 26, fp32 with its divisions 44 for 153 MB),
// the read-back 19.5 (100 and 68 %; fp32 40).  One token of 64 rows takes the launch, 2.4 us.
//
// One thread owns a stored word (8 channels of K or V of one head) and walks over a block's tokens, four of
// them in flight: 64 bytes a thread for half types, which is what covers the memory latency.  The four
// neighbouring threads of a scale group share its maximum by two shuffles.
#include "dependent.cuh"
#include "int4.cuh"
#include "ptx.cuh"

namespace tsa {

struct Int4Rows {
  ts_kv4_cache c;
  ts_view4 key, value;
  int steps;
  int64_t position;
  const int32_t* positions;
  int32_t* positions_out;
  const int32_t* lens;
  int tile;  // of the read-back: tokens past the tile that a row ends in are left alone, 0: none are
  uint32_t* fault;
  bool vec;          // unit channel stride, 16-byte aligned rows
  int page_log2;
  int tokens;        // of a block
  int token_blocks;  // blocks of a row
};

constexpr int kInFlight = 4;

template <typename T>
struct Raw8 {
  alignas(16) T x[8];
};

template <typename T>
__device__ __forceinline__ void load8(const T* src, int64_t stride, bool vec, Raw8<T>& r) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i)
      reinterpret_cast<uint4*>(r.x)[i] = reinterpret_cast<const uint4*>(src)[i];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) r.x[e] = src[e * stride];
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* dst, int64_t stride, bool vec, const Raw8<T>& r) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i)
      reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(r.x)[i];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) dst[e * stride] = r.x[e];
  }
}

__device__ __forceinline__ int sub_sat(int a, int b) {
  int r;
  asm("sub.sat.s32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The larger, or NaN if either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The largest |x| of 8 values, NaN if one is NaN: as pairs where the type allows it.
__device__ __forceinline__ float amax8(const Raw8<float>& r) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max_nan(m, fabsf(r.x[e]));
  return m;
}
__device__ __forceinline__ float amax8(const Raw8<__half>& r) {
  const __half2* p = reinterpret_cast<const __half2*>(r.x);
  const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(p[0]), __habs2(p[1])), __hmax2_nan(__habs2(p[2]), __habs2(p[3])));
  return max_nan(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float amax8(const Raw8<__nv_bfloat16>& r) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(r.x);
  const __nv_bfloat162 m =
      __hmax2_nan(__hmax2_nan(__habs2(p[0]), __habs2(p[1])), __hmax2_nan(__habs2(p[2]), __habs2(p[3])));
  return max_nan(__low2float(m), __high2float(m));
}

// The word of 8 channels whose group has the finite maximum amax <= 7 * kInt4ScaleMax, so that no quotient
// passes 7.  fp32 inputs divide; half types multiply by the reciprocal and correct the quotient once with its
// remainder (Markstein, IBM J. Res. Dev. 34, 1990), which yields the same correctly rounded quotient (checked
// for every scale and every 11-bit value) at a third of the instructions, two values at a time.
template <typename T>
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], float scale) {
  float inv;  // 1 / scale, correctly rounded: one Newton step from the approximation (checked for every scale)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
  inv = fmaf(fmaf(-scale, inv, 1.f), inv, inv);
  const uint64_t inv2 = ptx::f2pack(inv, inv), minus2 = ptx::f2pack(-scale, -scale);
  // Rounding half to even and adding 8 by a sum whose last place is 1: 1.5 * 2^23 + 8.  The eight sums' bits are
  // added up at their nibbles' places; what their common upper bits add is one constant.
  constexpr uint32_t kBits = 0x4B400000u;
  const uint64_t magic2 = ptx::f2pack(12582920.f, 12582920.f);
  uint32_t word = 0;
#pragma unroll
  for (int e = 6; e >= 0; e -= 2) {
    float lo, hi;
    if constexpr (sizeof(T) == 4) {
      lo = __fdiv_rn(x[e], scale) + 12582920.f;
      hi = __fdiv_rn(x[e + 1], scale) + 12582920.f;
    } else {
      const uint64_t v = ptx::f2pack(x[e], x[e + 1]);
      uint64_t n = ptx::fma2(v, inv2, 0ull);
      n = ptx::fma2(ptx::fma2(n, minus2, v), inv2, n);
      ptx::f2unpack(ptx::add2(n, magic2), lo, hi);
    }
    word = (word * 16u + __float_as_uint(hi)) * 16u + __float_as_uint(lo);
  }
  return word - kBits * 0x11111111u;
}

// The blocks of one head and kind that kInFlight tokens from p0 on fall into: two at most, as a page holds more.
struct Span {
  unsigned char *first, *second;  // nullptr: no page
};
__device__ __forceinline__ unsigned char* page_block(const ts_kv4_cache& c, int b, int slot, unsigned char* base) {
  const int page = int4_page(c, b, slot);
  return page < 0 ? nullptr : base + page * c.page_stride;
}
__device__ __forceinline__ Span token_span(const ts_kv4_cache& c, int b, int p0, int log2, unsigned char* base) {
  Span s;
  s.first = page_block(c, b, p0 >> log2, base);
  s.second = (p0 + kInFlight - 1) >> log2 != p0 >> log2 ? page_block(c, b, (p0 >> log2) + 1, base) : s.first;
  return s;
}

template <typename T>
__global__ void kv_append_int4_kernel(const __grid_constant__ Int4Rows a) {
  let_next_start();
  wait_for_previous();
  const ts_kv4_cache& c = a.c;
  const int b = blockIdx.x / a.token_blocks, t0 = (blockIdx.x - b * a.token_blocks) * a.tokens;
  const int t1 = min(a.steps, t0 + a.tokens);
  const int chunks = c.head_dim / 8, groups = c.head_dim / 32;
  const int items = c.kv_heads * 2 * chunks;  // a multiple of 4
  const int i = blockIdx.y * blockDim.x + threadIdx.x;
  const int pos = a.positions ? a.positions[b] : (int)a.position;
  if (t0 == 0 && i == 0 && a.positions_out) a.positions_out[b] = pos + a.steps;
  if (i >= items) return;
  const int chunk = i % chunks, kind = i / chunks & 1, h = i / (2 * chunks);
  const int g = chunk / 4, w = chunk % 4 * groups + g;
  const int block = int4_block_bytes(c.head_dim, c.page_size), row = c.head_dim / 2;
  const ts_view4& v = kind ? a.value : a.key;
  const T* src = reinterpret_cast<const T*>(v.data) + b * v.stride[0] + h * v.stride[1] + t0 * v.stride[2] +
                 (int64_t)chunk * 8 * v.stride[3];
  unsigned char* base = reinterpret_cast<unsigned char*>(c.pool) + (int64_t)h * block + kind * (block / 2);
  const int scales = c.page_size * row + g * 2, mask = c.page_size - 1;
  const uint32_t quad = 0xFu << (threadIdx.x & 28);
  for (int t = t0; t < t1; t += kInFlight) {
    Raw8<T> raw[kInFlight];
    const Span span = token_span(c, b, pos + t, a.page_log2, base);
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (t + u < t1) load8(src, v.stride[3], a.vec, raw[u]);
      src += v.stride[2];
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (t + u >= t1) break;
      float x[8], amax = amax8(raw[u]);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = Elem<T>::to_acc(raw[u].x[e]);
      amax = max_nan(amax, __shfl_xor_sync(quad, amax, 1));
      amax = max_nan(amax, __shfl_xor_sync(quad, amax, 2));
      if (!(amax <= 7.f * kInt4ScaleMax)) {  // saturate, NaN to 0
        amax = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = x[e] == x[e] ? fminf(fmaxf(x[e], -7.f * kInt4ScaleMax), 7.f * kInt4ScaleMax) : 0.f;
          amax = fmaxf(amax, fabsf(x[e]));
        }
        amax = fmaxf(amax, __shfl_xor_sync(quad, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(quad, amax, 2));
      }
      const float scale = int4_scale(amax);
      const uint32_t word = quantise8<T>(x, scale);
      const int p = pos + t + u, at = p & mask;
      unsigned char* dst = (p ^ (pos + t)) >> a.page_log2 ? span.second : span.first;
      if (!dst) {
        record_fault(a.fault, FAULT_PAGE);
        continue;
      }
      reinterpret_cast<uint32_t*>(dst + at * row)[w] = word;
      if (chunk % 4 == 0) *reinterpret_cast<__half*>(dst + scales + at * (row / 8)) = __float2half_rn(scale);
    }
  }
}

template <typename T>
__global__ void kv_gather_int4_kernel(const __grid_constant__ Int4Rows a) {
  let_next_start();
  wait_for_previous();
  const ts_kv4_cache& c = a.c;
  const int b = blockIdx.x / a.token_blocks, t0 = (blockIdx.x - b * a.token_blocks) * a.tokens;
  int t1 = min(a.steps, t0 + a.tokens);
  const int chunks = c.head_dim / 8, groups = c.head_dim / 32;
  const int items = c.kv_heads * 2 * chunks;
  const int i = blockIdx.y * blockDim.x + threadIdx.x;
  if (i >= items) return;
  const int pos = a.positions ? a.positions[b] : 0, len = a.lens ? a.lens[b] : INT32_MAX;
  if (a.tile > 0) t1 = min(t1, ceil_div(min(max(len, 0), a.steps), a.tile) * a.tile);
  const int chunk = i % chunks, kind = i / chunks & 1, h = i / (2 * chunks);
  const int g = chunk / 4, w = chunk % 4 * groups + g;
  const int block = int4_block_bytes(c.head_dim, c.page_size), row = c.head_dim / 2;
  const ts_view4& v = kind ? a.value : a.key;
  T* dst = reinterpret_cast<T*>(v.data) + b * v.stride[0] + h * v.stride[1] + t0 * v.stride[2] +
           (int64_t)chunk * 8 * v.stride[3];
  unsigned char* base = reinterpret_cast<unsigned char*>(c.pool) + (int64_t)h * block + kind * (block / 2);
  const int scales = c.page_size * row + g * 2, mask = c.page_size - 1;
  const int live = min(t1, max(t0, sub_sat(len, pos)));  // tokens from here on are zeros
  for (int t = t0; t < t1; t += kInFlight) {
    uint32_t word[kInFlight];
    float scale[kInFlight];
    Span span{nullptr, nullptr};
    if (t < live) span = token_span(c, b, pos + t, a.page_log2, base);
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      word[u] = 0x88888888u;
      scale[u] = 0.f;
      if (t + u >= live) continue;
      const int p = pos + t + u, at = p & mask;
      const unsigned char* src = (p ^ (pos + t)) >> a.page_log2 ? span.second : span.first;
      if (!src) {
        record_fault(a.fault, FAULT_PAGE);
        continue;
      }
      word[u] = reinterpret_cast<const uint32_t*>(src + at * row)[w];
      scale[u] = __half2float(*reinterpret_cast<const __half*>(src + scales + at * (row / 8)));
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (t + u >= t1) break;
      const uint64_t scale2 = ptx::f2pack(scale[u], scale[u]);
      Raw8<T> raw;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {  // the nibbles under 2^23's exponent: 2^23 + n + 8
        const uint64_t n = ptx::f2pack(__uint_as_float((word[u] >> (4 * e) & 15u) | 0x4B000000u),
                                       __uint_as_float((word[u] >> (4 * e + 4) & 15u) | 0x4B000000u));
        float lo, hi;
        ptx::f2unpack(ptx::fma2(ptx::add2(n, ptx::f2pack(-8388616.f, -8388616.f)), scale2, 0ull), lo, hi);
        raw.x[e] = Elem<T>::from_acc(lo);
        raw.x[e + 1] = Elem<T>::from_acc(hi);
      }
      store8(dst, v.stride[3], a.vec, raw);
      dst += v.stride[2];
    }
  }
}

static bool rows_vec(const ts_view4& v, int size) {
  return v.stride[3] == 1 && reinterpret_cast<uintptr_t>(v.data) % 16 == 0 && v.stride[0] * size % 16 == 0 &&
         v.stride[1] * size % 16 == 0 && v.stride[2] * size % 16 == 0;
}

// Blocks of up to 256 words; as many tokens each as leaves about eight blocks a SM.
static bool rows_grid(Int4Rows& a, dim3& grid, int& threads) {
  const int items = a.c.kv_heads * 2 * (a.c.head_dim / 8);
  threads = items >= 256 ? 256 : (items + 31) / 32 * 32;
  grid.y = (items + threads - 1) / threads;
  const int64_t each = (int64_t)a.c.batch * a.steps * grid.y / (148 * 8);
  a.tokens = each >= 16 ? 16 : each >= 4 ? (int)(each / kInFlight * kInFlight) : each < 1 ? 1 : (int)each;
  a.token_blocks = (a.steps + a.tokens - 1) / a.tokens;
  const int64_t blocks = (int64_t)a.c.batch * a.token_blocks;
  grid.x = (unsigned)blocks;
  a.page_log2 = a.c.page_size == 16 ? 4 : a.c.page_size == 32 ? 5 : 6;
  return blocks <= 0x7FFFFFFF && grid.y <= 65535;
}

cudaError_t kv_append_int4(const ts_view4& key, const ts_view4& value, int dtype, int steps, const ts_kv4_cache& c,
                           int64_t position, const int32_t* positions, int32_t* positions_out, uint32_t* fault,
                           cudaStream_t st) {
  const int size = dtype == TS_F32 ? 4 : 2;
  Int4Rows a{c, key, value, steps, position, positions, positions_out, nullptr, 0, fault,
             rows_vec(key, size) && rows_vec(value, size)};
  dim3 grid;
  int threads;
  if (!rows_grid(a, grid, threads)) return cudaErrorInvalidValue;
  switch (dtype) {
    case TS_F32: return launch_dependent(kv_append_int4_kernel<float>, grid, dim3(threads), 0, st, a);
    case TS_F16: return launch_dependent(kv_append_int4_kernel<__half>, grid, dim3(threads), 0, st, a);
    case TS_BF16: return launch_dependent(kv_append_int4_kernel<__nv_bfloat16>, grid, dim3(threads), 0, st, a);
  }
  return cudaErrorInvalidValue;
}

cudaError_t kv_gather_int4(const ts_kv4_cache& c, const int32_t* starts, const int32_t* lens, const ts_view4& key,
                           const ts_view4& value, int dtype, int length, int tile, uint32_t* fault, cudaStream_t st) {
  if (length == 0) return cudaSuccess;
  const int size = dtype == TS_F32 ? 4 : 2;
  Int4Rows a{c, key, value, length, 0, starts, nullptr, lens, tile, fault, rows_vec(key, size) && rows_vec(value, size)};
  dim3 grid;
  int threads;
  if (!rows_grid(a, grid, threads)) return cudaErrorInvalidValue;
  switch (dtype) {
    case TS_F32: return launch_dependent(kv_gather_int4_kernel<float>, grid, dim3(threads), 0, st, a);
    case TS_F16: return launch_dependent(kv_gather_int4_kernel<__half>, grid, dim3(threads), 0, st, a);
    case TS_BF16: return launch_dependent(kv_gather_int4_kernel<__nv_bfloat16>, grid, dim3(threads), 0, st, a);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tsa
