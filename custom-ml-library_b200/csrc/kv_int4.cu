// Quantising append into the pages of a 4-bit KV cache, and the read-back of its values.
// Both move each value once: 16 bits in and 4.5 out (the append), 4.5 in and 16 out (the gather),
// so HBM, or for a token of each row the launch, bounds them.
#include "int4.cuh"

namespace tsa {

struct Int4Rows {
  ts_kv4_cache c;
  ts_view4 key, value;
  int steps;
  int64_t position;
  const int32_t* positions;
  int32_t* positions_out;
  const int32_t* lens;
  uint32_t* fault;
  bool vec;  // unit channel stride, 16-byte aligned rows
};

template <typename T>
__device__ __forceinline__ void load8(const T* src, int64_t stride, bool vec, float (&x)[8]) {
  if (vec) {
    alignas(16) T raw[8];
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i)
      reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(src)[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = Elem<T>::to_acc(raw[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = Elem<T>::to_acc(src[e * stride]);
  }
}

// One block a (row, token); one thread 8 channels (a stored word) of a K or V row, so the four
// neighbouring threads of a scale group share its maximum by two shuffles.
template <typename T>
__global__ void kv_append_int4_kernel(Int4Rows a) {
  const ts_kv4_cache& c = a.c;
  const int b = blockIdx.x / a.steps, t = blockIdx.x - b * a.steps;
  const int64_t pos = (a.positions ? (int64_t)a.positions[b] : a.position) + t;
  const int chunks = c.head_dim / 8, groups = c.head_dim / 32;
  const int64_t slot = pos / c.page_size;
  const int page = pos < 0 || slot >= c.slots ? -1 : int4_page(c, b, (int)slot);
  if (t == 0 && threadIdx.x == 0 && a.positions_out) a.positions_out[b] = (int32_t)(pos + a.steps);
  if (page < 0) {
    if (threadIdx.x == 0) record_fault(a.fault, FAULT_PAGE);
    return;
  }
  const int at = (int)(pos - slot * c.page_size);
  const int block = int4_block_bytes(c.head_dim, c.page_size);
  const int items = c.kv_heads * 2 * chunks;  // a multiple of 4
  for (int i = threadIdx.x; i < items; i += blockDim.x) {
    const int chunk = i % chunks, kind = i / chunks & 1, h = i / (2 * chunks);
    const ts_view4& v = kind ? a.value : a.key;
    const T* src = reinterpret_cast<const T*>(v.data) + b * v.stride[0] + h * v.stride[1] + t * v.stride[2] +
                   (int64_t)chunk * 8 * v.stride[3];
    float x[8];
    load8(src, v.stride[3], a.vec, x);
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));
    const uint32_t quad = 0xFu << (threadIdx.x & 28);
    amax = fmaxf(amax, __shfl_xor_sync(quad, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(quad, amax, 2));
    const float scale = int4_scale(amax);
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) word |= int4_nibble(x[e], scale) << (4 * e);
    unsigned char* dst = reinterpret_cast<unsigned char*>(c.pool) + page * c.page_stride + (int64_t)h * block +
                         kind * (block / 2);
    const int g = chunk / 4, w = chunk % 4 * groups + g;
    reinterpret_cast<uint32_t*>(dst + (int64_t)at * (c.head_dim / 2))[w] = word;
    if (chunk % 4 == 0)
      reinterpret_cast<__half*>(dst + c.page_size * (c.head_dim / 2))[at * groups + g] = __float2half_rn(scale);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* dst, int64_t stride, bool vec, const float (&x)[8]) {
  if (vec) {
    alignas(16) T raw[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) raw[e] = Elem<T>::from_acc(x[e]);
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i)
      reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(raw)[i];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) dst[e * stride] = Elem<T>::from_acc(x[e]);
  }
}

// The same split as the append: one block a (row, token), one thread a word.
template <typename T>
__global__ void kv_gather_int4_kernel(Int4Rows a) {
  const ts_kv4_cache& c = a.c;
  const int b = blockIdx.x / a.steps, t = blockIdx.x - b * a.steps;
  const int64_t pos = (a.positions ? (int64_t)a.positions[b] : 0) + t;
  const int chunks = c.head_dim / 8, groups = c.head_dim / 32;
  const int64_t slot = pos / c.page_size;
  const bool past = a.lens && pos >= a.lens[b];
  const int page = past || pos < 0 || slot >= c.slots ? -1 : int4_page(c, b, (int)slot);
  if (page < 0 && !past && threadIdx.x == 0) record_fault(a.fault, FAULT_PAGE);
  const int at = (int)(pos - slot * c.page_size);
  const int block = int4_block_bytes(c.head_dim, c.page_size);
  const int items = c.kv_heads * 2 * chunks;
  for (int i = threadIdx.x; i < items; i += blockDim.x) {
    const int chunk = i % chunks, kind = i / chunks & 1, h = i / (2 * chunks);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    if (page >= 0) {
      const unsigned char* src = reinterpret_cast<const unsigned char*>(c.pool) + page * c.page_stride +
                                 (int64_t)h * block + kind * (block / 2);
      const int g = chunk / 4, w = chunk % 4 * groups + g;
      const uint32_t word = reinterpret_cast<const uint32_t*>(src + (int64_t)at * (c.head_dim / 2))[w];
      const float scale =
          __half2float(reinterpret_cast<const __half*>(src + c.page_size * (c.head_dim / 2))[at * groups + g]);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)((int)(word >> (4 * e) & 15u) - 8) * scale;
    }
    const ts_view4& v = kind ? a.value : a.key;
    T* dst = reinterpret_cast<T*>(v.data) + b * v.stride[0] + h * v.stride[1] + t * v.stride[2] +
             (int64_t)chunk * 8 * v.stride[3];
    store8(dst, v.stride[3], a.vec, x);
  }
}

static bool rows_vec(const ts_view4& v, int size) {
  return v.stride[3] == 1 && reinterpret_cast<uintptr_t>(v.data) % 16 == 0 && v.stride[0] * size % 16 == 0 &&
         v.stride[1] * size % 16 == 0 && v.stride[2] * size % 16 == 0;
}

static int row_threads(const ts_kv4_cache& c) {
  const int items = c.kv_heads * 2 * (c.head_dim / 8);
  return items >= 256 ? 256 : (items + 31) / 32 * 32;
}

cudaError_t kv_append_int4(const ts_view4& key, const ts_view4& value, int dtype, int steps, const ts_kv4_cache& c,
                           int64_t position, const int32_t* positions, int32_t* positions_out, uint32_t* fault,
                           cudaStream_t st) {
  const int size = dtype == TS_F32 ? 4 : 2;
  const Int4Rows a{c,   key,     value, steps, position, positions, positions_out, nullptr, fault,
                   rows_vec(key, size) && rows_vec(value, size)};
  const int64_t blocks = (int64_t)c.batch * steps;
  if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const int threads = row_threads(c);
  switch (dtype) {
    case TS_F32: kv_append_int4_kernel<float><<<(unsigned)blocks, threads, 0, st>>>(a); break;
    case TS_F16: kv_append_int4_kernel<__half><<<(unsigned)blocks, threads, 0, st>>>(a); break;
    case TS_BF16: kv_append_int4_kernel<__nv_bfloat16><<<(unsigned)blocks, threads, 0, st>>>(a); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

cudaError_t kv_gather_int4(const ts_kv4_cache& c, const int32_t* starts, const int32_t* lens, const ts_view4& key,
                           const ts_view4& value, int dtype, int length, uint32_t* fault, cudaStream_t st) {
  const int size = dtype == TS_F32 ? 4 : 2;
  const Int4Rows a{c, key, value, length, 0, starts, nullptr, lens, fault,
                   rows_vec(key, size) && rows_vec(value, size)};
  const int64_t blocks = (int64_t)c.batch * length;
  if (blocks == 0) return cudaSuccess;
  if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const int threads = row_threads(c);
  switch (dtype) {
    case TS_F32: kv_gather_int4_kernel<float><<<(unsigned)blocks, threads, 0, st>>>(a); break;
    case TS_F16: kv_gather_int4_kernel<__half><<<(unsigned)blocks, threads, 0, st>>>(a); break;
    case TS_BF16: kv_gather_int4_kernel<__nv_bfloat16><<<(unsigned)blocks, threads, 0, st>>>(a); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace tsa
