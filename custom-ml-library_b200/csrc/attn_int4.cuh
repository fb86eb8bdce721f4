// Attention over a paged 4-bit KV cache (see int4.cuh for the storage).
//
//   s_ij = scale * sum_c q_ic n_jc k_scale_j(c/32),   p_ij = softmax over the visible j,
//   o_ic = sum_j p_ij n_jc v_scale_j(c/32)
//
// One pass over the keys with the running maximum and sum of the softmax.  A step of one token a row
// reads 4.5 bits a cached value, so HBM bounds it as long as turning nibbles into operands and
// multiplying costs less than about 2.8 instruction slots a value on one SM (148 SMs, 128 lanes,
// 1.9 GHz against 6.4 TB/s).  CUDA-core arithmetic needs more than that (unpack, convert, and one
// multiply-add for every query); the tensor cores do the multiply-adds for 8 query columns at once:
//   S^T = K q^T    m16n8k16, A = 16 keys x 16 channels, B = 8 query columns
//   O^T = V^T P^T  m16n8k16, A = 16 channels x 16 keys, B = the same 8 columns
// (mma.sync: a fragment is built in registers straight from the nibbles, while tcgen05 would want
// the dequantised tile written to shared memory first, four times the bytes.)  Everything is fp16 in
// the products and fp32 in the sums and statistics:
//   n       by the exponent trick, 0x6400 | nibble = 1024 + nibble: one logic op and one subtraction
//           (or multiply-add) a pair; exact, and so is n * scale (8 significant bits)
//   K scale on the fp32 sum of each 32-channel group; V scale on the fp16 operand
//   q       times a power of two that puts its largest element in [2^14, 2^15): exact for bf16 and
//           fp16 rows except elements 2^-38 below the largest; fp32 rows as hi + lo (22 bits)
//   p       times 2^15, fp16; for fp16 and fp32 outputs hi + lo, since the 2^-12 of one fp16 part is
//           as large as the output's own rounding there
// The rows of the K tile are permuted within 8 tokens so that the P^T fragment (one transposing
// register move of S^T's) meets V rows whose shared-memory reads do not collide, see token_of_row.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "int4.cuh"
#include "ptx.cuh"

namespace tsa {

struct Int4Attn {
  ts_attn_params p;
  ts_kv4_cache c;
  int page_log2, block_bytes;
  int group;       // query heads of a KV head
  int cols;        // query columns of a KV head: group * q_len
  int col_blocks;  // grid slices of the columns
  int split_keys, max_splits;
  float* ws_acc;  // [rows, max_splits, D]
  float* ws_ml;   // [rows, max_splits, 2]
  uint32_t* fault;
};

// Columns of a KV head run token-major (column = token * group + head), so a block of columns
// covers few tokens.  [0, end) are the keys that any of the block's columns sees.
__device__ __forceinline__ void int4_range(const Int4Attn& a, int b, int col_end, int& len, int64_t& offset, int& end) {
  len = min(a.p.kv_len, max(0, a.p.kv_lens[b]));
  offset = (int64_t)len - a.p.q_len;
  end = len;
  if (a.p.is_causal) {
    const int last = (min(col_end, a.cols) - 1) / a.group;
    end = (int)i64max(0, i64min(len, offset + last + 1));
  }
}

constexpr float kInt4Log2e = 1.4426950408889634f;
constexpr float kInt4Ln2 = 0.6931471805599453f;

template <typename T>
__device__ __forceinline__ void int4_store_row(const Int4Attn& a, int b, int h, int i, int d, float value) {
  T* o = reinterpret_cast<T*>(a.p.o.data) + b * a.p.o.stride[0] + h * a.p.o.stride[1] + i * a.p.o.stride[2];
  o[d * a.p.o.stride[3]] = Elem<T>::from_acc(value);
}
__device__ __forceinline__ void int4_store_lse(const Int4Attn& a, int b, int h, int i, float m, float l) {
  if (a.p.lse)
    reinterpret_cast<float*>(a.p.lse)[b * a.p.lse_stride[0] + h * a.p.lse_stride[1] + i * a.p.lse_stride[2]] =
        l == 0.f ? -INFINITY : (m + log2f(l)) * kInt4Ln2;
}

namespace {

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }
__device__ __forceinline__ __half2 bits_h2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }

// (x & mask) | 1024's exponent in both halves, one three-input logic op.
__device__ __forceinline__ uint32_t magic_or(uint32_t x, uint32_t mask) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(0x64006400u));
  return y;
}
// Nibbles 0 and 4 of a word as the pair (n, n'); nibbles 1 and 5 without shifting: 1024 + 16 n.
__device__ __forceinline__ __half2 pair_low(uint32_t w) {
  return __hsub2(bits_h2(magic_or(w, 0x000F000Fu)), __float2half2_rn(1032.f));
}
__device__ __forceinline__ __half2 pair_high(uint32_t w) {
  return __hfma2(bits_h2(magic_or(w, 0x00F000F0u)), __float2half2_rn(0.0625f), __float2half2_rn(-72.f));
}

// Token (of 8) that row r of a K tile holds.  V slots 2t and 2t + 1 of lane t are then the tokens t
// and 4 + (t ^ 1): neighbouring key rows differ in parity and so do the lanes' V rows, which spreads
// both reads over the 32 banks at D = 128 (64-byte rows).
__device__ __forceinline__ int token_of_row(int r) { return r & 1 ? 4 + ((r >> 1) ^ 1) : r >> 1; }

}  // namespace

// T: type of q and o.  DG = D / 32.  NT: tiles of 8 query columns a block holds.  One warp streams
// its own stages of KT tokens through a ring of kStages; the block's kWarps take the stages of a split
// in turn and merge once at the end, so no barrier runs inside the loop.
template <typename T, int DG, int NT, int KT, int kStages, int kWarps>
__global__ void __launch_bounds__(kWarps * 32) attn_int4_kernel(const __grid_constant__ Int4Attn a) {
  constexpr int D = DG * 32;
  constexpr int QP = sizeof(T) == 4 ? 2 : 1;                                // fp16 parts of q
  constexpr int PP = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;         // fp16 parts of p
  constexpr int NW = (DG + 1) / 2;                                          // V words a lane takes of a row
  constexpr int kTiles = KT / 16;
  constexpr int kStageBytes = 2 * KT * (D / 2 + D / 16);
  constexpr int kRow = D / 2, kScaleRow = D / 16;

  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  unsigned char* ring = smem + warp * (kStages * kStageBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kWarps * kStages * kStageBytes) + warp * kStages;

  // Column blocks of one split are neighbours in the grid, so their reads of the cache meet in L2.
  int64_t idx = blockIdx.x;
  const int cb = (int)(idx % a.col_blocks);
  idx /= a.col_blocks;
  const int split = (int)(idx % a.max_splits);
  idx /= a.max_splits;
  const int hk = (int)(idx % a.p.kv_heads), b = (int)(idx / a.p.kv_heads);
  const int col0 = cb * NT * 8;
  int len, end;
  int64_t offset;
  int4_range(a, b, col0 + NT * 8, len, offset, end);
  const int n_splits = max(1, ceil_div(end, a.split_keys));
  if (split >= n_splits) return;
  const int k_begin = split * a.split_keys, k_end = min(end, k_begin + a.split_keys);
  const int stages = k_end > k_begin ? ceil_div(k_end - k_begin, KT) : 0;
  const int mine = stages > warp ? ceil_div(stages - warp, kWarps) : 0;

  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) ptx::mbar_init(&full[s], 1);
    ptx::fence_mbar_init();
  }
  __syncwarp();

  // Lane j fetches page j of a stage; its table entry is read one stage ahead.
  const int page_size = 1 << a.page_log2;
  const int stage_pages = KT >> a.page_log2 ? KT >> a.page_log2 : 1;
  const int32_t* table = a.c.table + b * a.c.table_stride;
  const unsigned char* pool = reinterpret_cast<const unsigned char*>(a.c.pool) + (int64_t)hk * a.block_bytes;
  auto stage_key = [&](int n) { return k_begin + (warp + n * kWarps) * KT; };
  auto entry = [&](int n) {
    const int key = stage_key(n) + lane * page_size;
    return n < mine && lane < stage_pages && key < k_end ? table[key >> a.page_log2] : -2;
  };
  auto issue = [&](int n, int page) {
    unsigned char* dst = ring + (n % kStages) * kStageBytes;
    uint64_t* bar = &full[n % kStages];
    const bool wanted = page != -2;
    const bool good = wanted && page >= 0 && page < a.c.pages;
    if (wanted && !good) record_fault(a.fault, FAULT_PAGE);
    if constexpr (KT >= 64) {  // whole pages (page_size <= 64)
      const int n_good = __popc(__ballot_sync(0xffffffffu, good));
      if (lane == 0) ptx::mbar_expect_tx(bar, (uint32_t)n_good * a.block_bytes);
      __syncwarp();
      if (good) ptx::bulk_g2s(dst + lane * a.block_bytes, pool + page * a.c.page_stride, a.block_bytes, bar);
    }
  };

  // Queries: B fragments (channels 32 gr + 8 t + {0,4}, {1,5}, {2,6}, {3,7} of column g).
  uint32_t qf[QP][NT][DG][4];
  float cs[NT][2];  // what turns a column's products into exponents of 2: columns 2t and 2t + 1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int col = col0 + nt * 8 + g;
    const bool live = col < a.cols;
    const int i = live ? col / a.group : 0, h = hk * a.group + (live ? col - i * a.group : 0);
    const T* qp = reinterpret_cast<const T*>(a.p.q.data) + b * a.p.q.stride[0] + h * a.p.q.stride[1] +
                  i * a.p.q.stride[2];
    float x[DG][8], amax = 0.f;
    bool odd = false;  // a NaN anywhere in the row
#pragma unroll
    for (int gr = 0; gr < DG; ++gr)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[gr][e] = live ? Elem<T>::to_acc(qp[(int64_t)(32 * gr + 8 * t + e) * a.p.q.stride[3]]) : 0.f;
        amax = fmaxf(amax, fabsf(x[gr][e]));
        odd |= x[gr][e] != x[gr][e];
      }
    if (odd) amax = INFINITY;
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // up = 2^(14 - floor(log2 amax)); the exponent field stays within normal numbers
    const int up_exp = min(253, max(1, 268 - (int)(__float_as_uint(amax) >> 23)));
    const float up = __uint_as_float((uint32_t)up_exp << 23);
    float unit = __uint_as_float((uint32_t)(254 - up_exp) << 23) * ((float)a.p.scale * kInt4Log2e);
    if (!(amax < INFINITY)) unit = __int_as_float(0x7fc00000);  // a non-finite query gives NaN, as its product would
#pragma unroll
    for (int j = 0; j < 2; ++j) cs[nt][j] = __shfl_sync(0xffffffffu, unit, (2 * t + j) * 4);
#pragma unroll
    for (int gr = 0; gr < DG; ++gr)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = x[gr][e] * up, hi = x[gr][e + 4] * up;
        const __half2 part = __floats2half2_rn(lo, hi);
        qf[0][nt][gr][e] = h2_bits(part);
        if constexpr (QP == 2)
          qf[1][nt][gr][e] = h2_bits(__floats2half2_rn(lo - __low2float(part), hi - __high2float(part)));
      }
  }
  // Last key each of this lane's columns sees, and the last that all of them see.
  int limit[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int col = min(col0 + nt * 8 + 2 * t + j, a.cols - 1);
      limit[nt][j] = a.p.is_causal ? (int)i64max(-1, i64min(len, offset + col / a.group + 1) - 1) : len - 1;
    }
  const int all_see = a.p.is_causal ? (int)i64max(-1, i64min(len, offset + col0 / a.group + 1) - 1) : len - 1;

  float acc[NT][4 * NW][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int k = 0; k < 4 * NW; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[nt][k][e] = 0.f;
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
  }

  int ahead = entry(0);
#pragma unroll
  for (int n = 0; n < kStages - 1; ++n) {
    if (n < mine) issue(n, ahead);
    ahead = entry(n + 1);
  }
  const int tok_a = token_of_row(g), tok_b = 8 + tok_a;
  bool ok = true;
  int issued = min(mine, kStages - 1);
  for (int n = 0; n < mine; ++n) {
    if (issued < mine) {
      issue(issued, ahead);
      ++issued;
      ahead = entry(issued);
    }
    ok = __all_sync(0xffffffffu, ptx::mbar_wait(&full[n % kStages], (n / kStages) & 1, a.fault, FAULT_DEC_FULL));
    if (!ok) break;
    const unsigned char* st = ring + (n % kStages) * kStageBytes;
    const int key0 = stage_key(n);

    float s[NT][kTiles][4];
#pragma unroll
    for (int tile = 0; tile < kTiles; ++tile) {
      const int in_page = (tile * 16) & (page_size - 1);
      const unsigned char* kb = st + ((tile * 16) >> a.page_log2) * a.block_bytes;
      const unsigned char* ks = kb + page_size * kRow + in_page * kScaleRow;
      kb += in_page * kRow + t * (DG * 4);
      uint32_t wa[DG], wb[DG];
      if constexpr (DG % 4 == 0) {
#pragma unroll
        for (int i = 0; i < DG / 4; ++i) {
          *reinterpret_cast<uint4*>(&wa[4 * i]) = reinterpret_cast<const uint4*>(kb + tok_a * kRow)[i];
          *reinterpret_cast<uint4*>(&wb[4 * i]) = reinterpret_cast<const uint4*>(kb + tok_b * kRow)[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < DG; ++i) {
          wa[i] = reinterpret_cast<const uint32_t*>(kb + tok_a * kRow)[i];
          wb[i] = reinterpret_cast<const uint32_t*>(kb + tok_b * kRow)[i];
        }
      }
#pragma unroll
      for (int gr = 0; gr < DG; ++gr) {
        const float sa = __half2float(reinterpret_cast<const __half*>(ks + tok_a * kScaleRow)[gr]);
        const float sb = __half2float(reinterpret_cast<const __half*>(ks + tok_b * kScaleRow)[gr]);
        const uint32_t a0 = h2_bits(pair_low(wa[gr])), a2 = h2_bits(pair_high(wa[gr]));
        const uint32_t a1 = h2_bits(pair_low(wb[gr])), a3 = h2_bits(pair_high(wb[gr]));
        const uint32_t c0 = h2_bits(pair_low(wa[gr] >> 8)), c2 = h2_bits(pair_high(wa[gr] >> 8));
        const uint32_t c1 = h2_bits(pair_low(wb[gr] >> 8)), c3 = h2_bits(pair_high(wb[gr] >> 8));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float dot[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = QP - 1; q >= 0; --q) {
            mma16816(dot, a0, a1, a2, a3, qf[q][nt][gr][0], qf[q][nt][gr][1]);
            mma16816(dot, c0, c1, c2, c3, qf[q][nt][gr][2], qf[q][nt][gr][3]);
          }
          float(&x)[4] = s[nt][tile];
          x[0] = gr ? fmaf(sa, dot[0], x[0]) : sa * dot[0];
          x[1] = gr ? fmaf(sa, dot[1], x[1]) : sa * dot[1];
          x[2] = gr ? fmaf(sb, dot[2], x[2]) : sb * dot[2];
          x[3] = gr ? fmaf(sb, dot[3], x[3]) : sb * dot[3];
        }
      }
    }
    // Softmax of the stage's KT keys, a column's keys spread over the 8 lanes of equal t.
    const bool edge = key0 + KT > min(k_end, all_see + 1);
    uint32_t pf[PP][NT][kTiles][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int tile = 0; tile < kTiles; ++tile)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float& x = s[nt][tile][e];
          x *= cs[nt][e & 1];
          if (edge) {
            const int key = key0 + tile * 16 + (e < 2 ? tok_a : tok_b);
            if (key >= k_end || key > limit[nt][e & 1]) x = -INFINITY;
          }
          top[e & 1] = fmaxf(top[e & 1], x);
        }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 4));
        top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 8));
        top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], 16));
      }
      if (__any_sync(0xffffffffu, top[0] > m[nt][0] || top[1] > m[nt][1])) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float up = fmaxf(m[nt][j], top[j]);
          const float f = up > m[nt][j] ? ptx::ex2(m[nt][j] - up) : 1.f;
          m[nt][j] = up;
          l[nt][j] *= f;
#pragma unroll
          for (int k = 0; k < 4 * NW; ++k) {
            acc[nt][k][j] *= f;
            acc[nt][k][j + 2] *= f;
          }
        }
      }
      const float base0 = (m[nt][0] == -INFINITY ? 0.f : m[nt][0]) - 15.f;
      const float base1 = (m[nt][1] == -INFINITY ? 0.f : m[nt][1]) - 15.f;
#pragma unroll
      for (int tile = 0; tile < kTiles; ++tile) {
        const float(&x)[4] = s[nt][tile];
        const float p0 = ptx::ex2(x[0] - base0), p1 = ptx::ex2(x[1] - base1);
        const float p2 = ptx::ex2(x[2] - base0), p3 = ptx::ex2(x[3] - base1);
        l[nt][0] += p0 + p2;
        l[nt][1] += p1 + p3;
        const __half2 ha = __floats2half2_rn(p0, p1), hb = __floats2half2_rn(p2, p3);
        pf[0][nt][tile][0] = transpose8x8(h2_bits(ha));
        pf[0][nt][tile][1] = transpose8x8(h2_bits(hb));
        if constexpr (PP == 2) {
          pf[1][nt][tile][0] = transpose8x8(h2_bits(__floats2half2_rn(p0 - __low2float(ha), p1 - __high2float(ha))));
          pf[1][nt][tile][1] = transpose8x8(h2_bits(__floats2half2_rn(p2 - __low2float(hb), p3 - __high2float(hb))));
        }
      }
    }
    // O^T += V^T P^T.  Lane (g, t) supplies the words g * NW + j of the tokens in its four slots.
#pragma unroll
    for (int tile = 0; tile < kTiles; ++tile) {
      const int in_page = (tile * 16) & (page_size - 1);
      const unsigned char* vb = st + ((tile * 16) >> a.page_log2) * a.block_bytes + (a.block_bytes >> 1);
      const unsigned char* vs = vb + page_size * kRow + in_page * kScaleRow;
      vb += in_page * kRow;
      const int slot[4] = {t, 4 + (t ^ 1), 8 + t, 12 + (t ^ 1)};
      uint32_t w[4][NW];
      __half sc[4][NW];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int j = 0; j < NW; ++j) {
          const int word = g * NW + j;
          if (DG % 2 == 0 || word < D / 8) {
            w[k][j] = reinterpret_cast<const uint32_t*>(vb + slot[k] * kRow)[word];
            sc[k][j] = reinterpret_cast<const __half*>(vs + slot[k] * kScaleRow)[word % DG];
          } else {
            w[k][j] = 0;
            sc[k][j] = __ushort_as_half(0);
          }
          // Past the end the page may hold anything; its nibbles are finite, its scale need not be.
          if (edge && key0 + tile * 16 + slot[k] >= k_end) sc[k][j] = __ushort_as_half(0);
        }
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        const __half2 sc0 = __halves2half2(sc[0][j], sc[1][j]), sc1 = __halves2half2(sc[2][j], sc[3][j]);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t x0 = __byte_perm(w[0][j], w[1][j], half ? 0x7632 : 0x5410);
          const uint32_t x1 = __byte_perm(w[2][j], w[3][j], half ? 0x7632 : 0x5410);
#pragma unroll
          for (int hi = 0; hi < 2; ++hi) {
            const uint32_t a0 = h2_bits(__hmul2(pair_low(x0 >> (8 * hi)), sc0));
            const uint32_t a1 = h2_bits(__hmul2(pair_high(x0 >> (8 * hi)), sc0));
            const uint32_t a2 = h2_bits(__hmul2(pair_low(x1 >> (8 * hi)), sc1));
            const uint32_t a3 = h2_bits(__hmul2(pair_high(x1 >> (8 * hi)), sc1));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int q = PP - 1; q >= 0; --q)
                mma16816(acc[nt][4 * j + 2 * half + hi], a0, a1, a2, a3, pf[q][nt][tile][0], pf[q][nt][tile][1]);
          }
        }
      }
    }
    __syncwarp();  // every lane is done with the stage before it is filled again
  }
  if (!ok) {  // let the copies that are still in flight land before the block ends
    for (int n = 0; n < issued; ++n) {
      if (n + kStages < issued) continue;
      ptx::mbar_wait(&full[n % kStages], (n / kStages) & 1, a.fault, FAULT_DEC_FULL);
    }
  }
  // Merge the warps' partial results through shared memory.
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 4);
      l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 8);
      l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 16);
    }
  constexpr int kCols = NT * 8;
  constexpr int kPad = D + 4;
  float* red = reinterpret_cast<float*>(smem);
  float* ml = red + kWarps * kCols * kPad;
  const bool all_ok = __syncthreads_and(ok);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < NW; ++j) {
      const int word = g * NW + j;
      if (DG % 2 == 0 || word < D / 8) {
        const int ch = 32 * (word % DG) + 8 * (word / DG);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            red[(warp * kCols + nt * 8 + 2 * t + (e & 1)) * kPad + ch + 2 * k + (e >> 1)] = acc[nt][4 * j + k][e];
      }
    }
    if (g == 0)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        ml[(warp * kCols + nt * 8 + 2 * t + j) * 2] = m[nt][j];
        ml[(warp * kCols + nt * 8 + 2 * t + j) * 2 + 1] = l[nt][j];
      }
  }
  __syncthreads();
  if (!all_ok) return;
  for (int i = threadIdx.x; i < kCols * D; i += kWarps * 32) {
    const int col = i / D, d = i - col * D;
    if (col0 + col >= a.cols) break;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[(w * kCols + col) * 2]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, out = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ptx::ex2(ml[(w * kCols + col) * 2] - base);
      sum += ml[(w * kCols + col) * 2 + 1] * f;
      out += red[(w * kCols + col) * kPad + d] * f;
    }
    const int tok = (col0 + col) / a.group, h = hk * a.group + (col0 + col) - tok * a.group;
    if (n_splits == 1) {
      int4_store_row<T>(a, b, h, tok, d, sum == 0.f ? 0.f : out / sum);
      if (d == 0) int4_store_lse(a, b, h, tok, top - 15.f, sum);
    } else {
      const int64_t row = ((int64_t)b * a.p.q_heads + h) * a.p.q_len + tok;
      a.ws_acc[(row * a.max_splits + split) * D + d] = out;
      if (d == 0) {
        a.ws_ml[(row * a.max_splits + split) * 2] = top;
        a.ws_ml[(row * a.max_splits + split) * 2 + 1] = sum;
      }
    }
  }
}

// One block an output row: merges its splits.
template <typename T>
__global__ void attn_int4_combine(const __grid_constant__ Int4Attn a, int block_cols) {
  const int64_t row = blockIdx.x;
  const int tok = (int)(row % a.p.q_len), h = (int)(row / a.p.q_len % a.p.q_heads);
  const int b = (int)(row / ((int64_t)a.p.q_len * a.p.q_heads));
  const int col = tok * a.group + h % a.group;
  int len, end;
  int64_t offset;
  int4_range(a, b, col / block_cols * block_cols + block_cols, len, offset, end);
  const int n = max(1, ceil_div(end, a.split_keys));
  if (n == 1) return;
  const float* ml = a.ws_ml + row * a.max_splits * 2;
  float top = -INFINITY;
  for (int s = 0; s < n; ++s) top = fmaxf(top, ml[2 * s]);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int s = 0; s < n; ++s) sum += ml[2 * s + 1] * ptx::ex2(ml[2 * s] - base);
  for (int d = threadIdx.x; d < a.p.head_dim; d += blockDim.x) {
    float out = 0.f;
    for (int s = 0; s < n; ++s)
      out += a.ws_acc[(row * a.max_splits + s) * a.p.head_dim + d] * ptx::ex2(ml[2 * s] - base);
    int4_store_row<T>(a, b, h, tok, d, sum == 0.f ? 0.f : out / sum);
  }
  if (threadIdx.x == 0) int4_store_lse(a, b, h, tok, top - 15.f, sum);
}

template <typename T>
cudaError_t attn_int4_launch(const Int4Attn& a, int nt, cudaStream_t st);

}  // namespace tsa
