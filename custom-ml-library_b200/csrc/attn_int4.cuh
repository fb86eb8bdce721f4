// Attention over a paged 4-bit KV cache (see int4.cuh for the storage).
//
//   s_ij = scale * sum_c q_ic n_jc k_scale_j(c/32),   p_ij = softmax over the visible j,
//   o_ic = sum_j p_ij n_jc v_scale_j(c/32)
//
// One pass over the keys with the running maximum and sum of the softmax.  A step of one token a row
// reads 4.5 bits a cached value, so HBM would bound it as long as turning nibbles into operands and
// multiplying costs less than about 2.8 instruction slots a value on one SM (148 SMs, 128 lanes,
// 1.9 GHz against 6.4 TB/s).  CUDA-core arithmetic needs more than that (unpack, convert, and one
// multiply-add for every query); the tensor cores do the multiply-adds for 8 query columns at once:
//   S^T = K q^T    m16n8k16, A = 16 keys x 16 channels, B = 8 query columns
//   O^T = V^T P^T  m16n8k16, A = 16 channels x 16 keys, B = the same 8 columns
// (mma.sync: a fragment is built in registers straight from the nibbles, while tcgen05 would want
// the dequantised tile written to shared memory first, four times the bytes.)  Everything is fp16 in
// the products and fp32 in the sums and statistics:
//   K       (one column tile, half types) the masked nibbles themselves: a nibble in the low bits of a half is the subnormal nibble * 2^-24, in
//           the next four bits nibble * 2^-20, so the queries of the odd ones are a sixteenth; one logic op a
//           pair.  What the nibbles' offset of 8 adds to a 32-channel group's product is a constant of the
//           column, the accumulator's start.  The group's scale goes on its fp32 sum.  (Two and three tiles
//           and fp32 subtract instead, as V does: 59 against 63 us for 20 columns)
//   V       needs its scale on the operand: the nibble in the mantissa of a power of two, 0x6400 | nibble = 1024 +
//           nibble or 0x5400 | nibble << 4 = 64 + nibble, then a subtraction and a product, both exact.  (As one
//           multiply-add, (64 + nibble) scale - 72 scale, the last term would leave fp16 from a scale of 910 on)
//   q       times a power of two that puts its largest element in [2^14, 2^15), rounded to fp16: by at most 2^-39
//           of that element, 2^-35 in the odd channels of the masked form.  So half types keep all their bits down
//           to 2^-31 (bf16) and 2^-28 (fp16) of the largest, odd channels to 2^-27 and 2^-24; fp32 rows as hi + lo
//           (22 bits)
//   p       times 2^7 of a reference within 2^8 of the maximum, fp16; for fp16 and fp32 outputs hi + lo,
//           since the 2^-12 of one fp16 part is as large as the output's own rounding there
// Measured, 64 rows x 32 heads of 1024-8192 keys, D = 128 (1.36 GB): 252 us in fp16, 246 in bf16, 313 in fp32: 84, 86
// and 67 % of the copy rate.  Issue bounds it: 299 warp instructions a tile of 16 keys at 62 % of the issue slots, no
// pipe above 51 %; the copies alone take 212 us, the arithmetic alone took about 228 with 11 instructions fewer.
// Twelve warps an SM fit (168 registers); 16 of 128 spill, and lost what they hid (308 against 253 us).
// The rows of the K tile are permuted within 8 tokens so that the P^T fragment (one transposing
// register move of S^T's) meets V rows whose shared-memory reads do not collide, see token_of_row.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "dependent.cuh"
#include "int4.cuh"
#include "ptx.cuh"

namespace tsa {

constexpr int kInt4MaxRows = 1024;  // rows of one launch: their prefix sums sit in shared memory
// Units of one launch's line of work (see Int4Shares), which the kernels count in 32 bits with room for a share
// more: a call with a longer line takes several launches.
constexpr int64_t kInt4MaxUnits = 1 << 30;

struct Int4Attn {
  ts_attn_params p;
  ts_kv4_cache c;
  int page_log2, block_bytes;
  int group;       // query heads of a KV head
  int cols;        // query columns of a KV head: group * q_len, token-major (column = token * group + head)
  int col_blocks;  // blocks of columns; one warp holds one at a time
  int slot_cols;   // columns of a block that can be live
  int tokens_left; // query tokens of a row from this launch's first on
  int blocks;      // that share the work
  bool by_pair;    // one block a (row, KV head, column block) instead of equal shares
  int parts;       // about how many warps share a row where rows are of one length
  bool q_vec, o_vec;  // rows of unit stride and 16-byte alignment
  float* ws_acc;   // [2 * warps of all blocks, slot_cols, D] partial results
  float* ws_ml;    // [2 * warps of all blocks, slot_cols, 2]
  int32_t* ws_first;  // [2, batch + 1] stages and units before each row
  uint32_t* fault;
};

__device__ __forceinline__ int int4_len(const Int4Attn& a, int b) { return min(a.p.kv_len, max(0, a.p.kv_lens[b])); }
// The same for the merge ahead of its wait.  What wrote the lengths has ended by then, though the attention kernel has
// not: that one's blocks let the merge start only after they have themselves waited for the kernels before them, whose
// writes are at device scope with that.  The load asks there, past this SM's L1, which promises nothing before the wait.
__device__ __forceinline__ int int4_len_early(const Int4Attn& a, int b) {
  int n;
  asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(n) : "l"(a.p.kv_lens + b) : "memory");
  return min(a.p.kv_len, max(0, n));
}
// The shares count n + 1 units for a pair (KV head and column block) of a row with n stages: entering it
// (its queries read, its result written) takes a warp about as long as a stage.  Unit 0 of a pair is the
// entry, unit i + 1 its stage i.  Worker w takes the units [w * share, (w + 1) * share): the first `block_warps`
// warps of each block, which are fewer than the block has where a short line would else leave SMs idle (but no
// fewer than four, whose parts merge on the SM).  Shares of one size leave some workers idle; shares that differ
// by a unit kept all of them busy and lost as much to the extra parts (two rows of up to 131072 keys: 29.1 against
// 29.2 us, 64 rows of 20 columns 143.7 against 142.6, 9 pairs of up to 701 keys 10.5 against 9.9).
struct Int4Shares {
  int block_warps, share;
};
__device__ __forceinline__ Int4Shares int4_shares(const Int4Attn& a, int units, int most_warps) {
  const int block_warps = min(most_warps, max(4, ceil_div(units, a.blocks)));  // at least one a scheduler
  return Int4Shares{block_warps, max(1, ceil_div(units, a.blocks * block_warps))};
}

constexpr float kInt4Log2e = 1.4426950408889634f;
constexpr float kInt4Ln2 = 0.6931471805599453f;

template <typename T>
__device__ __forceinline__ T* int4_out_row(const Int4Attn& a, int b, int h, int i) {
  return reinterpret_cast<T*>(a.p.o.data) + b * a.p.o.stride[0] + h * a.p.o.stride[1] + i * a.p.o.stride[2];
}
__device__ __forceinline__ void int4_store_lse(const Int4Attn& a, int b, int h, int i, float m, float l) {
  if (a.p.lse)
    reinterpret_cast<float*>(a.p.lse)[b * a.p.lse_stride[0] + h * a.p.lse_stride[1] + i * a.p.lse_stride[2]] =
        l == 0.f ? -INFINITY : (m + log2f(l)) * kInt4Ln2;
}

namespace {

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = A B + c, one c a column: an operand of its own, where writing it to d first would cost four moves.
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1, float2 c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }
__device__ __forceinline__ __half2 bits_h2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }

constexpr uint32_t kLow = 0x000F000Fu, kHigh = 0x00F000F0u;  // nibbles 0 and 4 of a word, 1 and 5

// (x & mask) | magic, one three-input logic op.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t magic) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(mask), "r"(magic));
  return y;
}
// Nibbles 0 and 4 of a word as the fp16 pair 1024 + nibble (the nibble in the last four mantissa bits),
// nibbles 1 and 5 as 64 + nibble (in the four bits above them, no shift).
__device__ __forceinline__ uint32_t biased_low(uint32_t w) { return and_or(w, kLow, 0x64006400u); }
__device__ __forceinline__ uint32_t biased_high(uint32_t w) { return and_or(w, kHigh, 0x54005400u); }
// The same pairs as the values n = nibble - 8.
__device__ __forceinline__ uint32_t value_low(uint32_t w) {
  return h2_bits(__hsub2(bits_h2(biased_low(w)), __float2half2_rn(1032.f)));
}
__device__ __forceinline__ uint32_t value_high(uint32_t w) {
  return h2_bits(__hsub2(bits_h2(biased_high(w)), __float2half2_rn(72.f)));
}

// Token (of 8) that row r of a K tile holds.  V slots 2t and 2t + 1 of lane t are then the tokens t
// and 4 + (t ^ 1): neighbouring key rows differ in parity and so do the lanes' V rows, which spreads
// both reads over the 32 banks at D = 128 (64-byte rows).
__device__ __forceinline__ int token_of_row(int r) { return r & 1 ? 4 + ((r >> 1) ^ 1) : r >> 1; }

}  // namespace

// What a lane holds of its query columns and of their running softmax.
// kTwin: at most 4 columns, each held twice; the second of a column takes the other fp16 part of p, so that
// one product serves both parts.
template <typename T, int DG, int NT, bool kTwin>
struct Int4State {
  static constexpr int QP = sizeof(T) == 4 ? 2 : 1;                          // fp16 parts of q
  static constexpr int PP = std::is_same<T, __nv_bfloat16>::value || kTwin ? 1 : 2;  // products with p's fp16 parts
  static constexpr int kColumns = kTwin ? 4 : 8 * NT;
  static constexpr int NW = (DG + 1) / 2;                                    // V words a lane takes of a row
  static constexpr bool kQueriesShared = NT > 1;  // several tiles' query fragments wait in shared memory
  // Tiles of 16 keys whose scores and probabilities are held at a time: what the registers leave room for.
  static constexpr int kChunk = NT == 1 ? 4 : NT == 2 ? 2 : 1;
  uint32_t qf[kQueriesShared ? 1 : QP][kQueriesShared ? 1 : DG][4];
  // One tile multiplies the masked nibbles (of several, the offsets below would cost more than they save).  fp32
  // rows keep subtracting: the offset cancels most of the fp32 sums' upper bits, 1.1e-6 of the output against 2e-7.
  static constexpr bool kMaskedK = NT == 1 && sizeof(T) == 2;
  float qb[kMaskedK ? DG : 1][2];  // what the nibbles' 8 takes from a group's products, columns 2t and 2t + 1
  uint32_t qs;  // shared address of [QP, NT, DG, 32 lanes] x 16 bytes, this lane's first
  __device__ __forceinline__ uint4 fragment(int part, int nt, int gr) const {
    if constexpr (kQueriesShared) {
      uint4 v;  // volatile: loaded where it is used, or the compiler keeps all of them in registers
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                   : "r"(qs + ((part * NT + nt) * DG + gr) * 512));
      return v;
    } else {
      return make_uint4(qf[part][gr][0], qf[part][gr][1], qf[part][gr][2], qf[part][gr][3]);
    }
  }
  float cs[NT][2];       // turns a column's products into exponents of 2; columns 2t and 2t + 1
  int limit[NT][2];      // last key a column sees
  float acc[NT][4 * NW][4];
  float m[NT][2], l[NT][2];
};

// N consecutive aligned 32-bit words from shared memory in the widest loads.
template <int N>
__device__ __forceinline__ void lds_words(const unsigned char* src, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 v = reinterpret_cast<const uint4*>(src)[i];
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 v = reinterpret_cast<const uint2*>(src)[i];
      w[2 * i] = v.x, w[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(src)[i];
  }
}
// N consecutive fp16 scales as pairs in words (an odd last one in the low half).
template <int N>
__device__ __forceinline__ void lds_scales(const unsigned char* src, uint32_t (&w)[(N + 1) / 2]) {
  if constexpr (N % 2 == 0) {
    lds_words<N / 2>(src, w);
  } else {
#pragma unroll
    for (int i = 0; i < (N + 1) / 2; ++i) {
      w[i] = reinterpret_cast<const uint16_t*>(src)[2 * i];
      if (2 * i + 1 < N) w[i] |= (uint32_t) reinterpret_cast<const uint16_t*>(src)[2 * i + 1] << 16;
    }
  }
}
__device__ __forceinline__ float scale_float(uint32_t pair, int i) {
  return i & 1 ? __high2float(bits_h2(pair)) : __low2float(bits_h2(pair));
}

// Where the 16-token tiles of a stage begin: a stage is `units` blocks of `unit` tokens, each laid out like
// a page, so tile 2 i + j starts i * pair + j * one bytes after tile 0.
struct Int4Tiles {
  int row_one, row_pair;      // nibble rows
  int scale_one, scale_pair;  // scales
  int scales;                 // from a block's rows to its scales
  int values;                 // from keys to values
};
__device__ __forceinline__ Int4Tiles int4_tiles(int unit, int row, int scale_row) {
  const int block = 2 * unit * (row + scale_row);
  return Int4Tiles{unit == 16 ? block : 16 * row,
                   unit == 64 ? 32 * row : unit == 32 ? block : 2 * block,
                   unit == 16 ? block : 16 * scale_row,
                   unit == 64 ? 32 * scale_row : unit == 32 ? block : 2 * block,
                   unit * row,
                   block / 2};
}

// One stage: KT tokens at st, the first of them key0.  kEdge: some column does not see
// all of them, or the split ends among them.
template <bool kEdge, typename T, int DG, int NT, bool kTwin, int KT>
__device__ __forceinline__ void int4_stage(Int4State<T, DG, NT, kTwin>& q, const unsigned char* st,
                                           const Int4Tiles& at, int key0, int k_end) {
  using State = Int4State<T, DG, NT, kTwin>;
  constexpr int D = DG * 32, NW = State::NW, kRow = D / 2, kScaleRow = D / 16;
  constexpr int kTiles = KT / 16 < State::kChunk ? KT / 16 : State::kChunk;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tok_a = token_of_row(g), tok_b = 8 + tok_a;

#pragma unroll 1
  for (int tile0 = 0; tile0 < KT / 16; tile0 += kTiles) {
  if (kEdge && tile0 > 0 && key0 + tile0 * 16 >= k_end) break;
  // S^T = K q^T, a 32-channel group at a time, the group's scale on its fp32 sum.
  float s[NT][kTiles][4];
#pragma unroll
  for (int tile = 0; tile < kTiles; ++tile) {
    if (kEdge && tile > 0 && key0 + (tile0 + tile) * 16 >= k_end) {  // none of its keys exists
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][tile][e] = -INFINITY;
      continue;
    }
    const int in = tile0 + tile;
    const unsigned char* kb = st + (in >> 1) * at.row_pair + (in & 1) * at.row_one + t * (DG * 4);
    const unsigned char* ks = st + at.scales + (in >> 1) * at.scale_pair + (in & 1) * at.scale_one;
    uint32_t wa[DG], wb[DG];
    uint32_t ha[(DG + 1) / 2], hb[(DG + 1) / 2];
    lds_words<DG>(kb + tok_a * kRow, wa);
    lds_words<DG>(kb + tok_b * kRow, wb);
    lds_scales<DG>(ks + tok_a * kScaleRow, ha);
    lds_scales<DG>(ks + tok_b * kScaleRow, hb);
#pragma unroll
    for (int gr = 0; gr < DG; ++gr) {
      const uint32_t va = wa[gr] >> 8, vb = wb[gr] >> 8;
      uint32_t k[8];
      float2 offset = make_float2(0.f, 0.f);
      if constexpr (State::kMaskedK) {
        k[0] = wa[gr] & kLow, k[1] = wb[gr] & kLow, k[2] = wa[gr] & kHigh, k[3] = wb[gr] & kHigh;
        k[4] = va & kLow, k[5] = vb & kLow, k[6] = va & kHigh, k[7] = vb & kHigh;
        offset = make_float2(q.qb[gr][0], q.qb[gr][1]);
      } else {
        k[0] = value_low(wa[gr]), k[1] = value_low(wb[gr]), k[2] = value_high(wa[gr]), k[3] = value_high(wb[gr]);
        k[4] = value_low(va), k[5] = value_low(vb), k[6] = value_high(va), k[7] = value_high(vb);
      }
      const float sa = scale_float(ha[gr / 2], gr), sb = scale_float(hb[gr / 2], gr);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float dot[4];
        constexpr int kLast = State::QP - 1;  // the smaller part first
        uint4 b = q.fragment(kLast, nt, gr);
        mma16816_first(dot, k[0], k[1], k[2], k[3], b.x, b.y, offset);
        mma16816(dot, k[4], k[5], k[6], k[7], b.z, b.w);
        if constexpr (kLast > 0) {
          b = q.fragment(0, nt, gr);
          mma16816(dot, k[0], k[1], k[2], k[3], b.x, b.y);
          mma16816(dot, k[4], k[5], k[6], k[7], b.z, b.w);
        }
        float(&x)[4] = s[nt][tile];
        x[0] = gr ? fmaf(sa, dot[0], x[0]) : sa * dot[0];
        x[1] = gr ? fmaf(sa, dot[1], x[1]) : sa * dot[1];
        x[2] = gr ? fmaf(sb, dot[2], x[2]) : sb * dot[2];
        x[3] = gr ? fmaf(sb, dot[3], x[3]) : sb * dot[3];
      }
    }
  }
  // Softmax; a column's keys lie in the 8 lanes of equal t.
  uint32_t pf[State::PP][NT][kTiles][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int tile = 0; tile < kTiles; ++tile) {
      float(&x)[4] = s[nt][tile];
      if constexpr (kEdge) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + (tile0 + tile) * 16 + (e < 2 ? tok_a : tok_b);
          if (key >= k_end || key > q.limit[nt][e & 1]) x[e] = -INFINITY;
        }
      }
      top[0] = ptx::max3(top[0], x[0], x[2]);
      top[1] = ptx::max3(top[1], x[1], x[3]);
    }
    // The reference m follows the maximum only when a score passes it by more than 2^8: p * 2^7 then
    // stays below 2^15, and most stages need no reduction over the lanes.  (Products round up and sums
    // down, so the fused x cs + base below cannot pass 15 however large the scores are.)
    if (__any_sync(0xffffffffu, __fmul_ru(top[0], q.cs[nt][0]) > __fadd_rd(q.m[nt][0], 8.f) ||
                                    __fmul_ru(top[1], q.cs[nt][1]) > __fadd_rd(q.m[nt][1], 8.f))) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float up = top[j];
        up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 4));
        up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 8));
        up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 16));
        up = fmaxf(q.m[nt][j], __fmul_ru(up, q.cs[nt][j]));
        const float f = up > q.m[nt][j] ? ptx::ex2(q.m[nt][j] - up) : 1.f;
        q.m[nt][j] = up;
        q.l[nt][j] *= f;
#pragma unroll
        for (int k = 0; k < 4 * NW; ++k) {
          q.acc[nt][k][j] *= f;
          q.acc[nt][k][j + 2] *= f;
        }
      }
    }
    const uint64_t base2 = ptx::f2pack(__fadd_rd(7.f, q.m[nt][0] == -INFINITY ? 0.f : -q.m[nt][0]),
                                       __fadd_rd(7.f, q.m[nt][1] == -INFINITY ? 0.f : -q.m[nt][1]));
    const uint64_t cs2 = ptx::f2pack(q.cs[nt][0], q.cs[nt][1]);
    uint64_t sum2 = ptx::f2pack(q.l[nt][0], q.l[nt][1]);
#pragma unroll
    for (int tile = 0; tile < kTiles; ++tile) {
      const float(&x)[4] = s[nt][tile];
      float p0, p1, p2, p3;
      ptx::f2unpack(ptx::fma2(ptx::f2pack(x[0], x[1]), cs2, base2), p0, p1);
      ptx::f2unpack(ptx::fma2(ptx::f2pack(x[2], x[3]), cs2, base2), p2, p3);
      p0 = ptx::ex2(p0), p1 = ptx::ex2(p1), p2 = ptx::ex2(p2), p3 = ptx::ex2(p3);
      sum2 = ptx::add2(sum2, ptx::add2(ptx::f2pack(p0, p1), ptx::f2pack(p2, p3)));
      __half2 ha = __floats2half2_rn(p0, p1), hb = __floats2half2_rn(p2, p3);
      if constexpr (kTwin) {  // the second columns (t >= 2) keep what the first ones' rounding leaves
        const float rest = t >= 2 ? -1.f : 0.f;
        ha = __floats2half2_rn(fmaf(rest, __low2float(ha), p0), fmaf(rest, __high2float(ha), p1));
        hb = __floats2half2_rn(fmaf(rest, __low2float(hb), p2), fmaf(rest, __high2float(hb), p3));
      }
      pf[0][nt][tile][0] = transpose8x8(h2_bits(ha));
      pf[0][nt][tile][1] = transpose8x8(h2_bits(hb));
      if constexpr (State::PP == 2) {
        pf[1][nt][tile][0] = transpose8x8(h2_bits(__floats2half2_rn(p0 - __low2float(ha), p1 - __high2float(ha))));
        pf[1][nt][tile][1] = transpose8x8(h2_bits(__floats2half2_rn(p2 - __low2float(hb), p3 - __high2float(hb))));
      }
    }
    ptx::f2unpack(sum2, q.l[nt][0], q.l[nt][1]);
  }
  // O^T += V^T P^T.  Lane (g, t) supplies the words g * NW + j of the tokens in its four slots, as
  // n * scale, exact over the whole range of scales: at most 8 bits, between 2^-20 and 64512.
  const int slot[4] = {t, 4 + (t ^ 1), 8 + t, 12 + (t ^ 1)};
#pragma unroll
  for (int tile = 0; tile < kTiles; ++tile) {
    if (kEdge && tile > 0 && key0 + (tile0 + tile) * 16 >= k_end) break;
    const int in = tile0 + tile;
    const unsigned char* vb = st + at.values + (in >> 1) * at.row_pair + (in & 1) * at.row_one;
    const unsigned char* vs = st + at.values + at.scales + (in >> 1) * at.scale_pair + (in & 1) * at.scale_one;
    uint32_t w[4][NW], sc[4][(NW + 1) / 2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (DG % 2 == 0) {
        lds_words<NW>(vb + slot[k] * kRow + g * (NW * 4), w[k]);
        lds_scales<NW>(vs + slot[k] * kScaleRow + (g * NW) % DG * 2, sc[k]);
      } else {
#pragma unroll
        for (int j = 0; j < (NW + 1) / 2; ++j) sc[k][j] = 0;
#pragma unroll
        for (int j = 0; j < NW; ++j) {
          const int word = g * NW + j;
          const bool in = word < D / 8;
          w[k][j] = in ? reinterpret_cast<const uint32_t*>(vb + slot[k] * kRow)[word] : 0;
          if (in) sc[k][j / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(vs + slot[k] * kScaleRow)[word % DG] << 16 * (j & 1);
        }
      }
      if constexpr (kEdge) {  // past the end a page may hold anything: its nibbles are finite, its scale need not be
        if (key0 + (tile0 + tile) * 16 + slot[k] >= k_end)
#pragma unroll
          for (int j = 0; j < (NW + 1) / 2; ++j) sc[k][j] = 0;
      }
    }
#pragma unroll
    for (int j = 0; j < NW; ++j) {
      const __half2 sc0 = bits_h2(__byte_perm(sc[0][j / 2], sc[1][j / 2], j & 1 ? 0x7632 : 0x5410));
      const __half2 sc1 = bits_h2(__byte_perm(sc[2][j / 2], sc[3][j / 2], j & 1 ? 0x7632 : 0x5410));
#pragma unroll
      for (int byte = 0; byte < 4; ++byte) {
        // byte `byte` of two tokens' words in the low bytes of the halves; the other bytes are masked off
        const uint32_t x0 = __byte_perm(w[0][j], w[1][j], 0x0400 + byte * 0x0101);
        const uint32_t x1 = __byte_perm(w[2][j], w[3][j], 0x0400 + byte * 0x0101);
        const uint32_t a0 = h2_bits(__hmul2(bits_h2(value_low(x0)), sc0));
        const uint32_t a1 = h2_bits(__hmul2(bits_h2(value_high(x0)), sc0));
        const uint32_t a2 = h2_bits(__hmul2(bits_h2(value_low(x1)), sc1));
        const uint32_t a3 = h2_bits(__hmul2(bits_h2(value_high(x1)), sc1));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int part = State::PP - 1; part >= 0; --part)
            mma16816(q.acc[nt][4 * j + byte], a0, a1, a2, a3, pf[part][nt][tile][0], pf[part][nt][tile][1]);
      }
    }
  }
  }
}

// A lane's elements of a block of query columns, as they are in memory.
template <typename T, int DG, int NT>
struct Int4Queries {
  alignas(16) T x[NT][DG][8];
};

template <typename T, int DG, int NT, bool kTwin>
__device__ __forceinline__ void int4_fetch_queries(const Int4Attn& a, Int4Queries<T, DG, NT>& raw, int b, int hk, int col0) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int col = kTwin ? g & 3 : col0 + nt * 8 + g;
    const bool live = col < a.cols;
    const int i = live ? col / a.group : 0, h = hk * a.group + (live ? col - i * a.group : 0);
    const T* qp = reinterpret_cast<const T*>(a.p.q.data) + b * a.p.q.stride[0] + h * a.p.q.stride[1] +
                  i * a.p.q.stride[2];
#pragma unroll
    for (int gr = 0; gr < DG; ++gr) {
      const T* src = qp + (int64_t)(32 * gr + 8 * t) * a.p.q.stride[3];
      if (a.q_vec) {
#pragma unroll
        for (int e = 0; e < (int)(8 * sizeof(T) / 16); ++e)
          reinterpret_cast<uint4*>(raw.x[nt][gr])[e] = reinterpret_cast<const uint4*>(src)[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) raw.x[nt][gr][e] = src[e * a.p.q.stride[3]];
      }
    }
  }
}

// Turns a block of query columns into operands and clears their running softmax.
template <typename T, int DG, int NT, bool kTwin>
__device__ __forceinline__ void int4_load_queries(const Int4Attn& a, Int4State<T, DG, NT, kTwin>& q,
                                                  const Int4Queries<T, DG, NT>& raw, int col0, int len) {
  using State = Int4State<T, DG, NT, kTwin>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const bool live = (kTwin ? g & 3 : col0 + nt * 8 + g) < a.cols;
    float x[DG][8], amax = 0.f;
    bool odd = false;  // a NaN anywhere in the row
#pragma unroll
    for (int gr = 0; gr < DG; ++gr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[gr][e] = live ? Elem<T>::to_acc(raw.x[nt][gr][e]) : 0.f;
        amax = fmaxf(amax, fabsf(x[gr][e]));
        odd |= x[gr][e] != x[gr][e];
      }
    }
    if (odd) amax = INFINITY;
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // up = 2^(14 - floor(log2 amax)); the exponent field stays within normal numbers.  The softmax scale's
    // sign goes to q, so that the largest product is the largest score; where the scale leaves nothing of
    // the products, q becomes zero (a zero factor would make NaN of a hidden key's -inf).
    const float scale = (float)a.p.scale * kInt4Log2e;
    const int up_exp = min(253, max(1, 268 - (int)(__float_as_uint(amax) >> 23)));
    // Products of masked nibbles come out times 2^-24.  (A query beyond 8e34 would take their factor past fp32; held at its end
    // it is still the largest score that stands alone.)
    float unit = fminf(__uint_as_float((uint32_t)(254 - up_exp) << 23) * fabsf(scale) * (State::kMaskedK ? 0x1p24f : 1.f), 3.4e38f);
    float up = __uint_as_float((uint32_t)up_exp << 23) * (scale < 0.f ? -1.f : 1.f);
    if (unit == 0.f) up = 0.f, unit = 1.f;
    if (!(amax < INFINITY)) unit = __int_as_float(0x7fc00000);  // a non-finite query gives NaN, as its product would
#pragma unroll
    for (int j = 0; j < 2; ++j) q.cs[nt][j] = __shfl_sync(0xffffffffu, unit, (2 * t + j) * 4);
    // B fragments: channels 32 gr + 8 t + {0,4}, {1,5}, {2,6}, {3,7} of column g
#pragma unroll
    for (int gr = 0; gr < DG; ++gr) {
      uint32_t f[State::QP][4];
      float sum = 0.f;  // of the parts as they are multiplied, the odd ones times 16
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float sixteenth = State::kMaskedK && e & 1 ? 0.0625f : 1.f, lo = x[gr][e] * up * sixteenth, hi = x[gr][e + 4] * up * sixteenth;
        const __half2 part = __floats2half2_rn(lo, hi);
        f[0][e] = h2_bits(part);
        float both = __low2float(part) + __high2float(part);
        if constexpr (State::QP == 2) {
          const __half2 rest = __floats2half2_rn(lo - __low2float(part), hi - __high2float(part));
          f[1][e] = h2_bits(rest);
          both += __low2float(rest) + __high2float(rest);
        }
        sum = fmaf(both, e & 1 ? 16.f : 1.f, sum);
      }
      if constexpr (State::kMaskedK) {
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum *= -8.f * 0x1p-24f;
#pragma unroll
        for (int j = 0; j < 2; ++j) q.qb[gr][j] = __shfl_sync(0xffffffffu, sum, (2 * t + j) * 4);
      }
      if constexpr (State::kQueriesShared) {  // read back by this lane alone
#pragma unroll
        for (int part = 0; part < State::QP; ++part)
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(q.qs + ((part * NT + nt) * DG + gr) * 512),
                       "r"(f[part][0]), "r"(f[part][1]), "r"(f[part][2]), "r"(f[part][3]));
      } else {
#pragma unroll
        for (int part = 0; part < State::QP; ++part)
#pragma unroll
          for (int e = 0; e < 4; ++e) q.qf[part][gr][e] = f[part][e];
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int mine = kTwin ? (2 * t + j) & 3 : col0 + nt * 8 + 2 * t + j;
      const int tok = min(mine, a.cols - 1) / a.group;
      q.limit[nt][j] = a.p.is_causal ? max(-1, len - a.tokens_left + tok) : len - 1;
      if (q.limit[nt][j] < 0) q.cs[nt][j] = 1.f;  // sees no key: its hidden scores stay -inf whatever the query holds
      q.m[nt][j] = -INFINITY;
      q.l[nt][j] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < 4 * State::NW; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) q.acc[nt][k][e] = 0.f;
  }
}

// Writes the columns' results: to the output when the warp saw all of their keys, else to a partial slot.
template <typename T, int DG, int NT, bool kTwin>
__device__ __forceinline__ void int4_store(const Int4Attn& a, Int4State<T, DG, NT, kTwin>& q, int b, int hk, int col0,
                                           int slot) {
  constexpr int D = DG * 32, NW = Int4State<T, DG, NT, kTwin>::NW;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float sum = q.l[nt][j];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const int local = nt * 8 + 2 * t + j, col = col0 + local;
      if constexpr (kTwin) {
#pragma unroll
        for (int k = 0; k < 4 * NW; ++k) {
          q.acc[nt][k][j] += __shfl_xor_sync(0xffffffffu, q.acc[nt][k][j], 2);
          q.acc[nt][k][j + 2] += __shfl_xor_sync(0xffffffffu, q.acc[nt][k][j + 2], 2);
        }
      }
      if (col >= a.cols || local >= Int4State<T, DG, NT, kTwin>::kColumns) continue;
      const int tok = col / a.group, h = hk * a.group + col - tok * a.group;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      float* part = slot < 0 ? nullptr : a.ws_acc + ((int64_t)slot * a.slot_cols + local) * D;
      T* row = int4_out_row<T>(a, b, h, tok);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const int word = g * NW + w, ch = 32 * (word % DG) + 8 * (word / DG);
        if (DG % 2 && word >= D / 8) continue;
        float x[8];  // channels ch..ch + 7
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = q.acc[nt][4 * w + e / 2][j + 2 * (e & 1)];
        if (slot >= 0) {
          reinterpret_cast<float4*>(part + ch)[0] = make_float4(x[0], x[1], x[2], x[3]);
          reinterpret_cast<float4*>(part + ch)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
          alignas(16) T y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = Elem<T>::from_acc(x[e] * inv);
          if (a.o_vec) {
#pragma unroll
            for (int e = 0; e < (int)(8 * sizeof(T) / 16); ++e)
              reinterpret_cast<uint4*>(row + ch)[e] = reinterpret_cast<const uint4*>(y)[e];
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) row[(ch + e) * a.p.o.stride[3]] = y[e];
          }
        }
      }
      if (g == 0) {
        if (slot >= 0)
          reinterpret_cast<float2*>(a.ws_ml)[(int64_t)slot * a.slot_cols + local] = make_float2(q.m[nt][j], sum);
        else
          int4_store_lse(a, b, h, tok, q.m[nt][j] - 7.f, sum);
      }
    }
}

// Shared memory of the warps' barriers.
__host__ __device__ constexpr int int4_barrier_bytes(int warps, int stages) {
  return (warps * stages * (int)sizeof(uint64_t) + 127) / 128 * 128;
}

// T: type of q and o.  DG = D / 32.  NT: tiles of 8 query columns a warp holds, 1 to 3.
//
// The work is a line of stages of KT tokens, ordered by (row, KV head, column block, key); rows differ in
// length, so every warp takes an equal share of the line instead of whole rows or splits of one size.  A
// share may begin and end inside a row: what it holds of such a row goes to one of the warp's two partial
// slots, and attn_int4_combine merges them.  (Where a pair has at most one stage for each warp of a block,
// by_pair gives every pair a block of its own: nothing is left to merge, so the second launch falls away.)  Each warp runs its own ring of bulk copies through its whole
// share, the next row's first stages in flight while it finishes the last one; no block barrier runs
// between the start and the merge.
// Beside its stages a call of 16 rows x 8 heads takes 1 us until the rows' lengths are summed up, 2.5 until its
// first copies are under way, 2 until they are there, 2 to write the parts and about 4 to merge them: 27 us in all,
// where the bytes alone would take 12.
template <typename T, int DG, int NT, bool kTwin, int KT, int kStages, int kWarps, int kMinBlocks>
__global__ void __launch_bounds__(kWarps * 32, kMinBlocks) attn_int4_kernel(const __grid_constant__ Int4Attn a) {
  constexpr int D = DG * 32;
  constexpr int kRowBytes = D / 2 + D / 16, kStageBytes = 2 * KT * kRowBytes;

  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // The barriers lie ahead of what the merge overlays: their words may hold nothing else while the block runs.
  constexpr int kBarriers = int4_barrier_bytes(kWarps, kStages);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem) + warp * kStages;
  unsigned char* rings = smem + kBarriers;
  unsigned char* ring = rings + warp * (kStages * kStageBytes);
  using State = Int4State<T, DG, NT, kTwin>;
  constexpr int kQueryBytes = State::kQueriesShared ? State::QP * NT * DG * 512 : 0;
  unsigned char* queries = rings + kWarps * kStages * kStageBytes;
  int* first = reinterpret_cast<int*>(queries + kWarps * kQueryBytes);
  const int pairs = a.p.kv_heads * a.col_blocks;

  const int unit = min(1 << a.page_log2, KT), units = KT / unit;  // 1, 2 or 4
  const Int4Tiles tiles = int4_tiles(unit, D / 2, D / 16);
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) ptx::mbar_init(&full[s], units);
    ptx::fence_mbar_init();
  }
  int* first_unit = first + a.p.batch + 1;
  wait_for_previous();
  let_next_start();  // the merge reads the lengths without waiting for this kernel's end: not before the wait above
  if (warp == 0 && !a.by_pair) {  // stages and units of the rows before b
    int stages = 0, rows = 0;
    for (int b0 = 0; b0 <= a.p.batch; b0 += 32) {
      const int b = b0 + lane;
      const int n = b < a.p.batch ? ceil_div(int4_len(a, b), KT) : 0;
      int before = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int below = __shfl_up_sync(0xffffffffu, before, off);
        if (lane >= off) before += below;
      }
      const uint32_t filled = __ballot_sync(0xffffffffu, n > 0);
      const int at = (stages + before - n) * pairs, unit_at = at + (rows + __popc(filled & ((1u << lane) - 1))) * pairs;
      if (b <= a.p.batch) {
        first[b] = at;
        first_unit[b] = unit_at;
        if (blockIdx.x == 0) a.ws_first[b] = at, a.ws_first[a.p.batch + 1 + b] = unit_at;
      }
      stages += __shfl_sync(0xffffffffu, before, 31);
      rows += __popc(filled);
    }
  }
  __syncthreads();
  struct Place {  // of a stage: row, column block and KV head, stage of the pair and their number
    int b, pair, st, n_st;
  };
  Place home, p;    // of the block's first stage, of this warp's next pair
  int begin, mine;  // this warp's first stage and their number
  int block_mine;   // the block's
  int block_id = 0, id = 0;  // the block's first worker, this warp's
  int total = 0, total_units = 0;
  auto row_of = [&](const int* starts, int i) {  // the last row that starts at or before i
    int lo = 0, hi = a.p.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (starts[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  auto stages_before = [&](int64_t u, Place& p) {  // of the units before u; p: where they end
    p = Place{0, 0, 0, 0};
    if (u >= total_units) return total;
    p.b = row_of(first_unit, (int)u);
    const int n = (first_unit[p.b + 1] - first_unit[p.b]) / pairs, at = (int)u - first_unit[p.b];
    p.pair = at / n;
    p.n_st = n - 1;
    p.st = max(0, at - p.pair * n - 1);
    return first[p.b] + p.pair * p.n_st + p.st;
  };
  auto from_lane = [](const Place& p, int l) {
    return Place{__shfl_sync(0xffffffffu, p.b, l), __shfl_sync(0xffffffffu, p.pair, l), __shfl_sync(0xffffffffu, p.st, l),
                 __shfl_sync(0xffffffffu, p.n_st, l)};
  };
  auto place = [&](int i) {
    Place p;
    if (a.by_pair) {
      p = home;
      p.st = i;
      return p;
    }
    p.b = row_of(first, i);
    p.n_st = (first[p.b + 1] - first[p.b]) / pairs;
    p.pair = (i - first[p.b]) / p.n_st;
    p.st = i - first[p.b] - p.pair * p.n_st;
    return p;
  };
  if (a.by_pair) {
    home.b = blockIdx.x / pairs;
    home.pair = blockIdx.x - home.b * pairs;
    home.st = 0;
    home.n_st = block_mine = ceil_div(int4_len(a, home.b), KT);
    const int share = ceil_div(block_mine, kWarps);
    begin = min(warp * share, block_mine);
    mine = min(share, block_mine - begin);
    p = home;
    p.st = begin;
  } else {
    total = first[a.p.batch];
    total_units = first_unit[a.p.batch];
    const Int4Shares shares = int4_shares(a, total_units, kWarps);
    const int share = shares.share;
    block_id = blockIdx.x * shares.block_warps;
    id = block_id + warp;
    // The four bounds on four lanes at once: one after the other these searches took 2 us of the start.
    const int worker = lane == 0 ? id : lane == 1 ? id + 1 : lane == 2 ? block_id : block_id + shares.block_warps;
    Place at;
    const int bound = stages_before((int64_t)worker * share, at);
    begin = __shfl_sync(0xffffffffu, bound, 0);
    mine = warp < shares.block_warps ? __shfl_sync(0xffffffffu, bound, 1) - begin : 0;
    block_mine = __shfl_sync(0xffffffffu, bound, 3) - __shfl_sync(0xffffffffu, bound, 2);
    if (block_mine <= 0) return;
    p = from_lane(at, 0);
    home = from_lane(at, 2);
  }

  // A stage is `units` whole pages, or part of one.  The sources of the next 32 units are worked out by one
  // lane each; that lane then issues its copies: the page's block, or of a part the keys, key scales, values
  // and value scales.
  const unsigned char* ahead = nullptr;  // this lane's unit: its block in the pool, nullptr: none
  int ahead_tok = 0;                     // its first token in the page
  auto look = [&](int n, const Place& p) {  // from stage n of the share on
    ahead = nullptr;
    if (n + lane / units < mine) {
      const int key = p.st * KT + lane % units * unit;
      if (key < int4_len(a, p.b)) {
        const int page = a.c.table[p.b * a.c.table_stride + (key >> a.page_log2)];
        ahead_tok = key & ((1 << a.page_log2) - 1);
        if (page >= 0 && page < a.c.pages)
          ahead = reinterpret_cast<const unsigned char*>(a.c.pool) + page * a.c.page_stride +
                  (int64_t)(p.pair / a.col_blocks) * a.block_bytes;
        else
          record_fault(a.fault, FAULT_PAGE);
      }
    }
    __syncwarp();
  };
  auto issue = [&](int n) {
    const int at = n * units & 31;
    if (at == 0 && n > 0) look(n, place(begin + min(n + lane / units, mine - 1)));
    const int u = lane - at;
    if ((unsigned)u < (unsigned)units) {
      unsigned char* dst = ring + (n % kStages) * kStageBytes;
      uint64_t* bar = &full[n % kStages];
      if (!ahead) {
        ptx::mbar_arrive(bar);
      } else if (unit == 1 << a.page_log2) {
        ptx::mbar_expect_tx(bar, kStageBytes / units);
        ptx::bulk_g2s(dst + u * (kStageBytes / units), ahead, kStageBytes / units, bar);
      } else {
        ptx::mbar_expect_tx(bar, kStageBytes);
        const unsigned char* rows = ahead + ahead_tok * (D / 2);
        const unsigned char* scales = ahead + ((D / 2) << a.page_log2) + ahead_tok * (D / 16);
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
          unsigned char* to = dst + kind * (kStageBytes / 2);
          ptx::bulk_g2s(to, rows + kind * (a.block_bytes / 2), KT * (D / 2), bar);
          ptx::bulk_g2s(to + KT * (D / 2), scales + kind * (a.block_bytes / 2), KT * (D / 16), bar);
        }
      }
    }
  };
  // The first queries are asked for before the first stages: behind them they took 3 us to come.  (The registers
  // that hold them cost several column tiles more than that: 65 against 59 us for 20 columns.)
  constexpr bool kEarly = NT == 1;
  int issued = 0;
  Int4Queries<T, DG, NT> raw;
  if (mine > 0) {
    Place at = p;
    const int i = min(lane / units, mine - 1);
    if (p.st + i < p.n_st) at.st += i;
    else at = place(begin + i);
    const int hk = p.pair / a.col_blocks;
    if constexpr (kEarly) int4_fetch_queries<T, DG, NT, kTwin>(a, raw, p.b, hk, (p.pair - hk * a.col_blocks) * NT * 8);
    look(0, at);
    while (issued < min(mine, kStages - 1)) issue(issued++);
  }
  // A block whose share lies within one pair merges its warps' parts before they leave the SM.
  const bool together = home.st + block_mine <= home.n_st;

  State q;
  q.qs = ptx::smem_u32(queries + warp * kQueryBytes) + lane * 16;
  bool ok = true;
  int n = 0;
  while (n < mine && ok) {
    if (n > 0) {  // the next pair with keys
      p.st = 0;
      if (++p.pair == pairs) {
        p.pair = 0;
        do ++p.b;
        while (first[p.b + 1] == first[p.b]);
        p.n_st = (first[p.b + 1] - first[p.b]) / pairs;
      }
    }
    const int len = int4_len(a, p.b), hk = p.pair / a.col_blocks, col0 = (p.pair - hk * a.col_blocks) * NT * 8;
    const int count = min(mine - n, p.n_st - p.st);
    if (!kEarly || n > 0) int4_fetch_queries<T, DG, NT, kTwin>(a, raw, p.b, hk, col0);
    int4_load_queries<T, DG, NT, kTwin>(a, q, raw, col0, len);
    // the first key that some column does not see
    const int plain = a.p.is_causal ? min(len, max(0, len - a.tokens_left + col0 / a.group + 1)) : len;
    int key0 = p.st * KT;
    for (int k = 0; k < count; ++k, ++n, key0 += KT) {
      if (issued < mine) issue(issued++);
      ok = __all_sync(0xffffffffu, ptx::mbar_wait(&full[n % kStages], (n / kStages) & 1, a.fault, FAULT_DEC_FULL));
      if (!ok) {  // let the copies that are still in flight land before the block ends
        for (int s = n + 1; s < issued; ++s)
          ptx::mbar_wait(&full[s % kStages], (s / kStages) & 1, a.fault, FAULT_DEC_FULL);
        break;
      }
      const unsigned char* st = ring + (n % kStages) * kStageBytes;
      if (key0 + KT <= plain)
        int4_stage<false, T, DG, NT, kTwin, KT>(q, st, tiles, key0, len);
      else
        int4_stage<true, T, DG, NT, kTwin, KT>(q, st, tiles, key0, len);
      __syncwarp();  // every lane is done with the stage before it is filled again
    }
    if (ok && !together)
      int4_store(a, q, p.b, hk, col0, count == p.n_st ? -1 : 2 * id + (n == count ? 0 : 1));
  }
  if (!together) return;

  // Merge through shared memory, over the rings: warp w's columns behind those of the warps before it.
  constexpr int kCols = NT * 8, kPad = D + 4, NW = State::NW;
  float* red = reinterpret_cast<float*>(rings);
  float2* ml = reinterpret_cast<float2*>(red + kWarps * kCols * kPad);
  const int g = lane >> 2, t = lane & 3;
  const int hk = home.pair / a.col_blocks, col0 = (home.pair - hk * a.col_blocks) * NT * 8;
  const int n_cols = min(State::kColumns, a.cols - col0);
  if (!__syncthreads_and(ok)) return;
  if (mine <= 0) {
    for (int i = lane; i < kCols; i += 32) ml[warp * kCols + i] = make_float2(-INFINITY, 0.f);
  } else {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = q.l[nt][j];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int col = warp * kCols + nt * 8 + 2 * t + j;
        if (g == 0) ml[col] = make_float2(q.m[nt][j], sum);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const int word = g * NW + w, ch = 32 * (word % DG) + 8 * (word / DG);
          if ((DG % 2 && word >= D / 8) || (kTwin ? (2 * t + j) & 3 : nt * 8 + 2 * t + j) >= n_cols) continue;
#pragma unroll
          for (int e = 0; e < 8; e += 4)
            *reinterpret_cast<float4*>(&red[col * kPad + ch + e]) =
                make_float4(q.acc[nt][4 * w + e / 2][j], q.acc[nt][4 * w + e / 2][j + 2],
                            q.acc[nt][4 * w + e / 2 + 1][j], q.acc[nt][4 * w + e / 2 + 1][j + 2]);
        }
      }
  }
  __syncthreads();
  const bool all = block_mine == home.n_st;
  for (int i = threadIdx.x; i < n_cols * D; i += kWarps * 32) {
    const int col = i / D, d = i - col * D;
    float top = -INFINITY, sum = 0.f, out = 0.f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w * kCols + col].x);
    const float base = top == -INFINITY ? 0.f : top;
    for (int w = 0; w < kWarps; ++w) {
      const float2 x = ml[w * kCols + col];
      if (x.x == -INFINITY && x.y == 0.f) continue;  // nothing there
      const float f = ptx::ex2(x.x - base);
      sum += x.y * f;
      out += red[(w * kCols + col) * kPad + d] * f;
      if (kTwin) out += red[(w * kCols + col + 4) * kPad + d] * f;
    }
    const int tok = (col0 + col) / a.group, h = hk * a.group + col0 + col - tok * a.group;
    if (all) {
      int4_out_row<T>(a, home.b, h, tok)[d * a.p.o.stride[3]] = Elem<T>::from_acc(sum == 0.f ? 0.f : out / sum);
      if (d == 0) int4_store_lse(a, home.b, h, tok, top - 7.f, sum);
    } else {
      const int64_t slot = (int64_t)2 * block_id * a.slot_cols + col;
      a.ws_acc[slot * D + d] = out;
      if (d == 0) reinterpret_cast<float2*>(a.ws_ml)[slot] = make_float2(top, sum);
    }
  }
}

// row_warps warps (1, 2, 4 or 8) merge an output row; rows without keys become zeros, and a row that was
// written whole is left alone.  What bounds it is one chain of dependent loads behind the first kernel's end, so up
// to 32 rows' places are worked out before it (from the lengths, for stages of `keys` tokens; of more rows the first
// kernel leaves the sums), and a warp has eight parts in flight.  Two rows of up to 131072 keys: 24.4 us a call against
// 29.6 with the places found behind the wait and four parts in flight, 18 heads of up to 701 keys 7.6 against 9.0.
template <typename T, int NT, int kWarps>
__global__ void __launch_bounds__(256) attn_int4_combine(const __grid_constant__ Int4Attn a, int row_warps, int keys) {
  constexpr int kFlight = 8, kChannels = 128;
  __shared__ float part[8][kChannels];
  __shared__ float2 part_ml[8];
  let_next_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = a.p.batch * a.p.q_heads * a.p.q_len;  // the host has checked that it fits
  const int64_t row64 = (int64_t)blockIdx.x * (8 / row_warps) + warp / row_warps;
  const int sub = warp % row_warps;
  if (row64 >= rows) return;  // all warps of a row, like every return below
  const int row = (int)row64, of_head = row / a.p.q_len, tok = row - of_head * a.p.q_len;
  const int b = of_head / a.p.q_heads, h = of_head - b * a.p.q_heads;
  const int hk = h / a.group, col = tok * a.group + h - hk * a.group;
  const int pairs = a.p.kv_heads * a.col_blocks, pair = hk * a.col_blocks + col / (NT * 8), local = col % (NT * 8);
  int n = 0;  // units of a pair: one more than its stages
  int head = 0, mid = 0, tail = 0, lo = 0, c0 = 0, c1 = 0, w0 = 0, w1 = 0;
  int warps = 0;  // of a block
  bool whole = false, late = false;
  // Finds the row's parts: of the first block's warps, of the blocks that merged theirs, of the last block's warps.
  auto locate = [&](int total, int row_first) {
    const int enter = row_first + pair * n;  // the pair's stages are the units enter + 1 .. enter + n - 1
    const Int4Shares shares = int4_shares(a, total, kWarps);
    const int share = shares.share;
    warps = shares.block_warps;
    w0 = (enter + 1) / share, w1 = (enter + n - 1) / share, c0 = w0 / warps, c1 = w1 / warps;
    auto merged = [&](int c) {  // no stage of the block's share is another pair's (the next one's entry may be)
      return (int64_t)c * warps * share >= enter &&
             i64min((int64_t)(c + 1) * warps * share, total) <= (int64_t)enter + n + 1;
    };
    const bool m0 = merged(c0), m1 = merged(c1);
    whole = w0 == w1 || (c0 == c1 && m0);
    head = m0 ? 0 : min(w1, c0 * warps + warps - 1) - w0 + 1;
    lo = m0 ? c0 : c0 + 1, mid = max(0, (m1 ? c1 : c1 - 1) - lo + 1);
    tail = c1 != c0 && !m1 ? w1 - c1 * warps + 1 : 0;
    late = (int64_t)w0 * share < enter;  // the row is not the first thing of its first worker
    lo *= warps, c1 *= warps;
  };
  const bool few = a.p.batch <= 32;
  if (few) {
    const int stages = lane < a.p.batch ? ceil_div(int4_len_early(a, lane), keys) : 0, units = stages ? stages + 1 : 0;
    n = __shfl_sync(0xffffffffu, units, b);
    const int total = __reduce_add_sync(0xffffffffu, units), before = __reduce_add_sync(0xffffffffu, lane < b ? units : 0);
    if (n) locate(total * pairs, before * pairs);
  }
  wait_for_previous();
  if (!few) {
    const int32_t* first_unit = a.ws_first + a.p.batch + 1;
    const int total = first_unit[a.p.batch], row_first = first_unit[b];
    n = (first_unit[b + 1] - row_first) / pairs;
    if (n) locate(total, row_first);
  }
  if (whole) return;
  auto slot = [&](int i) {
    const int w = i < head ? w0 + i : i < head + mid ? lo + (i - head) * warps : c1 + i - head - mid;
    return (int64_t)(2 * w + (late && w == w0)) * a.slot_cols + local;
  };
  const int parts = head + mid + tail;
  const float2* all_ml = reinterpret_cast<const float2*>(a.ws_ml);
  T* o = int4_out_row<T>(a, b, h, tok);
#pragma unroll 1
  for (int d0 = 0; d0 < a.p.head_dim; d0 += kChannels) {
    const int channels = min(kChannels, a.p.head_dim - d0);  // four of them a lane
    float m = -INFINITY, l = 0.f;
    float4 out = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = sub; i0 < parts; i0 += row_warps * kFlight) {
      float2 x[kFlight];
      float4 v[kFlight];
      float top = m;
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        const int i = i0 + u * row_warps;
        x[u] = make_float2(-INFINITY, 0.f);
        v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < parts) {
          const int64_t s = slot(i);
          x[u] = all_ml[s];
          if (lane * 4 < channels) v[u] = *reinterpret_cast<const float4*>(a.ws_acc + s * a.p.head_dim + d0 + lane * 4);
        }
      }
#pragma unroll
      for (int u = 0; u < kFlight; ++u) top = fmaxf(top, x[u].x);
      const float base = top == -INFINITY ? 0.f : top, f0 = ptx::ex2(m - base);
      m = top;
      l *= f0;
      out = make_float4(out.x * f0, out.y * f0, out.z * f0, out.w * f0);
#pragma unroll
      for (int u = 0; u < kFlight; ++u) {
        const float f = ptx::ex2(x[u].x - base);
        l += x[u].y * f;
        out.x += v[u].x * f, out.y += v[u].y * f, out.z += v[u].z * f, out.w += v[u].w * f;
      }
    }
    if (row_warps == 1) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float y[4] = {out.x, out.y, out.z, out.w};
      if (lane * 4 < channels)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[(d0 + lane * 4 + e) * a.p.o.stride[3]] = Elem<T>::from_acc(y[e] * inv);
    } else {  // every warp joins some of the channels
      const int w_row = warp - sub;
      auto row_sync = [&] {
        asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / row_warps), "r"(32 * row_warps) : "memory");
      };
      if (d0 > 0) row_sync();  // the part before has been read
      reinterpret_cast<float4*>(part[warp])[lane] = out;
      if (lane == 0) part_ml[warp] = make_float2(m, l);
      row_sync();
      m = -INFINITY, l = 0.f;
      for (int w = 0; w < row_warps; ++w) m = fmaxf(m, part_ml[w_row + w].x);
      const float base = m == -INFINITY ? 0.f : m;
      float f[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const float2 x = w < row_warps ? part_ml[w_row + w] : make_float2(-INFINITY, 0.f);
        f[w] = ptx::ex2(x.x - base);
        l += x.y * f[w];
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      for (int d = sub * 32 + lane; d < channels; d += row_warps * 32) {
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w)
          if (w < row_warps) y += part[w_row + w][d] * f[w];
        o[(d0 + d) * a.p.o.stride[3]] = Elem<T>::from_acc(y * inv);
      }
    }
    if (d0 == 0 && sub == 0 && lane == 0) int4_store_lse(a, b, h, tok, m - 7.f, l);
  }
}

// Shape of the kernel that takes a problem.
struct Int4Shape {
  int nt;      // column tiles of a warp
  int keys;    // tokens of a stage
  int warps;   // of a block
  int blocks;  // resident on an SM
  bool by_pair;
  bool twin;   // columns held twice
};
Int4Shape int4_shape(const ts_attn_params& p);

template <typename T>
cudaError_t attn_int4_launch(const Int4Attn& a, const Int4Shape& shape, int blocks, cudaStream_t st);
template <typename T>
cudaError_t attn_int4_launch_wide(const Int4Attn& a, const Int4Shape& shape, int blocks, cudaStream_t st);

}  // namespace tsa
