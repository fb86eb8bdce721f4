// Attention of drafted tokens over a contiguous KV cache on tcgen05 (bf16 / f16, head dimensions that are
// multiples of 8 up to 128): out = softmax(scale q K^T) V over the keys that tree.cuh's rule lets a node see.
//
// The T drafted tokens of the query heads that share a KV head are the rows of a 128-row tile, so that every
// key is read once for all of them.  The work is one line of 128-key tiles over (row, KV head, row tile), of
// which every SM takes an equal share; a unit that several CTAs share is joined by tree_merge_kernel.
// Per CTA, one pipeline over its whole share, across units:
//   warp 0      TMA producer, K and V tiles through one ring, in the order in which they are multiplied
//   warp 1      MMA issuer: S_t = Q K^T and O_t += P_t V for tile i, t = i mod 2
//   warps 2, 3  the rows of Q, packed by plain loads (any T, any strides), one unit ahead
//   warps 4-7   softmax of the even tiles, warps 8-11 of the odd ones: the same rows, a running maximum,
//               sum and accumulator of their own, thread r on row r
// The two softmax groups halve the time of a tile's exponentials, which one group alone would spend longer
// on (about 1850 clocks) than the tile's bytes take from memory per SM (about 1500 at two tiles in flight).
// P is rounded to the type of V, as in the prefill kernels; scores, sums and accumulators are fp32.
#include <type_traits>

#include "dependent.cuh"
#include "ptx.cuh"
#include "tc_util.cuh"
#include "tree.cuh"

namespace tsa {

namespace {

constexpr int kBM = 128, kBN = 128;
constexpr int kSlabBytes = 128 * 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescaleThreshold = 8.0f;  // log2 units

template <int D> struct TreeCfg {
  static constexpr int kSlabs = D / 64;
  static constexpr int kTileBytes = kSlabs * kSlabBytes;
  static constexpr int kStages = D == 128 ? 5 : 10;
  static constexpr int kOffKV = 2 * kTileBytes;  // behind the two buffers of Q
  static constexpr int kOffBar = kOffKV + kStages * kTileBytes;
  static constexpr int kSmem = kOffBar + 512 + 1024;  // barriers; alignment
  static constexpr uint32_t kColS = 0, kColO = 256;
};
constexpr int kMaxStages = 10;

struct TreeBars {
  uint64_t q_full[2], q_empty[2];
  uint64_t kv_full[kMaxStages], kv_empty[kMaxStages];
  uint64_t s_full[2], p_full[2], o_done[2], drain;
  int64_t rest, tiles;  // the share: its place within its first row, its length
  int row;
  uint32_t tmem_base;
};
static_assert(sizeof(TreeBars) <= 512, "barriers");

}  // namespace

template <int D, bool kBF16>
__global__ void __launch_bounds__(384, 1)
    attn_tree_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ TreeArgs args) {
  using C = TreeCfg<D>;
  constexpr int S = C::kStages;
  const ts_attn_params& p = args.p;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);
  TreeBars* bars = reinterpret_cast<TreeBars*>(smem + C::kOffBar);
  unsigned char* sQ = smem;
  unsigned char* sKV = smem + C::kOffKV;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(&bars->q_full[t], 2);
      ptx::mbar_init(&bars->q_empty[t], 1);
      ptx::mbar_init(&bars->s_full[t], 1);
      ptx::mbar_init(&bars->p_full[t], 4);
      ptx::mbar_init(&bars->o_done[t], 1);
    }
    for (int s = 0; s < S; ++s) {
      ptx::mbar_init(&bars->kv_full[s], 1);
      ptx::mbar_init(&bars->kv_empty[s], 1);
    }
    ptx::mbar_init(&bars->drain, 1);
    ptx::fence_mbar_init();
  }
  if (warp == 2) {
    ptx::tmem_alloc(&bars->tmem_base, 512);
    ptx::tmem_relinquish();
  }
  wait_for_previous();
  let_next_start();
  const TreeLine line(args, kBN);
  if (warp == 0) {
    int64_t before;
    const int64_t total = line_total(line, lane, 0, &before);
    const int ctas = (int)i64min(args.ctas, total);
    int row = 0;
    int64_t rest = 0, tiles = 0;
    if ((int)blockIdx.x < ctas) {
      const int64_t at = line_bound(blockIdx.x, total, ctas);
      tiles = line_bound(blockIdx.x + 1, total, ctas) - at;
      line_find(line, lane, at, &row, &rest);
    }
    if (lane == 0) {
      bars->row = row;
      bars->rest = rest;
      bars->tiles = fault_set(args.fault) ? 0 : tiles;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  const int64_t n_tiles = bars->tiles;
  LineWalk walk;
  walk.start(bars->row, bars->rest, n_tiles, line);

  if (warp < 4) {
    // 4 x 32 x 80 + 8 x 32 x 208 = 63488 of the 64512 registers of the launch
    ptx::setmaxnreg_dec<80>();
    if (warp == 0) {
      // ---------------------------- producer ------------------------------
      if (lane == 0 && n_tiles > 0) {
        ptx::prefetch_tensormap(&tm_k);
        ptx::prefetch_tensormap(&tm_v);
        LineWalk of[2] = {walk, walk};  // K is two tiles ahead of V
        int j[2] = {0, 0};
        int64_t f = 0;
        auto load = [&](int which) -> bool {
          LineWalk& w = of[which];
          if (j[which] == w.count) {
            if (!w.next(line)) return true;  // no tile left
            j[which] = 0;
          }
          const int s = (int)(f % S);
          if (f >= S && !wait_bar(&bars->kv_empty[s], (uint32_t)((f / S) - 1) & 1, args.fault, FAULT_FWD_EMPTY))
            return false;
          const int len = tree_len(p, w.b);
          const WindowTiles wt(args.win, (int64_t)len - p.q_len, len, kBN);
          const int key = wt.tile(w.first + j[which]) * kBN, hk = w.unit / args.row_tiles;
          ptx::mbar_expect_tx(&bars->kv_full[s], C::kTileBytes);
          for (int sl = 0; sl < C::kSlabs; ++sl)
            ptx::tma_load_4d(sKV + s * C::kTileBytes + sl * kSlabBytes, which ? &tm_v : &tm_k, 64 * sl, key, hk, w.b,
                             &bars->kv_full[s]);
          ++j[which];
          ++f;
          return true;
        };
        bool ok = load(0) && load(0);
        for (int64_t i = 0; i < n_tiles && ok; ++i) ok = load(1) && load(0);
        // Every issued copy must have landed before shared memory is released.
        for (int64_t g = i64max(0, f - S); g < f; ++g)
          (void)wait_bar(&bars->kv_full[g % S], (uint32_t)(g / S) & 1, nullptr, FAULT_FWD_DRAIN);
      }
    } else if (warp == 1) {
      // ---------------------------- MMA issuer ----------------------------
      if (lane == 0 && n_tiles > 0) {
        constexpr uint32_t idesc_qk = ptx::idesc_f16(kBF16, kBM, kBN, false, false);
        constexpr uint32_t idesc_pv = ptx::idesc_f16(kBF16, kBM, D, false, true);
        const uint32_t aQ = ptx::smem_u32(sQ), aKV = ptx::smem_u32(sKV);
        LineWalk ws = walk, wp = walk;  // of the next S and the next P.V
        int js = 0, jp = 0, seg = -1;   // tiles of their segments done; the S segment's number
        int64_t f = 0, is = 0, ip = 0;  // ring fills used, tiles done
        auto issue_s = [&]() -> bool {
          if (js == ws.count) {
            if (!ws.next(line)) return true;
            js = 0;
            ++seg;
            if (!wait_bar(&bars->q_full[seg & 1], (uint32_t)(seg >> 1) & 1, args.fault, FAULT_FWD_Q)) return false;
          }
          const int s = (int)(f % S);
          if (!wait_bar(&bars->kv_full[s], (uint32_t)(f / S) & 1, args.fault, FAULT_FWD_KV)) return false;
          ptx::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk >> 2) * kSlabBytes + (kk & 3) * 32;
            ptx::mma_f16_ss(tmem + C::kColS + (uint32_t)(is & 1) * kBN,
                            ptx::sw128_desc(aQ + (seg & 1) * C::kTileBytes + off, 16, 1024),
                            ptx::sw128_desc(aKV + s * C::kTileBytes + off, 16, 1024), idesc_qk, kk > 0 ? 1u : 0u);
          }
          ptx::mma_commit(&bars->s_full[is & 1]);
          ptx::mma_commit(&bars->kv_empty[s]);
          if (++js == ws.count) ptx::mma_commit(&bars->q_empty[seg & 1]);
          ++f;
          ++is;
          return true;
        };
        auto issue_pv = [&]() -> bool {
          if (jp == wp.count) {
            wp.next(line);
            jp = 0;
          }
          const int t = (int)(ip & 1), s = (int)(f % S);
          if (!wait_bar(&bars->kv_full[s], (uint32_t)(f / S) & 1, args.fault, FAULT_FWD_KV) ||
              !wait_bar(&bars->p_full[t], (uint32_t)(ip >> 1) & 1, args.fault, FAULT_FWD_P))
            return false;
          ptx::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < kBN / 16; ++kk)
            ptx::mma_f16_ts(tmem + C::kColO + (uint32_t)t * D, tmem + C::kColS + (uint32_t)t * kBN + 8 * kk,
                            ptx::sw128_desc(aKV + s * C::kTileBytes + kk * 16 * 128, kSlabBytes, 1024), idesc_pv,
                            (jp >= 2 || kk > 0) ? 1u : 0u);  // a segment's first tile of each group starts O_t
          ptx::mma_commit(&bars->kv_empty[s]);
          if (jp + 2 >= wp.count) ptx::mma_commit(&bars->o_done[t]);
          ++jp;
          ++f;
          ++ip;
          return true;
        };
        bool ok = issue_s() && issue_s();
        for (int64_t i = 0; i < n_tiles && ok; ++i) ok = issue_pv() && issue_s();
        ptx::mma_commit(&bars->drain);
        (void)wait_bar(&bars->drain, 0, nullptr, FAULT_FWD_DRAIN);
        if (!ok) record_fault(args.fault, FAULT_FWD_P);
      }
    } else {
      // ----------------------------- Q loaders ----------------------------
      using T = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
      const T* q = reinterpret_cast<const T*>(p.q.data);
      const int group = p.q_heads / p.kv_heads;
      constexpr int kChunks = D / 8;  // of 8 channels
      for (int seg = 0; walk.next(line); ++seg) {
        if (seg >= 2 && !__all_sync(0xffffffffu, wait_bar(&bars->q_empty[seg & 1], (uint32_t)((seg >> 1) - 1) & 1,
                                                          args.fault, FAULT_FWD_EMPTY)))
          break;
        const int hk = walk.unit / args.row_tiles, r0 = walk.unit % args.row_tiles * kBM;
        unsigned char* dst = sQ + (seg & 1) * C::kTileBytes;
        constexpr int kBatch = 8;  // loads in flight a thread
        for (int i0 = threadIdx.x - 64; i0 < kBM * kChunks; i0 += 64 * kBatch) {
          uint4 v[kBatch];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const int i = i0 + 64 * u, r = i / kChunks, c = i % kChunks;
            v[u] = make_uint4(0u, 0u, 0u, 0u);
            if (r0 + r < args.rows && 8 * c < p.head_dim) {
              const int h = hk * group + (r0 + r) / p.q_len, node = (r0 + r) % p.q_len;
              v[u] = *reinterpret_cast<const uint4*>(q + (int64_t)walk.b * p.q.stride[0] +
                                                     (int64_t)h * p.q.stride[1] + (int64_t)node * p.q.stride[2] +
                                                     8 * c);
            }
          }
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const int i = i0 + 64 * u, r = i / kChunks, c = i % kChunks;
            *reinterpret_cast<uint4*>(dst + (c >> 3) * kSlabBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[u];
          }
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&bars->q_full[seg & 1]);
      }
    }
  } else {
    // ------------------------- softmax warpgroups --------------------------
    ptx::setmaxnreg_inc<208>();
    const int t = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t t_row = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t col_s = C::kColS + (uint32_t)t * kBN;
    const uint32_t col_o = C::kColO + (uint32_t)t * D;
    const float qk_scale = (float)p.scale * kLog2e;
    int64_t i0 = 0;      // tiles of the share before this segment
    uint32_t done = 0;   // segments in which this group had a tile
    bool ok = true;
    while (ok && walk.next(line)) {
      const int r0 = walk.unit % args.row_tiles * kBM, b = walk.b;
      const int len = tree_len(p, b);
      const int64_t base = (int64_t)len - p.q_len;
      const WindowTiles wt(args.win, base, len, kBN);
      const bool live_warp = r0 + (warp & 3) * 32 < args.rows;  // some row of the warp is a query's
      const bool live = r0 + row < args.rows;
      const int32_t* parents = args.parents + b * args.parents_stride;
      NodeView view = tree_node((r0 + row) % p.q_len, base, !args.parents, args.win,
                                [&](int i) { return parents[i]; });
      if (!live) {
        view.end = 0;
        view.drafted = 0;
      }
      float m_run = -INFINITY, l_run = 0.f;
      const int j0 = (int)((t - i0) & 1);  // this group's first tile of the segment
      for (int j = j0; j < walk.count; j += 2) {
        const int64_t i = i0 + j;
        if (!__all_sync(0xffffffffu, wait_bar(&bars->s_full[t], (uint32_t)(i >> 1) & 1, args.fault, FAULT_FWD_S))) {
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        const int k0 = wt.tile(walk.first + j) * kBN;
        if (live_warp) {
          uint32_t r[kBN];
#pragma unroll
          for (int c = 0; c < kBN / 32; ++c)
            ptx::tmem_ld32(t_row + col_s + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(r + 32 * c));
          ptx::tmem_wait_ld();
          // Only tiles with drafted tokens, the cache's end, or an edge of some node's window are masked.
          const bool need_mask = k0 + kBN > base || (args.win.window > 0 && k0 + kBN > args.win.sinks &&
                                                     (int64_t)k0 <= (int64_t)len - 1 - args.win.window);
          uint32_t seen[4];
          float mx = -INFINITY;
          if (!need_mask) {
            float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
            for (int c = 0; c < kBN; c += 8) {
              m0 = ptx::max3(m0, __uint_as_float(r[c]), __uint_as_float(r[c + 1]));
              m1 = ptx::max3(m1, __uint_as_float(r[c + 2]), __uint_as_float(r[c + 3]));
              m2 = ptx::max3(m2, __uint_as_float(r[c + 4]), __uint_as_float(r[c + 5]));
              m3 = ptx::max3(m3, __uint_as_float(r[c + 6]), __uint_as_float(r[c + 7]));
            }
            mx = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
          } else {
#pragma unroll
            for (int w = 0; w < 4; ++w) seen[w] = view_bits(view, base, args.win.sinks, k0 + 32 * w);
#pragma unroll
            for (int c = 0; c < kBN; ++c)
              if ((seen[c >> 5] >> (c & 31)) & 1u) mx = fmaxf(mx, __uint_as_float(r[c]));
          }
          mx = mx == -INFINITY ? mx : mx * qk_scale;
          const float m_new = fmaxf(m_run, mx);
          const bool rescale =
              m_new > m_run + kRescaleThreshold || (m_run == -INFINITY && m_new != -INFINITY);
          float factor = 1.f;
          if (rescale) {
            factor = m_run == -INFINITY ? 0.f : ptx::ex2(m_run - m_new);
            m_run = m_new;
            l_run *= factor;
          }
          const float safe = m_run == -INFINITY ? 0.f : m_run;
          uint32_t pk[kBN / 2];
          uint64_t sum2[2] = {ptx::f2pack(0.f, 0.f), ptx::f2pack(0.f, 0.f)};
          const uint64_t sc2 = ptx::f2pack(qk_scale, qk_scale), ng2 = ptx::f2pack(-safe, -safe);
#pragma unroll
          for (int c = 0; c < kBN; c += 2) {
            float x0, x1;
            ptx::f2unpack(ptx::fma2(ptx::f2pack(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), sc2, ng2), x0, x1);
            float p0 = ptx::ex2(x0), p1 = ptx::ex2(x1);
            if (need_mask) {
              p0 = (seen[c >> 5] >> (c & 31)) & 1u ? p0 : 0.f;
              p1 = (seen[c >> 5] >> ((c & 31) + 1)) & 1u ? p1 : 0.f;
            }
            sum2[(c >> 1) & 1] = ptx::add2(sum2[(c >> 1) & 1], ptx::f2pack(p0, p1));
            pk[c / 2] = kBF16 ? ptx::pack_bf16(p0, p1) : ptx::pack_f16(p0, p1);
          }
          float a0, a1, b0, b1;
          ptx::f2unpack(sum2[0], a0, a1);
          ptx::f2unpack(sum2[1], b0, b1);
          l_run += (a0 + a1) + (b0 + b1);
          ptx::tmem_st32(t_row + col_s, *reinterpret_cast<const uint32_t(*)[32]>(pk));
          ptx::tmem_st32(t_row + col_s + 32, *reinterpret_cast<const uint32_t(*)[32]>(pk + 32));
          // S_t(i) was issued behind the group's last P.V, so O_t holds all of them: rescale it in place.
          if (j > j0 && __any_sync(0xffffffffu, rescale)) {
            if (!rescale) factor = 1.f;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              ptx::tmem_ld32(t_row + col_o + 32 * c, o);
              ptx::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
              ptx::tmem_st32(t_row + col_o + 32 * c, o);
            }
          }
          ptx::tmem_wait_st();
        }
        if (k0 + kBN > len) {
          // The cache may hold anything behind its last key: its values there become zeros, as 0 * NaN is NaN.
          const int64_t f = i64min(2 + 2 * i, 2 * n_tiles - 1);  // the fill that brought this tile's V
          unsigned char* v = sKV + (int)(f % S) * C::kTileBytes;
          if (!__all_sync(0xffffffffu,
                          wait_bar(&bars->kv_full[f % S], (uint32_t)(f / S) & 1, args.fault, FAULT_FWD_KV))) {
            ok = false;
            break;
          }
          const int gone = len - k0;  // first row to clear
          for (int x = row; x < (kBN - gone) * (D / 8); x += 128) {
            const int vr = gone + x / (D / 8), c = x % (D / 8);
            *reinterpret_cast<uint4*>(v + (c >> 3) * kSlabBytes + vr * 128 + ((c & 7) << 4)) =
                make_uint4(0u, 0u, 0u, 0u);
          }
          ptx::fence_proxy_async_smem();
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&bars->p_full[t]);
      }
      // The segment's partial result: channel quads of all rows, rows side by side.
      const bool any = j0 < walk.count;
      if (ok && any) {
        ok = __all_sync(0xffffffffu, wait_bar(&bars->o_done[t], done & 1, args.fault, FAULT_FWD_O));
        ++done;
      }
      ptx::tc_fence_after();
      const int64_t part = 2 * ((int64_t)b * line.units + walk.unit + blockIdx.x) + t;
      // A padded node has taken part in the tiles that need no mask: it has seen nothing.
      if (live) args.ml[part * args.part_rows + row] = view.depth < 0 ? make_float2(-INFINITY, 0.f) : make_float2(m_run, l_run);
      if (ok && any && live_warp) {
        float4* out = reinterpret_cast<float4*>(args.part + part * args.part_rows * p.head_dim);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          ptx::tmem_ld32(t_row + col_o + 32 * c, o);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (live && 32 * c + e < p.head_dim)
              out[(8 * c + e / 4) * args.part_rows + row] =
                  make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]),
                              __uint_as_float(o[e + 3]));
        }
      }
      // The next segment's first P_t must not start O_t over before it is read.
      ptx::tc_fence_before();
      i0 += walk.count;
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// Joining: out = sum_p 2^(m_p - m) O_p / sum_p 2^(m_p - m) l_p over the partial
// results p of a row.  One block a (unit, 8 rows); a thread holds one channel
// quad of a row over every kSplit-th part.
// ---------------------------------------------------------------------------
namespace {
constexpr int kMergeRows = 8, kMergeThreads = 256;
}

template <typename T>
__global__ void __launch_bounds__(kMergeThreads) tree_merge_kernel(const __grid_constant__ TreeArgs a, int tile_keys,
                                                                   int parts_of) {
  const ts_attn_params& p = a.p;
  __shared__ int64_t s_first, s_total;
  __shared__ float4 s_sum[kMergeThreads];
  wait_for_previous();
  let_next_start();
  const TreeLine line(a, tile_keys);
  const int unit = blockIdx.x % line.units, b = blockIdx.x / line.units;
  const int r0 = unit % a.row_tiles * a.tile_rows, row0 = blockIdx.y * kMergeRows;
  if (r0 + row0 >= a.rows) return;  // the last row tile is shorter
  if (threadIdx.x < 32) {
    int64_t before;
    const int64_t total = line_total(line, threadIdx.x, b, &before);
    if (threadIdx.x == 0) {
      s_first = before;
      s_total = total;
    }
  }
  __syncthreads();
  const int n = line.tiles(b);
  const int64_t total = s_total, at = s_first + (int64_t)unit * n;
  const int ctas = (int)i64min(a.ctas, total);
  int64_t part0 = 0;
  int parts = 0;
  if (n > 0) {
    const int c0 = line_owner(at, total, ctas), c1 = line_owner(at + n - 1, total, ctas);
    part0 = parts_of * ((int64_t)blockIdx.x + c0);
    parts = parts_of * (c1 - c0 + 1);
  }
  const int quads = part_quads(p);
  const int items = min(kMergeRows, a.rows - r0 - row0) * quads;  // (quad, row), rows fastest
  const int rows = items / quads;
  const int split = max(1, min(parts, kMergeThreads / max(1, items)));
  const int hk = unit / a.row_tiles, group = p.q_heads / p.kv_heads;
  for (int x0 = 0; x0 < items; x0 += kMergeThreads / split) {
    const int x = x0 + threadIdx.x % (kMergeThreads / split), s = threadIdx.x / (kMergeThreads / split);
    const bool mine = x < items && s < split;
    const int row = row0 + (mine ? x % rows : 0), quad = mine ? x / rows : 0;
    float m = -INFINITY, l = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mine) {
      const float2* ml = a.ml + part0 * a.part_rows + row;
      for (int i = 0; i < parts; ++i) m = fmaxf(m, ml[(int64_t)i * a.part_rows].x);
      if (m != -INFINITY) {
        for (int i = 0; i < parts; ++i) {
          const float2 v = ml[(int64_t)i * a.part_rows];
          if (v.x == -INFINITY) continue;
          const float w = ptx::ex2(v.x - m);
          l += w * v.y;
          if (i % split != s) continue;
          const float4 o = reinterpret_cast<const float4*>(
              a.part)[(part0 + i) * a.part_rows * quads + (int64_t)quad * a.part_rows + row];
          sum.x += w * o.x;
          sum.y += w * o.y;
          sum.z += w * o.z;
          sum.w += w * o.w;
        }
      }
    }
    s_sum[threadIdx.x] = sum;
    __syncthreads();
    if (mine && s == 0) {
      for (int i = 1; i < split; ++i) {
        const float4 o = s_sum[i * (kMergeThreads / split) + threadIdx.x];
        sum.x += o.x;
        sum.y += o.y;
        sum.z += o.z;
        sum.w += o.w;
      }
      const float inv = l > 0.f ? 1.f / l : 0.f;
      const int h = hk * group + (r0 + row) / p.q_len, node = (r0 + row) % p.q_len;
      T* out = reinterpret_cast<T*>(p.o.data) + (int64_t)b * p.o.stride[0] + (int64_t)h * p.o.stride[1] +
               (int64_t)node * p.o.stride[2] + (int64_t)(4 * quad) * p.o.stride[3];
      const float value[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * quad + e < p.value_dim) out[e * p.o.stride[3]] = Elem<T>::from_acc(value[e]);
      if (quad == 0 && p.lse)
        reinterpret_cast<float*>(p.lse)[(int64_t)b * p.lse_stride[0] + (int64_t)h * p.lse_stride[1] +
                                        (int64_t)node * p.lse_stride[2]] =
            l > 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int device_sms() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cached[dev] == 0) {
    int n = 0;
    cached[dev] =
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0 ? n : 148;
  }
  return cached[dev];
}

static bool rows16_ok(const ts_view4& v) {
  if (v.stride[3] != 1 || reinterpret_cast<uintptr_t>(v.data) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if ((v.stride[i] * 2) % 16) return false;
  return true;
}

bool tc_tree_supported(const ts_attn_params& p) {
  if (p.dtype != TS_BF16 && p.dtype != TS_F16) return false;
  if (p.head_dim != p.value_dim || p.head_dim % 8 || p.head_dim > 128) return false;
  if (!(p.scale > 0.0) || !rows16_ok(p.q) || !view_tma_ok(p.k) || !view_tma_ok(p.v)) return false;
  return encode_fn() != nullptr;
}

TreeArgs tree_args(const ts_attn_params& p, int tile_rows, int ctas, int parts_of, size_t* bytes) {
  TreeArgs a = {};
  a.p = p;
  a.rows = p.q_heads / p.kv_heads * p.q_len;
  a.tile_rows = tile_rows;
  a.row_tiles = ceil_div(a.rows, tile_rows);
  a.part_rows = min(a.rows, tile_rows);
  a.ctas = ctas;
  // Segments: one a unit, one more for every border between CTAs.
  const size_t parts = parts_of * ((size_t)p.batch * p.kv_heads * a.row_tiles + ctas);
  *bytes = parts * a.part_rows * (part_quads(p) * sizeof(float4) + sizeof(float2));
  return a;
}

void tree_place(TreeArgs* a, int parts_of, void* workspace) {
  const size_t parts = parts_of * ((size_t)a->p.batch * a->p.kv_heads * a->row_tiles + a->ctas);
  a->part = reinterpret_cast<float*>(workspace);
  a->ml = reinterpret_cast<float2*>(a->part + parts * a->part_rows * part_quads(a->p) * 4);
}

size_t tc_tree_workspace(const ts_attn_params& p) {
  size_t bytes;
  tree_args(p, kBM, device_sms(), 2, &bytes);
  return bytes;
}

cudaError_t tree_merge(const TreeArgs& a, int tile_keys, int parts_of, cudaStream_t st) {
  const dim3 grid((unsigned)(a.p.batch * a.p.kv_heads * a.row_tiles), (unsigned)ceil_div(a.part_rows, kMergeRows));
  switch (a.p.dtype) {
    case TS_F32: return launch_dependent(tree_merge_kernel<float>, grid, kMergeThreads, 0, st, a, tile_keys, parts_of);
    case TS_F16: return launch_dependent(tree_merge_kernel<__half>, grid, kMergeThreads, 0, st, a, tile_keys, parts_of);
    case TS_BF16:
      return launch_dependent(tree_merge_kernel<__nv_bfloat16>, grid, kMergeThreads, 0, st, a, tile_keys, parts_of);
  }
  return cudaErrorInvalidValue;
}

template <int D, bool BF16>
static cudaError_t launch_tree(const CUtensorMap& mk, const CUtensorMap& mv, const TreeArgs& a, cudaStream_t st) {
  auto kern = attn_tree_kernel<D, BF16>;
  const cudaError_t e = ensure_max_smem(reinterpret_cast<const void*>(kern), TreeCfg<D>::kSmem);
  if (e != cudaSuccess) return e;
  return launch_dependent(kern, dim3(a.ctas), dim3(384), TreeCfg<D>::kSmem, st, mk, mv, a);
}

cudaError_t tc_tree(const ts_attn_params& p, const int32_t* parents, int64_t parents_stride, const WindowArgs& win,
                    void* workspace, uint32_t* fault, cudaStream_t st) {
  size_t bytes;
  TreeArgs a = tree_args(p, kBM, device_sms(), 2, &bytes);
  tree_place(&a, 2, workspace);
  a.parents = parents;
  a.parents_stride = parents_stride;
  a.win = win;
  a.fault = fault;
  CUtensorMap mk, mv;
  if (!make_map(&mk, p.k, p.dtype, p.batch, p.kv_heads, p.kv_len, p.head_dim, kBN) ||
      !make_map(&mv, p.v, p.dtype, p.batch, p.kv_heads, p.kv_len, p.head_dim, kBN))
    return cudaErrorInvalidValue;
  const bool bf = p.dtype == TS_BF16;
  cudaError_t e;
  if (p.head_dim <= 64)
    e = bf ? launch_tree<64, true>(mk, mv, a, st) : launch_tree<64, false>(mk, mv, a, st);
  else
    e = bf ? launch_tree<128, true>(mk, mv, a, st) : launch_tree<128, false>(mk, mv, a, st);
  if (e != cudaSuccess) return e;
  return tree_merge(a, kBN, 2, st);
}

}  // namespace tsa
