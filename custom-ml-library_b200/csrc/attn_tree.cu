// Attention of drafted tokens over a contiguous KV cache on tcgen05 (bf16 / f16, head dimensions that are
// multiples of 8 up to 128): out = softmax(scale q K^T) V over the keys that tree.cuh's rule lets a node see.
//
// The T drafted tokens of the query heads that share a KV head are the rows of a 128-row tile, so that every
// key is read once for all of them.  The work is one line of 128-key tiles over (row, KV head, row tile), of
// which every SM takes an equal share; a unit that several CTAs share is joined by tree_merge_kernel.
// Per CTA, one pipeline over its whole share, across units:
//   warp 0      TMA producer, K and V tiles through one ring, in the order in which they are multiplied
//   warp 1      MMA issuer: S(i + 1) = Q K(i + 1)^T, then O_t += P_t(i) V(i) for the two halves t of the keys
//   warps 2, 3  the rows of Q, packed by plain loads (any T, any strides), one unit ahead
//   warps 4-7   softmax of the lower 64 keys of every tile, warps 8-11 of the upper ones: the same rows, a
//               running maximum, sum and accumulator of their own, thread r on row r; joined at a unit's end
// S is a tile ahead, so a V tile waits in the ring for its own P alone and the rest of the ring is in flight.
// (Groups on alternate whole tiles hold two V tiles back, and the ring then keeps too little in flight: 198
// against 150 us for 32 rows of 500 to 8192 keys, 16 nodes; six slots instead of five, with the queries of up to 64
// rows in half the room, 125.)
// Bounded by memory for long caches: those 32 rows read 578 MB, 89 us at the rate of a copy, in 116 us of this kernel,
// 14 of them until the first tile has come and 10 for the spread of the CTAs' ends; the join takes the other 9.  Few
// rows and short caches are a chain of latencies: 2.5 us to plan, 2 for the first keys, 2.5 for the first softmax
// (instructions come from L2), 1.8 a tile, 9 to join 37 parts (28 us for 2 rows of 32768 visible keys on 2 heads, 12 for
// 37 keys on 4).
// P is rounded to the type of V, as in the prefill kernels; scores, sums and accumulators are fp32.
#include <type_traits>

#include "dependent.cuh"
#include "ptx.cuh"
#include "tc_util.cuh"
#include "tree.cuh"

namespace tsa {

namespace {

constexpr int kBM = 128, kBN = 128, kHalf = kBN / 2;
constexpr int kUnitPlaces = 2;  // what a unit's start and end cost, in tiles (about 2.5 us; a tile takes 1.65)
constexpr int kSlabBytes = 128 * 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescaleThreshold = 8.0f;  // log2 units

template <int D> struct TreeCfg {
  static constexpr int kSlabs = D / 64;
  static constexpr int kTileBytes = kSlabs * kSlabBytes;
  // Two buffers of Q and a ring of K and V tiles share kTiles tiles' room.  Up to 64 rows the buffers of Q take half
  // of it each (the products then read other bytes for the rows behind, whose results are not used).
  static constexpr int kTiles = D == 128 ? 7 : 12;
  static constexpr int kOffBar = kTiles * kTileBytes;
  static constexpr int kSmem = kOffBar + 1536 + 1024;  // barriers; alignment
  static constexpr uint32_t kColS = 0, kColO = 256;
};
constexpr int kMaxStages = 11;

struct TreeBars {
  uint64_t q_full[2], q_empty[2];
  uint64_t kv_full[kMaxStages], kv_empty[kMaxStages];
  uint64_t s_full[2], p_full[2], o_done[2], drain;
  uint64_t halves, joined, o_read;  // at a segment's end: the upper half's sums, the factors, O read by both groups
  LinePlace from;  // the share's beginning
  int64_t tiles;   // and its tiles
  uint32_t tmem_base;
  float2 red[kBM];
};
static_assert(sizeof(TreeBars) <= 1536, "barriers");

}  // namespace

template <int D, bool kBF16>
__global__ void __launch_bounds__(384, 1)
    attn_tree_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ TreeArgs args) {
  using C = TreeCfg<D>;
  const ts_attn_params& p = args.p;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);
  TreeBars* bars = reinterpret_cast<TreeBars*>(smem + C::kOffBar);
  const bool low = args.part_rows <= kBM / 2;
  const int S = C::kTiles - (low ? 1 : 2);                        // slots of the ring
  const int q_slab = low ? kSlabBytes / 2 : kSlabBytes;           // 64 channels of a buffer's rows
  unsigned char* sQ = smem;                                       // buffer i at i * kSlabs * q_slab
  unsigned char* sKV = smem + (low ? 1 : 2) * C::kTileBytes;
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
    ptx::mbar_init(&bars->halves, 4);
    ptx::mbar_init(&bars->joined, 4);
    ptx::mbar_init(&bars->o_read, 8);
    ptx::fence_mbar_init();
  }
  if (warp == 2) {
    ptx::tmem_alloc(&bars->tmem_base, 512);
    ptx::tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&tm_k);
    ptx::prefetch_tensormap(&tm_v);
  }
  wait_for_previous();
  let_next_start();
  const TreeLine line(args, kBN, kUnitPlaces);
  if (warp == 0) {
    const bool faulted = fault_set(args.fault);  // under way during the planning
    LinePlace ends[2];
    line_share(line, lane, blockIdx.x, args.ctas, ends);
    if (lane == 0) {
      bars->from = ends[0];
      bars->tiles = faulted ? 0 : ends[1].tiles - ends[0].tiles;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  const int64_t n_tiles = bars->tiles;
  LineWalk walk;
  walk.start(bars->from, n_tiles, line);

  if (warp < 4) {
    // 4 x 32 x 80 + 8 x 32 x 208 = 63488 of the 64512 registers of the launch
    ptx::setmaxnreg_dec<80>();
    if (warp == 0) {
      // ---------------------------- producer ------------------------------
      if (lane == 0 && n_tiles > 0) {
        // K is a tile ahead of V: they walk along the share by themselves.
        struct Stream {
          LineWalk walk;
          int j, hk;
        } of[2] = {{walk, 0, 0}, {walk, 0, 0}};
        int slot = 0, fills = 0;
        uint32_t phase = 1;  // of kv_empty: the ring's first round finds every slot free
        auto load = [&](Stream& w, const CUtensorMap* map) -> bool {
          if (w.j == w.walk.count) {
            if (!w.walk.next(line)) return true;  // no tile left
            w.j = 0;
            w.hk = w.walk.unit / args.row_tiles;
          }
          if (fills >= S && !wait_bar(&bars->kv_empty[slot], phase, args.fault, FAULT_FWD_EMPTY)) return false;
          const int key = w.walk.list.tiles.tile(w.walk.first + w.j) * kBN;
          ptx::mbar_expect_tx(&bars->kv_full[slot], C::kTileBytes);
          for (int sl = 0; sl < C::kSlabs; ++sl)
            ptx::tma_load_4d(sKV + slot * C::kTileBytes + sl * kSlabBytes, map, 64 * sl, key, w.hk, w.walk.b,
                             &bars->kv_full[slot]);
          ++w.j;
          fills = min(fills + 1, S);
          if (++slot == S) slot = 0, phase ^= 1;
          return true;
        };
        bool ok = load(of[0], &tm_k);
        for (int64_t i = 0; i < n_tiles && ok; ++i) ok = load(of[0], &tm_k) && load(of[1], &tm_v);
        // Every issued copy must have landed before shared memory is released.  kv_full's phase of a round is the
        // opposite of kv_empty's for the round before; slots before `slot` were filled in the present round.
        for (int s = 0; s < S; ++s) {
          const uint32_t round = s < slot ? phase ^ 1 : phase;
          if (s < slot || fills == S) (void)wait_bar(&bars->kv_full[s], round, nullptr, FAULT_FWD_DRAIN);
        }
      }
    } else if (warp == 1) {
      // ---------------------------- MMA issuer ----------------------------
      if (lane == 0 && n_tiles > 0) {
        constexpr uint32_t idesc_qk = ptx::idesc_f16(kBF16, kBM, kBN, false, false);
        constexpr uint32_t idesc_pv = ptx::idesc_f16(kBF16, kBM, D, false, true);
        const uint32_t aQ = ptx::smem_u32(sQ), aKV = ptx::smem_u32(sKV);
        LineWalk ws = walk, wp = walk;  // of the next S and the next P.V
        int js = 0, jp = 0, seg = -1;   // tiles of their segments done; the S segment's number
        uint32_t is = 0, ip = 0;        // tiles done (their lowest bits count)
        int s = 0;                      // the ring's next slot
        uint32_t round = 0;
        auto used = [&] {
          if (++s == S) s = 0, round ^= 1;
        };
        auto issue_s = [&]() -> bool {
          if (js == ws.count) {
            if (!ws.next(line)) return true;
            js = 0;
            ++seg;
            if (!wait_bar(&bars->q_full[seg & 1], (uint32_t)(seg >> 1) & 1, args.fault, FAULT_FWD_Q)) return false;
          }
          if (!wait_bar(&bars->kv_full[s], round, args.fault, FAULT_FWD_KV)) return false;
          ptx::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            ptx::mma_f16_ss(
                tmem + C::kColS + (is & 1) * kBN,
                ptx::sw128_desc(aQ + ((seg & 1) * C::kSlabs + (kk >> 2)) * q_slab + (kk & 3) * 32, 16, 1024),
                ptx::sw128_desc(aKV + s * C::kTileBytes + (kk >> 2) * kSlabBytes + (kk & 3) * 32, 16, 1024), idesc_qk,
                kk > 0 ? 1u : 0u);
          ptx::mma_commit(&bars->s_full[is & 1]);
          ptx::mma_commit(&bars->kv_empty[s]);
          if (++js == ws.count) ptx::mma_commit(&bars->q_empty[seg & 1]);
          used();
          ++is;
          return true;
        };
        // P(i) V(i), the two halves of the tile's keys into their own accumulators.
        auto issue_pv = [&]() -> bool {
          if (jp == wp.count) {
            wp.next(line);
            jp = 0;
          }
          if (!wait_bar(&bars->kv_full[s], round, args.fault, FAULT_FWD_KV)) return false;
          for (int t = 0; t < 2; ++t) {
            if (!wait_bar(&bars->p_full[t], ip & 1, args.fault, FAULT_FWD_P)) return false;
            ptx::tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < kHalf / 16; ++kk)
              ptx::mma_f16_ts(tmem + C::kColO + (uint32_t)t * D,
                              tmem + C::kColS + (ip & 1) * kBN + t * kHalf + 8 * kk,
                              ptx::sw128_desc(aKV + s * C::kTileBytes + (t * kHalf + kk * 16) * 128, kSlabBytes, 1024),
                              idesc_pv, (jp > 0 || kk > 0) ? 1u : 0u);  // a segment's first tile starts O_t
            ptx::mma_commit(&bars->o_done[t]);
          }
          ptx::mma_commit(&bars->kv_empty[s]);
          ++jp;
          used();
          ++ip;
          return true;
        };
        bool ok = issue_s();
        for (int64_t i = 0; i < n_tiles && ok; ++i) ok = issue_s() && issue_pv();
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
        unsigned char* dst = sQ + (seg & 1) * C::kSlabs * q_slab;
        const int rows = min(kBM, args.rows - r0);  // what the rows behind them give is not used
        const int c = (threadIdx.x - 64) % kChunks;
        const T* from = q + (int64_t)walk.b * p.q.stride[0] + (int64_t)(hk * group) * p.q.stride[1] + 8 * c;
        for (int r = (threadIdx.x - 64) / kChunks; r < rows; r += 64 / kChunks) {
          unsigned char* to = dst + (c >> 3) * q_slab + r * 128 + (((c & 7) ^ (r & 7)) << 4);
          const int h = (r0 + r) / p.q_len, node = r0 + r - h * p.q_len;
          if (8 * c < p.head_dim)
            ptx::copy16_async(to, from + (int64_t)h * p.q.stride[1] + (int64_t)node * p.q.stride[2]);
          else
            *reinterpret_cast<uint4*>(to) = make_uint4(0u, 0u, 0u, 0u);
        }
        ptx::copies_done();
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&bars->q_full[seg & 1]);
      }
    }
  } else {
    // ------------------------- softmax warpgroups --------------------------
    ptx::setmaxnreg_inc<208>();
    const int t = (warp - 4) >> 2;  // half of a tile's keys
    const int row = (warp & 3) * 32 + lane;
    const uint32_t t_row = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t col_o = C::kColO + (uint32_t)t * D;
    const float qk_scale = (float)p.scale * kLog2e;
    int64_t i = 0;  // tile of the share
    NodeView view;
    uint64_t hidden = 0;  // of row view_b
    int view_b = -1, view_r0 = -1;
    bool ok = true;
    for (int seg = 0; ok && walk.next(line); ++seg) {
      const int r0 = walk.unit % args.row_tiles * kBM, b = walk.b;
      const int len = tree_len(p, b);
      const int64_t base = (int64_t)len - p.q_len;
      const WindowTiles& wt = walk.list.tiles;
      // Keys that all the tile's queries see: those before the first of a chain's tokens and it, a tree's committed ones.
      const int64_t common = args.parents ? base : walk.list.first + 1;
      const bool live_warp = r0 + (warp & 3) * 32 < args.rows;  // some row of the warp is a query's
      const bool live = r0 + row < args.rows;
      if (b != view_b || r0 != view_r0) {  // the heads of a row share it
        view = tree_node_of_warp((r0 + row) % p.q_len, p.q_len, base, args, b, lane, &hidden);
        if (!live) {
          view.end = 0;
          view.drafted = 0;
        }
        view_b = b;
        view_r0 = r0;
      }
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = 0; j < walk.count; ++j, ++i) {
        const uint32_t t_s = t_row + C::kColS + (uint32_t)(i & 1) * kBN + t * kHalf;
        if (!__all_sync(0xffffffffu, wait_bar(&bars->s_full[i & 1], (uint32_t)(i >> 1) & 1, args.fault, FAULT_FWD_S))) {
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        const int k0 = wt.tile(walk.first + j) * kBN, kh = k0 + t * kHalf;
        bool rescale = false;
        float factor = 1.f;
        if (live_warp) {
          uint32_t r[kHalf];
#pragma unroll
          for (int c = 0; c < kHalf / 32; ++c)
            ptx::tmem_ld32(t_s + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(r + 32 * c));
          ptx::tmem_wait_ld();
          // Only halves with drafted tokens, the cache's end, or an edge of some node's window are masked.
          const bool need_mask = kh + kHalf > common || (args.win.window > 0 && kh + kHalf > args.win.sinks &&
                                                         (int64_t)kh <= walk.list.last - args.win.window);
          uint32_t seen[2];
          float mx = -INFINITY;
          if (!need_mask) {
            float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
            for (int c = 0; c < kHalf; c += 4) {
              m0 = ptx::max3(m0, __uint_as_float(r[c]), __uint_as_float(r[c + 1]));
              m1 = ptx::max3(m1, __uint_as_float(r[c + 2]), __uint_as_float(r[c + 3]));
            }
            mx = fmaxf(m0, m1);
          } else {
#pragma unroll
            for (int w = 0; w < 2; ++w) seen[w] = view_bits(view, base, args.win.sinks, kh + 32 * w);
#pragma unroll
            for (int c = 0; c < kHalf; ++c)
              if ((seen[c >> 5] >> (c & 31)) & 1u) mx = fmaxf(mx, __uint_as_float(r[c]));
          }
          mx = mx == -INFINITY ? mx : mx * qk_scale;
          const float m_new = fmaxf(m_run, mx);
          rescale = m_new > m_run + kRescaleThreshold || (m_run == -INFINITY && m_new != -INFINITY);
          if (rescale) {
            factor = m_run == -INFINITY ? 0.f : ptx::ex2(m_run - m_new);
            m_run = m_new;
            l_run *= factor;
          }
          const float safe = m_run == -INFINITY ? 0.f : m_run;
          uint32_t pk[kHalf / 2];
          uint64_t sum2[2] = {ptx::f2pack(0.f, 0.f), ptx::f2pack(0.f, 0.f)};
          const uint64_t sc2 = ptx::f2pack(qk_scale, qk_scale), ng2 = ptx::f2pack(-safe, -safe);
#pragma unroll
          for (int c = 0; c < kHalf; c += 2) {
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
          // P over the first half of the scores that this thread has read.
          ptx::tmem_st32(t_s, *reinterpret_cast<const uint32_t(*)[32]>(pk));
        }
        // O_t holds the products up to the tile before once those have completed.  Warps without a live row wait as
        // well: S is a tile ahead, and what they say of one tile must not count for the tile before.
        if (j > 0 && !__all_sync(0xffffffffu,
                                 wait_bar(&bars->o_done[t], (uint32_t)(i - 1) & 1, args.fault, FAULT_FWD_O))) {
          ok = false;
          break;
        }
        if (live_warp) {
          if (j > 0 && __any_sync(0xffffffffu, rescale)) {
            ptx::tc_fence_after();
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
        const bool hides = hidden && kh + kHalf > base && kh < base + p.q_len;
        if (kh + kHalf > len || hides) {
          // The cache may hold anything behind its last key and in the slots of padded nodes: its values there become
          // zeros, as 0 * NaN is NaN.
          const int64_t f = i64min(2 + 2 * i, 2 * n_tiles - 1);  // the fill that brought this tile's V
          unsigned char* v = sKV + (int)(f % S) * C::kTileBytes;
          if (!__all_sync(0xffffffffu,
                          wait_bar(&bars->kv_full[f % S], (uint32_t)(f / S) & 1, args.fault, FAULT_FWD_KV))) {
            ok = false;
            break;
          }
          auto clear = [&](int hr, int c) {  // 8 channels of a row of the half
            *reinterpret_cast<uint4*>(v + (c >> 3) * kSlabBytes + (t * kHalf + hr) * 128 + ((c & 7) << 4)) =
                make_uint4(0u, 0u, 0u, 0u);
          };
          const int gone = max(len - kh, 0);  // first row behind the last key
          for (int x = row; x < (kHalf - gone) * (D / 8); x += 128) clear(gone + x / (D / 8), x % (D / 8));
          if (hides) {
            const uint64_t bits = gone_bits(hidden, base, len, kh);
            for (int x = row; x < kHalf * (D / 8); x += 128)
              if ((bits >> (x / (D / 8))) & 1u) clear(x / (D / 8), x % (D / 8));
          }
          ptx::fence_proxy_async_smem();
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&bars->p_full[t]);
      }
      // A padded node has taken part in the tiles that need no mask: it has seen nothing.
      if (view.depth < 0) m_run = -INFINITY, l_run = 0.f;
      // Join the halves: both groups learn the row's reference and sum and their accumulators' factors.
      if (ok && t == 1) bars->red[row] = make_float2(m_run, l_run);
      __syncwarp();
      if (t == 1 && lane == 0) ptx::mbar_arrive(&bars->halves);
      float own = 0.f, other = 0.f;  // factors of this group's accumulator and of the other one
      if (t == 0) {
        ok = __all_sync(0xffffffffu, wait_bar(&bars->halves, (uint32_t)seg & 1, args.fault, FAULT_FWD_O) && ok);
        const float2 high = bars->red[row];
        const float m = fmaxf(m_run, high.x), safe = m == -INFINITY ? 0.f : m;
        own = m_run == -INFINITY ? 0.f : ptx::ex2(m_run - safe);
        other = high.x == -INFINITY ? 0.f : ptx::ex2(high.x - safe);
        const int64_t part = (int64_t)b * line.units + walk.unit + blockIdx.x;
        if (live) args.ml[part * args.part_rows + row] = make_float2(m, own * l_run + other * high.y);
        bars->red[row] = make_float2(other, own);
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&bars->joined);
      } else {
        ok = __all_sync(0xffffffffu, wait_bar(&bars->joined, (uint32_t)seg & 1, args.fault, FAULT_FWD_O) && ok);
        const float2 factors = bars->red[row];
        own = factors.x;
        other = factors.y;
      }
      // The segment's partial result: channel quads of all rows, rows side by side; each group half of the channels.
      if (ok)
        ok = __all_sync(0xffffffffu,
                        wait_bar(&bars->o_done[0], (uint32_t)(i - 1) & 1, args.fault, FAULT_FWD_O) &&
                            wait_bar(&bars->o_done[1], (uint32_t)(i - 1) & 1, args.fault, FAULT_FWD_O));
      ptx::tc_fence_after();
      if (ok && live_warp) {
        const int64_t part = (int64_t)b * line.units + walk.unit + blockIdx.x;
        float4* out = reinterpret_cast<float4*>(args.part + part * args.part_rows * p.head_dim);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const int ch = t * (D / 2) + 32 * c;
          uint32_t o[32], x[32];
          ptx::tmem_ld32(t_row + col_o + ch, o);
          ptx::tmem_ld32(t_row + C::kColO + (uint32_t)(1 - t) * D + ch, x);
          ptx::tmem_wait_ld();
          auto joined = [&](int e) {  // an accumulator without a key may hold anything
            const float a = own == 0.f ? 0.f : own * __uint_as_float(o[e]);
            return other == 0.f ? a : fmaf(other, __uint_as_float(x[e]), a);
          };
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (live && ch + e < p.head_dim)
              out[((ch + e) / 4) * args.part_rows + row] =
                  make_float4(joined(e), joined(e + 1), joined(e + 2), joined(e + 3));
        }
      }
      // Both groups have read both accumulators before the next segment's first product starts them over.
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&bars->o_read);
      ok = __all_sync(0xffffffffu, wait_bar(&bars->o_read, (uint32_t)seg & 1, args.fault, FAULT_FWD_O) && ok);
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
// results p of a row.  blockIdx.y takes a share of a unit's (channel quad, row)
// items, rows fastest; where a share has fewer items than the block threads,
// several threads take every split-th partial result of an item.
// ---------------------------------------------------------------------------
namespace {
constexpr int kMergeThreads = 256, kFewParts = 4, kMergeParts = 8;  // partial results in flight a thread
}

template <typename T>
__global__ void __launch_bounds__(kMergeThreads)
    tree_merge_kernel(const __grid_constant__ TreeArgs a, int tile_keys, int start_places, int share) {
  const ts_attn_params& p = a.p;
  __shared__ int64_t s_first, s_total;
  __shared__ int s_tiles;
  __shared__ float2 s_row[kMergeThreads];  // reference and sum of every row, of several slices of its results first
  __shared__ float4 s_sum[kMergeThreads];
  const TreeLine line(a, tile_keys, start_places, true);
  const int unit = blockIdx.x % line.units, b = blockIdx.x / line.units;
  const int r0 = unit % a.row_tiles * a.tile_rows, rows = min(a.tile_rows, a.rows - r0);
  const int quads = part_quads(p), items = rows * quads, first = blockIdx.y * share;
  if (first >= items) {  // the last row tile is shorter
    wait_for_previous();
    return;
  }
  const int mine = min(share, items - first);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (warp == 0) {
    int64_t before;
    const int64_t total = line_total(line, lane, b, &before);
    if (lane == 0) {
      const int h = unit / line.row_tiles, t = unit % line.row_tiles;
      if (h > 0) {
        int64_t places, tiles;
        line.head(b, &places, &tiles);
        before += h * places;
      }
      for (int x = 0; x < t; ++x) before += line.places(line.list(b, x).count);
      s_tiles = line.list(b, t).count;
      s_first = before;
      s_total = total;
    }
  }
  __syncthreads();
  const int n = s_tiles;
  const int64_t total = s_total, at = s_first + start_places;  // its first tile's place
  const int ctas = (int)i64min(a.ctas, total);
  int64_t part0 = 0;
  int parts = 0;
  if (n > 0) {
    const int c0 = line_owner(at, total, ctas), c1 = line_owner(at + n - 1, total, ctas);
    part0 = (int64_t)blockIdx.x + c0;
    parts = c1 - c0 + 1;
  }
  wait_for_previous();
  let_next_start();
  const float2* ml = a.ml + part0 * a.part_rows;
  const int hk = unit / a.row_tiles, group = p.q_heads / p.kv_heads;
  const float4* from = reinterpret_cast<const float4*>(a.part) + part0 * a.part_rows * quads;
  auto write_lse = [&](int row, float m, float l) {
    const int h = hk * group + (r0 + row) / p.q_len, node = (r0 + row) % p.q_len;
    reinterpret_cast<float*>(p.lse)[(int64_t)b * p.lse_stride[0] + (int64_t)h * p.lse_stride[1] +
                                    (int64_t)node * p.lse_stride[2]] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  };
  // A quad of the output in one store, where its rows lie on such boundaries.
  const bool whole = p.o.stride[3] == 1 && p.value_dim % 4 == 0 &&
                     ((reinterpret_cast<uintptr_t>(p.o.data) / sizeof(T)) | p.o.stride[0] | p.o.stride[1] | p.o.stride[2]) % 4 == 0;
  auto write = [&](int row, int quad, float4 sum, float inv) {
    const int h = hk * group + (r0 + row) / p.q_len, node = (r0 + row) % p.q_len;
    T* out = reinterpret_cast<T*>(p.o.data) + (int64_t)b * p.o.stride[0] + (int64_t)h * p.o.stride[1] +
             (int64_t)node * p.o.stride[2] + (int64_t)(4 * quad) * p.o.stride[3];
    alignas(4 * sizeof(T)) const T value[4] = {Elem<T>::from_acc(sum.x * inv), Elem<T>::from_acc(sum.y * inv),
                                               Elem<T>::from_acc(sum.z * inv), Elem<T>::from_acc(sum.w * inv)};
    if (whole) {
      struct alignas(4 * sizeof(T)) Four {
        T v[4];
      };
      *reinterpret_cast<Four*>(out) = *reinterpret_cast<const Four*>(value);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * quad + e < p.value_dim) out[e * p.o.stride[3]] = value[e];
    }
  };
  // Of a result whose reference is x.  One without a reference has seen nothing, or NaN alone: 0 times its sum, 0 or
  // NaN, is what it adds to the row's.
  auto weight = [](float x, float m) { return x == -INFINITY ? 0.f : ptx::ex2(x - m); };
  auto add = [](float4& sum, float w, const float4& o) {
    if (w == 0.f) return;  // a part that has seen nothing may hold anything
    sum.x = fmaf(w, o.x, sum.x);
    sum.y = fmaf(w, o.y, sum.y);
    sum.z = fmaf(w, o.z, sum.z);
    sum.w = fmaf(w, o.w, sum.w);
  };
  if (parts <= kFewParts) {
    // Few results: a thread reads all that its item needs at once.
    for (int x = threadIdx.x; x < mine; x += kMergeThreads) {
      const int row = (first + x) % rows, quad = (first + x) / rows;
      float2 v[kFewParts];
      float4 o[kFewParts], sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kFewParts; ++i) {
        v[i] = make_float2(-INFINITY, 0.f);
        if (i < parts) {
          v[i] = ml[i * a.part_rows + row];
          o[i] = from[(int64_t)i * a.part_rows * quads + (int64_t)quad * a.part_rows + row];
        }
      }
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int i = 0; i < kFewParts; ++i) m = fmaxf(m, v[i].x);
#pragma unroll
      for (int i = 0; i < kFewParts; ++i) {
        const float w = weight(v[i].x, m);
        l = fmaf(w, v[i].y, l);
        add(sum, w, o[i]);
      }
      write(row, quad, sum, l > 0.f ? 1.f / l : l);  // a sum that is NaN stays one
      if (quad == 0 && p.lse) write_lse(row, m, l);
    }
    return;
  }
  // Threads over an item's results; the first of them are under way while the rows' numbers are found.
  const int split = max(1, min(parts, kMergeThreads / mine)), lanes = kMergeThreads / split;
  const int slot = threadIdx.x % lanes, s = threadIdx.x / lanes;
  float4 o[kMergeParts];
  auto load = [&](int x, int i0) {
    const int row = (first + x) % rows, quad = (first + x) / rows;
#pragma unroll
    for (int u = 0; u < kMergeParts; ++u)
      if (i0 + u * split < parts)
        o[u] = from[(int64_t)(i0 + u * split) * a.part_rows * quads + (int64_t)quad * a.part_rows + row];
  };
  if (slot < mine && s < split) load(slot, s);
  const int slices = kMergeThreads / rows, row_slice = threadIdx.x / rows;
  if (row_slice < slices) {
    const int row = threadIdx.x % rows;
    float m = -INFINITY, l = 0.f;
    for (int i0 = row_slice; i0 < parts; i0 += slices * kFewParts) {
      float2 v[kFewParts];
      float top = m;
#pragma unroll
      for (int u = 0; u < kFewParts; ++u) {
        const int i = i0 + u * slices;
        v[u] = i < parts ? ml[(int64_t)i * a.part_rows + row] : make_float2(-INFINITY, 0.f);
      }
#pragma unroll
      for (int u = 0; u < kFewParts; ++u) top = fmaxf(top, v[u].x);
      l *= weight(m, top);
#pragma unroll
      for (int u = 0; u < kFewParts; ++u) l = fmaf(weight(v[u].x, top), v[u].y, l);
      m = top;
    }
    s_row[threadIdx.x] = make_float2(m, l);
  }
  __syncthreads();
  for (int n = slices; n > 1;) {  // the slices' numbers, upper halves into lower ones
    const int half = (n + 1) / 2;
    if (row_slice < n - half) {
      const float2 x = s_row[threadIdx.x], y = s_row[threadIdx.x + half * rows];
      const float m = fmaxf(x.x, y.x);
      s_row[threadIdx.x] = make_float2(m, fmaf(weight(y.x, m), y.y, weight(x.x, m) * x.y));
    }
    __syncthreads();
    n = half;
  }
  if (blockIdx.y == 0 && p.lse && row_slice == 0) write_lse(threadIdx.x, s_row[threadIdx.x].x, s_row[threadIdx.x].y);
  for (int x0 = 0; x0 < mine; x0 += lanes) {
    const int x = x0 + slot;
    const bool live = x < mine && s < split;
    const float2 total = s_row[live ? (first + x) % rows : 0];
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live && total.x != -INFINITY) {
      const int row = (first + x) % rows;
      for (int i0 = s; i0 < parts; i0 += split * kMergeParts) {
        if (x0 > 0 || i0 > s) load(x, i0);
        float w[kMergeParts];
#pragma unroll
        for (int u = 0; u < kMergeParts; ++u) {
          const int i = i0 + u * split;
          w[u] = i < parts ? ptx::ex2(ml[(int64_t)i * a.part_rows + row].x - total.x) : 0.f;  // 0 where it has seen nothing
        }
#pragma unroll
        for (int u = 0; u < kMergeParts; ++u) add(sum, w[u], o[u]);
      }
    }
    if (split > 1) {
      s_sum[threadIdx.x] = sum;
      __syncthreads();
      if (live && s == 0)
        for (int i = 1; i < split; ++i) {
          const float4 y = s_sum[i * lanes + threadIdx.x];
          sum.x += y.x;
          sum.y += y.y;
          sum.z += y.z;
          sum.w += y.w;
        }
      __syncthreads();
    }
    if (live && s == 0) write((first + x) % rows, (first + x) / rows, sum, total.y > 0.f ? 1.f / total.y : total.y);
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

// Partial results: segments of the line, one a unit and one more for every border between CTAs.
static size_t tree_parts(const TreeArgs& a) {
  return (size_t)a.p.batch * a.p.kv_heads * a.row_tiles + a.ctas;
}

TreeArgs tree_args(const ts_attn_params& p, int tile_rows, int ctas, size_t* bytes) {
  TreeArgs a = {};
  a.p = p;
  a.rows = p.q_heads / p.kv_heads * p.q_len;
  a.tile_rows = tile_rows;
  a.row_tiles = ceil_div(a.rows, tile_rows);
  a.part_rows = min(a.rows, tile_rows);
  a.ctas = ctas;
  *bytes = tree_parts(a) * a.part_rows * (part_quads(p) * sizeof(float4) + sizeof(float2));
  return a;
}

void tree_place(TreeArgs* a, void* workspace) {
  a->part = reinterpret_cast<float*>(workspace);
  a->ml = reinterpret_cast<float2*>(a->part + tree_parts(*a) * a->part_rows * part_quads(a->p) * 4);
}

size_t tc_tree_workspace(const ts_attn_params& p) {
  size_t bytes;
  tree_args(p, kBM, device_sms(), &bytes);
  return bytes;
}

cudaError_t tree_merge(const TreeArgs& a, int tile_keys, int start_places, cudaStream_t st) {
  // Blocks for the SMs two or three times over, with shares of 64 items at least, or of so few that a thread reads all
  // that it takes of an item at once.
  const int units = a.p.batch * a.p.kv_heads * a.row_tiles, items = a.part_rows * part_quads(a.p);
  const int parts = ceil_div(a.ctas, units) + 1;  // of a unit of ordinary length
  const int least = max(8, min(64, kMergeThreads * kMergeParts / parts));
  const int share = max(least, ceil_div(items, max(1, 600 / units)));
  const dim3 grid((unsigned)units, (unsigned)ceil_div(items, share)), block(kMergeThreads);
  switch (a.p.dtype) {
    case TS_F32: return launch_dependent(tree_merge_kernel<float>, grid, block, 0, st, a, tile_keys, start_places, share);
    case TS_F16: return launch_dependent(tree_merge_kernel<__half>, grid, block, 0, st, a, tile_keys, start_places, share);
    case TS_BF16: return launch_dependent(tree_merge_kernel<__nv_bfloat16>, grid, block, 0, st, a, tile_keys, start_places, share);
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
  TreeArgs a = tree_args(p, kBM, device_sms(), &bytes);
  tree_place(&a, workspace);
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
  return tree_merge(a, kBN, kUnitPlaces, st);
}

}  // namespace tsa
