// Attention of drafted tokens (a tree, or a chain) over a contiguous KV cache: what the tensor-core kernel
// (attn_tree.cu) and the CUDA-core kernel (attn_rows.cuh) share.
//
// Row b's cache holds len = kv_lens[b] keys, the last T = q_len of them drafted: node i sits in slot
// len - T + i.  A node sees the committed keys [0, len - T), its ancestors and itself.  Its position, which
// the window and the rotation of queries and keys go by, is len - T + its depth.
#pragma once
#include "common.cuh"
#include "window.cuh"

namespace tsa {

constexpr int kTreeNodes = 64;  // of a tree: a node's ancestors are one 64-bit word

struct TreeArgs {
  ts_attn_params p;        // kv_lens set
  const int32_t* parents;  // [batch, T], or null: a chain
  int64_t parents_stride;
  WindowArgs win;
  int rows;       // query heads of a KV head times T: row r is head r / T of the group, node r % T
  int tile_rows;  // of a row tile
  int row_tiles;
  int part_rows;  // of a partial result: those of a tile that some KV head has
  int ctas;
  float* part;  // partial outputs, unnormalised
  float2* ml;   // their reference maxima (log2 units) and sums
  uint32_t* fault;
};

// Channel quads of a partial result's row.
__host__ __device__ __forceinline__ int part_quads(const ts_attn_params& p) { return ceil_div(p.value_dim, 4); }

// Keys of a row, without kv_lens those that the last of the q_len tokens behind causal_offset sees (a windowed chunk).
__device__ __forceinline__ int tree_len(const ts_attn_params& p, int b) {
  return min(p.kv_len, p.kv_lens ? max(0, p.kv_lens[b]) : (int)(p.causal_offset + p.q_len));
}
// The same from L2: for a kernel that asks before it has waited for the one in front of it (which has waited for what
// wrote the lengths).
__device__ __forceinline__ int tree_len_early(const ts_attn_params& p, int b) {
  return min(p.kv_len, p.kv_lens ? max(0, __ldcg(p.kv_lens + b)) : (int)(p.causal_offset + p.q_len));
}

// What a node sees: the slots [near, end), those below min(end, sinks), and `drafted`'s bits from slot `base` on.
struct NodeView {
  int64_t near, end;
  uint64_t drafted;
  int depth;  // -1: a padded node, or one whose slot lies before the cache
};

// `up(i)` gives node i's parent.
template <typename Up>
__device__ __forceinline__ NodeView tree_node(int node, int64_t base, bool chain, const WindowArgs& win, Up up) {
  NodeView v;
  v.near = v.end = 0;
  v.drafted = 0;
  v.depth = -1;
  if (chain) {
    const int64_t at = base + node;
    if (at < 0) return v;
    v.depth = node;
    v.end = at + 1;
    if (win.window > 0) v.near = i64max(0, v.end - win.window);
    return v;
  }
  int depth = 0;
  uint64_t drafted = 0;
  for (int i = node;;) {  // parents come before their children, so this ends
    if (base + i < 0) return v;
    drafted |= 1ull << i;
    const int above = up(i);
    if (above == -1) break;
    if (above < 0 || above >= i) return v;
    i = above;
    ++depth;
  }
  v.depth = depth;
  v.end = i64max(0, base);
  if (win.window > 0) {
    const int64_t at = base + depth;
    v.near = i64max(0, at + 1 - win.window);
    drafted = 0;
    int i = node;
    for (int d = 0; d <= depth && i >= 0; ++d) {
      if (d < win.window || at - d < win.sinks) drafted |= 1ull << i;
      if (d < depth) i = up(i);
    }
  }
  v.drafted = drafted;
  return v;
}

// The drafted slots of a row that nobody sees, as bits from slot `base` on: of padded nodes, and of children of those or
// of nodes without a slot.  Their values are not multiplied, as 0 * NaN is NaN.  One warp, lane l with the parents of
// nodes l and l + 32 (-1 behind the last).
__device__ __forceinline__ uint64_t hidden_nodes(int nodes, int64_t base, int low, int high, int lane) {
  auto ends = [&](int i, int above) { return i < nodes && (base + i < 0 || above < -1 || above >= i); };
  if (!__any_sync(0xffffffffu, ends(lane, low) || ends(lane + 32, high))) return 0;
  uint64_t seen = 0, last;
  auto hangs = [&](int i, int above) {
    return i < nodes && !ends(i, above) && (above == -1 || (last >> above & 1u));
  };
  do {  // a level more every time
    last = seen;
    const uint64_t upper = __ballot_sync(0xffffffffu, hangs(lane + 32, high));
    seen = upper << 32 | __ballot_sync(0xffffffffu, hangs(lane, low));
  } while (seen != last);
  return ~seen & (~0ull >> (64 - nodes));
}
// Bits k of [0, 64): slot `slot` + k lies at or behind `len`, or is one of `hidden`.
__device__ __forceinline__ uint64_t gone_bits(uint64_t hidden, int64_t base, int len, int slot) {
  const int kept = len - slot;
  uint64_t bits = kept >= 64 ? 0 : ~0ull << max(kept, 0);
  const int64_t o = slot - base;
  if (hidden && o < 64 && o > -64) bits |= o >= 0 ? hidden >> o : hidden << -o;
  return bits;
}

// The same as tree_node for 32 nodes of a row, one behind the other (from the last the first follows), and the slots that
// nobody sees.  Parents by shuffles: lane l holds those of nodes l and l + 32.
__device__ __forceinline__ NodeView tree_node_of_warp(int node, int nodes, int64_t base, const TreeArgs& a, int b,
                                                      int lane, uint64_t* hidden) {
  const bool chain = a.parents == nullptr;
  *hidden = 0;
  if (chain) return tree_node(node, base, true, a.win, [](int) { return -1; });
  const int32_t* parents = a.parents + b * a.parents_stride;
  const int low = lane < nodes ? parents[lane] : -1, high = lane + 32 < nodes ? parents[lane + 32] : -1;
  auto up = [&](int i) {  // all lanes
    const int x = __shfl_sync(0xffffffffu, low, i & 31), y = __shfl_sync(0xffffffffu, high, i & 31);
    return i < 32 ? x : y;
  };
  NodeView v;
  v.near = v.end = 0;
  v.drafted = 0;
  v.depth = -1;
  uint64_t drafted = 0;
  int i = node, depth = 0;
  bool going = base + i >= 0, live = going;
  while (__any_sync(0xffffffffu, going)) {  // parents come before their children, so this ends
    const int above = up(i);
    if (going) {
      drafted |= 1ull << i;
      if (above < 0 || above >= i || base + above < 0) {
        live = above == -1;
        going = false;
      } else {
        i = above;
        ++depth;
      }
    }
  }
  // Up to 32 nodes are all among the lanes' own (8 nodes over 37 keys: 11.5 us, with a walk over levels 12.1).
  *hidden = nodes <= 32 ? __reduce_or_sync(0xffffffffu, live ? 0u : 1u << node) : hidden_nodes(nodes, base, low, high, lane);
  if (a.win.window > 0 && __any_sync(0xffffffffu, live)) {
    const int64_t at = base + depth;
    drafted = 0;
    i = node;
    going = live;
    for (int d = 0; __any_sync(0xffffffffu, going); ++d) {
      if (going && (d < a.win.window || at - d < a.win.sinks)) drafted |= 1ull << i;
      going = going && d < depth;
      const int above = up(i);
      if (going) i = max(0, above);
    }
    v.near = i64max(0, at + 1 - a.win.window);
  }
  if (!live) return v;
  v.depth = depth;
  v.end = i64max(0, base);
  v.drafted = drafted;
  return v;
}

// Bits k of [0, 32): the node sees slot `slot` + k.
__device__ __forceinline__ uint32_t view_bits(const NodeView& v, int64_t base, int sinks, int64_t slot) {
  uint32_t bits = range_bits(v.near, v.end, slot) | range_bits(0, i64min(v.end, sinks), slot);
  const int64_t o = slot - base;
  if (v.drafted && o < 64 && o > -32) bits |= (uint32_t)(o >= 0 ? v.drafted >> o : v.drafted << -o);
  return bits;
}

// What a row tile of row b reads: the tiles of its list, for queries at positions [first, last].
struct TileList {
  WindowTiles tiles;
  int count;
  int64_t first, last;
};

// Units of work, (row b, KV head, row tile), stand in line one behind the other, each with the key tiles that it
// reads and, in front of them, `start` places for what a unit costs by itself (its queries, its epilogue); CTA c takes
// the places [c L / G, (c + 1) L / G) of L.
struct TreeLine {
  int batch, heads, row_tiles, units;  // units of a row b: unit h row_tiles + t is row tile t of KV head h
  int tile, start;                     // keys of a tile; places in front of a unit's tiles
  bool early;
  const TreeArgs* a;
  __device__ __forceinline__ TreeLine(const TreeArgs& args, int tile_keys, int start_places, bool asks_early = false)
      : batch(args.p.batch), heads(args.p.kv_heads), row_tiles(args.row_tiles), units(heads * row_tiles),
        tile(tile_keys), start(start_places), early(asks_early), a(&args) {}
  __device__ __forceinline__ TileList list(int b, int row_tile) const {
    const ts_attn_params& p = a->p;
    const int len = early ? tree_len_early(p, b) : tree_len(p, b);
    const int64_t base = (int64_t)len - p.q_len;
    // The tokens of a chain that lie within one head are consecutive positions; a tree's may be anywhere.
    int n0 = 0, n1 = p.q_len - 1;
    if (!a->parents && p.q_len > 1) {
      const int r0 = row_tile * a->tile_rows, r1 = min(r0 + a->tile_rows, a->rows) - 1, h = r0 / p.q_len;
      if (r1 / p.q_len == h) n0 = r0 - h * p.q_len, n1 = r1 - h * p.q_len;
    }
    const WindowTiles tiles(a->win, base + n0, len, tile);
    const int end = (int)i64max(0, i64min(len, base + n1 + 1));
    return TileList{tiles, tiles.count(ceil_div(end, tile)), base + n0, base + n1};
  }
  // Places of a unit with n tiles: none for one without a key.
  __device__ __forceinline__ int64_t places(int n) const { return n > 0 ? n + start : 0; }
  // Places and tiles of one KV head of row b.
  __device__ __forceinline__ void head(int b, int64_t* all_places, int64_t* all_tiles) const {
    *all_places = *all_tiles = 0;
    for (int t = 0; t < row_tiles; ++t) {
      const int n = list(b, t).count;
      *all_places += places(n);
      *all_tiles += n;
    }
  }
};
__device__ __forceinline__ int64_t line_bound(int c, int64_t total, int ctas) { return c * total / ctas; }
__device__ __forceinline__ int line_owner(int64_t at, int64_t total, int ctas) {
  return (int)(((at + 1) * ctas - 1) / total);
}

__device__ __forceinline__ int64_t warp_sum(int64_t x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// One warp: the line's places, and those before the units of row `b`.
__device__ __forceinline__ int64_t line_total(const TreeLine& line, int lane, int b, int64_t* before) {
  int64_t sum = 0, first = 0;
  for (int i = lane; i < line.batch; i += 32) {
    int64_t n, tiles;
    line.head(i, &n, &tiles);
    sum += n;
    if (i < b) first += n;
  }
  *before = warp_sum(first) * line.heads;
  return warp_sum(sum) * line.heads;
}

// A place of the line: the unit it belongs to, its place within the unit, and the tiles in front of it.
struct LinePlace {
  int row, unit;
  int64_t rest, tiles;
};

// One warp: the two ends of CTA `c`'s share of the line (both at its beginning for a CTA without one).
__device__ __forceinline__ void line_share(const TreeLine& line, int lane, int c, int max_ctas, LinePlace (&ends)[2]) {
  int64_t own = 0, own_tiles = 0;  // of one KV head of row `lane`: kept for batches of up to 32 rows
  if (lane < line.batch) line.head(lane, &own, &own_tiles);
  int64_t total = own;
  for (int i = lane + 32; i < line.batch; i += 32) {
    int64_t n, tiles;
    line.head(i, &n, &tiles);
    total += n;
  }
  total = warp_sum(total) * line.heads;
  const int ctas = (int)i64min(max_ctas, total);
  ends[0] = ends[1] = LinePlace{0, 0, 0, 0};
  if (c >= ctas) return;
  const int64_t at[2] = {line_bound(c, total, ctas), line_bound(c + 1, total, ctas)};
  int64_t places = 0, tiles = 0;  // in front of this step's rows
  bool found[2] = {false, false};
  for (int b0 = 0; b0 < line.batch && !(found[0] && found[1]); b0 += 32) {
    if (b0 > 0) {
      own = own_tiles = 0;
      if (b0 + lane < line.batch) line.head(b0 + lane, &own, &own_tiles);
    }
    const int64_t mine = own * line.heads, mine_tiles = own_tiles * line.heads;
    int64_t up_to = mine, up_tiles = mine_tiles;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, up_to, off), y = __shfl_up_sync(0xffffffffu, up_tiles, off);
      if (lane >= off) up_to += x, up_tiles += y;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      // the row that holds the first place, and the last one
      const uint32_t past = __ballot_sync(0xffffffffu, places + up_to > at[e] - e);
      if (found[e] || !past) continue;
      const int l = __ffs(past) - 1;
      found[e] = true;
      int64_t rest = at[e] - places - __shfl_sync(0xffffffffu, up_to - mine, l);
      const int64_t size = __shfl_sync(0xffffffffu, own, l), size_tiles = __shfl_sync(0xffffffffu, own_tiles, l);
      LinePlace at_e = {b0 + l, 0, 0, tiles + __shfl_sync(0xffffffffu, up_tiles - mine_tiles, l)};
      const int64_t h = rest / size;
      rest -= h * size;
      at_e.tiles += h * size_tiles;
      int t = 0;
      for (; t < line.row_tiles; ++t) {
        const int n = line.list(b0 + l, t).count;
        if (rest < line.places(n)) break;
        rest -= line.places(n);
        at_e.tiles += n;
      }
      at_e.unit = (int)h * line.row_tiles + t;
      at_e.rest = rest;
      at_e.tiles += i64max(0, rest - line.start);
      ends[e] = at_e;
    }
    places += __shfl_sync(0xffffffffu, up_to, 31);
    tiles += __shfl_sync(0xffffffffu, up_tiles, 31);
  }
}

// A CTA's walk along its tiles, segment by segment (one unit each).
struct LineWalk {
  int b, unit, first;  // of the present segment: row, unit of the row, first tile of the unit's list
  int count;           // its tiles; 0 before the first segment
  int64_t left;        // tiles behind it
  TileList list;
  __device__ __forceinline__ void start(const LinePlace& from, int64_t tiles, const TreeLine& line) {
    b = from.row;
    unit = from.unit;
    first = (int)i64max(0, from.rest - line.start);
    count = 0;
    left = tiles;
  }
  __device__ __forceinline__ bool next(const TreeLine& line) {
    if (left == 0) return false;
    if (count) {
      first = 0;
      ++unit;
    }
    for (;;) {  // units without a key take no place in the line
      if (unit >= line.units) {
        unit = 0;
        ++b;
      }
      if (b >= line.batch) return false;  // not reached while the lengths stay as they are
      list = line.list(b, unit % line.row_tiles);
      if (list.count > first) break;
      first = 0;
      ++unit;
    }
    count = (int)i64min(left, list.count - first);
    left -= count;
    return true;
  }
};

// Row tiles of `tile_rows` rows, with partial results in a workspace of *bytes.
TreeArgs tree_args(const ts_attn_params& p, int tile_rows, int ctas, size_t* bytes);
// Where a workspace holds them.
void tree_place(TreeArgs* a, void* workspace);
// Joins the partial results of a line of work over tiles of `tile_keys` keys.
cudaError_t tree_merge(const TreeArgs& a, int tile_keys, int start_places, cudaStream_t st);

// attn_tree.cu: half types on the tensor cores.
bool tc_tree_supported(const ts_attn_params& p);
size_t tc_tree_workspace(const ts_attn_params& p);
cudaError_t tc_tree(const ts_attn_params& p, const int32_t* parents, int64_t parents_stride, const WindowArgs& win,
                    void* workspace, uint32_t* fault, cudaStream_t st);
int device_sms();

}  // namespace tsa
