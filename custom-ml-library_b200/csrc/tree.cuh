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

__device__ __forceinline__ int tree_len(const ts_attn_params& p, int b) {
  return min(p.kv_len, max(0, p.kv_lens[b]));
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

// Bits k of [0, 32): the node sees slot `slot` + k.
__device__ __forceinline__ uint32_t view_bits(const NodeView& v, int64_t base, int sinks, int64_t slot) {
  uint32_t bits = range_bits(v.near, v.end, slot) | range_bits(0, i64min(v.end, sinks), slot);
  const int64_t o = slot - base;
  if (v.drafted && o < 64 && o > -32) bits |= (uint32_t)(o >= 0 ? v.drafted >> o : v.drafted << -o);
  return bits;
}

// Units of work, (row b, KV head, row tile), stand in line one behind the other, each with the key tiles that it
// reads; CTA c takes [c L / G, (c + 1) L / G) of the L tiles.
struct TreeLine {
  int batch, units;  // units of a row b
  int tile;          // keys of a tile
  const ts_attn_params* p;
  WindowArgs win;
  __device__ __forceinline__ TreeLine(const TreeArgs& a, int tile_keys)
      : batch(a.p.batch), units(a.p.kv_heads * a.row_tiles), tile(tile_keys), p(&a.p), win(a.win) {}
  __device__ __forceinline__ int tiles(int b) const {
    const int len = tree_len(*p, b);
    return WindowTiles(win, (int64_t)len - p->q_len, len, tile).count(ceil_div(len, tile));
  }
};
__device__ __forceinline__ int64_t line_bound(int c, int64_t total, int ctas) { return c * total / ctas; }
__device__ __forceinline__ int line_owner(int64_t at, int64_t total, int ctas) {
  return (int)(((at + 1) * ctas - 1) / total);
}

// One warp: tiles of all rows' units, and of those before row `b`.
__device__ __forceinline__ int64_t line_total(const TreeLine& line, int lane, int b, int64_t* before) {
  int64_t sum = 0, first = 0;
  for (int i = lane; i < line.batch; i += 32) {
    const int n = line.tiles(i);
    sum += n;
    if (i < b) first += n;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, off);
    first += __shfl_xor_sync(0xffffffffu, first, off);
  }
  *before = first * line.units;
  return sum * line.units;
}

// One warp: the row b, and the place within its tiles, of the line's position `at`.
__device__ __forceinline__ void line_find(const TreeLine& line, int lane, int64_t at, int* row, int64_t* rest) {
  int64_t before = 0;
  for (int b0 = 0; b0 < line.batch; b0 += 32) {
    const int64_t n = b0 + lane < line.batch ? (int64_t)line.tiles(b0 + lane) * line.units : 0;
    int64_t up_to = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t other = __shfl_up_sync(0xffffffffu, up_to, off);
      if (lane >= off) up_to += other;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + up_to > at);
    if (past) {
      const int l = __ffs(past) - 1;
      *row = b0 + l;
      *rest = at - before - __shfl_sync(0xffffffffu, up_to - n, l);
      return;
    }
    before += __shfl_sync(0xffffffffu, up_to, 31);
  }
  *row = line.batch;
  *rest = 0;
}

// A CTA's walk along its part of the line, segment by segment (one unit each).
struct LineWalk {
  int b, unit, first;  // of the present segment: row, unit of the row, first tile of the unit's list
  int count;           // its tiles; 0 before the first segment
  int64_t left;        // tiles behind it
  __device__ __forceinline__ void start(int row, int64_t rest, int64_t tiles, const TreeLine& line) {
    b = row;
    count = 0;
    left = tiles;
    unit = first = 0;
    if (tiles > 0) {
      const int n = line.tiles(row);
      unit = (int)(rest / n);
      first = (int)(rest % n);
    }
  }
  __device__ __forceinline__ bool next(const TreeLine& line) {
    if (left == 0) return false;
    if (count) {
      first = 0;
      if (++unit == line.units) {
        unit = 0;
        ++b;
      }
    }
    int n = 0;
    while (b < line.batch && (n = line.tiles(b)) == 0) ++b;  // rows without a key take no place in the line
    if (n <= first) return false;                              // not reached while the lengths stay as they are
    count = (int)i64min(left, n - first);
    left -= count;
    return true;
  }
};

// Row tiles of `tile_rows` rows, partial results for `parts_of` a segment in a workspace of *bytes.
TreeArgs tree_args(const ts_attn_params& p, int tile_rows, int ctas, int parts_of, size_t* bytes);
// Where a workspace holds them.
void tree_place(TreeArgs* a, int parts_of, void* workspace);
// Joins the partial results of a line of work over tiles of `tile_keys` keys.
cudaError_t tree_merge(const TreeArgs& a, int tile_keys, int parts_of, cudaStream_t st);

// attn_tree.cu: half types on the tensor cores.
bool tc_tree_supported(const ts_attn_params& p);
size_t tc_tree_workspace(const ts_attn_params& p);
cudaError_t tc_tree(const ts_attn_params& p, const int32_t* parents, int64_t parents_stride, const WindowArgs& win,
                    void* workspace, uint32_t* fault, cudaStream_t st);
int device_sms();

}  // namespace tsa
