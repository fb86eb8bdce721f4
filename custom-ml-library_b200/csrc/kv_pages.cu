// Pages of a paged KV cache: sharing rows (fork, reorder, free), handing out pages with
// copy-on-write, copying pages and closing up a pool.
//
// A page table is int32 [rows, slots] with -1 where a row has no page; refs[p] counts the table
// entries (and whatever pins a caller adds) that hold page p, and a page with refs 0 is free.
// counters = {free pages, a page number below which no page is free, error bits, unused}.
// Every result is a function of the inputs alone: integer sums commute, pages are handed out
// lowest first in the order of (row, slot), and of the writers that share a page the last keeps it.
// The one exception is counters[1] after a fork: a page that passes from row to row may be counted as
// free for a moment, so how far the bound lies below the lowest free page depends on the order of blocks.
//
// The pages themselves are opaque bytes.  Copies are bound by HBM (each byte read and written once): 2.65 GB of a
// compaction's pages move in 442 us, 93 % of the measured copy rate.  The table work is a chain of small launches,
// bound by the latency of their dependent loads: fork and reserve of 8 rows 9 us, a compaction of 160 pages 8, so
// each starts while the one before it ends.
#include "dependent.cuh"
#include "int4.cuh"

namespace tsa {

namespace {
constexpr int kErrPages = 1;   // not enough free pages: nothing was changed
constexpr int kErrIndex = 2;   // an index, page or row outside its range was skipped
constexpr int kErrSlots = 4;   // a row would need more slots than the table has: nothing was changed
constexpr int kScanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kCopyChunk = kCopyThreads * 16 * 4;  // bytes one block moves per step

// Exclusive sum over the block; `total` receives the sum of all threads' values.
__device__ __forceinline__ int block_scan(int v, int& total, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += up;
  }
  __syncthreads();  // the previous call's readers are done
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int s = lane < (int)(blockDim.x >> 5) ? warp_sums[lane] : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, s, off);
      if (lane >= off) s += up;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  total = warp_sums[(blockDim.x >> 5) - 1];
  return inc - v + (warp ? warp_sums[warp - 1] : 0);
}
}  // namespace

// ---------------------------------------------------------------------------
// Copies
// ---------------------------------------------------------------------------
// Item i moves page from[i * stride] of `src` to page to[i * stride] of `dst` in every layer; a
// negative entry is skipped.  Blocks stride over (item, layer, 16 KB chunk), 64 bytes in flight a
// thread.  n_dev, when given, holds the number of items.
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(ts_page_pool src, ts_page_pool dst,
                                                                 const int32_t* from, const int32_t* to, int stride,
                                                                 int n, const int32_t* n_dev) {
  let_next_start();
  wait_for_previous();
  if (n_dev) n = min(n, *n_dev);
  const int chunks = (int)((src.page_bytes + kCopyChunk - 1) / kCopyChunk);
  const int64_t work = (int64_t)n * src.layers * chunks;
  for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const int chunk = (int)(w % chunks);
    const int64_t rest = w / chunks;
    const int layer = (int)(rest % src.layers);
    const int64_t i = rest / src.layers;
    const int a = from[i * stride], b = to[i * stride];
    if (a < 0 || b < 0 || a >= src.pages || b >= dst.pages) continue;
    const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned char*>(src.data) +
                                                    layer * src.layer_stride + a * src.page_stride);
    uint4* d = reinterpret_cast<uint4*>(reinterpret_cast<unsigned char*>(dst.data) + layer * dst.layer_stride +
                                        b * dst.page_stride);
    const int64_t vecs = src.page_bytes / 16;
    const int64_t v0 = (int64_t)chunk * (kCopyChunk / 16) + threadIdx.x;
    uint4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (v0 + k * kCopyThreads < vecs) x[k] = s[v0 + k * kCopyThreads];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (v0 + k * kCopyThreads < vecs) d[v0 + k * kCopyThreads] = x[k];
  }
}

// dependent: the kernel before it on the stream is one of this file's that made the list.
static cudaError_t launch_copy(const ts_page_pool& src, const ts_page_pool& dst, const int32_t* from,
                               const int32_t* to, int stride, int n, const int32_t* n_dev, bool dependent,
                               cudaStream_t st) {
  const int64_t work = (int64_t)n * src.layers * ((src.page_bytes + kCopyChunk - 1) / kCopyChunk);
  if (work == 0) return cudaSuccess;
  const int64_t most = 148 * 8;  // every block of a full GPU; they stride over the rest
  const dim3 grid((unsigned)(work < most ? work : most));
  if (dependent) return launch_dependent(page_copy_kernel, grid, dim3(kCopyThreads), 0, st, src, dst, from, to, stride, n, n_dev);
  page_copy_kernel<<<grid, kCopyThreads, 0, st>>>(src, dst, from, to, stride, n, n_dev);
  return cudaGetLastError();
}

cudaError_t kv_pages_copy(const ts_page_pool& src, const ts_page_pool& dst, const int32_t* from, const int32_t* to,
                          int count, cudaStream_t st) {
  return launch_copy(src, dst, from, to, 1, count, nullptr, false, st);
}

// ---------------------------------------------------------------------------
// Fork / reorder / free: new row r takes over (shares) the pages of old row index[r]
// ---------------------------------------------------------------------------
// One block an old and a new row: the new row's pages gain a reference, the old row's lose one.
// A page's count may pass zero on the way; the free counter follows every crossing, so it ends at
// the right number whatever the order.
__global__ void kv_fork_kernel(const int32_t* table, int64_t table_stride, const int32_t* lens, int rows,
                               const int32_t* index, int32_t* table_out, int64_t table_out_stride, int32_t* lens_out,
                               int rows_out, int slots, int page_size, int32_t* refs, int pages, int32_t* counters) {
  let_next_start();
  const int r = blockIdx.x;
  int freed = 0, lowest = pages;
  if (r < rows_out) {
    const int src = index[r];
    if (src >= rows && threadIdx.x == 0) atomicOr(&counters[2], kErrIndex);
    const bool live = src >= 0 && src < rows;
    const int len = live ? max(0, lens[src]) : 0;
    const int used = (int)(((int64_t)len + page_size - 1) / page_size);
    for (int s = threadIdx.x; s < slots; s += blockDim.x) {
      int page = live && s < used ? table[src * table_stride + s] : -1;
      if (page >= pages) {
        page = -1;
        atomicOr(&counters[2], kErrIndex);
      }
      if (page >= 0 && atomicAdd(&refs[page], 1) == 0) --freed;
      table_out[r * table_out_stride + s] = page < 0 ? -1 : page;
    }
    if (threadIdx.x == 0) lens_out[r] = len;
  }
  if (r < rows) {
    for (int s = threadIdx.x; s < slots; s += blockDim.x) {
      const int page = table[r * table_stride + s];
      if (page >= 0 && page < pages && atomicSub(&refs[page], 1) == 1) {
        ++freed;
        lowest = min(lowest, page);
      }
    }
  }
  freed = __reduce_add_sync(0xffffffffu, freed);
  lowest = __reduce_min_sync(0xffffffffu, lowest);
  if ((threadIdx.x & 31) == 0) {
    if (freed) atomicAdd(&counters[0], freed);
    if (lowest < pages) atomicMin(&counters[1], lowest);
  }
}

cudaError_t kv_pages_fork(const int32_t* table, int64_t table_stride, const int32_t* lens, int rows,
                          const int32_t* index, int32_t* table_out, int64_t table_out_stride, int32_t* lens_out,
                          int rows_out, int slots, int page_size, int32_t* refs, int pages, int32_t* counters,
                          cudaStream_t st) {
  const int n = rows > rows_out ? rows : rows_out;
  const int threads = slots >= 256 ? 256 : (slots + 31) / 32 * 32;
  kv_fork_kernel<<<n, threads, 0, st>>>(table, table_stride, lens, rows, index, table_out, table_out_stride, lens_out,
                                        rows_out, slots, page_size, refs, pages, counters);
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// Reserve: pages for the tokens [len, len + steps) of every row
// ---------------------------------------------------------------------------
struct ReserveArgs {
  int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* row_steps;
  int32_t* refs;
  int32_t* counters;
  int32_t* writers;  // [pages] rows that write to a page they may share
  int32_t* last;     // [pages] the last of them, plus one
  int32_t* list;     // [pages] the pages handed out
  int32_t* offs;     // [rows]  a row's first place in the list
  int32_t* pairs;    // [rows, 2] copy-on-write: from, to (-1: none)
  int rows, slots, pages, page_size, steps;
};

__device__ __forceinline__ int reserve_steps(const ReserveArgs& a, int r) {
  return max(0, a.row_steps ? a.row_steps[r] : a.steps);
}
// The page that row r's next token falls into when that page is partly filled, or -1.
__device__ __forceinline__ int reserve_partial(const ReserveArgs& a, int r) {
  const int len = a.lens[r];
  if (len <= 0 || len % a.page_size == 0 || reserve_steps(a, r) == 0 || len / a.page_size >= a.slots) return -1;
  const int page = a.table[r * a.table_stride + len / a.page_size];
  return page >= 0 && page < a.pages ? page : -1;
}

// One block: the tables are small and the order of the hand-out runs through all rows.  What bounds it is the
// chain of dependent loads, so a thread keeps what it knows of its first row.
__global__ void __launch_bounds__(kScanThreads) kv_reserve_kernel(ReserveArgs a) {
  __shared__ int warp_sums[32];
  __shared__ int too_long;
  let_next_start();
  wait_for_previous();
  const int tid = threadIdx.x;
  if (tid == 0) too_long = 0;
  const int own_page = tid < a.rows ? reserve_partial(a, tid) : -1;
  auto partial = [&](int r) { return r == tid ? own_page : reserve_partial(a, r); };
  const int first_free = a.counters[1], n_free = a.counters[0];
  for (int r = tid; r < a.rows; r += kScanThreads) {
    const int page = partial(r);
    if (page >= 0) a.writers[page] = a.last[page] = 0;
  }
  __syncthreads();
  for (int r = tid; r < a.rows; r += kScanThreads) {
    const int page = partial(r);
    if (page >= 0) {
      atomicAdd(&a.writers[page], 1);
      atomicMax(&a.last[page], r + 1);
    }
  }
  __syncthreads();
  // How many pages each row needs: one in the place of a shared partial page, one per empty slot.
  int total = 0;
  for (int base = 0; base < a.rows; base += kScanThreads) {
    const int r = base + tid;
    int need = 0;
    bool copy = false;
    if (r < a.rows) {
      const int page = partial(r);
      copy = page >= 0 && (a.refs[page] > a.writers[page] || r + 1 < a.last[page]);
      need = copy ? 1 : 0;
      const int64_t len = max(0, a.lens[r]), stop = len + reserve_steps(a, r);
      const int64_t end = (stop + a.page_size - 1) / a.page_size;
      if (end > a.slots) atomicOr(&too_long, 1);
      const int slot_end = (int)i64min(end, a.slots);
#pragma unroll 4
      for (int s = (int)((len + a.page_size - 1) / a.page_size); s < slot_end; ++s)
        need += a.table[r * a.table_stride + s] < 0;
    }
    int sum;
    const int before = block_scan(need, sum, warp_sums);
    if (r < a.rows) {
      a.offs[r] = total + before;
      a.pairs[2 * r] = copy ? 0 : -1;
      a.pairs[2 * r + 1] = -1;
    }
    total += sum;
  }
  __syncthreads();
  const bool short_of_pages = total > n_free;
  if (too_long || short_of_pages) {
    if (tid == 0) atomicOr(&a.counters[2], too_long ? kErrSlots : kErrPages);
    return;  // pairs[][1] is -1 everywhere, so nothing is copied either
  }
  // The lowest free pages.
  int found = 0;
  for (int64_t base = first_free; found < total && base < a.pages; base += kScanThreads * 4) {
    int free4 = 0, ex;
    const int64_t p0 = base + tid * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (p0 + k < a.pages && a.refs[p0 + k] == 0) free4 |= 1 << k;
    int sum;
    ex = found + block_scan(__popc(free4), sum, warp_sums);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (free4 >> k & 1) {
        if (ex < total) a.list[ex] = (int)(p0 + k);
        ++ex;
      }
    found += sum;
  }
  __syncthreads();
  if (found < total) {  // the counter promised more than the pool holds
    if (tid == 0) atomicOr(&a.counters[2], kErrPages);
    return;
  }
  for (int r = tid; r < a.rows; r += kScanThreads) {
    int at = a.offs[r];
    int32_t* row = a.table + r * a.table_stride;
    const int64_t len = max(0, a.lens[r]), stop = len + reserve_steps(a, r);
    if (a.pairs[2 * r] >= 0) {
      const int slot = (int)(len / a.page_size), page = row[slot], own = a.list[at++];
      a.pairs[2 * r] = page;
      a.pairs[2 * r + 1] = own;
      row[slot] = own;
      a.refs[own] = 1;
      atomicSub(&a.refs[page], 1);
    }
    for (int s = (int)((len + a.page_size - 1) / a.page_size); s < (int)((stop + a.page_size - 1) / a.page_size); ++s)
      if (row[s] < 0) {
        const int own = a.list[at++];
        row[s] = own;
        a.refs[own] = 1;
      }
  }
  if (tid == 0 && total > 0) {
    a.counters[0] = n_free - total;
    a.counters[1] = a.list[total - 1] + 1;
  }
}

size_t kv_pages_reserve_workspace(int pages, int rows) {
  return ((size_t)3 * pages + (size_t)3 * rows) * sizeof(int32_t);
}

cudaError_t kv_pages_reserve(const ts_page_pool& pool, int32_t* table, int64_t table_stride, const int32_t* lens,
                             int rows, int slots, int page_size, int steps, const int32_t* row_steps, int32_t* refs,
                             int32_t* counters, void* ws, cudaStream_t st) {
  ReserveArgs a;
  a.table = table;
  a.table_stride = table_stride;
  a.lens = lens;
  a.row_steps = row_steps;
  a.refs = refs;
  a.counters = counters;
  a.writers = reinterpret_cast<int32_t*>(ws);
  a.last = a.writers + pool.pages;
  a.list = a.last + pool.pages;
  a.offs = a.list + pool.pages;
  a.pairs = a.offs + rows;
  a.rows = rows;
  a.slots = slots;
  a.pages = pool.pages;
  a.page_size = page_size;
  a.steps = steps;
  // usually right behind a fork, whose end it may await on the SM
  const cudaError_t e = launch_dependent(kv_reserve_kernel, dim3(1), dim3(kScanThreads), 0, st, a);
  if (e != cudaSuccess) return e;
  return launch_copy(pool, pool, a.pairs, a.pairs + 1, 2, rows, nullptr, true, st);
}

// ---------------------------------------------------------------------------
// Compaction: with n live pages, the live ones at or above n move into the holes below n, the
// highest page into the lowest hole
// ---------------------------------------------------------------------------
namespace {
constexpr int kRankPages = kScanThreads * 4;
}

__global__ void __launch_bounds__(kScanThreads) compact_count_kernel(const int32_t* refs, int pages, int32_t* counts) {
  __shared__ int warp_sums[32];
  let_next_start();
  const int64_t p0 = (int64_t)blockIdx.x * kRankPages + threadIdx.x * 4;
  int n = 0, total;
#pragma unroll
  for (int k = 0; k < 4; ++k) n += p0 + k < pages && refs[p0 + k] > 0;
  block_scan(n, total, warp_sums);
  if (threadIdx.x == 0) counts[blockIdx.x] = total;
}

// Ranks every page among the live ones and lists the moves: from[i] -> to[i], rank[p] = i.
__global__ void __launch_bounds__(kScanThreads) compact_rank_kernel(const int32_t* refs, int32_t* refs_out, int pages,
                                                                    const int32_t* counts, int32_t* from, int32_t* to,
                                                                    int32_t* rank, int32_t* moves, int32_t* counters) {
  __shared__ int warp_sums[32];
  let_next_start();
  wait_for_previous();
  int before = 0, live = 0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kScanThreads) {
    const int n = counts[i];
    live += n;
    before += i < (int)blockIdx.x ? n : 0;
  }
  block_scan(live, live, warp_sums);
  block_scan(before, before, warp_sums);
  const int64_t p0 = (int64_t)blockIdx.x * kRankPages + threadIdx.x * 4;
  int r[4], n = 0, total;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    r[k] = p0 + k < pages ? refs[p0 + k] : 0;
    n += r[k] > 0;
  }
  int ex = before + block_scan(n, total, warp_sums);  // live pages below p0 + k
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int p = (int)(p0 + k);
    if (p0 + k >= pages) break;
    if (p == live) *moves = live - ex;
    const bool moves_down = r[k] > 0 && p >= live;
    if (moves_down) from[live - 1 - ex] = p;
    rank[p] = moves_down ? live - 1 - ex : -1;
    if (r[k] <= 0 && p < live) to[p - ex] = p;
    // Holes and movers get their counts with the move.
    if (refs_out != refs) refs_out[p] = r[k] > 0 && p < live ? r[k] : 0;
    ex += r[k] > 0;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (live == pages) *moves = 0;
    counters[1] = live;
  }
}

__global__ void compact_tables_kernel(const int32_t* table, int32_t* table_out, int rows, int slots,
                                      int64_t table_stride, int64_t table_out_stride, const int32_t* refs,
                                      int32_t* refs_out, int pages, const int32_t* from, const int32_t* to,
                                      const int32_t* rank, const int32_t* moves, const int32_t* counters) {
  let_next_start();
  wait_for_previous();
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int live = counters[1];
  if (i < *moves) {
    const int n = refs[from[i]];
    refs_out[to[i]] = n;
    if (refs_out == refs) refs_out[from[i]] = 0;
  }
  if (i < (int64_t)rows * slots) {
    const int64_t r = i / slots, s = i - r * slots;
    int page = table[r * table_stride + s];
    if (page >= live) page = page < pages && rank[page] >= 0 ? to[rank[page]] : -1;  // a free page is nobody's
    table_out[r * table_out_stride + s] = page < 0 ? -1 : page;
  }
}

size_t kv_pages_compact_workspace(int pages) {
  return ((size_t)3 * pages + (pages + kRankPages - 1) / kRankPages + 1) * sizeof(int32_t);
}

cudaError_t kv_pages_compact(const ts_page_pool& pool, const int32_t* table, int32_t* table_out, int rows, int slots,
                             int64_t table_stride, int64_t table_out_stride, const int32_t* refs, int32_t* refs_out,
                             int32_t* counters, void* ws, cudaStream_t st) {
  const int pages = pool.pages, blocks = (pages + kRankPages - 1) / kRankPages;
  int32_t* from = reinterpret_cast<int32_t*>(ws);
  int32_t *to = from + pages, *rank = to + pages, *counts = rank + pages, *moves = counts + blocks;
  compact_count_kernel<<<blocks, kScanThreads, 0, st>>>(refs, pages, counts);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess)
    e = launch_dependent(compact_rank_kernel, dim3(blocks), dim3(kScanThreads), 0, st, refs, refs_out, pages, counts, from,
                         to, rank, moves, counters);
  const int64_t most = (int64_t)rows * slots > pages ? (int64_t)rows * slots : pages;
  if (e == cudaSuccess)
    e = launch_dependent(compact_tables_kernel, dim3((unsigned)((most + 255) / 256)), dim3(256), 0, st, table, table_out,
                         rows, slots, table_stride, table_out_stride, refs, refs_out, pages, from, to, rank, moves,
                         counters);
  if (e != cudaSuccess) return e;
  return launch_copy(pool, pool, from, to, 1, pages, moves, true, st);
}

}  // namespace tsa
