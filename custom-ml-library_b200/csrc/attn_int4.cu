// Host side of the attention over a 4-bit cache: what the kernels take, how the work is shared.
#include <cstdlib>

#include "attn_int4.cuh"

namespace tsa {

namespace {
int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
      n <= 0)
    n = 148;
  return n;
}

bool rows_vec(const ts_view4& v, int size) {
  return v.stride[3] == 1 && reinterpret_cast<uintptr_t>(v.data) % 16 == 0 && v.stride[0] * size % 16 == 0 &&
         v.stride[1] * size % 16 == 0 && v.stride[2] * size % 16 == 0;
}

int64_t max_units() {
  const char* lower = std::getenv("TS_INT4_LINE");
  const int64_t n = lower ? std::atoll(lower) : 0;
  return n > 0 && n < kInt4MaxUnits ? n : kInt4MaxUnits;
}

struct Part {  // rows and query tokens of a launch; no tokens: one token of one row is too much already
  int rows, tokens;
};
Part part_of(const ts_attn_params& p, const Int4Shape& shape) {
  const int64_t limit = max_units(), columns = shape.nt * 8, group = p.q_heads / p.kv_heads;
  const int64_t pair = (int64_t)ceil_div(p.kv_len, shape.keys) + 1, blocks = limit / (pair * p.kv_heads);
  const int64_t tokens = i64min(p.q_len, i64min(blocks * columns / group, kInt4MaxUnits / p.q_heads));
  if (tokens <= 0) return Part{0, 0};
  const int64_t row = pair * p.kv_heads * ((tokens * group + columns - 1) / columns);
  const int64_t rows = i64min(limit / row, kInt4MaxUnits / (p.q_heads * tokens));  // its output rows are counted too
  return Part{(int)i64min(i64min(p.batch, kInt4MaxRows), rows), (int)tokens};
}

void set_tokens(const Int4Shape& shape, int tokens, Int4Attn& a) {
  a.cols = a.group * tokens;
  a.col_blocks = ceil_div(a.cols, shape.nt * 8);
}

// Fills what follows from the problem and its parts; returns the grid's blocks.
int plan(const ts_attn_params& p, Int4Attn& a, Int4Shape& shape, Part& part) {
  shape = int4_shape(p);
  part = part_of(p, shape);
  if (part.tokens <= 0) return 0;
  a.group = p.q_heads / p.kv_heads;
  set_tokens(shape, part.tokens, a);
  a.slot_cols = a.cols < shape.nt * 8 ? a.cols : shape.nt * 8;
  const int64_t pairs = (int64_t)part.rows * p.kv_heads * a.col_blocks;
  a.by_pair = shape.by_pair;
  // One wave of blocks that fill the GPU, fewer where a warp would be left without a stage.
  const int blocks = a.by_pair ? (int)pairs
                               : (int)i64min(pairs * ceil_div(p.kv_len, shape.keys), (int64_t)sm_count() * shape.blocks);
  a.blocks = blocks;
  a.parts = (int)i64min((int64_t)blocks * shape.warps / pairs, 1 << 20);
  return blocks;
}

size_t partial_bytes(const Int4Attn& a, const Int4Shape& shape, int head_dim) {
  return (size_t)2 * a.blocks * shape.warps * a.slot_cols * (head_dim + 2) * sizeof(float);
}
}  // namespace

Int4Shape int4_shape(const ts_attn_params& p) {
  const int cols = p.q_heads / p.kv_heads * p.q_len;
  const bool twin = cols <= 4 && p.dtype != TS_BF16;
  if (p.head_dim > 128) return {1, 32, 4, 2, false, twin};
  // Several column tiles share the operands made from the nibbles, with their queries in shared memory.  Three
  // where that saves a second pass (16 rows x 8 KV heads, up to 8192 keys, 20 columns: 51 against 60 us with two,
  // 64 rows 144 against 193; 12 columns: 47 against 39).  Four spill: 32 columns took 78 us against 71 with two
  // passes of two.  Stages of 32 tokens keep too little in flight: 173 against 143 us for 64 rows
  // of 20 columns.
  if (cols > 8) return {cols > 16 && cols <= 24 && p.dtype != TS_F32 ? 3 : 2, 64, 4, 2, false, false};
  // Stages of 16 tokens where those of 64 would leave most warps without one: 7.5 against 9.6 us for 18 heads
  // of up to 701 keys (fp32); with more the two meet (16 heads of 2048 keys: 8.8 against 9.2).  With two stages
  // and more for every warp, one block of 12 warps a SM against three of 4: its merged parts are fewer (64 x 32
  // heads of 1024-8192 keys: 251 against 258 us, 4 heads of up to 131072: 26 against 29; 16 heads of 2048 keys, one
  // stage a warp: 9.6 against 9.2).
  const int64_t stages = (int64_t)p.batch * p.kv_heads * ((cols + 7) / 8) * ceil_div(p.kv_len, 64);
  if (p.kv_len <= 64 || stages <= 148 * 3) return {1, 16, 4, 3, p.kv_len <= 4 * 16, twin};
  if (stages >= 148 * 12 * 2) return {1, 64, 12, 1, false, twin};
  return {1, 64, 4, 3, false, twin};
}

bool attn_int4_workspace(const ts_attn_params& p, size_t* bytes) {
  Int4Attn a;
  Int4Shape shape;
  Part part;
  plan(p, a, shape, part);
  if (part.tokens <= 0) return false;
  *bytes = a.by_pair ? 0 : partial_bytes(a, shape, p.head_dim) + (size_t)2 * (part.rows + 1) * sizeof(int32_t);
  return true;
}

cudaError_t attn_int4_forward(const ts_attn_params& p, const ts_kv4_cache& c, void* ws, uint32_t* fault,
                              cudaStream_t st) {
  Int4Attn a;
  Int4Shape shape;
  Part each;
  int blocks = plan(p, a, shape, each);
  if (each.tokens <= 0) return cudaErrorInvalidValue;
  a.p = p;
  a.c = c;
  a.page_log2 = c.page_size == 16 ? 4 : c.page_size == 32 ? 5 : 6;
  a.block_bytes = int4_block_bytes(p.head_dim, c.page_size);
  a.ws_acc = reinterpret_cast<float*>(ws);
  a.ws_ml = a.by_pair ? nullptr : a.ws_acc + (size_t)2 * a.blocks * shape.warps * a.slot_cols * p.head_dim;
  a.ws_first = a.by_pair ? nullptr : reinterpret_cast<int32_t*>(a.ws_ml + (size_t)2 * a.blocks * shape.warps * a.slot_cols * 2);
  a.fault = fault;
  const int size = p.dtype == TS_F32 ? 4 : 2;
  a.q_vec = rows_vec(p.q, size);
  a.o_vec = rows_vec(p.o, size);
  for (int token = 0; token < p.q_len; token += each.tokens)  // launches follow one another on the stream
    for (int row = 0; row < p.batch; row += each.rows) {
      Int4Attn part = a;
      part.p.batch = (int)i64min(p.batch - row, each.rows);
      part.p.q_len = (int)i64min(p.q_len - token, each.tokens);
      part.tokens_left = p.q_len - token;
      set_tokens(shape, part.p.q_len, part);
      part.p.q.data = reinterpret_cast<unsigned char*>(p.q.data) + (row * p.q.stride[0] + token * p.q.stride[2]) * size;
      part.p.o.data = reinterpret_cast<unsigned char*>(p.o.data) + (row * p.o.stride[0] + token * p.o.stride[2]) * size;
      if (p.lse) part.p.lse = reinterpret_cast<float*>(p.lse) + row * p.lse_stride[0] + token * p.lse_stride[2];
      part.p.kv_lens = p.kv_lens + row;
      part.c.table = c.table + row * c.table_stride;
      cudaError_t e = cudaErrorInvalidValue;
      if (a.by_pair) blocks = part.p.batch * p.kv_heads * part.col_blocks;
      switch (p.dtype) {
        case TS_BF16: e = attn_int4_launch<__nv_bfloat16>(part, shape, blocks, st); break;
        case TS_F16: e = attn_int4_launch<__half>(part, shape, blocks, st); break;
        case TS_F32: e = attn_int4_launch<float>(part, shape, blocks, st); break;
      }
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

}  // namespace tsa
