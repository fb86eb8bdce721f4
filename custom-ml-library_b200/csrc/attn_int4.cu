// Host side of the attention over a 4-bit cache: what the kernels take, how the keys are split.
#include "attn_int4.cuh"

namespace tsa {

bool attn_int4_supported(const ts_attn_params& p, const ts_kv4_cache& c) {
  if (p.dtype != TS_BF16 && p.dtype != TS_F16 && p.dtype != TS_F32) return false;
  return c.page_size == 16 || c.page_size == 32 || c.page_size == 64;
}

static int int4_tiles(const ts_attn_params& p) {
  const int cols = p.q_heads / p.kv_heads * p.q_len;
  return cols > 8 && p.dtype != TS_F32 && p.head_dim <= 128 ? 2 : 1;
}

// Keys of one split: enough blocks for two rounds of three a SM, and at least one stage for every
// warp of a block.
static int int4_split_keys(const ts_attn_params& p, int col_blocks) {
  const int64_t work = (int64_t)p.batch * p.kv_heads * col_blocks * p.kv_len;
  const int64_t target = 148 * 3 * 2;
  const int64_t s = (work + target - 1) / target;
  return (int)i64max(256, i64min((s + 255) / 256 * 256, 1 << 20));
}

static void int4_plan(const ts_attn_params& p, Int4Attn& a, int& nt) {
  nt = int4_tiles(p);
  a.group = p.q_heads / p.kv_heads;
  a.cols = a.group * p.q_len;
  a.col_blocks = ceil_div(a.cols, nt * 8);
  a.split_keys = int4_split_keys(p, a.col_blocks);
  a.max_splits = max(1, ceil_div(p.kv_len, a.split_keys));
}

size_t attn_int4_workspace(const ts_attn_params& p, const ts_kv4_cache&) {
  Int4Attn a;
  int nt;
  int4_plan(p, a, nt);
  if (a.max_splits == 1) return 0;
  return (size_t)p.batch * p.q_heads * p.q_len * a.max_splits * (p.head_dim + 2) * sizeof(float);
}

cudaError_t attn_int4_forward(const ts_attn_params& p, const ts_kv4_cache& c, void* ws, size_t ws_bytes,
                              uint32_t* fault, cudaStream_t st) {
  Int4Attn a;
  int nt;
  int4_plan(p, a, nt);
  a.p = p;
  a.c = c;
  a.page_log2 = c.page_size == 16 ? 4 : c.page_size == 32 ? 5 : 6;
  a.block_bytes = int4_block_bytes(p.head_dim, c.page_size);
  a.ws_acc = reinterpret_cast<float*>(ws);
  a.ws_ml = a.ws_acc ? a.ws_acc + (size_t)p.batch * p.q_heads * p.q_len * a.max_splits * p.head_dim : nullptr;
  a.fault = fault;
  if (ws_bytes < attn_int4_workspace(p, c)) return cudaErrorInvalidValue;
  switch (p.dtype) {
    case TS_BF16: return attn_int4_launch<__nv_bfloat16>(a, nt, st);
    case TS_F16: return attn_int4_launch<__half>(a, nt, st);
    case TS_F32: return attn_int4_launch<float>(a, nt, st);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tsa
