// extern "C" entry points of libts_attn.so (declared in include/ts_attn.h):
// argument validation, kernel selection and the device fault word.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>

#include "common.cuh"
#include "decode.cuh"
#include "int4.cuh"
#include "int8.cuh"
#include "kv_cache.cuh"
#include "rope.cuh"
#include "rows.cuh"
#include "simt.cuh"
#include "symbols.cuh"
#include "tc_bwd.cuh"
#include "tc_fwd.cuh"
#include "token_logprobs.cuh"

namespace {

// Fault word written by kernels whose bounded waits gave up (per device).
__device__ uint32_t g_fault_word;

uint32_t* fault_ptr() { return static_cast<uint32_t*>(tsa::device_symbol_address(&g_fault_word)); }

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

int from_cuda(cudaError_t e) {
  if (e == cudaSuccess) return TS_OK;
  if (e == cudaErrorInvalidValue) return TS_ERR_INVALID_ARGUMENT;
  return TS_ERR_LAUNCH;
}

bool dtype_ok(int d) { return d == TS_F32 || d == TS_F16 || d == TS_BF16 || d == TS_F64; }

int check_params(const ts_attn_params* p) {
  if (!p) return TS_ERR_INVALID_ARGUMENT;
  if (!dtype_ok(p->dtype)) return TS_ERR_UNSUPPORTED;
  if (p->batch <= 0 || p->q_heads <= 0 || p->kv_heads <= 0 || p->q_len <= 0 || p->kv_len <= 0 ||
      p->head_dim <= 0 || p->value_dim <= 0)
    return TS_ERR_INVALID_ARGUMENT;
  if (p->q_heads % p->kv_heads) return TS_ERR_INVALID_ARGUMENT;
  if (p->head_dim > 256 || p->value_dim > 256) return TS_ERR_UNSUPPORTED;
  if (!p->q.data || !p->k.data || !p->v.data || !p->o.data) return TS_ERR_INVALID_ARGUMENT;
  if (p->causal_offset < 0) return TS_ERR_INVALID_ARGUMENT;
  if (!(p->scale == p->scale) || p->scale > 1.0e300 || p->scale < -1.0e300) return TS_ERR_INVALID_ARGUMENT;
  if (p->mask_kind < TS_MASK_NONE || p->mask_kind > TS_MASK_ADD_F32) return TS_ERR_INVALID_ARGUMENT;
  if (p->mask_kind != TS_MASK_NONE && !p->mask) return TS_ERR_INVALID_ARGUMENT;
  return TS_OK;
}

}  // namespace

namespace tsa {

void* device_symbol_address(const void* symbol) {
  // CUresult cuCtxGetId(CUcontext ctx, unsigned long long* id); ctx = NULL: the current context.
  typedef int (*CtxGetIdFn)(void*, unsigned long long*);
  struct Entry {
    const void* symbol;
    unsigned long long ctx;
    void* ptr;
  };
  constexpr int kEntries = 256;
  static Entry cache[kEntries];
  static int used = 0;
  static CtxGetIdFn ctx_get_id = nullptr;
  static std::once_flag once;
  static std::mutex lock;
  std::call_once(once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuCtxGetId", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      ctx_get_id = reinterpret_cast<CtxGetIdFn>(fn);
  });
  std::lock_guard<std::mutex> guard(lock);
  unsigned long long ctx = 0;
  bool have_ctx = ctx_get_id && ctx_get_id(nullptr, &ctx) == 0;
  if (have_ctx)
    for (int i = 0; i < used; ++i)
      if (cache[i].symbol == symbol && cache[i].ctx == ctx) return cache[i].ptr;
  void* ptr = nullptr;
  if (cudaGetSymbolAddress(&ptr, symbol) != cudaSuccess || ptr == nullptr) return nullptr;
  // The lookup above makes the device's primary context current if nothing was.
  if (!have_ctx) have_ctx = ctx_get_id && ctx_get_id(nullptr, &ctx) == 0;
  if (have_ctx && used < kEntries) cache[used++] = Entry{symbol, ctx, ptr};
  return ptr;
}

}  // namespace tsa

extern "C" {

int ts_attn_abi_version(void) { return TS_ATTN_ABI_VERSION; }

#ifndef TS_SOURCE_DIGEST
#define TS_SOURCE_DIGEST "unknown"
#endif
const char* ts_attn_source_digest(void) { return TS_SOURCE_DIGEST; }

const char* ts_attn_strerror(int status) {
  switch (status) {
    case TS_OK: return "ok";
    case TS_ERR_INVALID_ARGUMENT: return "invalid argument (shape, stride, pointer or value)";
    case TS_ERR_UNSUPPORTED: return "unsupported dtype / dimension combination";
    case TS_ERR_WORKSPACE: return "workspace missing or too small";
    case TS_ERR_LAUNCH: return "CUDA kernel launch or driver call failed";
    case TS_ERR_DEVICE_TIMEOUT: return "a bounded wait inside an engine kernel gave up";
    case TS_ERR_CAPACITY: return "KV-cache capacity exceeded or empty append";
    case TS_ERR_PAGE: return "a page table entry outside its pool";
  }
  return "unknown status";
}

int ts_attn_fwd_path(const ts_attn_params* p, int decode) {
  const int st = check_params(p);
  if (st != TS_OK) return st;
  ts_attn_params view;
  if (decode && tsa::gqa_decode_view(*p, &view)) return TS_PATH_TCGEN05;
  if (decode && tsa::decode_supported(*p)) return TS_PATH_DECODE;
  if (tsa::tc_fwd_supported(*p)) return TS_PATH_TCGEN05;
  return TS_PATH_SIMT;
}

int ts_attn_fwd(const ts_attn_params* p, void* stream) {
  const int st = check_params(p);
  if (st != TS_OK) return st;
  if (tsa::tc_fwd_supported(*p)) return from_cuda(tsa::tc_forward(*p, fault_ptr(), as_stream(stream)));
  return from_cuda(tsa::simt_forward(*p, as_stream(stream)));
}

size_t ts_attn_decode_workspace_size(const ts_attn_params* p) {
  ts_attn_params view;
  if (check_params(p) != TS_OK || tsa::gqa_decode_view(*p, &view) || !tsa::decode_supported(*p)) return 0;
  return tsa::decode_workspace(*p);
}

int ts_attn_decode(const ts_attn_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  const int st = check_params(p);
  if (st != TS_OK) return st;
  // A grouped-query step over enough (batch, KV head) pairs runs on the
  // tensor cores, the query heads of each KV head as the rows of one tile.
  ts_attn_params view;
  if (tsa::gqa_decode_view(*p, &view)) return from_cuda(tsa::tc_forward(view, fault_ptr(), as_stream(stream)));
  // Problems the split-K kernels do not take (many query rows, explicit masks,
  // value_dim != head_dim) go where ts_attn_fwd would send them; neither path
  // needs a workspace.
  if (!tsa::decode_supported(*p)) return ts_attn_fwd(p, stream);
  const size_t need = tsa::decode_workspace(*p);
  if (need && (!workspace || workspace_bytes < need)) return TS_ERR_WORKSPACE;
  return from_cuda(tsa::decode_forward(*p, workspace, workspace_bytes, fault_ptr(), as_stream(stream)));
}

size_t ts_attn_bwd_workspace_size(const ts_attn_bwd_params* bp) {
  if (!bp || check_params(&bp->fwd) != TS_OK) return 0;
  if (tsa::tc_bwd_supported(*bp)) return tsa::tc_bwd_workspace(*bp);
  return tsa::simt_backward_workspace(*bp);
}

int ts_attn_bwd_path(const ts_attn_bwd_params* bp) {
  if (!bp) return TS_ERR_INVALID_ARGUMENT;
  const int st = check_params(&bp->fwd);
  if (st != TS_OK) return st;
  return tsa::tc_bwd_supported(*bp) ? TS_PATH_TCGEN05 : TS_PATH_SIMT;
}

int ts_attn_bwd(const ts_attn_bwd_params* bp, void* workspace, size_t workspace_bytes, void* stream) {
  if (!bp) return TS_ERR_INVALID_ARGUMENT;
  const int st = check_params(&bp->fwd);
  if (st != TS_OK) return st;
  if (!bp->fwd.lse || !bp->dout.data || !bp->dq.data || !bp->dk.data || !bp->dv.data)
    return TS_ERR_INVALID_ARGUMENT;
  if (tsa::tc_bwd_supported(*bp)) {
    if (!workspace || workspace_bytes < tsa::tc_bwd_workspace(*bp)) return TS_ERR_WORKSPACE;
    return from_cuda(tsa::tc_backward(*bp, workspace, workspace_bytes, fault_ptr(), as_stream(stream)));
  }
  const size_t need = tsa::simt_backward_workspace(*bp);
  if (!workspace || workspace_bytes < need) return TS_ERR_WORKSPACE;
  return from_cuda(tsa::simt_backward(*bp, workspace, as_stream(stream)));
}

int ts_kv_append(const ts_kv_append_params* p, void* stream) {
  if (!p) return TS_ERR_INVALID_ARGUMENT;
  if (!dtype_ok(p->src_dtype) || !dtype_ok(p->cache_dtype)) return TS_ERR_UNSUPPORTED;
  if (p->batch <= 0 || p->heads <= 0 || p->head_dim <= 0 || p->value_dim <= 0 || p->capacity <= 0)
    return TS_ERR_INVALID_ARGUMENT;
  if (!p->key.data || !p->value.data || !p->key_cache.data || !p->value_cache.data)
    return TS_ERR_INVALID_ARGUMENT;
  if (p->steps <= 0) return TS_ERR_CAPACITY;
  if (!p->positions && (p->position < 0 || p->position + p->steps > p->capacity)) return TS_ERR_CAPACITY;
  return from_cuda(tsa::kv_append(*p, as_stream(stream)));
}

int ts_rope(ts_view4 x, ts_view4 y, int32_t dtype, int32_t batch, int32_t heads, int32_t seq, int32_t channels,
            int32_t rotary_dim, int64_t offset, const int32_t* positions, const float* inv_freq, int32_t inverse,
            void* stream) {
  if (!dtype_ok(dtype)) return TS_ERR_UNSUPPORTED;
  if (!x.data || !y.data || !inv_freq || batch <= 0 || heads <= 0 || seq <= 0 || channels <= 0)
    return TS_ERR_INVALID_ARGUMENT;
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > channels || offset < 0) return TS_ERR_INVALID_ARGUMENT;
  return from_cuda(tsa::rope_apply(x, y, dtype, batch, heads, seq, channels, rotary_dim, offset, positions, inv_freq,
                                   inverse, as_stream(stream)));
}

int ts_kv_append_rope(const ts_kv_append_params* p, const float* inv_freq, int32_t rotary_dim, void* stream) {
  if (!p) return TS_ERR_INVALID_ARGUMENT;
  if (!dtype_ok(p->src_dtype) || !dtype_ok(p->cache_dtype)) return TS_ERR_UNSUPPORTED;
  if (p->batch <= 0 || p->heads <= 0 || p->head_dim <= 0 || p->value_dim <= 0 || p->capacity <= 0 || !inv_freq)
    return TS_ERR_INVALID_ARGUMENT;
  if (!p->key.data || !p->value.data || !p->key_cache.data || !p->value_cache.data) return TS_ERR_INVALID_ARGUMENT;
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > p->head_dim) return TS_ERR_INVALID_ARGUMENT;
  if (p->steps <= 0) return TS_ERR_CAPACITY;
  if (!p->positions && (p->position < 0 || p->position + p->steps > p->capacity)) return TS_ERR_CAPACITY;
  return from_cuda(tsa::kv_append_rope(*p, inv_freq, rotary_dim, as_stream(stream)));
}

int ts_kv_reorder(ts_view4 src, ts_view4 dst, int32_t dtype, int32_t batch, int32_t heads, int32_t length,
                  int32_t channels, const int32_t* index, void* stream) {
  if (!dtype_ok(dtype) && dtype != TS_I8) return TS_ERR_UNSUPPORTED;
  if (!src.data || !dst.data || !index || batch <= 0 || heads <= 0 || length < 0 || channels <= 0)
    return TS_ERR_INVALID_ARGUMENT;
  return from_cuda(tsa::kv_reorder(src, dst, dtype, batch, heads, length, channels, index, as_stream(stream)));
}

}  // extern "C"

namespace {
bool make_dropout(const ts_dropout* d, tsa::DropoutArgs& out) {
  if (!d || !(d->p >= 0.0) || !(d->p < 1.0)) return false;
  out.p = (float)d->p;
  out.keep_min = (uint32_t)std::ceil(d->p * 65536.0);
  out.inv_keep_f = 1.0f / (float)(1.0 - d->p);
  out.inv_keep_d = 1.0 / (1.0 - d->p);
  out.seed = d->seed;
  out.offset = d->offset;
  return true;
}
}  // namespace

extern "C" {

int ts_attn_fwd_dropout(const ts_attn_params* p, const ts_dropout* d, void* stream) {
  const int st = check_params(p);
  if (st != TS_OK) return st;
  tsa::DropoutArgs args;
  if (!make_dropout(d, args)) return TS_ERR_INVALID_ARGUMENT;
  if (d->p == 0.0) return ts_attn_fwd(p, stream);  // no dropout: the plain path selection
  if (tsa::tc_fwd_supported(*p)) return from_cuda(tsa::tc_forward(*p, fault_ptr(), as_stream(stream), &args));
  return from_cuda(tsa::simt_forward(*p, as_stream(stream), &args));
}

size_t ts_attn_bwd_dropout_workspace_size(const ts_attn_bwd_params* bp) {
  if (!bp || check_params(&bp->fwd) != TS_OK) return 0;
  const size_t simt = tsa::simt_backward_workspace(*bp);
  if (!tsa::tc_bwd_supported(*bp)) return simt;
  const size_t tc = tsa::tc_bwd_workspace(*bp);
  return tc > simt ? tc : simt;
}

int ts_attn_bwd_dropout(const ts_attn_bwd_params* bp, const ts_dropout* d, void* workspace, size_t workspace_bytes,
                        void* stream) {
  if (!bp) return TS_ERR_INVALID_ARGUMENT;
  const int st = check_params(&bp->fwd);
  if (st != TS_OK) return st;
  if (!bp->fwd.lse || !bp->dout.data || !bp->dq.data || !bp->dk.data || !bp->dv.data)
    return TS_ERR_INVALID_ARGUMENT;
  tsa::DropoutArgs args;
  if (!make_dropout(d, args)) return TS_ERR_INVALID_ARGUMENT;
  if (d->p == 0.0) return ts_attn_bwd(bp, workspace, workspace_bytes, stream);  // the plain path selection
  if (tsa::tc_bwd_supported(*bp)) {
    if (!workspace || workspace_bytes < tsa::tc_bwd_workspace(*bp)) return TS_ERR_WORKSPACE;
    return from_cuda(tsa::tc_backward(*bp, workspace, workspace_bytes, fault_ptr(), as_stream(stream), &args));
  }
  if (!workspace || workspace_bytes < tsa::simt_backward_workspace(*bp)) return TS_ERR_WORKSPACE;
  return from_cuda(tsa::simt_backward(*bp, workspace, as_stream(stream), &args));
}

int ts_attn_dropout_mask(const ts_dropout* d, int32_t batch, int32_t heads, int32_t q_len, int32_t kv_len,
                         uint8_t* mask, void* stream) {
  tsa::DropoutArgs args;
  if (!make_dropout(d, args) || !mask || batch <= 0 || heads <= 0 || q_len <= 0 || kv_len <= 0)
    return TS_ERR_INVALID_ARGUMENT;
  return from_cuda(tsa::dropout_mask(args, batch, heads, q_len, kv_len, mask, as_stream(stream)));
}

int ts_kv_append_int8(const ts_kv_append_params* p, float* key_scales, float* value_scales, void* stream) {
  if (!p) return TS_ERR_INVALID_ARGUMENT;
  if (!dtype_ok(p->src_dtype) || !dtype_ok(p->cache_dtype)) return TS_ERR_UNSUPPORTED;
  if (p->batch <= 0 || p->heads <= 0 || p->head_dim <= 0 || p->value_dim <= 0 || p->capacity <= 0)
    return TS_ERR_INVALID_ARGUMENT;
  if (!p->key.data || !p->value.data || !p->key_cache.data || !p->value_cache.data || !key_scales || !value_scales)
    return TS_ERR_INVALID_ARGUMENT;
  if (p->steps <= 0) return TS_ERR_CAPACITY;
  if (!p->positions && (p->position < 0 || p->position + p->steps > p->capacity)) return TS_ERR_CAPACITY;
  return from_cuda(tsa::kv_append_int8(*p, key_scales, value_scales, as_stream(stream)));
}

int ts_kv_dequant_int8(ts_view4 src, const float* scales, int64_t scale_capacity, ts_view4 dst, int32_t dtype,
                       int32_t batch, int32_t heads, int32_t length, int32_t channels, void* stream) {
  if (!dtype_ok(dtype)) return TS_ERR_UNSUPPORTED;
  if (!src.data || !dst.data || !scales || batch <= 0 || heads <= 0 || length < 0 || channels <= 0 ||
      scale_capacity < length)
    return TS_ERR_INVALID_ARGUMENT;
  return from_cuda(tsa::kv_dequant_int8(src, scales, scale_capacity, dst, dtype, batch, heads, length, channels,
                                        as_stream(stream)));
}

size_t ts_attn_decode_int8_workspace_size(const ts_attn_params* p) {
  if (check_params(p) != TS_OK || !tsa::decode_int8_supported(*p)) return 0;
  return tsa::decode_int8_workspace(*p);
}

int ts_attn_decode_int8(const ts_attn_params* p, const float* key_scales, const float* value_scales,
                        int64_t scale_capacity, void* workspace, size_t workspace_bytes, void* stream) {
  const int st = check_params(p);
  if (st != TS_OK) return st;
  if (!key_scales || !value_scales || scale_capacity < p->kv_len) return TS_ERR_INVALID_ARGUMENT;
  if (!tsa::decode_int8_supported(*p)) return TS_ERR_UNSUPPORTED;
  const size_t need = tsa::decode_int8_workspace(*p);
  if (need && (!workspace || workspace_bytes < need)) return TS_ERR_WORKSPACE;
  return from_cuda(tsa::decode_int8_forward(*p, key_scales, value_scales, scale_capacity, workspace,
                                            workspace_bytes, fault_ptr(), as_stream(stream)));
}

}  // extern "C"

namespace {

bool int4_shape_ok(int head_dim, int page_size) {
  return head_dim > 0 && head_dim <= 256 && head_dim % 32 == 0 &&
         (page_size == 16 || page_size == 32 || page_size == 64);
}

int check_int4_cache(const ts_kv4_cache* c) {
  if (!c || !c->pool || !c->table || reinterpret_cast<uintptr_t>(c->pool) % 16) return TS_ERR_INVALID_ARGUMENT;
  if (c->batch <= 0 || c->slots <= 0 || c->pages <= 0 || c->kv_heads <= 0) return TS_ERR_INVALID_ARGUMENT;
  if (!int4_shape_ok(c->head_dim, c->page_size)) return TS_ERR_UNSUPPORTED;
  if ((int64_t)c->slots * c->page_size > 0x7FFFFF00) return TS_ERR_INVALID_ARGUMENT;  // token numbers are int32
  if (c->page_stride % 16 ||
      c->page_stride < (int64_t)c->kv_heads * tsa::int4_block_bytes(c->head_dim, c->page_size))
    return TS_ERR_INVALID_ARGUMENT;
  return TS_OK;
}

bool int4_dtype_ok(int d) { return d == TS_F32 || d == TS_F16 || d == TS_BF16; }

int check_int4_attn(const ts_attn_params* p, const ts_kv4_cache* c) {
  if (!p) return TS_ERR_INVALID_ARGUMENT;
  const int st = check_int4_cache(c);
  if (st != TS_OK) return st;
  if (!int4_dtype_ok(p->dtype) || p->mask_kind != TS_MASK_NONE) return TS_ERR_UNSUPPORTED;
  if (p->batch != c->batch || p->kv_heads != c->kv_heads || p->head_dim != c->head_dim ||
      p->value_dim != c->head_dim)
    return TS_ERR_INVALID_ARGUMENT;
  if (p->q_heads <= 0 || p->q_len <= 0 || p->kv_len <= 0 || p->q_heads % p->kv_heads) return TS_ERR_INVALID_ARGUMENT;
  if (p->kv_len > (int64_t)c->slots * c->page_size) return TS_ERR_INVALID_ARGUMENT;
  if (!p->q.data || !p->o.data || !p->kv_lens) return TS_ERR_INVALID_ARGUMENT;
  if (!(p->scale == p->scale) || p->scale > 1.0e300 || p->scale < -1.0e300) return TS_ERR_INVALID_ARGUMENT;
  if ((int64_t)p->q_heads / p->kv_heads * p->q_len > 0x40000000) return TS_ERR_UNSUPPORTED;
  return TS_OK;
}

// The prefill route dequantises the keys and values of this many rows and KV heads at a time: as many as fit the
// bytes of the pool, or 1 GiB where that is more, and one head of one row at the least.  (A row takes its room up
// to kv_len, so a batch with one long row would otherwise ask for many times what its pages hold.)
struct Int4Chunk {
  int rows, heads;
};
int64_t int4_head_bytes(const ts_attn_params& p) { return (int64_t)4 * p.kv_len * p.head_dim; }  // keys and values
Int4Chunk int4_chunk(const ts_attn_params& p, const ts_kv4_cache& c) {
  const int64_t limit = tsa::i64max((int64_t)1 << 30, c.pages * c.page_stride);
  const int64_t fit = tsa::i64max(1, limit / int4_head_bytes(p));
  if (fit < p.kv_heads) return Int4Chunk{1, (int)fit};
  return Int4Chunk{(int)tsa::i64min(tsa::i64min(p.batch, 32768), fit / p.kv_heads), p.kv_heads};
}
size_t int4_prefill_bytes(const ts_attn_params& p, const ts_kv4_cache& c) {
  const Int4Chunk chunk = int4_chunk(p, c);
  return (size_t)int4_head_bytes(p) * chunk.rows * chunk.heads;
}

// Rows [row, row + chunk.rows) and KV heads [head, head + chunk.heads) of the problem over contiguous keys and
// values of q's type at `ws`.
ts_attn_params int4_prefill_params(const ts_attn_params& p, Int4Chunk chunk, int row, int head, void* ws) {
  ts_attn_params d = p;
  const int group = p.q_heads / p.kv_heads;
  d.batch = (int)tsa::i64min(chunk.rows, p.batch - row);
  d.kv_heads = (int)tsa::i64min(chunk.heads, p.kv_heads - head);
  d.q_heads = d.kv_heads * group;
  auto from = [&](const ts_view4& v) {
    return reinterpret_cast<unsigned char*>(v.data) + (row * v.stride[0] + (int64_t)head * group * v.stride[1]) * 2;
  };
  d.q.data = from(p.q);
  d.o.data = from(p.o);
  if (p.lse)
    d.lse = reinterpret_cast<float*>(p.lse) + row * p.lse_stride[0] + (int64_t)head * group * p.lse_stride[1];
  d.kv_lens = p.kv_lens ? p.kv_lens + row : nullptr;
  const int64_t stride = p.head_dim, keys = stride * p.kv_len, all = keys * d.kv_heads * d.batch;
  d.k = ts_view4{ws, {keys * d.kv_heads, keys, stride, 1}};
  d.v = ts_view4{reinterpret_cast<unsigned char*>(ws) + 2 * all, {keys * d.kv_heads, keys, stride, 1}};
  d.causal_offset = 0;
  return d;
}

// Whether dequantising the pages and running the prefill kernel is the faster way, by what each costs a cached
// key in nanoseconds (fitted at D = 128, bf16, 2 and 16 rows of 8 KV heads, groups of 1, 4 and 8 query heads,
// 64, 128 and 256 query columns a KV head).  Over the pages the time grows with the columns (group x tokens):
// 1.95e-3 a KV head and column.  The other way writes and reads the dequantised rows, 0.133 a KV head, and then
// runs one query tile a block: 6.1 a wave of 128-row tiles, 13.4 of 256-row ones (more than 128 tokens), however
// few of a tile's rows are filled; a chunk of the batch starts a wave of its own.  Rows of 8000 keys: 16 rows, 64
// columns 186 against 225 to 625 us by group; 256 columns 686 against 261, 414 and 626; 2 rows, 256 columns 102
// against 145, 93 and 94.  The same numbers serve f16 (its pages cost 1.16 times as much) and D = 64 (pages 0.65,
// tiles 0.86): over these sizes and 1024 columns the way taken is the faster one or within 1.08 (bf16, D = 128),
// 1.23 (f16, D = 128) and 1.20 (D = 64) of it.
bool int4_prefill_faster(const ts_attn_params& p, const ts_kv4_cache& c) {
  const double heads = (double)p.batch * p.kv_heads, columns = (double)(p.q_heads / p.kv_heads) * p.q_len;
  const int rows = p.q_len > 128 ? 256 : 128;
  const Int4Chunk chunk = int4_chunk(p, c);
  const int64_t tiles = (int64_t)chunk.rows * chunk.heads * (p.q_heads / p.kv_heads) * ((p.q_len + rows - 1) / rows);
  const int64_t chunks = (int64_t)((p.batch + chunk.rows - 1) / chunk.rows) * ((p.kv_heads + chunk.heads - 1) / chunk.heads);
  const double waves = (double)(chunks * ((tiles + 147) / 148));
  return 1.95e-3 * heads * columns > 0.133 * heads + waves * (rows == 256 ? 13.4 : 6.1);
}

bool int4_prefill(const ts_attn_params& p, const ts_kv4_cache& c) {
  if (!int4_dtype_ok(p.dtype) || p.dtype == TS_F32) return false;
  alignas(16) static unsigned char aligned[16];  // stands for the workspace, which must be 16-byte aligned
  if (!tsa::tc_fwd_supported(int4_prefill_params(p, int4_chunk(p, c), 0, 0, aligned))) return false;
  const char* force = std::getenv("TS_INT4_KERNEL");
  if (force && !std::strcmp(force, "pages")) return false;
  if (force && !std::strcmp(force, "prefill")) return true;
  return int4_prefill_faster(p, c);
}

// The checked problem's route and the workspace it needs.
int int4_plan(const ts_attn_params* p, const ts_kv4_cache* c, bool* prefill, size_t* bytes) {
  const int st = check_int4_attn(p, c);
  if (st != TS_OK) return st;
  *prefill = int4_prefill(*p, *c);
  if (*prefill) *bytes = int4_prefill_bytes(*p, *c);
  else if (!tsa::attn_int4_workspace(*p, bytes)) return TS_ERR_UNSUPPORTED;
  return TS_OK;
}

int check_page_pool(const ts_page_pool* p) {
  if (!p || !p->data || p->layers <= 0 || p->pages <= 0 || p->page_bytes <= 0) return TS_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(p->data) % 16 || p->page_bytes % 16 || p->page_stride % 16 ||
      p->layer_stride % 16 || p->page_stride < p->page_bytes)
    return TS_ERR_INVALID_ARGUMENT;
  return TS_OK;
}

// A table that is written to: its rows share no entry.
bool table_rows_apart(int64_t stride, int rows, int slots) { return rows == 1 || stride >= slots; }

}  // namespace

extern "C" {

size_t ts_kv4_block_bytes(int32_t head_dim, int32_t page_size) {
  return int4_shape_ok(head_dim, page_size) ? (size_t)tsa::int4_block_bytes(head_dim, page_size) : 0;
}

int ts_kv_append_int4(ts_view4 key, ts_view4 value, int32_t dtype, int32_t steps, const ts_kv4_cache* cache,
                      int64_t position, const int32_t* positions, int32_t* positions_out, void* stream) {
  const int st = check_int4_cache(cache);
  if (st != TS_OK) return st;
  if (!int4_dtype_ok(dtype)) return TS_ERR_UNSUPPORTED;
  if (!key.data || !value.data) return TS_ERR_INVALID_ARGUMENT;
  // a row's blocks read its position while one of them writes the next one
  if (positions && positions_out && positions < positions_out + cache->batch && positions_out < positions + cache->batch)
    return TS_ERR_INVALID_ARGUMENT;
  if (steps <= 0) return TS_ERR_CAPACITY;
  if (!positions && (position < 0 || position + steps > (int64_t)cache->slots * cache->page_size))
    return TS_ERR_CAPACITY;
  return from_cuda(tsa::kv_append_int4(key, value, dtype, steps, *cache, position, positions, positions_out,
                                       fault_ptr(), as_stream(stream)));
}

int ts_kv_gather_int4(const ts_kv4_cache* cache, const int32_t* starts, const int32_t* lens, ts_view4 key,
                      ts_view4 value, int32_t dtype, int32_t length, void* stream) {
  const int st = check_int4_cache(cache);
  if (st != TS_OK) return st;
  if (!int4_dtype_ok(dtype)) return TS_ERR_UNSUPPORTED;
  if (!key.data || !value.data || length < 0) return TS_ERR_INVALID_ARGUMENT;
  if (!starts && length > (int64_t)cache->slots * cache->page_size) return TS_ERR_INVALID_ARGUMENT;
  return from_cuda(tsa::kv_gather_int4(*cache, starts, lens, key, value, dtype, length, 0, fault_ptr(),
                                       as_stream(stream)));
}

int ts_attn_int4_path(const ts_attn_params* p, const ts_kv4_cache* cache) {
  bool prefill = false;
  size_t bytes = 0;
  const int st = int4_plan(p, cache, &prefill, &bytes);
  return st != TS_OK ? st : prefill ? TS_PATH_TCGEN05 : TS_PATH_DECODE;
}

size_t ts_attn_int4_workspace_size(const ts_attn_params* p, const ts_kv4_cache* cache) {
  bool prefill = false;
  size_t bytes = 0;
  return int4_plan(p, cache, &prefill, &bytes) == TS_OK ? bytes : 0;
}

int ts_attn_int4(const ts_attn_params* p, const ts_kv4_cache* cache, void* workspace, size_t workspace_bytes,
                 void* stream) {
  bool prefill = false;
  size_t need = 0;
  const int st = int4_plan(p, cache, &prefill, &need);
  if (st != TS_OK) return st;
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return TS_ERR_WORKSPACE;
  if (!prefill) return from_cuda(tsa::attn_int4_forward(*p, *cache, workspace, fault_ptr(), as_stream(stream)));
  const Int4Chunk chunk = int4_chunk(*p, *cache);
  for (int row = 0; row < p->batch; row += chunk.rows)  // one after the other on the stream, in the same workspace
    for (int head = 0; head < p->kv_heads; head += chunk.heads) {
      const ts_attn_params d = int4_prefill_params(*p, chunk, row, head, workspace);
      ts_kv4_cache c = *cache;
      c.pool = reinterpret_cast<unsigned char*>(c.pool) + (int64_t)head * tsa::int4_block_bytes(c.head_dim, c.page_size);
      c.kv_heads = d.kv_heads;
      c.table += row * c.table_stride;
      c.batch = d.batch;
      cudaError_t e = tsa::kv_gather_int4(c, nullptr, d.kv_lens, d.k, d.v, d.dtype, d.kv_len, tsa::kTcKeyTile,
                                          fault_ptr(), as_stream(stream));
      if (e == cudaSuccess) e = tsa::tc_forward(d, fault_ptr(), as_stream(stream));
      if (e != cudaSuccess) return from_cuda(e);
    }
  return TS_OK;
}

int ts_kv_pages_copy(const ts_page_pool* src, const ts_page_pool* dst, const int32_t* from, const int32_t* to,
                     int32_t count, void* stream) {
  if (check_page_pool(src) != TS_OK || check_page_pool(dst) != TS_OK) return TS_ERR_INVALID_ARGUMENT;
  if (src->page_bytes != dst->page_bytes || src->layers != dst->layers || count < 0 || (count && (!from || !to)))
    return TS_ERR_INVALID_ARGUMENT;
  return from_cuda(tsa::kv_pages_copy(*src, *dst, from, to, count, as_stream(stream)));
}

int ts_kv_pages_fork(const int32_t* table, int64_t table_stride, const int32_t* lens, int32_t rows,
                     const int32_t* index, int32_t* table_out, int64_t table_out_stride, int32_t* lens_out,
                     int32_t rows_out, int32_t slots, int32_t page_size, int32_t* refs, int32_t pages,
                     int32_t* counters, void* stream) {
  if (!table || !lens || !index || !table_out || !lens_out || !refs || !counters || table == table_out ||
      lens == lens_out)
    return TS_ERR_INVALID_ARGUMENT;
  if (rows <= 0 || rows_out <= 0 || slots <= 0 || page_size <= 0 || pages <= 0) return TS_ERR_INVALID_ARGUMENT;
  if (!table_rows_apart(table_out_stride, rows_out, slots)) return TS_ERR_INVALID_ARGUMENT;
  return from_cuda(tsa::kv_pages_fork(table, table_stride, lens, rows, index, table_out, table_out_stride, lens_out,
                                      rows_out, slots, page_size, refs, pages, counters, as_stream(stream)));
}

size_t ts_kv_pages_reserve_workspace_size(int32_t pages, int32_t rows) {
  return pages > 0 && rows > 0 ? tsa::kv_pages_reserve_workspace(pages, rows) : 0;
}

int ts_kv_pages_reserve(const ts_page_pool* pool, int32_t* table, int64_t table_stride, const int32_t* lens,
                        int32_t rows, int32_t slots, int32_t page_size, int32_t steps, const int32_t* row_steps,
                        int32_t* refs, int32_t* counters, void* workspace, size_t workspace_bytes, void* stream) {
  const int st = check_page_pool(pool);
  if (st != TS_OK) return st;
  if (!table || !lens || !refs || !counters || rows <= 0 || slots <= 0 || page_size <= 0 || steps < 0)
    return TS_ERR_INVALID_ARGUMENT;
  if (!table_rows_apart(table_stride, rows, slots)) return TS_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < tsa::kv_pages_reserve_workspace(pool->pages, rows) ||
      reinterpret_cast<uintptr_t>(workspace) % sizeof(int32_t))
    return TS_ERR_WORKSPACE;
  return from_cuda(tsa::kv_pages_reserve(*pool, table, table_stride, lens, rows, slots, page_size, steps, row_steps,
                                         refs, counters, workspace, as_stream(stream)));
}

size_t ts_kv_pages_compact_workspace_size(int32_t pages) {
  return pages > 0 ? tsa::kv_pages_compact_workspace(pages) : 0;
}

int ts_kv_pages_compact(const ts_page_pool* pool, const int32_t* table, int64_t table_stride, int32_t* table_out,
                        int64_t table_out_stride, int32_t rows, int32_t slots, const int32_t* refs,
                        int32_t* refs_out, int32_t* counters, void* workspace, size_t workspace_bytes,
                        void* stream) {
  const int st = check_page_pool(pool);
  if (st != TS_OK) return st;
  if (!table || !table_out || !refs || !refs_out || !counters || rows <= 0 || slots <= 0)
    return TS_ERR_INVALID_ARGUMENT;
  if (!table_rows_apart(table_out_stride, rows, slots)) return TS_ERR_INVALID_ARGUMENT;
  if (!workspace || workspace_bytes < tsa::kv_pages_compact_workspace(pool->pages) ||
      reinterpret_cast<uintptr_t>(workspace) % sizeof(int32_t))
    return TS_ERR_WORKSPACE;
  return from_cuda(tsa::kv_pages_compact(*pool, table, table_out, rows, slots, table_stride, table_out_stride, refs,
                                         refs_out, counters, workspace, as_stream(stream)));
}

}  // extern "C"

namespace {

// One of the four instantiations of a family of kernels.
template <typename F32, typename F64, typename F16, typename BF16, typename... A>
cudaError_t by_dtype(int dtype, F32 f32, F64 f64, F16 f16, BF16 bf16, A&&... a) {
  switch (dtype) {
    case TS_F32: return f32(a...);
    case TS_F64: return f64(a...);
    case TS_F16: return f16(a...);
    case TS_BF16: return bf16(a...);
  }
  return cudaErrorInvalidValue;
}

constexpr int kGridMax = 65535;  // of a grid's second and third dimension
constexpr int kMaxKeys = 1 << 30;  // tiles' ends behind the last key stay 32-bit numbers

int check_window(const ts_attn_params* p, const ts_window* w) {
  const int st = check_params(p);
  if (st != TS_OK) return st;
  if (!w || w->window < 1 || w->sinks < 0 || !p->is_causal) return TS_ERR_INVALID_ARGUMENT;
  if (p->causal_offset > (int64_t)1 << 62) return TS_ERR_INVALID_ARGUMENT;  // positions behind it stay 64-bit numbers
  if (p->mask_kind != TS_MASK_NONE) return TS_ERR_UNSUPPORTED;
  if (p->q_heads > kGridMax || p->batch > kGridMax || (int64_t)p->kv_heads * p->batch > 0x7fffffff ||
      p->kv_len > kMaxKeys)
    return TS_ERR_UNSUPPORTED;
  return TS_OK;
}
tsa::WindowArgs window_args(const ts_window* w) {
  tsa::WindowArgs a;
  a.window = w->window;
  a.sinks = w->sinks;
  return a;
}

int check_window_bwd(const ts_attn_bwd_params* bp, const ts_window* w) {
  if (!bp) return TS_ERR_INVALID_ARGUMENT;
  const int st = check_window(&bp->fwd, w);
  if (st != TS_OK) return st;
  if (!bp->fwd.lse || !bp->dout.data || !bp->dq.data || !bp->dk.data || !bp->dv.data) return TS_ERR_INVALID_ARGUMENT;
  // Tiles of 128 keys are a grid's second dimension on the tensor cores, those with sinks in up to 64 parts (only while
  // there are fewer of them than SMs).
  if (bp->fwd.kv_len > 64 * kGridMax || (int64_t)bp->fwd.batch * bp->fwd.q_heads > 0x7fffffff ||
      (int64_t)bp->fwd.batch * bp->fwd.q_heads * bp->fwd.q_len > (int64_t)1 << 33)
    return TS_ERR_UNSUPPORTED;
  return TS_OK;
}
cudaError_t rows_window_bwd(const ts_attn_bwd_params& bp, const tsa::WindowArgs& win, size_t* bytes, void* ws,
                            cudaStream_t st) {
  return by_dtype(bp.fwd.dtype, tsa::rows_window_bwd_f32, tsa::rows_window_bwd_f64, tsa::rows_window_bwd_f16,
                  tsa::rows_window_bwd_bf16, bp, win, bytes, ws, st);
}
size_t window_bwd_workspace(const ts_attn_bwd_params& bp, const tsa::WindowArgs& win) {
  if (tsa::tc_bwd_window_supported(bp)) return tsa::tc_bwd_window_workspace(bp, win);
  size_t bytes = 0;
  (void)rows_window_bwd(bp, win, &bytes, nullptr, nullptr);
  return bytes;
}

int check_tree(const ts_attn_params* p, const ts_tree* t) {
  if (!t || !p || !p->kv_lens) return TS_ERR_INVALID_ARGUMENT;
  ts_attn_params q = *p;  // the rule is the tree's, whatever the causal fields hold
  q.causal_offset = 0;
  const int st = check_params(&q);
  if (st != TS_OK) return st;
  if (t->window < 0 || t->sinks < 0) return TS_ERR_INVALID_ARGUMENT;
  if (p->mask_kind != TS_MASK_NONE) return TS_ERR_UNSUPPORTED;
  if (t->parents && p->q_len > TS_TREE_MAX_NODES) return TS_ERR_UNSUPPORTED;
  if (p->kv_len > kMaxKeys) return TS_ERR_UNSUPPORTED;
  if ((int64_t)p->q_heads / p->kv_heads * p->q_len > 0x40000000 ||
      (int64_t)p->batch * p->q_heads * p->q_len > 0x40000000)
    return TS_ERR_UNSUPPORTED;
  return TS_OK;
}
cudaError_t rows_tree(const ts_attn_params& p, tsa::TreeArgs* a, size_t* bytes, void* ws, cudaStream_t st) {
  return by_dtype(p.dtype, tsa::rows_tree_f32, tsa::rows_tree_f64, tsa::rows_tree_f16, tsa::rows_tree_bf16, p, a,
                  bytes, ws, st);
}
size_t tree_workspace(const ts_attn_params& p) {
  if (tsa::tc_tree_supported(p)) return tsa::tc_tree_workspace(p);
  size_t bytes = 0;
  if (p.dtype != TS_F64) (void)rows_tree(p, nullptr, &bytes, nullptr, nullptr);
  return bytes;
}
cudaError_t tree_run(const ts_attn_params& p, const int32_t* parents, int64_t parents_stride, const tsa::WindowArgs& win,
                     void* workspace, cudaStream_t st) {
  if (tsa::tc_tree_supported(p)) return tsa::tc_tree(p, parents, parents_stride, win, workspace, fault_ptr(), st);
  tsa::TreeArgs a = {};
  a.parents = parents;
  a.parents_stride = parents_stride;
  a.win = win;
  size_t bytes;
  return rows_tree(p, &a, &bytes, workspace, st);
}

// Whether a windowed forward is shared along its keys (ts_attn_tree's kernels over a chain) rather than given to one
// block a query tile, by what both take in microseconds.  On the tensor cores a tile of 128 keys takes a query tile's
// CTA 1.45 and an SM's share of the line 2.5, which also starts, waits and merges for 14 and 0.16 a row (one token of
// 32 / 8 heads of 128 over a window of 4096: 19 against 51; 16 tokens 30 against 51, 128 tokens 67 against 52; one
// token, a window of 100: 12 against 9).  On CUDA cores a block's tile takes 4.5 while its SM has no other, the line's
// 25 (64 keys, up to 64 channels) or 16 (32 keys) behind 15 (one token of 8 heads of 64, a window of 500: 23 against
// 45, 500 tokens 75 against 59; 300 tokens of 8 / 2 heads of 128, a window of 2000: 156 against 311).
bool window_split_faster(const ts_attn_params& p, const tsa::WindowArgs& win, bool tc) {
  const int dim = p.head_dim > p.value_dim ? p.head_dim : p.value_dim, sms = tsa::device_sms();
  const int group = p.q_heads / p.kv_heads, keys = tc ? 128 : dim <= 64 ? 64 : 32, line_rows = tc ? 128 : 64;
  const int64_t heads = (int64_t)p.q_heads * p.batch;
  const int rt = tc ? 8 : tsa::rows_rt(p.q_len, heads, tsa::rows_widest(dim));
  const int64_t rows = (int64_t)group * p.q_len, units = (rows + line_rows - 1) / line_rows * p.kv_heads * p.batch;
  // Key tiles of a block of `queries` tokens.
  auto tiles = [&](int64_t queries) {
    const int64_t all = (p.kv_len + keys - 1) / keys;
    const int64_t near = (win.window + tsa::i64min(queries, p.q_len) + keys - 2) / keys + 1;
    return (double)tsa::i64min(all, near + ((int64_t)win.sinks + keys - 1) / keys);
  };
  const int64_t blocks = (p.q_len + 16 * rt - 1) / (16 * rt) * heads, waves = (blocks + sms - 1) / sms;
  const double line = (double)units * (tiles(line_rows) + (tc ? 2 : 0)) / (tc ? sms : 2 * sms);
  if (tc) return 14 + 2.5 * line + 0.16 * (rows < 128 ? rows : 128) < 0.9 * (5 + 1.45 * waves * tiles(128));
  const double share = waves * (8.0 + rt) / 13;
  return 15 + (keys == 64 ? 25 : 16) * (line > 1 ? line : 1) < 0.9 * (5 + 4.5 * tiles(16 * rt) * (share > 1 ? share : 1));
}

bool window_split(const ts_attn_params& p, const tsa::WindowArgs& win) {
  if (p.dtype == TS_F64) return false;
  if (!p.kv_lens && p.causal_offset + p.q_len > p.kv_len) return false;  // a chain's tokens are the last of the keys
  const bool tc = tsa::tc_window_supported(p);
  if (tc != tsa::tc_tree_supported(p) || (int64_t)p.q_heads * p.q_len * p.batch > 0x40000000) return false;
  const char* force = std::getenv("TS_WINDOW_KERNEL");
  if (force && !std::strcmp(force, "split")) return true;
  if (force && (!std::strcmp(force, "tile") || !std::strcmp(force, "pair"))) return false;
  return window_split_faster(p, win, tc);
}

}  // namespace

extern "C" {

int ts_attn_window_path(const ts_attn_params* p, const ts_window* w) {
  const int st = check_window(p, w);
  if (st != TS_OK) return st;
  return tsa::tc_window_supported(*p) ? TS_PATH_TCGEN05 : TS_PATH_SIMT;
}

size_t ts_attn_fwd_window_workspace_size(const ts_attn_params* p, const ts_window* w) {
  return check_window(p, w) == TS_OK && window_split(*p, window_args(w)) ? tree_workspace(*p) : 0;
}

int ts_attn_fwd_window(const ts_attn_params* p, const ts_window* w, void* workspace, size_t workspace_bytes,
                       void* stream) {
  const int st = check_window(p, w);
  if (st != TS_OK) return st;
  const tsa::WindowArgs win = window_args(w);
  if (window_split(*p, win)) {  // a chain of tokens over the keys
    if (!workspace || workspace_bytes < tree_workspace(*p) || reinterpret_cast<uintptr_t>(workspace) % 16)
      return TS_ERR_WORKSPACE;
    return from_cuda(tree_run(*p, nullptr, 0, win, workspace, as_stream(stream)));
  }
  if (tsa::tc_window_supported(*p)) return from_cuda(tsa::tc_forward_window(*p, win, fault_ptr(), as_stream(stream)));
  const tsa::RowsWindow a = {*p, win};
  return from_cuda(by_dtype(p->dtype, tsa::rows_window_fwd_f32, tsa::rows_window_fwd_f64, tsa::rows_window_fwd_f16,
                            tsa::rows_window_fwd_bf16, a, as_stream(stream)));
}

size_t ts_attn_bwd_window_workspace_size(const ts_attn_bwd_params* bp, const ts_window* w) {
  return check_window_bwd(bp, w) == TS_OK ? window_bwd_workspace(*bp, window_args(w)) : 0;
}

int ts_attn_bwd_window(const ts_attn_bwd_params* bp, const ts_window* w, void* workspace, size_t workspace_bytes,
                       void* stream) {
  const int st = check_window_bwd(bp, w);
  if (st != TS_OK) return st;
  const tsa::WindowArgs win = window_args(w);
  if (!workspace || workspace_bytes < window_bwd_workspace(*bp, win) || reinterpret_cast<uintptr_t>(workspace) % 16)
    return TS_ERR_WORKSPACE;
  if (tsa::tc_bwd_window_supported(*bp))
    return from_cuda(
        tsa::tc_backward(*bp, workspace, workspace_bytes, fault_ptr(), as_stream(stream), nullptr, &win));
  size_t bytes;
  return from_cuda(rows_window_bwd(*bp, win, &bytes, workspace, as_stream(stream)));
}

int ts_attn_tree_path(const ts_attn_params* p, const ts_tree* t) {
  const int st = check_tree(p, t);
  if (st != TS_OK) return st;
  return tsa::tc_tree_supported(*p) ? TS_PATH_TCGEN05 : TS_PATH_SIMT;
}

size_t ts_attn_tree_workspace_size(const ts_attn_params* p, const ts_tree* t) {
  return check_tree(p, t) == TS_OK ? tree_workspace(*p) : 0;
}

int ts_attn_tree(const ts_attn_params* p, const ts_tree* t, void* workspace, size_t workspace_bytes, void* stream) {
  const int st = check_tree(p, t);
  if (st != TS_OK) return st;
  const size_t need = tree_workspace(*p);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
    return TS_ERR_WORKSPACE;
  tsa::WindowArgs win;
  win.window = t->window;
  win.sinks = t->sinks;
  return from_cuda(tree_run(*p, t->parents, t->parents_stride, win, workspace, as_stream(stream)));
}

int ts_tree_positions(const int32_t* parents, int64_t parents_stride, const int32_t* lens, int32_t batch,
                      int32_t nodes, int32_t* positions, void* stream) {
  if (!parents || !lens || !positions || batch <= 0 || nodes <= 0) return TS_ERR_INVALID_ARGUMENT;
  return from_cuda(tsa::tree_positions(parents, parents_stride, lens, batch, nodes, positions, as_stream(stream)));
}

int ts_rope_at(ts_view4 x, ts_view4 y, int32_t dtype, int32_t batch, int32_t heads, int32_t seq, int32_t channels,
               int32_t rotary_dim, const int32_t* positions, const float* inv_freq, int32_t inverse, void* stream) {
  if (!dtype_ok(dtype)) return TS_ERR_UNSUPPORTED;
  if (!x.data || !y.data || !inv_freq || !positions || batch <= 0 || heads <= 0 || seq <= 0 || channels <= 0)
    return TS_ERR_INVALID_ARGUMENT;
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > channels) return TS_ERR_INVALID_ARGUMENT;
  if (batch > kGridMax) return TS_ERR_UNSUPPORTED;
  return from_cuda(tsa::rope_apply(x, y, dtype, batch, heads, seq, channels, rotary_dim, 0, positions, inv_freq,
                                   inverse, as_stream(stream), true));
}

int ts_kv_keep(const ts_kv_keep_params* p, void* stream) {
  if (!p || !p->keys || !p->values || !p->base || !p->path || !p->counts) return TS_ERR_INVALID_ARGUMENT;
  if (!dtype_ok(p->dtype) && p->dtype != TS_I8) return TS_ERR_UNSUPPORTED;
  if (p->layers <= 0 || p->batch <= 0 || p->heads <= 0 || p->head_dim <= 0 || p->value_dim <= 0 || p->capacity <= 0 ||
      p->nodes <= 0 || p->key_stride[3] != 1 || p->value_stride[3] != 1)
    return TS_ERR_INVALID_ARGUMENT;
  if (p->batch > kGridMax) return TS_ERR_UNSUPPORTED;
  const int size = p->dtype == TS_F64 ? 8 : p->dtype == TS_F32 ? 4 : p->dtype == TS_I8 ? 1 : 2;
  tsa::KvKeep a = {};
  for (int i = 0; i < 3; ++i) {
    a.stride[0][i] = p->key_stride[i] * size;
    a.stride[1][i] = p->value_stride[i] * size;
  }
  a.row_bytes[0] = p->head_dim * size;
  a.row_bytes[1] = p->value_dim * size;
  a.batch = p->batch;
  a.heads = p->heads;
  a.nodes = p->nodes;
  a.capacity = p->capacity;
  a.base = p->base;
  a.path = p->path;
  a.counts = p->counts;
  a.path_stride = p->path_stride;
  for (int l = 0; l < p->layers; ++l)
    if (!p->keys[l] || !p->values[l]) return TS_ERR_INVALID_ARGUMENT;
  for (int l0 = 0; l0 < p->layers; l0 += tsa::kKeepTensors / 2) {
    a.tensors = 0;
    for (int l = l0; l < p->layers && a.tensors < tsa::kKeepTensors; ++l) {
      a.data[a.tensors++] = p->keys[l];
      a.data[a.tensors++] = p->values[l];
    }
    const cudaError_t e = tsa::kv_keep(a, as_stream(stream));
    if (e != cudaSuccess) return from_cuda(e);
  }
  return TS_OK;
}

}  // extern "C"

namespace {

int check_logprobs(const ts_token_logprobs* p) {
  if (!p || !p->logits || p->rows <= 0 || p->vocab <= 0 || p->top < 0 || p->top > p->vocab)
    return TS_ERR_INVALID_ARGUMENT;
  if ((p->dtype != TS_F32 && p->dtype != TS_F16 && p->dtype != TS_BF16) || p->top > TS_TOP_TOKENS_MAX)
    return TS_ERR_UNSUPPORTED;
  const int size = p->dtype == TS_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(p->logits) % size || (p->rows > 1 && p->stride < 0)) return TS_ERR_INVALID_ARGUMENT;
  return TS_OK;
}

}  // namespace

extern "C" {

int ts_token_logprobs_fwd(const ts_token_logprobs* p, void* stream) {
  const int st = check_logprobs(p);
  if (st != TS_OK) return st;
  if ((p->logprob && !p->targets) || (p->top && (!p->top_logprobs || !p->top_indices))) return TS_ERR_INVALID_ARGUMENT;
  return from_cuda(tsa::token_logprobs(*p, as_stream(stream)));
}

int ts_token_logprobs_bwd(const ts_token_logprobs* p, const float* grad_logprob, const float* grad_entropy,
                          const float* grad_top, void* grad_logits, int64_t grad_stride, void* stream) {
  const int st = check_logprobs(p);
  if (st != TS_OK) return st;
  if (!p->targets || !p->norm || !p->entropy || !grad_logits || grad_logits == p->logits ||
      (grad_top && p->top && !p->top_indices) || (p->rows > 1 && grad_stride < p->vocab))
    return TS_ERR_INVALID_ARGUMENT;
  if ((int64_t)p->rows * (p->vocab / 4096 + 1) > 0x7fffffff) return TS_ERR_UNSUPPORTED;
  return from_cuda(tsa::token_logprobs_bwd(*p, grad_logprob, grad_entropy, grad_top, grad_logits, grad_stride,
                                           as_stream(stream)));
}

int ts_attn_device_status(void* stream, uint32_t* info) {
  uint32_t* f = fault_ptr();
  if (!f) return TS_ERR_LAUNCH;
  uint32_t host = 0;
  cudaStream_t s = as_stream(stream);
  if (cudaMemcpyAsync(&host, f, sizeof(uint32_t), cudaMemcpyDeviceToHost, s) != cudaSuccess) return TS_ERR_LAUNCH;
  if (cudaStreamSynchronize(s) != cudaSuccess) return TS_ERR_LAUNCH;
  if (info) *info = host;
  if (host) {
    const uint32_t zero = 0;
    if (cudaMemcpyAsync(f, &zero, sizeof(uint32_t), cudaMemcpyHostToDevice, s) != cudaSuccess ||
        cudaStreamSynchronize(s) != cudaSuccess)
      return TS_ERR_LAUNCH;
    return host == tsa::FAULT_PAGE ? TS_ERR_PAGE : TS_ERR_DEVICE_TIMEOUT;
  }
  return TS_OK;
}

}  // extern "C"
