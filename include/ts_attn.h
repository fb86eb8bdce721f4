/*
 * ts_attn.h -- C ABI of the B200 attention engine for tensorsmith.
 *
 * The engine replaces the compute behind tensorsmith's attention path
 * (tensorsmith 0.3.0; file:line below are relative to the tensorsmith project
 * root).  Every entry point takes plain device pointers, element strides and
 * sizes; the caller owns all memory (outputs and workspaces included).  Calls
 * are asynchronous on the given CUDA stream (a cudaStream_t passed as void*,
 * NULL = legacy default stream) of the current device.  Every entry point
 * returns TS_OK (0) or a negative ts_status and never aborts the process.
 *
 * Layout convention: a 4-D view [batch, heads, sequence, channels] is a base
 * pointer plus four ELEMENT strides, so tensors coming from tensorsmith's
 * reshape/permute (nn/transformer.py:124-138, memory order B,T,H,D) are
 * accepted without a copy.
 */
#ifndef TS_ATTN_H
#define TS_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TS_ATTN_ABI_VERSION 1

#if defined(__GNUC__)
#define TS_ATTN_API __attribute__((visibility("default")))
#else
#define TS_ATTN_API
#endif

/* Element types.  Half types compute in fp32 with fp32 softmax statistics,
 * as the reference does (nn/attention.py:63); fp64 computes in fp64. */
typedef enum ts_dtype { TS_F32 = 0, TS_F16 = 1, TS_BF16 = 2, TS_F64 = 3, TS_I8 = 4 } ts_dtype;
/* TS_I8 is a storage type only: the int8 KV cache of nn/cache.py:47-52
 * (ts_kv_append_int8, ts_kv_dequant_int8, ts_kv_reorder and the K/V views of
 * ts_attn_decode_int8).  No attention entry point computes in it. */

/* Optional attention mask of nn/attention.py:64-76, 105-107:
 * BOOL  -- uint8 0/1, True (1) = allowed, False -> score -inf;
 * ADD   -- values added to the scaled scores: fp32, or fp64 when dtype is TS_F64. */
typedef enum ts_mask_kind { TS_MASK_NONE = 0, TS_MASK_BOOL = 1, TS_MASK_ADD_F32 = 2 } ts_mask_kind;

typedef enum ts_status {
  TS_OK = 0,
  TS_ERR_INVALID_ARGUMENT = -1, /* shape / stride / pointer / value check failed */
  TS_ERR_UNSUPPORTED = -2,      /* combination not implemented by any kernel */
  TS_ERR_WORKSPACE = -3,        /* workspace missing or smaller than required */
  TS_ERR_LAUNCH = -4,           /* kernel launch or driver call failed */
  TS_ERR_DEVICE_TIMEOUT = -5,   /* a bounded wait inside a kernel gave up */
  TS_ERR_CAPACITY = -6,         /* KV-cache append would exceed the capacity */
  TS_ERR_PAGE = -7              /* a kernel met a page table entry outside the pool */
} ts_status;

/* Which kernel family ts_attn_fwd would run (for tests and diagnostics). */
typedef enum ts_fwd_path {
  TS_PATH_NONE = 0,
  TS_PATH_TCGEN05 = 1, /* bf16/f16 tensor-core prefill (tcgen05 + TMEM + TMA) */
  TS_PATH_SIMT = 2,    /* generic CUDA-core path (any dtype/dim/mask) */
  TS_PATH_DECODE = 3   /* split-K HBM-streaming decode */
} ts_fwd_path;

/* A [B, H, T, C] view: base pointer + element strides (b, h, t, c). */
typedef struct ts_view4 {
  void* data;
  int64_t stride[4];
} ts_view4;

/* Forward / decode problem.  Mirrors the arguments of
 * scaled_dot_product_attention (nn/attention.py:16-29). */
typedef struct ts_attn_params {
  ts_view4 q;  /* [B, Hq,  Tq, D]  */
  ts_view4 k;  /* [B, Hkv, Tk, D]  */
  ts_view4 v;  /* [B, Hkv, Tk, Dv] */
  ts_view4 o;  /* [B, Hq,  Tq, Dv] output, same dtype as q */
  /* optional [B, Hq, Tq] natural-log normaliser (-inf = fully masked row);
   * fp32, or fp64 when dtype is TS_F64 */
  void* lse;
  int64_t lse_stride[3];
  int32_t dtype; /* ts_dtype of q, k, v and o */
  int32_t batch, q_heads, kv_heads, q_len, kv_len, head_dim, value_dim;
  double scale;          /* softmax scale; the reference default is 1/sqrt(D) (nn/attention.py:60) */
  int32_t is_causal;     /* key j visible to query i iff i + offset >= j (nn/attention.py:108-111) */
  int64_t causal_offset; /* absolute position of query 0 in the key sequence */
  /* Optional per-row valid key count [B] (int32, device).  Keys j >= kv_lens[b]
   * are masked.  When set together with is_causal, the queries of row b sit at
   * the end of its valid keys: offset_b = kv_lens[b] - q_len (causal_offset is
   * then ignored).  Expresses tensorsmith's padded-cache + key-valid-mask idiom
   * (docs/transformers.md:52-55) without a mask tensor. */
  const int32_t* kv_lens;
  int32_t mask_kind;  /* ts_mask_kind */
  const void* mask;   /* [B, Hq, Tq, Tk] with broadcast (0) strides allowed */
  int64_t mask_stride[4];
} ts_attn_params;

/* Backward problem: the forward problem plus upstream and gradient views. */
typedef struct ts_attn_bwd_params {
  ts_attn_params fwd; /* q, k, v, o (forward output) and lse (required) */
  ts_view4 dout;      /* [B, Hq,  Tq, Dv] upstream gradient, dtype of q */
  ts_view4 dq;        /* [B, Hq,  Tq, D]  */
  ts_view4 dk;        /* [B, Hkv, Tk, D]  (summed over the query-head group) */
  ts_view4 dv;        /* [B, Hkv, Tk, Dv] */
} ts_attn_bwd_params;

/* KV-cache append: write a [B, H, steps, C] chunk at positions
 * [pos_b, pos_b + steps) of [B, H, capacity, C] caches. */
typedef struct ts_kv_append_params {
  ts_view4 key, value;             /* new chunk */
  ts_view4 key_cache, value_cache; /* preallocated storage */
  int32_t src_dtype;               /* ts_dtype of key/value (cast on write) */
  int32_t cache_dtype;             /* ts_dtype of the caches */
  int32_t batch, heads, steps, head_dim, value_dim, capacity;
  int64_t position;          /* write offset for every row when positions == NULL */
  const int32_t* positions;  /* optional [B] per-row write offsets (device) */
  int32_t* positions_out;    /* optional [B]: receives positions[b] + steps */
} ts_kv_append_params;

/* ABI version (TS_ATTN_ABI_VERSION) of the loaded library. */
TS_ATTN_API int ts_attn_abi_version(void);

/* Static description of a status code. */
TS_ATTN_API const char* ts_attn_strerror(int status);

/* Build provenance (no counterpart in tensorsmith): SHA-256, as 64 hex digits,
 * of the sources this library was compiled from -- every csrc/*.cu, csrc/*.cuh
 * and include/*.h, hashed in file-name order as name, NUL, contents, NUL.  The
 * Python loader refuses a library whose digest differs from the tree's. */
TS_ATTN_API const char* ts_attn_source_digest(void);

/* Kernel family ts_attn_fwd / ts_attn_decode would select (ts_fwd_path), or a
 * negative ts_status when the parameters are invalid. */
TS_ATTN_API int ts_attn_fwd_path(const ts_attn_params* params, int decode);

/* Prefill / training forward: O and (optionally) LSE.  Replaces the dense,
 * streaming and native forwards of nn/attention.py:132-198 (the native slot
 * :146-174 is where tensorsmith plugs a vendor kernel).  On the tensor-core
 * path the library picks the kernel by shape (two query tiles per CTA for two
 * or more 128-row tiles); the environment variable TS_FWD_KERNEL = "pair",
 * "tile" or "persistent", read at every call, forces one for tests and
 * measurements.  Results are the same within the stated tolerances. */
TS_ATTN_API int ts_attn_fwd(const ts_attn_params* params, void* stream);

/* Workspace bytes ts_attn_bwd needs (fp32 row statistics, plus an fp32 dQ
 * accumulator on the tensor-core path). */
TS_ATTN_API size_t ts_attn_bwd_workspace_size(const ts_attn_bwd_params* params);

/* Kernel family ts_attn_bwd would run (TS_PATH_TCGEN05 or TS_PATH_SIMT), or a
 * negative ts_status when the parameters are invalid. */
TS_ATTN_API int ts_attn_bwd_path(const ts_attn_bwd_params* params);

/* Backward: dQ, dK, dV from recomputed probabilities (LSE of the forward).
 * Replaces the dense / blockwise VJP and the GQA reduction of
 * nn/attention.py:200-248. */
TS_ATTN_API int ts_attn_bwd(const ts_attn_bwd_params* params, void* workspace, size_t workspace_bytes,
                void* stream);

/* Workspace bytes ts_attn_decode needs (per-split partial results). */
TS_ATTN_API size_t ts_attn_decode_workspace_size(const ts_attn_params* params);

/* Cached decode: a few query tokens against a long KV cache, split along the
 * keys and combined.  Same semantics as ts_attn_fwd; replaces the cached call
 * of nn/transformer.py:144-154 into nn/attention.py:132-145.  A grouped-query
 * step (one query token, 2-128 query heads per KV head, no mask, at least 64
 * (batch, KV head) pairs) runs on the tcgen05 prefill kernel with the query
 * heads of each KV head as the rows of one tile (ts_attn_fwd_path(params, 1)
 * then returns TS_PATH_TCGEN05).  Problems neither kernel family takes
 * (ts_attn_fwd_path(params, 1) != TS_PATH_DECODE) run exactly as ts_attn_fwd;
 * only TS_PATH_DECODE needs a workspace. */
TS_ATTN_API int ts_attn_decode(const ts_attn_params* params, void* workspace, size_t workspace_bytes,
                   void* stream);

/* KVCache.append slice write (nn/cache.py:54-86, unquantized storage). */
TS_ATTN_API int ts_kv_append(const ts_kv_append_params* params, void* stream);

/* Interleaved-pair rotary embedding of nn/attention.py:255-296 on a
 * [B, H, T, C] view: y = rope(x) at positions (positions[b] or offset) + t,
 * first rotary_dim (even) channels, inv_freq[i] = base^(-2i/rotary_dim) as
 * fp32 (rotary_dim/2 entries, device).  inverse != 0 applies the inverse
 * rotation (the VJP of :287-293).  y may alias x. */
TS_ATTN_API int ts_rope(ts_view4 x, ts_view4 y, int32_t dtype, int32_t batch, int32_t heads, int32_t seq,
                        int32_t channels, int32_t rotary_dim, int64_t offset, const int32_t* positions,
                        const float* inv_freq, int32_t inverse, void* stream);

/* KVCache.append with the key rotation of the attention module fused into the
 * write (nn/transformer.py:139-142 followed by nn/cache.py:54-86): keys are
 * rotated at their cache positions, values copied. */
TS_ATTN_API int ts_kv_append_rope(const ts_kv_append_params* params, const float* inv_freq, int32_t rotary_dim,
                                  void* stream);

/* KVCache.reorder batch gather (nn/cache.py:110-123): dst[b] = src[index[b]].
 * src and dst must not overlap. */
TS_ATTN_API int ts_kv_reorder(ts_view4 src, ts_view4 dst, int32_t dtype, int32_t batch, int32_t heads,
                  int32_t length, int32_t channels, const int32_t* index, void* stream);

/* Size of the fixed device scratch ts_attn_decode_noalloc uses (8 MiB per GPU). */
#define TS_ATTN_NOALLOC_SCRATCH_BYTES ((size_t)8 << 20)

/* Decode for callers that cannot allocate device memory (no counterpart in
 * tensorsmith): e.g. a serving loop whose allocator already gave all free HBM
 * to KV-cache pages, or host code that must not call cudaMalloc (which may
 * synchronise the device) between decode steps.  Same semantics and kernels as
 * ts_attn_decode, but the split partials live in a fixed library-owned device
 * array of TS_ATTN_NOALLOC_SCRATCH_BYTES on every GPU that loads the library,
 * held until exit.  The first call in a CUDA context looks up the array's
 * device address (make it before any stream capture; a context recreated after
 * cudaDeviceReset looks it up again); calls that overlap on the GPU share the
 * array and race.  Returns TS_ERR_WORKSPACE, launching nothing, when
 * the problem needs more scratch than that.  Allocates nothing. */
TS_ATTN_API int ts_attn_decode_noalloc(const ts_attn_params* params, void* stream);

/* Attention dropout of nn/attention.py:140-144 (forward) and :212-216
 * (backward): P.V uses p * keep / (1 - p) with keep = (u >= p), u uniform on
 * the 2^16 points k * 2^-16 of [0, 1) per (batch, query head, query row, key);
 * dP is multiplied by the same factor; LSE stays the softmax normaliser.  u
 * comes from a counter-based generator (Philox4x32-10, 16 bits per key) keyed
 * by (seed, offset), so a backward given the forward's (seed, offset)
 * regenerates its mask without storing it. */
typedef struct ts_dropout {
  double p;        /* drop probability, 0 <= p < 1 */
  uint64_t seed;   /* generator key */
  uint64_t offset; /* call counter; a forward and its backward pass the same value */
} ts_dropout;

/* ts_attn_fwd with dropout: the tcgen05 kernel where ts_attn_fwd would use it,
 * the generic CUDA-core kernels otherwise (every dtype / shape / mask of
 * ts_attn_fwd).  p = 0 is exactly ts_attn_fwd (same kernel selection). */
TS_ATTN_API int ts_attn_fwd_dropout(const ts_attn_params* params, const ts_dropout* dropout, void* stream);

/* Workspace bytes ts_attn_bwd_dropout needs. */
TS_ATTN_API size_t ts_attn_bwd_dropout_workspace_size(const ts_attn_bwd_params* params);

/* ts_attn_bwd for a forward made by ts_attn_fwd_dropout with the same dropout
 * arguments (p = 0 is exactly ts_attn_bwd). */
TS_ATTN_API int ts_attn_bwd_dropout(const ts_attn_bwd_params* params, const ts_dropout* dropout, void* workspace,
                                    size_t workspace_bytes, void* stream);

/* The keep mask those calls use, as uint8 0/1 [batch, heads, q_len, kv_len]
 * (contiguous; heads = query heads). */
TS_ATTN_API int ts_attn_dropout_mask(const ts_dropout* dropout, int32_t batch, int32_t heads, int32_t q_len,
                                     int32_t kv_len, uint8_t* mask, void* stream);

/* Quantising KVCache.append of nn/cache.py:54-86 with quantized=True.
 * key_cache / value_cache are int8 views; params->cache_dtype is the cache's
 * compute dtype (rows are rounded to it first, :68).  Per row:
 * scale = max(max|x| / 127, 1e-8) in fp32, q = round_half_even(x / scale)
 * (:70-75).  key_scales / value_scales are contiguous fp32 [batch, heads,
 * capacity] (the reference's [B, H, capacity, 1]). */
TS_ATTN_API int ts_kv_append_int8(const ts_kv_append_params* params, float* key_scales, float* value_scales,
                                  void* stream);

/* KVCache.get of a quantized cache (nn/cache.py:88-99):
 * dst[b, h, t, c] = dtype(float(src[b, h, t, c]) * scales[b, h, t]) for
 * t < length; scales contiguous [batch, heads, scale_capacity]. */
TS_ATTN_API int ts_kv_dequant_int8(ts_view4 src, const float* scales, int64_t scale_capacity, ts_view4 dst,
                                   int32_t dtype, int32_t batch, int32_t heads, int32_t length, int32_t channels,
                                   void* stream);

/* Workspace bytes ts_attn_decode_int8 needs (0 when one split suffices). */
TS_ATTN_API size_t ts_attn_decode_int8_workspace_size(const ts_attn_params* params);

/* Decode straight from an int8 KV cache (replaces nn/cache.py:91-99 followed
 * by nn/attention.py:132-145): params->k / params->v are int8 views (element
 * strides = bytes), params->dtype is the dtype of q and o, scales as in
 * ts_kv_append_int8 with `scale_capacity` keys per (row, head).  Scores are
 * k_scale * (q . k8) and probabilities meet v_scale * v8, in fp32; the
 * dequantised rows are never written.  Same masking rules as ts_attn_decode
 * (causal, causal_offset, kv_lens; no explicit mask).  TS_ERR_UNSUPPORTED when
 * the shape is outside the kernel (head_dim = value_dim in {64, 128, 256},
 * 16-byte aligned rows): dequantise with ts_kv_dequant_int8 and call
 * ts_attn_fwd instead. */
TS_ATTN_API int ts_attn_decode_int8(const ts_attn_params* params, const float* key_scales,
                                    const float* value_scales, int64_t scale_capacity, void* workspace,
                                    size_t workspace_bytes, void* stream);

/* ---- A paged KV cache held in 4 bits (no counterpart in tensorsmith, whose
 * smallest cache is int8, nn/cache.py:47-52) ----
 *
 * A page holds page_size tokens of every KV head, keys and values.  The block of
 * one page and head is contiguous:
 *   K nibbles [page_size, D/2] | K scales fp16 [page_size, D/32] | V nibbles | V scales
 * A row's D/8 words are ordered so that word t * (D/32) + g holds the channels
 * 32 g + 8 t + e in nibble e (bits 4e..4e+3).  One scale serves 32 channels of a
 * token: scale = max|x| / 7 rounded up to 5 significant bits, held in
 * [2^-20, 9216]; n = round_half_even(x / scale) in [-7, 7] is stored as n + 8.
 * n * scale is exact in bf16 and fp16.  Inputs beyond +-64512 saturate, NaN is
 * stored as 0.  4.5 bits a value. */
typedef struct ts_kv4_cache {
  void* pool;           /* uint8 [pages, kv_heads, block], 16-byte aligned */
  int64_t page_stride;  /* bytes between pages: at least kv_heads * block, a multiple of 16 */
  const int32_t* table; /* [batch, slots] (device): the page of each page_size tokens of a row, -1 none */
  int64_t table_stride; /* entries between rows */
  int32_t batch, slots, pages, kv_heads;
  int32_t head_dim;  /* a multiple of 32, at most 256 */
  int32_t page_size; /* 16, 32 or 64 */
} ts_kv4_cache;

/* Bytes of the block of one page and KV head, 0 for a head_dim or page_size the
 * cache does not take. */
TS_ATTN_API size_t ts_kv4_block_bytes(int32_t head_dim, int32_t page_size);

/* Quantising append: tokens [pos_b, pos_b + steps) of every row receive the rows
 * of key / value [batch, kv_heads, steps, D] (dtype F32, F16 or BF16), with
 * pos_b = positions[b], or position for every row when positions is NULL.
 * positions_out (optional, [batch]) receives pos_b + steps; it must not overlap
 * positions.  The table must already hold a page for every token written
 * (ts_kv_pages_reserve); a token without one is not written and sets the fault
 * word (TS_ERR_PAGE). */
TS_ATTN_API int ts_kv_append_int4(ts_view4 key, ts_view4 value, int32_t dtype, int32_t steps,
                                  const ts_kv4_cache* cache, int64_t position, const int32_t* positions,
                                  int32_t* positions_out, void* stream);

/* The values of `length` tokens of every row, from token starts[b] (0 when
 * starts is NULL), into key / value [batch, kv_heads, length, D].  Tokens at or
 * past lens[b] (optional) are written as zeros. */
TS_ATTN_API int ts_kv_gather_int4(const ts_kv4_cache* cache, const int32_t* starts, const int32_t* lens,
                                  ts_view4 key, ts_view4 value, int32_t dtype, int32_t length, void* stream);

/* Kernel family ts_attn_int4 would run: TS_PATH_DECODE (straight over the pages)
 * or TS_PATH_TCGEN05 (pages dequantised into the workspace, then the prefill
 * kernel), or a negative ts_status.  The environment variable TS_INT4_KERNEL =
 * "pages" or "prefill", read at every call, forces one where it supports the
 * problem, for tests and measurements. */
TS_ATTN_API int ts_attn_int4_path(const ts_attn_params* params, const ts_kv4_cache* cache);

/* Workspace bytes ts_attn_int4 needs.  (A problem over the pages whose line of
 * work passes 2^30 stages runs in several launches; the environment variable
 * TS_INT4_LINE lowers that limit, for tests.) */
TS_ATTN_API size_t ts_attn_int4_workspace_size(const ts_attn_params* params, const ts_kv4_cache* cache);

/* Attention of q [batch, Hq, Tq, D] over the cache: params as for ts_attn_decode,
 * with k and v ignored, kv_lens required and kv_len an upper bound of them that
 * the table can hold (kv_len <= slots * page_size); no explicit mask, no fp64.
 * Any number of query tokens: one token a row, a few drafted ones, or a chunk of
 * a prompt whose tokens are already in the cache.  The route decides how the
 * probabilities enter the product with V: over the pages in fp16 relative to the
 * row's maximum (two parts, 22 bits, for F16 and F32 outputs), on the prefill route
 * in q's type, as ts_attn_fwd has them (BF16: 8 bits; F16: 11 bits, and 2^-25 of the
 * largest at the least). */
TS_ATTN_API int ts_attn_int4(const ts_attn_params* params, const ts_kv4_cache* cache, void* workspace,
                             size_t workspace_bytes, void* stream);

/* ---- Pages of a paged cache (any storage: a page is opaque bytes) ----
 * refs[p] counts the table entries that hold page p (and pins a caller adds); a
 * page with refs 0 is free.  counters is int32 [4] on the device: {free pages, a
 * page number below which none is free (0 is always right; after a fork the engine's
 * may vary from run to run), error bits, unused};
 * error bits, set and never cleared by the engine: 1 not enough free pages, 2 an
 * index or page out of range was skipped, 4 a row would need more slots than the
 * table has.  A reserve that sets 1 or 4 changes nothing.  The rows of a table
 * that a call writes to must not overlap. */
typedef struct ts_page_pool {
  void* data;                        /* 16-byte aligned */
  int64_t layer_stride, page_stride; /* bytes, multiples of 16 */
  int64_t page_bytes;                /* contiguous bytes of a page, a multiple of 16 */
  int32_t layers, pages;             /* a page number means the same page of every layer */
} ts_page_pool;

/* Page from[i] of src is copied to page to[i] of dst, in every layer; a pair with
 * a negative or out-of-range entry is skipped.  No page may be both read and
 * written, and none written twice. */
TS_ATTN_API int ts_kv_pages_copy(const ts_page_pool* src, const ts_page_pool* dst, const int32_t* from,
                                 const int32_t* to, int32_t count, void* stream);

/* Row r of the new table shares the pages that hold the lens[index[r]] tokens of
 * old row index[r] (fork, beam reorder); index[r] < 0 leaves the row empty (free).
 * Pages that no row holds any longer become free, pages reserved past a row's
 * tokens too.  refs and counters are updated in place; table_out and lens_out
 * must not alias table and lens. */
TS_ATTN_API int ts_kv_pages_fork(const int32_t* table, int64_t table_stride, const int32_t* lens, int32_t rows,
                                 const int32_t* index, int32_t* table_out, int64_t table_out_stride,
                                 int32_t* lens_out, int32_t rows_out, int32_t slots, int32_t page_size,
                                 int32_t* refs, int32_t pages, int32_t* counters, void* stream);

/* Workspace bytes ts_kv_pages_reserve needs. */
TS_ATTN_API size_t ts_kv_pages_reserve_workspace_size(int32_t pages, int32_t rows);

/* Gives every row pages of its own for the tokens [lens[r], lens[r] + steps)
 * (row_steps[r] in place of steps when given): empty slots get free pages, and a
 * partly filled page that others hold too is replaced by a copy (in every layer of
 * the pool); of its holders that write, the last keeps it if no other row has it.
 * Pages are handed out lowest first, in the order of (row, slot).  lens stays.
 * Slots past a row's tokens must be -1 or pages of its own: after shortening a
 * row, ts_kv_pages_fork onto itself drops the ones it no longer needs. */
TS_ATTN_API int ts_kv_pages_reserve(const ts_page_pool* pool, int32_t* table, int64_t table_stride,
                                    const int32_t* lens, int32_t rows, int32_t slots, int32_t page_size,
                                    int32_t steps, const int32_t* row_steps, int32_t* refs, int32_t* counters,
                                    void* workspace, size_t workspace_bytes, void* stream);

/* Workspace bytes ts_kv_pages_compact needs. */
TS_ATTN_API size_t ts_kv_pages_compact_workspace_size(int32_t pages);

/* Moves the pool's n live pages into its first n: the highest page into the lowest
 * hole, and so on.  table_out / refs_out receive the tables and counts (they may
 * be table / refs themselves). */
TS_ATTN_API int ts_kv_pages_compact(const ts_page_pool* pool, const int32_t* table, int64_t table_stride,
                                    int32_t* table_out, int64_t table_out_stride, int32_t rows, int32_t slots,
                                    const int32_t* refs, int32_t* refs_out, int32_t* counters, void* workspace,
                                    size_t workspace_bytes, void* stream);

/* ---- Attention under a sliding window with sinks (no counterpart in tensorsmith, whose causal rule is
 * nn/attention.py:108-111) ----
 * A query at position i (causal_offset + its index; kv_lens[b] - q_len + its index where kv_lens is set) sees the
 * keys j <= i with i - j < window or j < sinks. */
typedef struct ts_window {
  int32_t window; /* at least 1; 0 where a call takes it as "no window" */
  int32_t sinks;  /* first keys that stay visible, at least 0 */
} ts_window;

/* ts_attn_fwd under a window: is_causal must be set, no explicit mask, no dropout.  Keys between the sinks and the
 * window of a block of queries are not read, but for those that share a tile (128 keys at most) with one that is seen:
 * their values must be finite, as 0 * NaN is NaN.  Half types with equal head dimensions that are multiples of 8 up to 128
 * run on the tcgen05 kernels (P in q's type, as ts_attn_fwd), everything else on CUDA cores.  Chunks too short to give
 * every SM a block are shared along their keys as in ts_attn_tree and then need the workspace; the environment variable
 * TS_WINDOW_KERNEL = "split", "tile" or "pair" (a block for 128 or 256 queries), read at every call, forces one way where
 * it supports the problem, for tests and measurements. */
TS_ATTN_API int ts_attn_fwd_window(const ts_attn_params* params, const ts_window* window, void* workspace,
                                   size_t workspace_bytes, void* stream);
TS_ATTN_API size_t ts_attn_fwd_window_workspace_size(const ts_attn_params* params, const ts_window* window);
/* Kernel family of both directions: TS_PATH_TCGEN05 or TS_PATH_SIMT, or a negative ts_status. */
TS_ATTN_API int ts_attn_window_path(const ts_attn_params* params, const ts_window* window);
TS_ATTN_API size_t ts_attn_bwd_window_workspace_size(const ts_attn_bwd_params* params, const ts_window* window);
/* ts_attn_bwd for a forward made by ts_attn_fwd_window with the same window. */
TS_ATTN_API int ts_attn_bwd_window(const ts_attn_bwd_params* params, const ts_window* window, void* workspace,
                                   size_t workspace_bytes, void* stream);

/* ---- Drafted tokens over a KV cache: a tree of them, or a chain (no counterpart in tensorsmith) ----
 * The last q_len of row b's kv_lens[b] keys are drafted tokens: node i sits in slot kv_lens[b] - q_len + i.  A node
 * sees every committed key (before them), its ancestors and itself; under a window, those of them that the rule of
 * ts_window lets it see, its position being the number of committed keys plus its depth.  Nodes whose slot would lie
 * before the cache do not exist. */
typedef struct ts_tree {
  const int32_t* parents; /* [batch, q_len] (device): node i's parent, a node before it, or -1: the committed tokens.
                             Any other value marks a padded node: it and its children give zeros (LSE -inf) and are
                             seen by nobody, whatever their slots hold.  NULL: a chain, node i's parent is node i - 1. */
  int64_t parents_stride; /* entries between rows */
  int32_t window, sinks;  /* ts_window; window 0: none */
} ts_tree;
#define TS_TREE_MAX_NODES 64 /* q_len with parents; chains may be longer */

/* Attention of q [batch, Hq, q_len, D] over the cache k, v: params as for ts_attn_decode with kv_lens required;
 * is_causal and causal_offset are ignored, no explicit mask, kv_len is 2^30 at most.  Slots at and behind kv_lens[b] are not used, whatever
 * they hold; the values of the others must be finite (one that is not may reach nodes that do not see it).  Half types with equal head dimensions that are multiples of 8 up to 128 run on the tcgen05 kernel. */
TS_ATTN_API int ts_attn_tree(const ts_attn_params* params, const ts_tree* tree, void* workspace,
                             size_t workspace_bytes, void* stream);
TS_ATTN_API int ts_attn_tree_path(const ts_attn_params* params, const ts_tree* tree);
TS_ATTN_API size_t ts_attn_tree_workspace_size(const ts_attn_params* params, const ts_tree* tree);

/* positions[b, i] = lens[b] + depth of node i (int32 [batch, nodes], contiguous), -1 for padded nodes: what ts_rope_at
 * rotates the queries and keys of drafted tokens by.  lens: committed tokens. */
TS_ATTN_API int ts_tree_positions(const int32_t* parents, int64_t parents_stride, const int32_t* lens, int32_t batch,
                                  int32_t nodes, int32_t* positions, void* stream);
/* ts_rope with a position of its own for every token: positions int32 [batch, seq], contiguous. */
TS_ATTN_API int ts_rope_at(ts_view4 x, ts_view4 y, int32_t dtype, int32_t batch, int32_t heads, int32_t seq,
                           int32_t channels, int32_t rotary_dim, const int32_t* positions, const float* inv_freq,
                           int32_t inverse, void* stream);

/* Closes caches behind the accepted path: slot base[b] + path[b, k] moves to slot base[b] + k for k < counts[b], in
 * the key and value caches of every layer, each in memory of its own.  path ascends (nodes of one root-to-leaf path do);
 * entries that would read past the capacity are skipped. */
typedef struct ts_kv_keep_params {
  void* const* keys; /* host arrays of `layers` device pointers, all with the strides below */
  void* const* values;
  int64_t key_stride[4], value_stride[4]; /* elements between rows, heads, slots, channels (1) */
  int32_t dtype;                          /* any ts_dtype, TS_I8 included */
  int32_t layers, batch, heads, head_dim, value_dim, capacity, nodes;
  const int32_t* base;   /* [batch] committed tokens */
  const int32_t* path;   /* [batch, nodes] */
  const int32_t* counts; /* [batch], at most nodes are used */
  int64_t path_stride;
} ts_kv_keep_params;
TS_ATTN_API int ts_kv_keep(const ts_kv_keep_params* params, void* stream);

/* ---- Log probabilities of given tokens (a language model's loss is their mean, negated) ----
 * logprob[r] = x[r, targets[r]] - lse(x[r]); 0 where targets[r] == ignore_index, NaN where it lies outside the
 * vocabulary.  entropy[r] = -sum p log p, in nats.  The `top` largest logits, in descending order, equal ones by
 * index (NaN is the largest): their log probabilities and indices.  A row of -inf has log probabilities of -inf,
 * entropy 0 and no gradient; NaN and +inf give NaN. */
typedef struct ts_token_logprobs {
  const void* logits; /* [rows, vocab], contiguous rows */
  int64_t stride;     /* elements between rows */
  int32_t dtype;      /* F32, F16 or BF16; sums in fp32 */
  int32_t rows, vocab;
  int32_t top; /* 0 to TS_TOP_TOKENS_MAX, at most vocab */
  const int64_t* targets;
  int64_t ignore_index;
  float* logprob;       /* [rows] */
  float* entropy;       /* [rows] */
  float* norm;          /* [rows, 2]: the largest logit m and log sum e^(x - m) (-inf: a row of -inf); optional */
  float* top_logprobs;  /* [rows, top] */
  int64_t* top_indices; /* [rows, top] */
} ts_token_logprobs;
#define TS_TOP_TOKENS_MAX 32
TS_ATTN_API int ts_token_logprobs_fwd(const ts_token_logprobs* params, void* stream);
/* grad_logits [rows, vocab] (dtype of the logits, another buffer) from the gradients of logprob, entropy and
 * top_logprobs (each optional, fp32, contiguous), given the forward's norm, entropy and top_indices.  A row with an
 * ignored target, to which the latter two give 0 or nothing, has a gradient of 0 whatever its logits are. */
TS_ATTN_API int ts_token_logprobs_bwd(const ts_token_logprobs* params, const float* grad_logprob,
                                      const float* grad_entropy, const float* grad_top, void* grad_logits,
                                      int64_t grad_stride, void* stream);

/* Reads and clears the device fault word written by kernels whose bounded
 * waits gave up, or that met a page outside the pool.  Synchronises `stream`.
 * Returns TS_OK, TS_ERR_DEVICE_TIMEOUT or TS_ERR_PAGE; *info (optional) receives
 * the recorded site code. */
TS_ATTN_API int ts_attn_device_status(void* stream, uint32_t* info);

#ifdef __cplusplus
}
#endif

#endif /* TS_ATTN_H */
