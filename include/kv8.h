/*
 * rhinoforge_amd -- attention over an int8 paged cache for MI355X (gfx950).
 *
 * C ABI of what a decoder layer does between its q/k/v projections and its o
 * projection: norms and rotation of the query and key heads, block tables and
 * slots from request lengths, the quantizing append, and attention over the
 * cache.  Same manner as w8a16.h: plain pointers and sizes, a HIP stream as
 * `void*` (NULL = the null stream), an rf_w8a16_status from every entry point,
 * refusals before any launch, no CPU computation, no synchronization and no
 * allocation.
 *
 * The cache of one layer
 *   A block holds `block_size` (32, 64 or 128) consecutive tokens of one
 *   request for all key/value heads; head_dim is 64, 128 or 256.
 *   k, v        : bytes [num_blocks][kv_heads][block_size * head_dim]
 *   k_scale,
 *   v_scale     : fp32 [num_blocks][kv_heads]
 *   A stored byte u stands for (u - 128) * scale, |u - 128| <= 127.
 *   Scales are +0 or positive; attention gives NaN where a query sees tokens of a
 *   block whose scale is negative, infinite or NaN.
 *   slot = block * block_size + token within the block.
 *
 * Byte order inside one head's block (RF_KV8_TILE): groups of 32 tokens, each
 * head_dim / 32 tiles of 1024 bytes; lane l (0..63) of a wavefront owns bytes
 * [16 l, 16 l + 16) of a tile, which are its operands of the matrix
 * instructions (Dt = head_dim / 64):
 *   k tile (tt * Dt + kb), byte 16 l + j   : token 16 tt + l % 16,
 *                                            dimension 64 kb + 16 (l / 16) + j
 *   v tile dt, byte 16 l + 8 e + 4 h + c   : dimension 32 dt + 16 e + l % 16,
 *                                            token 16 h + 4 (l / 16) + c
 * A wavefront reads a tile with one 16-byte load per lane.  The scores of 32
 * tokens leave the first product with each lane holding tokens 4 (l/16) + c
 * and 16 + 4 (l/16) + c of one query row, which is the order in which the
 * second product takes v: probabilities never move between lanes.
 */
#ifndef RHINOFORGE_AMD_KV8_H_
#define RHINOFORGE_AMD_KV8_H_

#include "w8a16.h"

#ifdef __cplusplus
extern "C" {
#endif

#define RF_KV8_GROUP 32          /* tokens of one group of tiles                */
#define RF_KV8_MAX_REQUESTS 8192 /* requests of one rf_kv8_plan call            */

/* One layer's cache. */
typedef struct rf_kv8_cache {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int64_t num_blocks;
  int32_t kv_heads;
  int32_t head_dim;   /* 64, 128 or 256  */
  int32_t block_size; /* 32, 64 or 128   */
} rf_kv8_cache;

/* A [tokens][heads][head_dim] operand: strides in elements, unit innermost
 * stride, pointer 16-byte aligned and strides multiples of 8. */
typedef struct rf_kv8_heads {
  const void* data;
  int64_t token_stride;
  int64_t head_stride;
  int32_t heads;
} rf_kv8_heads;

/* Norms and rotation of query and key heads, one pass:
 *   y = x / sqrt(mean(x^2) + eps) * weight      (per head; weight NULL: y = x)
 *   (a, b) <- (a cos - b sin, b cos + a sin)    for each of rot / 2 pairs
 * pair i is (i, i + rot / 2), or (2i, 2i + 1) with `interleaved`; dimensions
 * from rot on are not rotated.  Computed in fp32, rounded once.
 *   dtype      RF_W8A16_DTYPE_F16 or _BF16 of q, k, the weights and the outputs
 *   cos, sin   fp32 [table_rows][rot / 2]; row positions[t] (int64 where
 *              positions64, else int32), row t where positions is NULL.  A
 *              position outside the table gives a token of NaN.
 *   q_out, k_out  contiguous [tokens][heads][head_dim]; may not overlap inputs
 * head_dim a multiple of 8 up to 512; rot a multiple of 16 up to head_dim
 * (0: no rotation, cos and sin unused). */
typedef struct rf_kv8_rope_args {
  rf_kv8_heads q, k;
  void* q_out;
  void* k_out;
  const void* q_weight;
  const void* k_weight;
  const float* cos;
  const float* sin;
  const void* positions;
  int64_t tokens;
  int64_t table_rows;
  int32_t head_dim;
  int32_t rot;
  int32_t dtype;
  int32_t positions64;
  int32_t interleaved;
  float eps;
} rf_kv8_rope_args;
int rf_kv8_qk_norm_rope(const rf_kv8_rope_args* args, void* stream);

/* The same with positions of several axes (images and video: time, height,
 * width).  Pair i turns by row positions[axis(i) * axis_stride + t], column i.
 *   axes       1 .. RF_KV8_MAX_AXES
 *   sections   pairs of each axis (0 or more), rot / 2 together
 *   mixed 0    the axes' pairs one after the other: sections[0] of axis 0, then
 *              sections[1] of axis 1, ..
 *   mixed 1    in turn: pair i belongs to axis i % axes while i / axes is below
 *              that axis' section, to axis 0 from there on; sections have to be
 *              such that all pairs of the axes above 0 are there
 * positions are needed, and rot > 0.  A position of any axis outside the table
 * gives a token of NaN.  axis_stride: elements between axes, at least tokens. */
#define RF_KV8_MAX_AXES 4
typedef struct rf_kv8_mrope_args {
  rf_kv8_rope_args rope;
  int64_t axis_stride;
  int32_t axes;
  int32_t mixed;
  int32_t sections[RF_KV8_MAX_AXES];
} rf_kv8_mrope_args;
int rf_kv8_qk_norm_mrope(const rf_kv8_mrope_args* args, void* stream);

/* Block tables and slots of a batch, from its lengths (negative: taken as 0).
 * Request i holds cached[i] tokens and gets fresh[i] new ones; its blocks
 * [ceil(cached / bs), ceil((cached + fresh) / bs)) are taken from `free_blocks`
 * in order, request by request, from index *free_start on, and entered in
 * block_table[i] (row stride table_stride, `width` entries a row).
 *   slots[t]     of new token t of the batch (requests one after the other);
 *                -1 where its block is missing (free blocks or the table's
 *                width ran out) and for t past the batch's new tokens
 *   positions[t] cached + its index within the request (0 past the batch)
 *   cu[i]        new tokens before request i, cu[requests] = all of them
 *   kv_lens[i]   cached + fresh
 *   *free_next   *free_start + blocks needed; above num_free they ran out (the
 *                entries of blocks that were not there are -1)
 * All arrays int32.  requests <= RF_KV8_MAX_REQUESTS, tokens (the length of
 * slots and positions) >= 0.  Every workgroup reads all lengths and *free_start
 * while others write, so slots, positions, cu, kv_lens and free_next may not
 * overlap cached, fresh, free_blocks or free_start (RF_W8A16_EINVAL): the next
 * call's lengths are another array, or a copy made after this call. */
typedef struct rf_kv8_plan_args {
  int32_t* block_table;
  const int32_t* cached;
  const int32_t* fresh;
  const int32_t* free_blocks;
  const int32_t* free_start;
  int32_t* slots;
  int32_t* positions;
  int32_t* cu;
  int32_t* kv_lens;
  int32_t* free_next;
  int64_t requests;
  int64_t width;
  int64_t table_stride;
  int64_t num_free;
  int64_t tokens;
  int32_t block_size;
} rf_kv8_plan_args;
int rf_kv8_plan(const rf_kv8_plan_args* args, void* stream);

/* Quantizes new tokens into the cache: token t of k and v into slots[t]
 * (int32; negative or past the cache: skipped).  Per block, head and side:
 *   step = max(the block's scale if it holds tokens before the new ones,
 *              amax(new) / 127)      (amax below 2^-100 counts as 0)
 *   new  q = rint(x / step);  held q = rint(q * old step / step)
 * The new tokens of one block have to be consecutive slots, consecutive in the
 * batch.  An infinity or NaN among the new values makes the block's scale, and
 * so every value of that head and block, not finite. */
int rf_kv8_append(const rf_kv8_cache* cache, const rf_kv8_heads* k, const rf_kv8_heads* v,
                  int32_t dtype, const int32_t* slots, int64_t tokens, void* stream);

/* Cached tokens as the values they stand for: k_out, v_out contiguous
 * [n][kv_heads][head_dim] of dtype F16, BF16 or F32.  A slot that is negative
 * or past the cache gives zeros. */
int rf_kv8_read(const rf_kv8_cache* cache, const int32_t* slots, int64_t n, int32_t dtype,
                void* k_out, void* v_out, void* stream);

/* Attention of a ragged batch's queries over the cache.
 *   q     [tokens][heads][head_dim] F16 or BF16, heads a multiple of kv_heads;
 *         query head h reads key/value head h / (heads / kv_heads)
 *   cu_q  int32 [requests + 1], rising from 0: request i's queries are tokens
 *         cu_q[i] .. cu_q[i + 1] - 1 (tokens from cu_q[requests] on get zeros);
 *         NULL: tokens / requests queries each
 *   kv_lens int32 [requests]: tokens of request i in the cache, its queries'
 *         own among them; token j is in block block_table[i][j / block_size].
 *         Query n of N has position kv_len - N + n; it sees tokens at or before
 *         its position (causal; else all) and, with window > 0 (causal only),
 *         after position - window.  A query that sees nothing gets zeros and
 *         lse -inf.  A block id outside the cache gives NaN.
 *   out   contiguous, q's type; lse (may be NULL) fp32 [tokens][heads], natural log
 *   scale > 0 and finite
 *   Scores, sums and softmax statistics are fp32 (a score past what fp32 holds, in
 *   units of ln 2, counts as infinite).  A token's weight times its
 *   block's v_scale is rounded to fp16, relative to the largest such product that
 *   the row sees: to 2^-11 of itself, or 2^-32 of that largest one.
 *   tokens * heads < 2^31, (requests + 1) * kv_heads + tokens * heads / 16 < 2^31
 *   and width * block_size <= 2^30.
 *   max_q_len, max_kv_len  the largest of each, as far as the caller knows (0:
 *         not known).  They choose the launch; results are right without them.
 *   scratch  for calls whose tokens are split over workgroups: counters as
 *         every split launch has them (zero between calls, rf_w8a16_scratch),
 *         and rf_kv8_attention_workspace(args) bytes of partials (0: scratch
 *         may be NULL).  Missing or too small: RF_W8A16_EWORKSPACE, before any
 *         launch.  Calls that run at the same time need one each. */
typedef struct rf_kv8_attention_args {
  rf_kv8_cache cache;
  rf_kv8_heads q;
  const int32_t* cu_q;
  const int32_t* kv_lens;
  const int32_t* block_table;
  void* out;
  float* lse;
  const rf_w8a16_scratch* scratch;
  int64_t tokens;
  int64_t requests;
  int64_t width;        /* entries of a block_table row */
  int64_t table_stride; /* elements between rows        */
  int64_t max_q_len;
  int64_t max_kv_len;
  int32_t dtype;
  int32_t causal;
  int64_t window;
  float scale;
} rf_kv8_attention_args;
size_t rf_kv8_attention_workspace(const rf_kv8_attention_args* args);
int rf_kv8_attention(const rf_kv8_attention_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* RHINOFORGE_AMD_KV8_H_ */
