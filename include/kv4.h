/*
 * rhinoforge_amd -- attention over a 4-bit paged cache for MI355X (gfx950).
 *
 * C ABI of the cache that holds keys and values in 4 bits: the quantizing
 * append, the read-back, and attention over it.  Block tables, slots and
 * positions are those of kv8.h (rf_kv8_plan), and so are the manner of the
 * calls and the attention's arguments.
 *
 * The cache of one layer
 *   A block holds `block_size` (32, 64 or 128) consecutive tokens of one
 *   request for all key/value heads; head_dim is 64, 128 or 256.
 *   k, v  : bytes [num_blocks][kv_heads][block_size * head_dim / 2]
 *   rows  : 16-bit words [num_blocks][kv_heads][block_size / 32][2][32], one for
 *           each token: of the keys, then of the values
 *   Token, head and side (keys or values) hold head_dim numbers n of 0..15 and
 *   one word: bits 4..15 are those of the step s, a positive fp16 number whose
 *   last four mantissa bits are 0, and bits 0..3 are the zero point z.  They
 *   stand for (n - z) * s, which is an fp16 number exactly (s <= 4352).
 *   Word 0x7e00 (s not a number) in the keys marks a token that stands for NaN,
 *   keys and values; words of the values are always finite.
 *   slot = block * block_size + token within the block.
 *
 * Order inside one head's block: groups of 32 tokens, each head_dim / 64 tiles of
 * 1024 bytes for 64 dimensions; lane l (0..63) of a wavefront owns bytes
 * [16 l, 16 l + 16) of a tile, in dwords (w = 0..3):
 *   k  dword w: token 8 ((l % 16) / 4) + 4 (w / 2) + l % 4, dimensions
 *      16 (l / 16) + 8 (w % 2) + 0..7; dimension e of these at bits 4 p .. 4 p + 3,
 *      p = e / 2 + 4 (e % 2)
 *   v  dword w: half h (0, 1) is token 8 (l / 16) + 2 w + h, dimensions
 *      4 (l % 16) + 0..3 at bits 4 b .. 4 b + 3 of the half
 * A wavefront reads a tile with one 16-byte load per lane, and every AND with
 * 0x000f000f leaves two operands of a matrix instruction: of the keys, dimensions
 * that follow each other, of the values, tokens that do.
 */
#ifndef RHINOFORGE_AMD_KV4_H_
#define RHINOFORGE_AMD_KV4_H_

#include "kv8.h"

#ifdef __cplusplus
extern "C" {
#endif

#define RF_KV4_NAN 0x7e00   /* word of a token that stands for NaN        */
#define RF_KV4_EMPTY 0x0010 /* word of the least step, zero point 0       */

/* One layer's cache. */
typedef struct rf_kv4_cache {
  void* k;
  void* v;
  uint16_t* rows;
  int64_t num_blocks;
  int32_t kv_heads;
  int32_t head_dim;   /* 64, 128 or 256  */
  int32_t block_size; /* 32, 64 or 128   */
} rf_kv4_cache;

/* Quantizes new tokens into the cache: token t of k and v into slots[t] (int32;
 * negative or past the cache: skipped).  For each token, head and side:
 *   span = max(x, 0) - min(x, 0)                                  (in fp32)
 *   s    = the least step with 15 s >= span, 2^-20 <= s <= 4352
 *   z    = rint(-min(x, 0) / s)    n = rint(x / s) + z, within 0..15
 * so |value - x| <= s / 2 as long as span <= 65280.  An infinity or NaN among a
 * token's keys or values of a head makes all of these NaN.  Tokens do not touch
 * each other; the slots of one call are different from each other. */
int rf_kv4_append(const rf_kv4_cache* cache, const rf_kv8_heads* k, const rf_kv8_heads* v,
                  int32_t dtype, const int32_t* slots, int64_t tokens, void* stream);

/* Cached tokens as the values they stand for: k_out, v_out contiguous
 * [n][kv_heads][head_dim] of dtype F16 (exact), BF16 or F32 (exact).  A slot that
 * is negative or past the cache gives zeros. */
int rf_kv4_read(const rf_kv4_cache* cache, const int32_t* slots, int64_t n, int32_t dtype,
                void* k_out, void* v_out, void* stream);

/* Attention of a ragged batch's queries over the cache: the fields, the masks, the
 * limits and the workspace of rf_kv8_attention_args.  Scores, sums and softmax
 * statistics are fp32, and scores count by their differences, whatever their size (two
 * of more than fp32 holds in units of ln 2 may count as equal); a token's weight
 * (times its value step, where few rows share a token) is rounded to fp16, to 2^-11 of
 * itself or 2^-32 of the largest one that the row sees.  A query that sees a token
 * which stands for NaN, or one behind a block id outside the cache, gives NaN. */
typedef struct rf_kv4_attention_args {
  rf_kv4_cache cache;
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
} rf_kv4_attention_args;
size_t rf_kv4_attention_workspace(const rf_kv4_attention_args* args);
int rf_kv4_attention(const rf_kv4_attention_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* RHINOFORGE_AMD_KV4_H_ */
