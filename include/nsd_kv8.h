/*
 * nsd_kv8.h -- C ABI of the paged KV cache in 8 bits: written by prompts and
 * decode/verify rows, read back, and attended by decode/verify rows.
 *
 * A block is 16 tokens of one sequence.  For every layer and kv head it holds
 * 16 x 128 codes of 8 bits and one scale byte s for K, and the same for V.  A
 * value is code * 2^(s - 127):
 *
 *   NSD_KV8_E4M3  E4M3 (largest 448), s - 127 from -15 to 8
 *   NSD_KV8_INT8  whole numbers from -127 to 127, s - 127 from -24 to 9
 *
 * The scale of a set of values is the smallest power of two of the range that
 * leaves the largest finite magnitude no more than the largest code's.  Values
 * round to the nearest code, ties to the even one; E4M3 values end at 61440 and
 * whole numbers at 127.  So every value of a cache is an fp16 value: reading
 * back loses nothing, nor does the attention where it multiplies in fp16.  The
 * powers at the ranges' ends lose nothing either: below them codes are finer
 * than fp16's own steps.
 *
 * A value that is not finite has the NaN code in E4M3 and 0 in whole numbers,
 * counts for no scale, and raises NSD_STATUS_NONFINITE; an E4M3 NaN raises it
 * again whenever its block is written and its token stays.
 *
 * Rows stored at position p go to slot p % 16 of their block.  A prompt's blocks
 * are written whole, slots behind its last token as zeros.  Decode/verify rows
 * join the tokens that the block already holds, which are those of the slots
 * below the highest one written: the block's scale is that of these tokens'
 * values and the new rows together, and the tokens' codes are rounded again
 * where it changes.  Slots above hold no token (rows of a rejected draft, or of
 * the block's earlier owner), count for nothing and keep their codes (V's end as
 * zeros under the largest scale, where a code past the largest value would be an
 * infinity).  A scale that grows at least doubles, so however often a token is
 * rounded again it ends from its value by less than one step of the largest scale
 * that its block has had since (E4M3: of the value's own steps under that scale);
 * a scale that shrinks loses nothing, and brings nothing back.  Free scales would
 * let every append cost another half step.
 *
 * So rows that are written over later, a rejected draft's, leave the tokens below
 * them, and accepted rows of their own call, on the grid of their scale.  Where
 * tokens must not depend on them, the bytes of the sequence's last block are copied
 * before such a call and put back after it, and the accepted rows stored again.
 *
 * Layout: codes [num_blocks, num_layers, num_kv_heads, 2048 bytes], scales
 * uint8 [num_blocks, num_layers, num_kv_heads], each for K and for V, so that a
 * block's bytes are one run, as in the fp16 caches.  A tile's 2048 bytes lie as
 * the attention's matrix instructions take them, 64 lanes x 16 bytes at a time:
 *   K  unit 16 c + t (c < 8, token t): dims 8c .. 8c+7, then 64+8c .. 64+8c+7
 *   V  unit 64 h + 16 g + i (h < 2, g < 4, i < 16): byte 4 m + j is dim
 *      8 i + 4 h + m of token 4 g + j
 * and whole numbers are held as code + 128.
 *
 * Every entry point follows nsd_attn.h's contract: stream-ordered, no host
 * synchronisation, no allocation, an int status, nsd_last_error(); head_dim is
 * 128 and a block 16 tokens.  Pointers are 16-byte aligned (scales and int32
 * arrays need not be).  Metadata that points outside the cache, the block table
 * or the rows is skipped and flagged in *status (NULL: not flagged).  A block is
 * written for one sequence in a call, but any number of its rows, in any order;
 * of rows with the same position the last one stays.  Calls that write the same
 * block, or read what another writes, are ordered by the caller.
 */
#ifndef NSD_KV8_H
#define NSD_KV8_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NSD_KV8_E4M3 0
#define NSD_KV8_INT8 1

#define NSD_STATUS_NONFINITE 8  /* an infinity or a NaN was stored */

/* A cache: device buffers of the caller. */
typedef struct {
  void* k;
  void* v;
  void* k_scales;
  void* v_scales;
  int64_t num_blocks;
  int32_t num_layers;
  int32_t num_kv_heads;
  int32_t codes; /* NSD_KV8_* */
} nsd_kv8_cache;

/*
 * nsd_kv8_store: nsd_store_kvcache into an 8-bit cache (row r of k, v fp16
 * [n_rows, Hkv, 128] to position seq_lens[r] - 1 of block_table[seq_ids[r]]).
 * nsd_kv8_store_prefill: nsd_store_kvcache_prefill, of k, v [n_tokens, Hkv, 128].
 * Every decode/verify row is compared with every other: at most 65536 rows a call,
 * here and in the prologues, and time by their square from about 500 on.
 */
int nsd_kv8_store(const void* k, const void* v, const nsd_kv8_cache* cache, const int32_t* block_table,
                  int64_t bt_rows, int64_t bt_stride, const int32_t* seq_ids, const int32_t* seq_lens,
                  int64_t n_rows, int layer, int32_t* status, void* stream);
int nsd_kv8_store_prefill(const void* k, const void* v, int64_t n_tokens, const nsd_kv8_cache* cache,
                          const int32_t* block_table, int64_t bt_rows, int64_t bt_stride, const int32_t* seq_ids,
                          const int32_t* start_locs, const int32_t* prefill_lens, int64_t n_seqs,
                          int64_t max_prefill_len, int layer, int32_t* status, void* stream);

/*
 * nsd_qk_norm_rope_store_strided into an 8-bit cache, one launch: q normalised
 * and rotated into q_out [n_rows, Hq, 128] (which may be q itself, if it is
 * contiguous), k normalised and rotated (the same fp16 rows), k and v stored as
 * nsd_kv8_store does.  k and v are only read.  Row strides in elements,
 * multiples of 8.  A row past the RoPE tables is flagged and skipped whole.
 */
int nsd_kv8_qk_norm_rope_store(const void* q, int64_t q_row_stride, void* q_out, const void* k,
                               int64_t k_row_stride, const void* v, int64_t v_row_stride, const void* q_norm_w,
                               const void* k_norm_w, float eps, const void* cos_cache, const void* sin_cache,
                               int64_t n_positions, const nsd_kv8_cache* cache, const int32_t* block_table,
                               int64_t bt_rows, int64_t bt_stride, const int32_t* seq_ids, const int32_t* seq_lens,
                               int64_t n_rows, int layer, int num_q_heads, int32_t* status, void* stream);

/*
 * nsd_qk_norm_rope_store_partials into an 8-bit cache: q, k and v as the split
 * partials [splits][n_rows][(Hq + 2 Hkv) 128] (1 to 8 splits) of their one
 * projection, each value their sum rounded once to fp16.
 */
int nsd_kv8_qk_norm_rope_store_partials(const float* partials, int splits, void* q_out, const void* q_norm_w,
                                        const void* k_norm_w, float eps, const void* cos_cache,
                                        const void* sin_cache, int64_t n_positions, const nsd_kv8_cache* cache,
                                        const int32_t* block_table, int64_t bt_rows, int64_t bt_stride,
                                        const int32_t* seq_ids, const int32_t* seq_lens, int64_t n_rows, int layer,
                                        int num_q_heads, int32_t* status, void* stream);

/*
 * The values of cached tokens: token first[s] + i of block_table[seq_ids[s]]
 * (i < lens[s] <= max_len; first NULL: 0) to row start_locs[s] + i of k, v fp16
 * [n_tokens, Hkv, 128].  Other rows are left as they are.
 */
int nsd_kv8_load(void* k, void* v, int64_t n_tokens, const nsd_kv8_cache* cache, const int32_t* block_table,
                 int64_t bt_rows, int64_t bt_stride, const int32_t* seq_ids, const int32_t* first,
                 const int32_t* start_locs, const int32_t* lens, int64_t n_seqs, int64_t max_len, int layer,
                 int32_t* status, void* stream);

/*
 * nsd_paged_attention over an 8-bit cache: the same contract, and the attention
 * over the values that the cache holds, with fp32 scores, softmax and sums; a
 * weight meets the values as two fp16 numbers, 22 bits of it.  softmax_scale is a
 * positive number.  A NaN in the cache reaches the rows that attend its token and
 * no others.
 *
 * nsd_kv8_plan_build: its plan (nsd_attn_plan_build's words and checks) for a
 * device of `compute_units`; nsd_attn_plan_bound gives the words for n_workers =
 * 2 * compute_units.  Plans of nsd_attn_plan_build serve too, not as fast.  Parts
 * of a segment are merged in fp32: the workspace is nsd_kv8_attn_workspace bytes,
 * not those of nsd_attn_plan_build.
 */
int nsd_kv8_plan_build(const int32_t* seq_ids, const int32_t* seq_lens, int64_t n_rows, int num_q_heads,
                       int num_kv_heads, int64_t bt_rows, int64_t bt_stride, int compute_units, int max_group_rows,
                       int32_t* plan, int64_t plan_capacity, int64_t* plan_words);
int nsd_kv8_attn_workspace(const int32_t* plan_host, int64_t* bytes);
int nsd_kv8_paged_attention(const void* q, void* o, float* lse, const nsd_kv8_cache* cache, int layer,
                            int num_q_heads, const int32_t* block_table, int64_t bt_rows, int64_t bt_stride,
                            const int32_t* plan_host, const int32_t* plan_dev, void* workspace,
                            int64_t workspace_bytes, float softmax_scale, int32_t* status, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NSD_KV8_H */
