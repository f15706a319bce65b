/*
 * C ABI of the 8-bit paged KV cache (libb2attn.so): the append that quantises
 * new tokens, the decode step and the batched-prompt attention over the cache.
 * Conventions and error codes as in b2_decode_attn.h; the same model shapes
 * (16 query heads, 8 KV heads, head_dim 64, 64-token blocks).
 *
 *   k_pool   e4m3 [num_blocks][8][64 tokens][64 dims]   4 KiB per (block, head)
 *   v_pool   e4m3 [num_blocks][8][64 dims][64 tokens]   (dim-major: the product
 *            P . V reads the tokens of a dim together, as Q . K^T reads the
 *            dims of a token)
 *   k_scale, v_scale  fp32 [num_blocks][8]
 *
 * A stored code stands for code * scale of its (block, head).  Scales are
 * powers of two, so they cost an 8-bit float no relative precision and codes
 * move from one scale to another without a second rounding (but for codes that
 * become subnormal): the smallest with 448 * scale >= |x| for every value of
 * the (block, head), at least 2^-100.  Tokens appended to a block that already
 * holds some (the rows in front of them) raise its scale where they need a
 * larger one, and the codes in front of them are rounded again at the new
 * scale; the first row of a block sets the scale afresh.  Rows behind the
 * last appended token are left as they were, and no result depends on them.
 * An infinite value counts as the largest finite bf16; NaN is stored as NaN,
 * counts for no scale and reaches the tokens that see it, no others.
 *
 * One block may receive tokens of one sequence only in a call (blocks are not
 * shared between sequences that append).  2 KiB of cache hold one token of
 * one layer in bf16, 1 KiB (and 1 bit per 64 of it) here.
 */
#ifndef B2_KV8_H
#define B2_KV8_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Append of new tokens: q/k RMSNorm and RoPE (mode bits B2_NORM_QK and
 * B2_ROPE_QK, the arithmetic of b2_append_rope, bf16 results) and, with
 * B2_STORE_KV, their k/v quantised into the cache.
 *
 * qkv        bf16 [rows][row_stride], a row starts q[16][64] | k[8][64] | v[8][64].
 * The rows' places, one of
 *   slots      int32 [rows]: block * 64 + row of the block (what
 *              b2_tables_extend and b2_slot_map write); a negative slot is a
 *              row to skip.  Rows of one block follow one another without
 *              skipped rows between them, at consecutive slots: one warp
 *              writes them.  Others of the block, as far as skipped rows or a
 *              jump part them from its first ones, are not stored
 *              (B2_DEV_BAD_SLOT); rows of a block that those of another block
 *              part are a race that no check finds.
 *              positions int32 [rows] are the RoPE positions (B2_ROPE_QK).
 *   slots NULL rows = batch * tokens, row b * tokens + t at position
 *              past_lens[b] + t, for t < chunk_lens[b] (NULL: tokens), through
 *              block_tables [batch][max_blocks_per_seq].  A sequence with
 *              a negative length, more than `tokens` new tokens or more tokens
 *              than its table holds is refused whole (B2_DEV_BAD_LENGTH).
 * q_out      bf16 [rows][16][64] normalised and rotated query, or NULL; rows
 *            that are skipped are left as they were.
 */
int b2_kv8_append(const uint16_t *qkv, int64_t row_stride, int32_t rows,
                  const int32_t *slots, const int32_t *positions,
                  const int32_t *past_lens, const int32_t *chunk_lens, int32_t tokens,
                  const int32_t *block_tables, int32_t max_blocks_per_seq,
                  const uint16_t *gamma_q, const uint16_t *gamma_k, float eps,
                  const uint16_t *rope_cos, const uint16_t *rope_sin, int32_t rope_rows,
                  uint8_t *k_pool, uint8_t *v_pool, float *k_scale, float *v_scale,
                  int32_t num_blocks, uint16_t *q_out, int32_t mode,
                  int32_t *dev_err, void *stream);

/*
 * One decode step of 1 to 4 new tokens per sequence: the append above and
 * attention of token t over past_lens[b] + t + 1 tokens.  Without B2_STORE_KV
 * the new tokens' k/v are in the cache already.
 *
 * qkv        rows of row_stride, `rows` of them; token t of sequence b is row
 *            row_start[b] + t (NULL: b * tokens + t).  chunk_lens[b] (0 ..
 *            tokens; NULL: tokens) tokens are there; a sequence with none is
 *            skipped whatever its length and row, one that would leave the
 *            rows is refused (B2_DEV_BAD_LENGTH).
 * out        bf16 [rows][16][64]; rows of no token are left as they were.
 * workspace  b2_kv8_workspace_bytes() bytes, 16-byte aligned, zeroed once; a
 *            call that completes leaves it ready for the next.  Calls that
 *            share a workspace must not overlap on the GPU.  After a device
 *            error, zero it again.
 */
int b2_kv8_decode_step(const uint16_t *qkv, int64_t row_stride, int32_t rows, const int32_t *row_start,
                       int32_t tokens, const int32_t *chunk_lens,
                       const uint16_t *gamma_q, const uint16_t *gamma_k, float eps,
                       const uint16_t *rope_cos, const uint16_t *rope_sin, int32_t rope_rows,
                       const int32_t *past_lens, const int32_t *block_tables, int32_t max_blocks_per_seq,
                       uint8_t *k_pool, uint8_t *v_pool, float *k_scale, float *v_scale, int32_t num_blocks,
                       int32_t batch, float scale, int32_t mode, uint16_t *out,
                       void *workspace, int64_t workspace_bytes, int32_t *dev_err, void *stream);

int64_t b2_kv8_workspace_bytes(void);

/*
 * Batched-prompt attention over the cache, the chunk's tokens appended before:
 * token t of sequence b attends past_lens[b] + t + 1 tokens.
 *
 * q          bf16, row r at q + r * q_stride: the 16 x 64 query (q_out of
 *            b2_kv8_append, q_stride 1024, or rows of qkv whose q is
 *            normalised and rotated already).
 * row_start  int32 [batch]: the row of a sequence's first token (packed
 *            prompts); NULL: b * tokens.
 * chunk_lens int32 [batch], 0 .. tokens; NULL: tokens.
 * tokens     the longest chunk; batch * ceil(tokens / 64) * 8 < 2^31.
 * rows       rows of q and out; a sequence that would leave them is refused
 *            (B2_DEV_BAD_LENGTH).
 * out        bf16 [rows][16][64]; rows of no token are left as they were.
 */
int b2_kv8_prefill_attn(const uint16_t *q, int64_t q_stride, int32_t rows, const int32_t *row_start,
                        const int32_t *past_lens, const int32_t *chunk_lens, int32_t tokens,
                        const int32_t *block_tables, int32_t max_blocks_per_seq,
                        const uint8_t *k_pool, const uint8_t *v_pool,
                        const float *k_scale, const float *v_scale, int32_t num_blocks,
                        int32_t batch, float scale, uint16_t *out,
                        void *workspace, int64_t workspace_bytes, int32_t *dev_err, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* B2_KV8_H */
