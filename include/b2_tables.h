/*
 * C ABI of the block tables and slot maps built on the GPU (libb2attn.so):
 * a scheduler that hands out 64-token blocks of a paged pool from request
 * lengths, without the host, inside a captured graph.  Conventions and error
 * codes as in b2_decode_attn.h.
 *
 *   block_tables int32 [batch][max_blocks_per_seq]  logical -> pool block
 *   held         int32 [batch]       blocks that a request's row holds
 *   free_list    int32 [num_blocks]  ids of the free blocks in [0, *free_count)
 *   free_count   int32 [1]
 */
#ifndef B2_TABLES_H
#define B2_TABLES_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Blocks for new_lens[b] new tokens behind past_lens[b] cached ones, and the
 * place of every new token.  Request b needs
 *   max(0, ceil((past_lens[b] + new_lens[b]) / 64) - held[b])
 * blocks.  Requests are served in order of b, each block from the end of the
 * free list; the first request that does not fit and all later ones that need
 * a block are refused: they get no block and granted[b] = 0.
 *
 * held_out       int32 [batch], may be held itself.
 * free_count_out int32 [1], may be free_count itself.
 * granted        int32 [batch]: new_lens[b], or 0 (the chunk_lens of the
 *                append and attention calls that follow).
 * row_start      int32 [batch]: the row of request b's first new token.
 * slots          int32 [rows]: block * 64 + row of the block; -1 for the rows
 *                of a refused request and for rows of no token.
 * positions      int32 [rows]: past_lens[b] + t; 0 for rows of no token.
 * tokens_per_seq 0: rows are packed, request b's behind request b - 1's.  T:
 *                row b * T + t (rows == batch * T).
 * block_tables   gets the new entries; all others stay as they were.
 *
 * A request with a negative length, more than max_blocks_per_seq blocks, more
 * than tokens_per_seq new tokens or rows behind the last one is refused and
 * sets B2_DEV_BAD_LENGTH; an id outside [0, num_blocks) on the free list sets
 * B2_DEV_BAD_BLOCK.  Both calls are deterministic.
 */
int b2_tables_extend(int32_t *block_tables, int32_t max_blocks_per_seq, const int32_t *held,
                     const int32_t *free_list, int32_t num_blocks, const int32_t *free_count,
                     const int32_t *past_lens, const int32_t *new_lens, int32_t batch,
                     int32_t *held_out, int32_t *free_count_out, int32_t *granted, int32_t *row_start,
                     int32_t *slots, int32_t *positions, int32_t rows, int32_t tokens_per_seq,
                     int32_t *dev_err, void *stream);

/*
 * The slots and positions alone, from tables whose blocks are there:
 * row_start[b] + t (NULL: b * tokens_per_seq + t) for t < new_lens[b].  With
 * row_start the starts ascend and requests do not overlap.  A request that
 * b2_tables_extend would refuse for its lengths, or whose first row is
 * negative, gets no slot at all (-1) and sets B2_DEV_BAD_LENGTH.
 */
int b2_slot_map(const int32_t *block_tables, int32_t max_blocks_per_seq, int32_t num_blocks,
                const int32_t *past_lens, const int32_t *new_lens, const int32_t *row_start, int32_t batch,
                int32_t *slots, int32_t *positions, int32_t rows, int32_t tokens_per_seq,
                int32_t *dev_err, void *stream);

/*
 * The blocks of every request with finished[b] != 0 back to the end of the
 * free list (by request, then by logical block); its row of the table becomes
 * -1 and held[b] 0.  B2_DEV_BAD_LENGTH, and nothing released, when the list
 * would hold more than num_blocks ids.
 */
int b2_tables_release(int32_t *block_tables, int32_t max_blocks_per_seq, int32_t *held, int32_t *free_list,
                      int32_t num_blocks, int32_t *free_count, const uint8_t *finished, int32_t batch,
                      int32_t *dev_err, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* B2_TABLES_H */
