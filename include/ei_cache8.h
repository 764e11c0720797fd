/*
 * ei_cache8.h — a paged cache of 8-bit keys and values, trees of drafted tokens, and moving what was accepted.
 *
 * Conventions as in ei_attn.h and ei_packed.h (status codes, device pointers, streams, alignment, limits):
 * queries and outputs fp32, head_dim 128, GQA groups of 1 to 8, nothing allocated, no host
 * synchronisation, capturable.  No counterpart in the reference, whose cache is fp32 (src/cuda/model_cuda.cu:1571)
 * and whose decode takes one token at a time (:1648-1658).
 *
 * Every call is over a batch that ei_packed_plan laid out with kv_len: rows cu_rows[s] .. cu_rows[s+1] - 1 are the n
 * new rows of sequence s, row i of them stands at slot kv_len[s] - n + i of its cache; of rows past the last
 * sequence's nothing is used, and nothing is written for them.  A call whose n_seq, rows or heads differ from the
 * plan's writes nothing.  Lengths must not pass the plan's max_kv: attention takes a longer sequence as ei_packed.h
 * says, as one of max_kv keys, the last n of which count as its new rows (masks too), while rows at slots from max_kv
 * on are not stored and ei_cache_keep moves what those slots hold.
 * A call whose outputs, workspace or pools overlap anything else that it reads or writes is refused.
 */
#ifndef EI_CACHE8_H
#define EI_CACHE8_H

#include <stddef.h>
#include <stdint.h>

#include "ei_packed.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------ the 8-bit pool
 * n_blocks pages of block_size rows (a power of two >= 32), one head after another in a page: the 128 codes of key
 * t of KV head h in page b at k + (((size_t)b*n_head_kv + h)*block_size + t)*128, its scale at
 * k_scale[((size_t)b*n_head_kv + h)*block_size + t]; values likewise.  A code stands for code * scale.
 * A head row y of largest magnitude a is stored as
 *   EI_CACHE_INT8  scale a / 127, codes rint(y * (127 / a)), signed bytes
 *   EI_CACHE_E4M3  scale a / 448, codes y * (448 / a) rounded to the nearest e4m3 (4 exponent bits of bias 7, 3 of
 *                  fraction, no infinities, 0x7F and 0xFF are NaN), ties to even
 * each operation in fp32, rounded once: off by a/254 or half a step of e4m3, and by those roundings.  a < 2^-110:
 * scale and codes 0.  a not finite: scale NaN, codes 0 (every value of that head row reads as NaN).
 * 264 bytes per key and KV head, against 1024 of the fp32 pool. */
enum { EI_CACHE_E4M3 = 1, EI_CACHE_INT8 = 2 };
typedef struct ei_cache8 {
    void* k;         /* [n_blocks][n_head_kv][block_size][128] */
    void* v;
    float* k_scale;  /* [n_blocks][n_head_kv][block_size] */
    float* v_scale;
    int kind;        /* EI_CACHE_* */
    int n_blocks, block_size;
} ei_cache8;

/* Quantises the batch's new keys and values into their pages.  qkv row b is [Q | K | V] at qkv + b*row_stride, read
 * only.  Q and K heads are normed and turned first, to position turn_at[b] (device int32 [rows]), or with
 * turn_at NULL to the row's slot, as in ei_packed_step_paged (half layout, table cs of n_pos positions); Q goes
 * to q_out [rows][n_head][128], or nowhere if that is NULL.  A row whose slot is < 0, >= the plan's max_kv or past
 * its sequence's pages (block_table entry not in [0, n_blocks)) stores nothing, nor does one whose position is < 0 or
 * >= n_pos, whose query is copied as it is; so is that of a row at a slot < 0 or >= max_kv.
 * Blocks that are written must belong to one sequence alone. */
int ei_cache8_store(ei_stream_t stream, const float* qkv, long row_stride, float* q_out, const ei_cache8* cache,
                    const int* block_table, int max_blocks, int n_seq, int rows, int n_head, int n_head_kv,
                    int head_dim, const float* q_gamma, const float* k_gamma, const float* cs, int n_pos,
                    const int* turn_at, int rope_dim, float eps, const void* plan, size_t plan_bytes);

/* Reads the cache rows of the batch's new rows back: row b's keys, code * scale, to k_out + b*out_stride
 * ([n_head_kv][128]), its values to v_out.  A plan whose cu_rows count any last part of the sequences reads that.
 * Rows at slots < 0, past the sequence's pages or of pages outside the pool are zeros. */
int ei_cache8_load(ei_stream_t stream, const ei_cache8* cache, const int* block_table, int max_blocks, float* k_out,
                   float* v_out, long out_stride, int n_seq, int rows, int n_head, int n_head_kv, int head_dim,
                   const void* plan, size_t plan_bytes);

/* ------------------------------------------------------------------ trees of drafted tokens
 * mask (device [rows][mask_words] of 64-bit words, or NULL: causal): row i of a sequence's n new rows sees all
 * keys before the new rows, and of the new ones key j <= i if bit j%64 of word j/64 of its mask row is set (its
 * ancestors and itself, in a tree whose tokens come parents first); bits of words that are not there count
 * as unset, bits j > i are not looked at.  A row that sees no key gets zeros.
 * A token's position is the length before the new rows plus its depth (turn_at), its slot its place in the batch.
 *
 * Attention over the fp32 pool: ei_attn_packed_paged with a mask, and the step from raw projections,
 * ei_packed_step_paged with a mask and positions (NULL: the rows' slots).  A row at a position < 0 or >= n_pos
 * appends nothing, its query is neither normed nor turned. */
int ei_attn_tree_paged(ei_stream_t stream, const float* q, long q_stride, float* out, const float* kc,
                       const float* vc, int n_blocks, const int* block_table, int max_blocks, int block_size,
                       int n_seq, int rows, int n_head, int n_head_kv, int head_dim, const uint64_t* mask,
                       int mask_words, float scale, const void* plan, size_t plan_bytes, void* ws, size_t ws_bytes);
int ei_tree_step_paged(ei_stream_t stream, const float* qkv, long row_stride, float* out, float* kc, float* vc,
                       int n_blocks, const int* block_table, int max_blocks, int block_size, int n_seq, int rows,
                       int n_head, int n_head_kv, int head_dim, const float* q_gamma, const float* k_gamma,
                       const float* cs, int n_pos, const int* turn_at, int rope_dim, float eps, const uint64_t* mask,
                       int mask_words, float scale, const void* plan, size_t plan_bytes, void* ws, size_t ws_bytes);

/* ------------------------------------------------------------------ attention over the 8-bit pool
 * The batch's new rows (single tokens, drafts, trees, chunks), q row b at q + b*q_stride ([n_head][128], normed and
 * turned), over their sequences' pages, the new rows' own keys already stored.  Keys past the table's span, and
 * of a block whose entry is not in [0, n_blocks), count as zeros: nothing is read there.
 *
 * Codes are exact in binary16; q and the weights, each times the value's scale, are two binary16 planes, which keep
 * 22 bits of 24 down to 2^-39 of a query's largest value and of a row's largest weight times scale so far (2^-38 where
 * keys are taken again).  Sums and softmax in fp32; weights below 2^-116 of a row's largest may count as zero, and
 * outputs below fp32's normal numbers.  Scales of keys up to 2^96 are provided for (larger ones give infinities and
 * NaN), and all that values can have.  Where a scale above 2^20 is among the values, or none of a row's weights times
 * scales reaches 2^-82, the workgroup takes those keys again, three to five times slower.  Key and value rows that a
 * row does not see never reach it, whatever they hold; a NaN scale that it does see makes its output NaN, a NaN code of
 * a key too, and one of a value that column of it.  A batch called twice gives the same bits; they differ in the last
 * ones with the batch a sequence is in. */
int ei_attn_packed_cache8(ei_stream_t stream, const float* q, long q_stride, float* out, const ei_cache8* cache,
                          const int* block_table, int max_blocks, int n_seq, int rows, int n_head, int n_head_kv,
                          int head_dim, const uint64_t* mask, int mask_words, float scale, const void* plan,
                          size_t plan_bytes, void* ws, size_t ws_bytes);

/* ei_cache8_store, then ei_attn_packed_cache8 on its queries. */
int ei_packed_step_cache8(ei_stream_t stream, const float* qkv, long row_stride, float* out, const ei_cache8* cache,
                          const int* block_table, int max_blocks, int n_seq, int rows, int n_head, int n_head_kv,
                          int head_dim, const float* q_gamma, const float* k_gamma, const float* cs, int n_pos,
                          const int* turn_at, int rope_dim, float eps, const uint64_t* mask, int mask_words,
                          float scale, const void* plan, size_t plan_bytes, void* ws, size_t ws_bytes);

/* ------------------------------------------------------------------ the accepted path
 * Moves the cache rows of the new rows that are kept together: of sequence s, key and value rows of new row
 * kept[s*max_kept + j] go to new row j's slot, j = 0, 1, ... n_kept[s] - 1 (device int32 [n_seq][max_kept]
 * and [n_seq]).  kept must rise, within the sequence's new rows: a list is taken up to its first entry that is not
 * above the one before it or not one of the sequence's n rows.  Rows whose slots are < 0 or whose pages are not in the
 * pool do not move.  new_len[s] (device int32 [n_seq], not NULL) is the length with the rows that were taken; it may
 * be the kv_len that the plan was made from.  Blocks that are written must belong to one sequence alone. */
int ei_cache_keep(ei_stream_t stream, float* kc, float* vc, int n_blocks, const int* block_table, int max_blocks,
                  int block_size, int n_seq, int rows, int n_head, int n_head_kv, int head_dim, const int* kept,
                  int max_kept, const int* n_kept, int* new_len, const void* plan, size_t plan_bytes);
int ei_cache8_keep(ei_stream_t stream, const ei_cache8* cache, const int* block_table, int max_blocks, int n_seq,
                   int rows, int n_head, int n_head_kv, int head_dim, const int* kept, int max_kept,
                   const int* n_kept, int* new_len, const void* plan, size_t plan_bytes);

#ifdef __cplusplus
}
#endif

#endif /* EI_CACHE8_H */
