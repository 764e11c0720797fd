/*
 * ei_packed.h — the new rows of several sequences in one call: rotary positions row by row, causal
 * attention over packed prompts, and over chunks whose keys sit in a paged pool.
 *
 * Conventions as in ei_attn.h (status codes, device pointers, streams, alignment, limits): fp32,
 * head_dim 128, GQA groups of 1 to 8, nothing allocated, no host synchronisation, capturable.
 * No counterpart in the reference, which runs one sequence at a time (src/cuda/model_cuda.cu:1648-1658).
 *
 * A batch holds n_seq sequences whose new rows follow one another: rows cu_rows[s] ..
 * cu_rows[s+1] - 1 (device int32 [n_seq + 1], from 0 up, never falling, cu_rows[n_seq] <= rows) belong
 * to sequence s, which may have none.  Rows from cu_rows[n_seq] on belong to nobody: nothing is
 * written there, and it does not matter what they hold.
 *
 * A call whose outputs, workspace, plan or (in the step) pools overlap anything that it reads is refused.
 */
#ifndef EI_PACKED_H
#define EI_PACKED_H

#include <stddef.h>
#include <stdint.h>

#include "ei_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------ rotary positions
 * Frequencies f_i = theta^(-2i/rope_dim), i < rope_dim/2, or scaled for positions beyond the n_trained
 * a model was trained for by `factor` (>= 1):
 *   EI_ROPE_LINEAR  f_i / factor (positions squeezed into the trained range)
 *   EI_ROPE_NTK     f_i of the base theta * factor^(rope_dim / (rope_dim - 2)): the slowest pair is
 *                   slowed by factor, the fastest not at all (rope_dim > 2)
 *   EI_ROPE_YARN    f_i / factor for the pairs that make at most beta_slow turns over n_trained
 *                   positions, f_i for those that make beta_fast or more, a ramp over the pair index
 *                   between; cos and sin times 0.1 ln(factor) + 1, or times attn_factor if that is > 0
 * Fields a kind does not use are ignored. */
enum { EI_ROPE_NONE = 0, EI_ROPE_LINEAR = 1, EI_ROPE_NTK = 2, EI_ROPE_YARN = 3 };
typedef struct ei_rope_scaling {
    int kind;           /* EI_ROPE_* */
    double factor;      /* context extension, >= 1 */
    int n_trained;      /* EI_ROPE_YARN: positions the model was trained for */
    double beta_fast;   /* EI_ROPE_YARN: 32 as published */
    double beta_slow;   /* EI_ROPE_YARN: 1 as published */
    double attn_factor; /* EI_ROPE_YARN: factor on cos and sin; <= 0: 0.1 ln(factor) + 1 */
} ei_rope_scaling;

/* Fills the device table cs[p][i] = (float(m cos(p f_i)), float(m sin(p f_i))), [n_pos][rope_dim/2][2],
 * angles, cosines and sines in double, rounded once.  scaling NULL: EI_ROPE_NONE, the values of
 * ei_rope_table_fill.  Every entry point that takes a table takes this one.  rope_dim even, <= 128. */
int ei_rope_table_scaled(ei_stream_t stream, float* cs, int n_pos, int rope_dim, double theta,
                         const ei_rope_scaling* scaling);

/* Turns n_heads heads of `rows` rows, each row at its own position pos[b] (device int32 [rows]):
 * head h of row b at x + b*x_stride + h*128, written to y + b*y_stride + h*128.  y may be x with the
 * same stride (in place), or other columns of one buffer; any overlap of their rows is refused, and y over
 * cs, pos or gamma.  gamma (128 values, or NULL): each head is RMS-normed first, as in ei_headnorm_rope.
 * Pairs of the first rope_dim elements:
 *   EI_ROPE_HALF         (i, i + rope_dim/2)
 *   EI_ROPE_INTERLEAVED  (2i, 2i + 1)
 * elements from rope_dim on are only normed.  y columns past the heads are not written.  A row whose
 * position lies outside the table, pos[b] < 0 or >= n_pos (padding), is copied as it is, without
 * norm.  Strides are multiples of 4 floats, pointers 16-byte aligned (pos 4). */
enum { EI_ROPE_HALF = 0, EI_ROPE_INTERLEAVED = 1 };
int ei_rope_rows(ei_stream_t stream, const float* x, long x_stride, float* y, long y_stride, int rows, int n_heads,
                 int head_dim, const float* gamma, float eps, const float* cs, int n_pos, const int* pos,
                 int rope_dim, int layout);

/* ------------------------------------------------------------------ the plan of a batch
 * ei_packed_plan lays the batch's attention out over the GPU from its lengths (one small launch):
 * made once for a batch, it serves every layer, on any stream that the plan's launch comes before.
 * kv_len (device int32 [n_seq]): keys of sequence s after its new rows are appended, so that its
 * row i of n sees keys 0 .. kv_len[s] - n + i; a row that sees none (kv_len[s] < n) gets zeros.
 * kv_len NULL: whole prompts, kv_len[s] = n.  max_kv (<= 2^30) must be at least the longest length, prompts'
 * own lengths too: attention takes a longer sequence as one of max_kv keys, whose rows see as many keys fewer
 * as it is longer (and the first rows of a prompt none), and the step appends nothing at positions from
 * max_kv on.  Lengths below 0 count as 0.
 * A call of the entry points below whose n_seq, rows, heads differ from the plan's writes nothing, and so
 * does one on a plan whose cu_rows count more rows than `rows`.
 * The plan of n_seq sequences and `rows` rows takes ei_packed_plan_bytes(n_seq, rows, ...) bytes (0
 * for invalid shapes); 1 <= n_seq <= 65535, rows <= 2^20, rows * n_head <= 2^28. */
size_t ei_packed_plan_bytes(int n_seq, int rows, int n_head, int n_head_kv);
int ei_packed_plan(ei_stream_t stream, const int* cu_rows, const int* kv_len, int n_seq, int rows, int max_kv,
                   int n_head, int n_head_kv, void* plan, size_t plan_bytes);

/* Workspace of the calls below: sequences whose keys are split over workgroups, and the step's normed
 * queries.  It needs no initialisation; calls that share one must not overlap in time. */
size_t ei_packed_ws_bytes(int rows, int n_head, int n_head_kv);

/* ------------------------------------------------------------------ attention over packed prompts
 * Causal attention of every sequence over its own rows: q row b at q + b*q_stride ([n_head][128],
 * normed and turned), k and v rows at k + b*kv_stride ([n_head_kv][128]); views of one [Q | K | V]
 * buffer are fine; kv_stride at most 2^22.  out [rows][n_head][128], which must not overlap the inputs.
 * The plan must be one of whole prompts (kv_len NULL).
 *
 * Arithmetic of this call and the two below: sums and softmax in fp32, and for the last few rows of a
 * sequence (single tokens, drafts) the products too.  Other rows' are made of two binary16 planes per
 * operand, which keep 22 bits of 24 (the product of two low planes is left out, another 2^-22 at most), and
 *   V        to 2^-39 of the largest value in its 32 columns (0 .. 31, ...) at the keys before and beside it: a
 *            column far below those keeps fewer bits, at 2^-20 of them 17 to 19;
 *   q and K  so that a score is off by 2^-18 of a log2 unit at most;
 *   weights  so that an output is off by 2^-17 of the row's largest at most.
 * Where more is lost, the waves that notice it take their keys again in fp32, three to five times slower
 * (bad values beside 17 to 32 flat rows of a KV head: up to fourteen times):
 * V's largest values 2^17 times a row's outputs; weights that are nearly all at keys without a value; the
 * largest q of some neighbouring rows times the largest K of a key, times scale, above 2^12; infinite or NaN
 * values in K or V.  Outputs differ from ei_attn_prefill's, which keeps all 24 bits, and ei_attn_decode's in
 * the last bits, and with the batch a sequence is in; a batch called twice gives the same bits.  Key and
 * value rows that a row does not see never reach it, whatever they hold. */
int ei_attn_packed(ei_stream_t stream, const float* q, long q_stride, const float* k, const float* v,
                   long kv_stride, float* out, int n_seq, int rows, int n_head, int n_head_kv, int head_dim,
                   float scale, const void* plan, size_t plan_bytes, void* ws, size_t ws_bytes);

/* ------------------------------------------------------------------ attention over a paged pool
 * As ei_attn_packed, with the keys of sequence s in the pool kc, vc of n_blocks blocks: key t in pool
 * row block_table[s*max_blocks + t/block_size]*block_size + t%block_size (rows of n_head_kv*128
 * floats, block_size a power of two >= 32).  The new rows' keys must already be there.  Sequences may
 * share blocks.  Keys past the table's span, and keys of a block whose entry is not in
 * [0, n_blocks), count as zeros: nothing is read there. */
int ei_attn_packed_paged(ei_stream_t stream, const float* q, long q_stride, float* out, const float* kc,
                         const float* vc, int n_blocks, const int* block_table, int max_blocks, int block_size,
                         int n_seq, int rows, int n_head, int n_head_kv, int head_dim, float scale,
                         const void* plan, size_t plan_bytes, void* ws, size_t ws_bytes);

/* The whole step from raw projections: qkv row b is [Q | K | V] at qkv + b*row_stride, read only.
 * Row i of n of sequence s stands at position kv_len[s] - n + i: its Q and K heads are normed and
 * turned there (half layout, full or partial rope_dim, table cs of n_pos positions; as
 * ei_qkv_prepare), K and V appended to the sequence's pool row, then attention as
 * ei_attn_packed_paged.  A row at a position < 0, >= n_pos, >= the plan's max_kv or past its sequence's
 * pages appends nothing; at a position < 0, >= n_pos or >= max_kv its query is neither normed nor turned.
 * Blocks that are written must belong to one sequence alone. */
int ei_packed_step_paged(ei_stream_t stream, const float* qkv, long row_stride, float* out, float* kc, float* vc,
                         int n_blocks, const int* block_table, int max_blocks, int block_size, int n_seq, int rows,
                         int n_head, int n_head_kv, int head_dim, const float* q_gamma, const float* k_gamma,
                         const float* cs, int n_pos, int rope_dim, float eps, float scale, const void* plan,
                         size_t plan_bytes, void* ws, size_t ws_bytes);

#ifdef __cplusplus
}
#endif

#endif /* EI_PACKED_H */
