/*
 * ikv_batch.h — C-ABI of a step over several sequences on the MI355X (gfx950):
 * the append of packed rows to a paged KV cache, causal attention over packed
 * prompts, the decode attention of one new token of each sequence, the same
 * where sequences share a prefix, and a cache of 8 bits an element with its
 * append, its decode attention and its way back to floats. The rules on every row
 * of logits and their sampler are in ikv_model.h, the single-sequence forms in
 * ikv.h and there; the reference runs one sequence at a time (src/model.cpp:
 * 164-311) and samples greedily (src/sampler.cpp:42-65), so these entry points
 * have no counterpart there. Conventions as in ikv.h: device pointers, stream
 * as void*, 0 / negative errno / positive hipError_t, nothing allocates, frees
 * or synchronises, F32 row-major.
 *
 * The sequences' sizes are device data, read by the kernels: a call is planned
 * from the totals that the host knows, and may be captured in a HIP graph and
 * replayed with other sizes within them. Sizes that are out of range never
 * fault: IKV_STATUS_POSITION is raised in the status word, when one is given,
 * and the sequence that they belong to is skipped; where row_start descends or
 * leaves [0, n_rows] it is raised, too, and which rows are taken is undefined
 * (no access leaves the operands).
 *
 * Launches run on the current device; every operand is on it.
 */
#ifndef IKV_BATCH_H
#define IKV_BATCH_H

#include <stddef.h>
#include <stdint.h>

#include "ikv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------------
 * The paged KV cache of n_seq sequences: one pool per K and V as for
 * ikv_kv_pages (ikv.h), and a block table per sequence. Logical token t of
 * sequence s lives in pool row
 *     block_tables[s * table_stride + t / block_tokens] * block_tokens
 *         + t % block_tokens;
 * a sequence holds at most table_stride * block_tokens tokens. Only entries of
 * blocks that hold tokens of the call are read. An entry outside
 * [0, n_pool_blocks) is treated as by ikv_kv_pages: reads take block 0's rows,
 * writes are dropped, IKV_STATUS_BLOCK is raised in *status. Sequences may
 * share blocks that none of them writes in the call.
 * Checked before any launch (-EINVAL): n_pool_blocks positive, block_tokens a
 * positive multiple of 64, table_stride and n_seq not negative, and where there
 * are sequences block_tables not NULL and table_stride positive; -EOVERFLOW:
 * pool rows past 2^31, n_seq past 2^20, a table_stride * block_tokens past 2^28.
 * 0 sequences: nothing is launched, and 0 is returned where the rest is right.
 * ------------------------------------------------------------------- */
typedef struct ikv_kv_batch {
    const int32_t *block_tables; /* [n_seq][table_stride] */
    int64_t table_stride;
    int64_t block_tokens;
    int64_t n_pool_blocks;
    int64_t n_seq;
    int32_t *status;
} ikv_kv_batch;

/* ---------------------------------------------------------------------
 * Append of packed rows: rows [row_start[s], row_start[s+1]) of k_rows and
 * v_rows (row_bytes each: one token's K or V of all KV heads) become sequence
 * s's logical tokens first_token[s], first_token[s] + 1, ... in the pools.
 * row_start [n_seq + 1] int32 ascending from 0, row_start[n_seq] <= n_rows;
 * first_token [n_seq] int32, or NULL for zeros. Byte-exact; nothing else is
 * written, and rows behind row_start[n_seq] are not read. A token past the
 * sequence's table, or a negative one, is dropped and raises
 * IKV_STATUS_POSITION. Two rows of one call must not name the same pool row.
 * row_bytes: a multiple of 4; 4-byte aligned pointers (-EINVAL).
 * ------------------------------------------------------------------- */
int ikv_append_packed_f32(void *k_pool, void *v_pool, const void *k_rows, const void *v_rows,
                          const ikv_kv_batch *batch, const int32_t *row_start,
                          const int32_t *first_token, int64_t n_rows, size_t row_bytes,
                          void *stream);

/* ---------------------------------------------------------------------
 * Causal attention over packed prompts: rows [row_start[s], row_start[s+1])
 * of q [n_rows][n_head][head_dim] are sequence s's query tokens 0, 1, ...;
 * token t sees the sequence's keys 0 .. t. k, v [n_rows][n_head_kv][head_dim]
 * are packed alike; no row sees another sequence's keys. row_start [n_seq + 1]
 * int32 ascending from 0, row_start[n_seq] <= n_rows: rows behind it are
 * neither read nor written, and a sequence may have none. Head sizes,
 * grouping, scale and results as for ikv_attn_prefill_f32 (any head_dim up to
 * 512, any n_head that n_head_kv divides; else -ENOTSUP / -EINVAL; no
 * workspace), any alignment of 4 bytes. status: device int, or NULL.
 * A result depends on n_seq and n_rows, and in the paged form on the tables' width
 * and the other sequences' lengths, by the order of its sums (the kernel's form and
 * the parts of the keys follow from them), and on nothing else of the other
 * sequences; equal calls give equal bits.
 * -EOVERFLOW: n_rows * n_head past 2^27, or too many blocks for one launch.
 * ------------------------------------------------------------------- */
int ikv_attn_prefill_packed_f32(const float *q, const float *k, const float *v,
                                const int32_t *row_start, int64_t n_seq, int64_t n_rows, float *out,
                                int n_head, int n_head_kv, int head_dim, float scale,
                                int32_t *status, void *stream);

/* The same over a paged cache: sequence s's query tokens come behind n_past[s]
 * cached ones ([n_seq] int32, or NULL for zeros), and token t sees the cached
 * keys 0 .. n_past[s] + t. The pools already hold the new tokens' rows
 * (ikv_append_packed_f32); rows behind a sequence's last token are not read. A
 * sequence that does not fit its table, or of a negative n_past, raises
 * IKV_STATUS_POSITION and its rows are not written.
 *   workspace  NULL, or device memory, 16-byte aligned (else -EINVAL), for the
 *            parts of sequences of few rows behind long histories, whose keys
 *            are then split over several workgroups (a second launch joins the
 *            parts). ikv_attn_prefill_packed_paged_workspace_bytes() says how
 *            much is used at most for these sizes (max_tokens: table_stride *
 *            block_tokens); 0, or less memory than that: nothing is split.
 *            Nothing is expected in it or left in it. Launches that share it
 *            must be ordered.
 * The histories' lengths are device data: that no sequence is longer than a few
 * hundred tokens, for which the call has a faster kernel, shows only in tables
 * that cover no more (768), or in n_past NULL with so few rows. */
size_t ikv_attn_prefill_packed_paged_workspace_bytes(int64_t n_seq, int64_t n_rows,
                                                     int64_t max_tokens, int n_head, int n_head_kv,
                                                     int head_dim);
int ikv_attn_prefill_packed_paged_f32(const float *q, const float *k_pool, const float *v_pool,
                                      const ikv_kv_batch *batch, const int32_t *row_start,
                                      const int32_t *n_past, int64_t n_rows, float *out, int n_head,
                                      int n_head_kv, int head_dim, float scale, void *workspace,
                                      size_t workspace_bytes, void *stream);

/* ---------------------------------------------------------------------
 * Decode attention of one new token of each sequence over a paged cache, the
 * contexts' total length split over the compute units and joined.
 *   q, out   [n_seq][n_head][head_dim]
 *   n_kv     [n_seq] int32: the keys of each sequence, its new token's among
 *            them. 0 is an idle slot: its out row is zeros and nothing else of
 *            it is read or written. A negative length or one that the table
 *            does not cover raises IKV_STATUS_POSITION and is taken for 0.
 *   k_new, v_new  NULL, or the new tokens' rows [n_seq][n_head_kv][head_dim]:
 *            row n_kv[s] - 1 of sequence s is then read from them and written
 *            to the pools (other sequences' rows of the call must not be among
 *            the rows that are written; a row whose block entry is outside the
 *            pool is read and not written).
 *   scale    softmax scale; <= 0 selects 1/sqrtf(head_dim)
 *   workspace  device memory of ikv_attn_decode_batch_workspace_bytes() bytes,
 *            16-byte aligned, for the parts of split contexts and a counter per
 *            workgroup. It must be zero-filled before its first use; every
 *            launch leaves the counters at zero again, so it serves every later
 *            launch of any shape that it is large enough for. Its size does not
 *            depend on the number of sequences or their lengths. Launches that
 *            share it must be ordered (one stream); concurrent ones race.
 * Any head_dim up to 512 (else -ENOTSUP) and any n_head that n_head_kv divides;
 * 4-byte aligned operands. A result depends on the other sequences' lengths by
 * the order of its sums, and on nothing else of them; equal calls give equal
 * bits. -EINVAL: a missing or small workspace; -EOVERFLOW: n_head_kv * head_dim
 * past 2^23.
 * ------------------------------------------------------------------- */
size_t ikv_attn_decode_batch_workspace_bytes(int n_head, int n_head_kv, int head_dim);

int ikv_attn_decode_batch_f32(const float *q, float *k_pool, float *v_pool,
                              const ikv_kv_batch *batch, const int32_t *n_kv, const float *k_new,
                              const float *v_new, float *out, int n_head, int n_head_kv,
                              int head_dim, float scale, void *workspace, size_t workspace_bytes,
                              void *stream);

/* ---------------------------------------------------------------------
 * A paged KV cache of 8 bits an element: codes and, for each row of head_dim
 * elements (a token's K or V of one KV head), an F32 scale. A code stands for
 * code * scale. With top the row's largest magnitude,
 *     IKV_Q8_INT8  scale = top / 127, code = 127 x / top, an integer;
 *     IKV_Q8_E4M3  scale = top / 448, code = 448 x / top in 1-4-3 bits (the
 *                  largest 448, no infinities), from the quotient as a float;
 * the quotient in 64 bits, rounded to nearest, ties to even. A row of zeros has
 * scale 0; one with an element that is not finite has a NaN scale and codes 0, so
 * it reads back as NaNs. The block of ikv_kv_batch's table entry b holds
 *     codes  [b][n_head_kv][block_tokens][head_dim] bytes
 *     scales [b][n_head_kv][block_tokens] floats
 * in each of the K and V arrays, head by head, so that a head's rows of a block
 * are contiguous. codes and scales 16-byte aligned (else -EINVAL); head_dim a multiple
 * of 16 up to 256 (else -ENOTSUP); -EOVERFLOW: n_head_kv * head_dim past 2^23.
 * ------------------------------------------------------------------- */
#define IKV_Q8_INT8 0
#define IKV_Q8_E4M3 1

typedef struct ikv_kv_q8 {
    void *k_codes;
    float *k_scales;
    void *v_codes;
    float *v_scales;
    int32_t n_head_kv;
    int32_t head_dim;
    int32_t format; /* IKV_Q8_* */
} ikv_kv_q8;

/* ikv_append_packed_f32 into such a cache: rows [row_start[s], row_start[s+1]) of
 * k_rows and v_rows [n_rows][n_head_kv][head_dim] (16-byte aligned) become
 * sequence s's logical tokens first_token[s], first_token[s] + 1, ... */
int ikv_append_packed_q8(const ikv_kv_q8 *cache, const float *k_rows, const float *v_rows,
                         const ikv_kv_batch *batch, const int32_t *row_start,
                         const int32_t *first_token, int64_t n_rows, void *stream);

/* The way back: rows [row_start[s], row_start[s+1]) of k_rows and v_rows become
 * the values (code * scale, rounded once) of sequence s's logical tokens
 * first_token[s], first_token[s] + 1, ...; tokens from n_kv[s] on ([n_seq] int32,
 * or NULL: none are) leave their rows as they were, as do rows behind
 * row_start[n_seq]. With row_start at multiples of block_tokens k_rows and v_rows
 * are themselves pools of ikv_kv_batch, sequence s's blocks one behind the other
 * from row_start[s] / block_tokens on: so ikv_attn_prefill_packed_paged_f32 attends
 * over a history that is held in 8 bits. */
int ikv_read_packed_q8(const ikv_kv_q8 *cache, float *k_rows, float *v_rows,
                       const ikv_kv_batch *batch, const int32_t *row_start,
                       const int32_t *first_token, const int32_t *n_kv, int64_t n_rows,
                       void *stream);

/* ikv_attn_decode_batch_f32 over such a cache; q and out are F32, sums and softmax
 * F32. With k_new and v_new (F32 [n_seq][n_head_kv][head_dim]) row n_kv[s] - 1 of
 * sequence s is quantised, written and attended to as it is held: the result is
 * that of ikv_append_packed_q8 and a call without them. q, k_new, v_new and out
 * 16-byte aligned (else -EINVAL). The workspace is used as there (zero-filled
 * once; one of this form serves only this form).
 * Queries, and weights times V's scales, are multiplied as three bf16 pieces: V scales
 * below 2^-100 lose bits that F32 would keep, and with scales above 2^80 sums may leave
 * F32's range, as scores do whose query and key are too large for it. (All of them are
 * held and read back as they are.) */
size_t ikv_attn_decode_batch_q8_workspace_bytes(int n_head, int n_head_kv, int head_dim);

int ikv_attn_decode_batch_q8(const float *q, const ikv_kv_q8 *cache, const ikv_kv_batch *batch,
                             const int32_t *n_kv, const float *k_new, const float *v_new,
                             float *out, int n_head, float scale, void *workspace,
                             size_t workspace_bytes, void *stream);

/* ---------------------------------------------------------------------
 * ikv_attn_decode_batch_f32 where groups of sequences share their first blocks (a
 * system prompt, one document under many questions): those blocks' keys are read
 * once for a group, not once for each of its sequences.
 *   group_start    [n_groups + 1] int32, ascending from 0 to n_seq: group g is the
 *                  sequences [group_start[g], group_start[g + 1])
 *   shared_blocks  [n_groups] int32: the leading entries that the tables of group
 *                  g's sequences have in common (an idle slot's table is not
 *                  read). 0: nothing is shared.
 * Every sequence has a key of its own: one of n_kv[s] <= shared_blocks[g] *
 * block_tokens that is not idle (0) raises IKV_STATUS_POSITION and is taken for 0,
 * as is one of no group within [0, n_seq]. A group of a negative shared_blocks, or of
 * more than the table's width, raises it, too, and shares nothing. Rows that k_new and
 * v_new bring must not lie in blocks that any other sequence reads.
 *   workspace  as for ikv_attn_decode_batch_f32 (zero-filled once), of
 *              ikv_attn_decode_shared_workspace_bytes() bytes for at least these
 *              n_seq and n_groups.
 * Heads of over 128 dims, or of a number of dims that 8 does not divide, operands
 * that are not 16-byte aligned, and calls whose tables hold so few keys (96 MB, all
 * sequences' together) that a launch for the shared ones takes longer than reading
 * them have their shared blocks read once for each sequence, from its own table. That
 * goes by table_stride, so tables of another width may give results that differ by
 * roundings. n_groups 0: nothing is shared.
 * ------------------------------------------------------------------- */
size_t ikv_attn_decode_shared_workspace_bytes(int64_t n_seq, int64_t n_groups, int n_head,
                                              int n_head_kv, int head_dim);

int ikv_attn_decode_shared_f32(const float *q, float *k_pool, float *v_pool,
                               const ikv_kv_batch *batch, const int32_t *group_start,
                               const int32_t *shared_blocks, int64_t n_groups, const int32_t *n_kv,
                               const float *k_new, const float *v_new, float *out, int n_head,
                               int n_head_kv, int head_dim, float scale, void *workspace,
                               size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* IKV_BATCH_H */
