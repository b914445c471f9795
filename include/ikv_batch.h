/*
 * ikv_batch.h — C-ABI of a step over several sequences on the MI355X (gfx950):
 * the append of packed rows to a paged KV cache, causal attention over packed
 * prompts, the decode attention of one new token of each sequence, and the
 * sampler of every row of logits. The single-sequence forms are in ikv.h and
 * ikv_model.h; the reference runs one sequence at a time (src/model.cpp:
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

#ifdef __cplusplus
}
#endif

#endif /* IKV_BATCH_H */
