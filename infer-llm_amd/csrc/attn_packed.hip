// attn_packed.hip — causal attention over several prompts, packed one behind
// the other (ikv_attn_prefill_packed_f32 and its paged form): the checks, and
// the choice among the three kernels that run them: short prompts with heads of
// 128 that leave each block a CU take the F32 MFMA one (attn_prefill.hip), others
// the bf16-piece one (attn_bf16x3.hip) and, for head sizes and alignments that it
// does not take, the generic one (attn_generic.hip). Each workgroup finds its
// sequence from row_start (packed_block in batch.hpp) and then works as on a
// prompt alone. In the bf16-piece kernel, up to 64 sequences, where the blocks are
// more than fit the card, those with the most keys start first; where they are
// fewer, the keys of the long ones are split (part_tiles). It takes prompts of every
// length: 16 of 64 tokens, 16 heads of 128, 17 us against 33 in the generic one, one
// token 10.2 against 13.0.
// Measured (MI355X, us): 5 prompts of 8192 tokens together, 32 heads of 128 over
// 8, behind up to 2000: 1620-1750, 173-187 TFLOP/s, 1.1 PFLOP/s of pieces; 16
// prompts of 7001 tokens, 16 heads of 128: 162-173; 9 chunks of 1999 tokens, 12
// heads of 64, behind up to 1500: 61-64 (in two launches); 6 prompts of 160, 16
// heads of 128: 11 (the call; the kernel 9.7), with histories and tables of 4096
// tokens, so on the bf16-piece kernel, 18. The generic kernel, 16 prompts behind up
// to 500, each case with the time of its flops at 154 TFLOP/s: 3605 tokens, 8 heads
// of 200 over 4, 1160 (71); 2692, of 256, 740 (53); 3082, of 512 over 2, 1780 (153);
// 1744, 16 heads of 65 over 8, 600 (17).
#include "attn_bf16x3.hpp"
#include "attn_generic.hpp"
#include "attn_prefill.hpp"
#include "batch.hpp"

namespace {

int prefill_packed(const float *q, const float *k, const float *v, const ikv::Pages *pages,
                   ikv::PackedSeqs seqs, int64_t n_rows, float *out, int n_head, int n_head_kv,
                   int head_dim, float scale, size_t space_bytes, void *stream) {
  if (n_head <= 0 || n_head_kv <= 0 || n_head % n_head_kv != 0 || head_dim <= 0 || n_rows < 0) return -EINVAL;
  if (!ikv::generic_attn_shape(n_head, n_head_kv, head_dim)) return -ENOTSUP;
  if (n_rows == 0 || seqs.n_seq == 0) return 0;
  if (!q || !k || !v || !out || !seqs.row_start) return -EINVAL;
  if (n_rows > INT_MAX / 16 / n_head) return -EOVERFLOW;
  seqs.n_rows = static_cast<int>(n_rows);
  hipStream_t s = static_cast<hipStream_t>(stream);
  int rc = ikv::attn_prefill_packed(q, k, v, pages, out, n_head, n_head_kv, head_dim, seqs, scale, s);
  if (rc != -ENOTSUP) return rc;
  rc = ikv::attn_bf16x3_packed(q, k, v, pages, out, n_head, n_head_kv, head_dim, seqs, scale,
                               space_bytes, s);
  if (rc != -ENOTSUP) return rc;
  return ikv::attn_generic_packed(q, k, v, pages, out, n_head, n_head_kv, head_dim, seqs, scale, s);
}

}  // namespace

extern "C" int ikv_attn_prefill_packed_f32(const float *q, const float *k, const float *v,
                                           const int32_t *row_start, int64_t n_seq, int64_t n_rows,
                                           float *out, int n_head, int n_head_kv, int head_dim,
                                           float scale, int32_t *status, void *stream) {
  if (n_seq < 0) return -EINVAL;
  if (n_seq > ikv::kMaxSeqs) return -EOVERFLOW;
  ikv::PackedSeqs seqs;
  seqs.row_start = row_start;
  seqs.n_seq = static_cast<int>(n_seq);
  seqs.capacity = static_cast<int>(ikv::kMaxSeqTokens) - 1;
  seqs.status = status;
  return prefill_packed(q, k, v, nullptr, seqs, n_rows, out, n_head, n_head_kv, head_dim, scale, 0, stream);
}

extern "C" int ikv_attn_prefill_packed_paged_f32(const float *q, const float *k_pool, const float *v_pool,
                                                 const ikv_kv_batch *batch, const int32_t *row_start,
                                                 const int32_t *n_past, int64_t n_rows, float *out,
                                                 int n_head, int n_head_kv, int head_dim, float scale,
                                                 void *workspace, size_t workspace_bytes, void *stream) {
  ikv::BatchPages b;
  if (const int rc = ikv::batch_arg(batch, b)) return rc;
  ikv::PackedSeqs seqs;
  seqs.row_start = row_start;
  seqs.n_past = n_past;
  seqs.n_seq = b.n_seq;
  seqs.capacity = b.capacity;
  seqs.stride = b.stride;
  seqs.status = b.status;
  if (workspace && !ikv::aligned16(workspace)) return -EINVAL;
  seqs.space = static_cast<float *>(workspace);
  const ikv::Pages pages{b.tables, b.bt, b.n_blocks, b.status};
  return prefill_packed(q, k_pool, v_pool, &pages, seqs, n_rows, out, n_head, n_head_kv, head_dim, scale,
                        workspace ? workspace_bytes : 0, stream);
}

extern "C" size_t ikv_attn_prefill_packed_paged_workspace_bytes(int64_t n_seq, int64_t n_rows, int64_t max_tokens,
                                                                int n_head, int n_head_kv, int head_dim) {
  if (n_head <= 0 || n_head_kv <= 0 || n_head % n_head_kv != 0 || n_seq <= 0 || n_seq > ikv::kMaxSeqs ||
      n_rows <= 0 || n_rows > INT_MAX / 16 / n_head || max_tokens <= 0 || max_tokens > ikv::kMaxSeqTokens ||
      head_dim <= 0 || head_dim > 128 || head_dim % 4 != 0)
    return 0;
  ikv::PackedSeqs seqs;
  seqs.n_past = reinterpret_cast<const int32_t *>(16);  // (histories; not read)
  seqs.n_seq = static_cast<int>(n_seq);
  seqs.n_rows = static_cast<int>(n_rows);
  seqs.capacity = static_cast<int>(max_tokens);
  return ikv::attn_bf16x3_packed_bytes(n_head, n_head_kv, head_dim, seqs);
}
