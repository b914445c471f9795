// attn_decode_batch.hip — one new token of each of several sequences over a
// paged KV cache (ikv_attn_decode_batch_f32). The kernel is in attn_decode_batch.hpp.
#include "attn_decode_batch.hpp"

extern "C" size_t ikv_attn_decode_batch_workspace_bytes(int n_head, int n_head_kv, int head_dim) {
  if (n_head <= 0 || n_head_kv <= 0 || n_head % n_head_kv != 0 || head_dim <= 0 || head_dim > kMaxDim) return 0;
  const Form f = form_of(n_head / n_head_kv, head_dim);
  return ikv::parts_bytes(f.gq, f.lpk * f.nv * 4);
}

extern "C" int ikv_attn_decode_batch_f32(const float *q, float *k_pool, float *v_pool,
                                         const ikv_kv_batch *batch, const int32_t *n_kv,
                                         const float *k_new, const float *v_new, float *out, int n_head,
                                         int n_head_kv, int head_dim, float scale, void *workspace,
                                         size_t workspace_bytes, void *stream) {
  Args a;
  if (const int rc = ikv::batch_arg(batch, a.b)) return rc;
  if (n_head <= 0 || n_head_kv <= 0 || n_head % n_head_kv != 0 || head_dim <= 0) return -EINVAL;
  if (head_dim > kMaxDim) return -ENOTSUP;
  if (a.b.n_seq == 0) return 0;
  if (!q || !k_pool || !v_pool || !n_kv || !out || (k_new == nullptr) != (v_new == nullptr)) return -EINVAL;
  if (!workspace || !ikv::aligned16(workspace) ||
      workspace_bytes < ikv_attn_decode_batch_workspace_bytes(n_head, n_head_kv, head_dim))
    return -EINVAL;
  // a unit's rows are one buffer range; a sequence's heads index in int
  if (n_head_kv > INT_MAX / (64 * 4) / head_dim || n_head > INT_MAX / head_dim) return -EOVERFLOW;
  const Form f = form_of(n_head / n_head_kv, head_dim);
  set_args(a, q, k_pool, v_pool, n_kv, k_new, v_new, out, n_head, n_head_kv, head_dim, scale, workspace);
  bool vec = head_dim % 4 == 0;
  for (const void *x : {static_cast<const void *>(q), static_cast<const void *>(k_pool),
                        static_cast<const void *>(v_pool), static_cast<const void *>(k_new),
                        static_cast<const void *>(v_new)})
    vec = vec && ikv::aligned16(x);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (f.lpk == 32) return launch_heads<32, 4>(a, f.gq, vec, s);
  if (f.lpk == 16) return launch_heads<16, 4>(a, f.gq, vec, s);
  return launch_narrow(a, f, vec, s);
}
