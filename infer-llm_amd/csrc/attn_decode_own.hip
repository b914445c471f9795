// attn_decode_own.hip — the batched decode's kernel (attn_decode_batch.hpp) over the
// keys of each sequence behind those that it shares, for ikv_attn_decode_shared_f32
// (attn_decode_shared.hip has the shared ones).
#include "attn_decode_batch.hpp"

namespace ikv {

int decode_behind_shared(const float *q, float *k_pool, float *v_pool, const BatchPages &b, const float *k_new,
                         const float *v_new, float *out, int n_head, int n_head_kv, int head_dim, float scale,
                         void *workspace, const SharedParts &parts, hipStream_t s) {
  SharedArgs a;
  a.b = b;
  a.shared = parts;
  set_args(a, q, k_pool, v_pool, nullptr, k_new, v_new, out, n_head, n_head_kv, head_dim, scale, workspace);
  return launch_narrow(a, form_of(n_head / n_head_kv, head_dim), true, s);
}

}  // namespace ikv
