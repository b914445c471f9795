// attn_decode_shared.hip — one new token of each of several sequences where groups
// of sequences share their first blocks (ikv_attn_decode_shared_f32).
#include "batch.hpp"

namespace {

constexpr int kThreads = 256;

// The keys of each sequence, 0 where it has none of its own behind those it shares.
__global__ __launch_bounds__(kThreads) void shared_lengths_kernel(ikv::BatchPages b, const int32_t *group_start,
                                                                  const int32_t *shared_blocks, int n_groups,
                                                                  const int32_t *n_kv, int32_t *keys) {
  const int seq = blockIdx.x * kThreads + threadIdx.x;
  if (seq >= b.n_seq) return;
  int shared = n_groups == 0 ? 0 : -1;
  if (n_groups > 0) {
    int lo = 0, hi = n_groups;  // the last group that begins at or before seq is in [lo, hi)
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (group_start[mid] <= seq)
        lo = mid;
      else
        hi = mid;
    }
    const int first = group_start[lo], end = group_start[lo + 1];
    if (first >= 0 && first <= seq && seq < end && end <= b.n_seq) {
      const int blocks = shared_blocks[lo];
      shared = blocks >= 0 && blocks <= b.stride ? blocks * b.bt : 0;
      if (shared == 0 && blocks != 0) ikv::raise_status(b.status, IKV_STATUS_POSITION);
    }
  }
  const int n = n_kv[seq];
  const bool fits = shared >= 0 && n > shared && n <= b.capacity;
  if (!fits && n != 0) ikv::raise_status(b.status, IKV_STATUS_POSITION);
  keys[seq] = fits ? n : 0;
}

}  // namespace

extern "C" size_t ikv_attn_decode_shared_workspace_bytes(int64_t n_seq, int64_t n_groups, int n_head, int n_head_kv,
                                                         int head_dim) {
  const size_t parts = ikv_attn_decode_batch_workspace_bytes(n_head, n_head_kv, head_dim);
  if (parts == 0 || n_seq < 0 || n_seq > ikv::kMaxSeqs || n_groups < 0 || n_groups > ikv::kMaxSeqs) return 0;
  return parts + static_cast<size_t>(n_seq) * sizeof(int32_t);
}

extern "C" int ikv_attn_decode_shared_f32(const float *q, float *k_pool, float *v_pool, const ikv_kv_batch *batch,
                                          const int32_t *group_start, const int32_t *shared_blocks, int64_t n_groups,
                                          const int32_t *n_kv, const float *k_new, const float *v_new, float *out,
                                          int n_head, int n_head_kv, int head_dim, float scale, void *workspace,
                                          size_t workspace_bytes, void *stream) {
  ikv::BatchPages b;
  if (const int rc = ikv::batch_arg(batch, b)) return rc;
  if (n_groups < 0 || n_head <= 0 || n_head_kv <= 0 || n_head % n_head_kv != 0 || head_dim <= 0) return -EINVAL;
  if (head_dim > 512) return -ENOTSUP;
  if (n_groups > ikv::kMaxSeqs) return -EOVERFLOW;
  if (b.n_seq == 0) return 0;
  if (!q || !k_pool || !v_pool || !out || (k_new == nullptr) != (v_new == nullptr)) return -EINVAL;
  if (n_head_kv > INT_MAX / (64 * 4) / head_dim || n_head > INT_MAX / head_dim) return -EOVERFLOW;
  if (!n_kv || (n_groups > 0 && (!group_start || !shared_blocks))) return -EINVAL;
  if (!workspace || !ikv::aligned16(workspace) ||
      workspace_bytes < ikv_attn_decode_shared_workspace_bytes(b.n_seq, n_groups, n_head, n_head_kv, head_dim))
    return -EINVAL;
  const size_t parts = ikv_attn_decode_batch_workspace_bytes(n_head, n_head_kv, head_dim);
  int32_t *const keys = reinterpret_cast<int32_t *>(static_cast<char *>(workspace) + parts);
  shared_lengths_kernel<<<(b.n_seq + kThreads - 1) / kThreads, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
      b, group_start, shared_blocks, static_cast<int>(n_groups), n_kv, keys);
  return ikv_attn_decode_batch_f32(q, k_pool, v_pool, batch, keys, k_new, v_new, out, n_head, n_head_kv, head_dim,
                                   scale, workspace, parts, stream);
}
