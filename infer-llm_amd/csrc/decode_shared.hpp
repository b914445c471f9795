// decode_shared.hpp — what the two launches of the decode with a shared prefix
// (ikv_attn_decode_shared_f32) pass on: the sums over each group's shared keys
// (attn_decode_shared.hip), which the decode over each sequence's own keys
// (attn_decode_batch.hip) joins with its own.
#pragma once

#include "batch.hpp"

namespace ikv {

// A sequence: its own keys (0: idle, or flagged), those that it shares in front of
// them, its group, and its first row (query head of its first KV head) among the
// group's rows of a KV head.
struct SharedSeq {
  int keys, shared, group, row;
};

// A group's items, (rows of a chunk, KV head) with the chunks outer: the first one,
// its first unit, and the units of each.
struct SharedGroup {
  unsigned long long begin;
  int item, tiles;
};

// The parts of the sums. Run r of item i left them at slot i + r (each next (item,
// run) that there is has more of one or of both, so no two share a slot):
// [slot][row][2] maximum and sum, [slot][row][dims] values.
struct SharedParts {
  const SharedSeq *seqs;
  const SharedGroup *groups;
  const unsigned long long *chunk;  // units of a run
  const float *ml, *o;
  int rows, dims, slots;  // of a slot; slots that there are
  int n_head_kv;
};

// (x, y), sums of a row's own keys at maximum `top` and sum `all`, and those of the
// keys that it shares, divided. h: the query head, counted from the KV head's first;
// d: dims d and d + 1.
__device__ __forceinline__ float2 join_shared(const SharedParts &p, int seq, int g, int h, int d, float top, float all,
                                              float x, float y) {
  const SharedSeq s = p.seqs[seq];
  if (s.shared > 0 && d < p.dims) {
    const SharedGroup grp = p.groups[s.group];
    const int row = s.row + h, item = row / p.rows * p.n_head_kv + g, at = row % p.rows;
    const unsigned long long begin = grp.begin + static_cast<unsigned long long>(item) * grp.tiles;
    const unsigned long long end = begin + grp.tiles - 1, chunk = *p.chunk;
    int w0, n;
    if ((end | chunk) >> 32) {
      w0 = static_cast<int>(begin / chunk);
      n = static_cast<int>(end / chunk) - w0 + 1;
    } else {
      w0 = static_cast<int>(static_cast<unsigned>(begin) / static_cast<unsigned>(chunk));
      n = static_cast<int>(static_cast<unsigned>(end) / static_cast<unsigned>(chunk)) - w0 + 1;
    }
    const int slot = grp.item + item + w0;
    n = max(0, min(n, p.slots - slot));  // (all of them, unless the groups overlap)
    constexpr int kParts = 8;  // loaded at once
    for (int j = 0; j < n; j += kParts) {
      float2 ml[kParts], v[kParts];
#pragma unroll
      for (int z = 0; z < kParts; ++z) {
        const size_t r = static_cast<size_t>(slot + min(j + z, n - 1)) * p.rows + at;
        ml[z] = *reinterpret_cast<const float2 *>(p.ml + r * 2);
        v[z] = *reinterpret_cast<const float2 *>(p.o + r * p.dims + d);
      }
      float next = top;
#pragma unroll
      for (int z = 0; z < kParts; ++z) next = fmaxf(next, ml[z].x);
      const float f = top == -INFINITY ? 0.f : fast_exp2(top - next);
      all *= f, x *= f, y *= f;
      top = next;
#pragma unroll
      for (int z = 0; z < kParts; ++z) {
        if (j + z >= n) continue;
        const float w = ml[z].x == -INFINITY ? 0.f : fast_exp2(ml[z].x - top);
        all = fmaf(w, ml[z].y, all);
        x = fmaf(w, v[z].x, x);
        y = fmaf(w, v[z].y, y);
      }
    }
  }
  return make_float2(x / all, y / all);
}

// The decode over each sequence's own keys, joined with `parts`: operands as for
// ikv_attn_decode_batch_f32, checked, 16-byte aligned, head_dim a multiple of 4 up to
// 128, workspace of ikv_attn_decode_batch_workspace_bytes().
int decode_behind_shared(const float *q, float *k_pool, float *v_pool, const BatchPages &b, const float *k_new,
                         const float *v_new, float *out, int n_head, int n_head_kv, int head_dim, float scale,
                         void *workspace, const SharedParts &parts, hipStream_t s);

}  // namespace ikv
