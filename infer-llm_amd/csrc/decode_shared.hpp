// decode_shared.hpp — what the two launches of the decode with a shared prefix
// (ikv_attn_decode_shared_f32) pass on: the sums over each group's shared keys
// (attn_decode_shared.hip), which the decode over each sequence's own keys
// (attn_decode_batch.hip) joins with its own.
#pragma once

#include "batch.hpp"

namespace ikv {

// A sequence: its own keys (0: idle, or flagged), those that it shares in front of
// them, its first row (query head of its first KV head) among its group's rows of a
// KV head, and its group's items, (chunk of rows, KV head) with the chunks outer: the
// first one's place among all, its first unit, the units of each, and those of a run.
struct alignas(16) SharedSeq {
  int keys, shared, row, item;
  unsigned long long begin, chunk;
  int tiles, unused[3];
};

// The parts of the sums. Run r of item i left them at slot i + r (each next (item,
// run) that there is has more of one or of both, so no two share a slot):
// [slot][row][2] maximum and sum, [slot][row][dims] values.
struct SharedParts {
  const SharedSeq *seqs;
  const float *ml, *o;
  int rows, dims, slots;  // of a slot; slots that there are
  int n_head_kv;
};

// The slots and the row in them of a sequence's query head h, counted from KV head
// g's first.
struct SharedRow {
  int slot, n, at;
  __device__ __forceinline__ SharedRow(const SharedParts &p, const SharedSeq &s, int g, int h) {
    if (s.shared == 0) {
      n = 0;
      return;
    }
    const int row = s.row + h, item = row / p.rows * p.n_head_kv + g;
    at = row % p.rows;
    const unsigned long long begin = s.begin + static_cast<unsigned long long>(item) * s.tiles;
    const unsigned long long end = begin + s.tiles - 1;
    int w0, w1;
    if ((end | s.chunk) >> 32) {
      w0 = static_cast<int>(begin / s.chunk);
      w1 = static_cast<int>(end / s.chunk);
    } else {
      w0 = static_cast<int>(static_cast<unsigned>(begin) / static_cast<unsigned>(s.chunk));
      w1 = static_cast<int>(static_cast<unsigned>(end) / static_cast<unsigned>(s.chunk));
    }
    slot = s.item + item + w0;
    // (all of them, unless the groups overlap)
    n = static_cast<unsigned>(slot) < static_cast<unsigned>(p.slots) ? min(w1 - w0 + 1, p.slots - slot) : 0;
  }
};

// (x, y), sums of a row's own keys at maximum `top` and sum `all`, and those of the
// keys that it shares, divided: dims d and d + 1.
__device__ __forceinline__ float2 join_shared(const SharedParts &p, const SharedRow &s, int d, float top, float all,
                                              float x, float y) {
  constexpr int kParts = 16;  // loaded at once
  for (int j = 0; j < s.n; j += kParts) {
    float2 ml[kParts], v[kParts];
#pragma unroll
    for (int z = 0; z < kParts; ++z) {
      const size_t r = static_cast<size_t>(s.slot + min(j + z, s.n - 1)) * p.rows + s.at;
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
      if (j + z >= s.n) continue;
      const float w = ml[z].x == -INFINITY ? 0.f : fast_exp2(ml[z].x - top);
      all = fmaf(w, ml[z].y, all);
      x = fmaf(w, v[z].x, x);
      y = fmaf(w, v[z].y, y);
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
