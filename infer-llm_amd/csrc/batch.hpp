// batch.hpp — several sequences in one launch: the descriptors of
// include/ikv_batch.h as the kernels see them, and the search for the sequence
// that a packed row or block belongs to.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/ikv_batch.h"
#include "ikv_common.hpp"

namespace ikv {

constexpr int64_t kMaxSeqs = 1 << 20;       // n_seq
constexpr int64_t kMaxWorkgroups = (1 << 24) - 1;  // of 256 threads: 2^32 in a launch
constexpr int64_t kMaxSeqTokens = 1 << 28;  // tokens of one sequence

// Block tables of several sequences (ikv_kv_batch).
struct BatchPages {
  const int32_t *tables = nullptr;
  int64_t stride = 0;  // entries per sequence
  int bt = 0;
  int n_blocks = 0;
  int capacity = 0;  // tokens that a table covers
  int n_seq = 0;
  int *status = nullptr;
};

inline int batch_arg(const ikv_kv_batch *b, BatchPages &out) {
  if (!b || b->table_stride < 0 || b->block_tokens <= 0 || b->block_tokens % 64 != 0 || b->n_pool_blocks <= 0 ||
      b->n_seq < 0)
    return -EINVAL;
  // (no sequences: an empty table has no address, and perhaps no columns)
  if (b->n_seq > 0 && (!b->block_tables || b->table_stride == 0)) return -EINVAL;
  if (b->block_tokens > INT_MAX / b->n_pool_blocks || b->n_seq > kMaxSeqs ||
      b->block_tokens > kMaxSeqTokens / std::max<int64_t>(b->table_stride, 1))
    return -EOVERFLOW;
  out.tables = b->block_tables;
  out.stride = b->table_stride;
  out.bt = static_cast<int>(b->block_tokens);
  out.n_blocks = static_cast<int>(b->n_pool_blocks);
  out.capacity = static_cast<int>(b->table_stride * b->block_tokens);
  out.n_seq = static_cast<int>(b->n_seq);
  out.status = b->status;
  return 0;
}

// One sequence's table.
__device__ __forceinline__ Pages pages_of(const BatchPages &b, int seq) {
  return Pages{b.tables + seq * b.stride, b.bt, b.n_blocks, b.status};
}

// A value that the whole wave has, in scalar registers, where the compiler does not
// see it: a buffer resource of vector registers is looped over, load by load.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  const unsigned lo = __builtin_amdgcn_readfirstlane(static_cast<int>(x));
  const int hi = __builtin_amdgcn_readfirstlane(static_cast<int>(x >> 32));
  return static_cast<int64_t>(hi) << 32 | lo;
}

// The last i in [0, n) for which at_most(i) holds, or -1, for a predicate that
// holds up to some i and not behind it; by a whole wave, 64 probes a round (two
// rounds up to 4096). Whatever the predicate says, the result is in [-1, n).
template <class F>
__device__ __forceinline__ int wave_find_last(int n, F &&at_most) {
  const int lane = threadIdx.x & 63;
  int lo = 0, span = n;
  for (;;) {
    const int step = (span + 63) / 64;
    const bool hit = lane * step < span && at_most(lo + lane * step);
    const int hits = __builtin_popcountll(__builtin_amdgcn_ballot_w64(hit));
    if (hits == 0) return lo - 1;  // (in the first round only, if at all)
    lo += (hits - 1) * step;
    if (step == 1) return lo;
    span = min(step, span - (hits - 1) * step);
  }
}

// By the first workgroup of a launch: IKV_STATUS_POSITION where row_start does
// not ascend within [0, n_rows].
__device__ __forceinline__ void check_row_start(const int32_t *row_start, int n_seq, int64_t n_rows, int *status) {
  if (blockIdx.x != 0 || !status) return;
  bool bad = false;
  for (int s = threadIdx.x; s < n_seq; s += blockDim.x)
    bad |= row_start[s] < 0 || row_start[s + 1] < row_start[s] || row_start[s + 1] > n_rows;
  if (bad) raise_status(status, IKV_STATUS_POSITION);
}

// Prompts packed one behind the other: sequence s has rows [row_start[s],
// row_start[s + 1]) of q, behind n_past[s] cached tokens.
struct PackedSeqs {
  const int32_t *row_start = nullptr;
  const int32_t *n_past = nullptr;  // NULL: none
  int n_seq = 0;
  int n_rows = 0;    // of q, all sequences
  int capacity = 0;  // tokens that a sequence may have
  int64_t stride = 0;  // block table entries per sequence
  int *status = nullptr;
  bool longest_first = false;  // the blocks' order (packed_block_longest)
  int parts = 1;               // of a block's keys, at most (attn_bf16x3.hip),
  int part_slots = 0;          // and the workgroups that fit the card
  float *space = nullptr;      // the parts' sums
};

// One block of `block` query rows (row = token * G + query head of the group)
// of one sequence.
struct PackedBlock {
  int seq, first, rows, past;  // the sequence, its first row, its rows, its history
  int n_blocks, item;          // its blocks, and which of them
};

// An upper bound on the blocks of all sequences: block_base(n_seq).
__host__ __device__ inline int64_t packed_blocks(int64_t n_rows, int64_t n_seq, int G, int block) {
  return n_rows * G / block + n_seq;
}

constexpr int kLaneSeqs = 64;  // up to so many, a sequence a lane

// One sequence of each lane: its first row, its rows and its history; no rows
// where its sizes are out of range (flagged).
struct LaneSeq {
  int first = 0, rows = 0, past = 0;
  __device__ explicit LaneSeq(const PackedSeqs &p) {
    const int lane = threadIdx.x & 63;
    if (lane >= p.n_seq) return;
    const int at = p.row_start[lane], end = p.row_start[lane + 1], before = p.n_past ? p.n_past[lane] : 0;
    if (at < 0 || end < at || end > p.n_rows) return;  // (check_row_start raises)
    first = at;
    if (before < 0 || before > p.capacity - (end - at)) {
      if (end > at && blockIdx.x == 0 && threadIdx.x < 64) raise_status(p.status, IKV_STATUS_POSITION);
      return;
    }
    rows = end - at;
    past = before;
  }
};

// The block that workgroup `item` takes, or false where there is none. Sequence
// s may take items from row_start[s] * G / block + s on: that leaves it at least
// the blocks that it has, whatever the lengths, so no list of blocks is needed.
template <int BLOCK>
__device__ __forceinline__ bool packed_block(const PackedSeqs &p, int G, int item, PackedBlock &b) {
  check_row_start(p.row_start, p.n_seq, p.n_rows, p.status);
  auto base = [&](int start, int s) { return min(max(start, 0), p.n_rows) * G / BLOCK + s; };
  if (p.n_seq <= kLaneSeqs) {
    // (one round of loads where the search and its result take two)
    const int lane = threadIdx.x & 63;
    const LaneSeq mine(p);
    const int from = lane < p.n_seq ? base(p.row_start[lane], lane) : INT_MAX;
    const unsigned long long upto = __builtin_amdgcn_ballot_w64(from <= item);
    if (upto == 0) return false;
    b.seq = 63 - __builtin_clzll(upto);
    b.first = __builtin_amdgcn_readlane(mine.first, b.seq);
    b.rows = __builtin_amdgcn_readlane(mine.rows, b.seq);
    b.past = __builtin_amdgcn_readlane(mine.past, b.seq);
    b.item = item - __builtin_amdgcn_readlane(from, b.seq);
  } else {
    b.seq = wave_find_last(p.n_seq, [&](int s) { return base(p.row_start[s], s) <= item; });
    if (b.seq < 0) return false;
    b.first = p.row_start[b.seq];
    const int end = p.row_start[b.seq + 1];
    b.past = p.n_past ? p.n_past[b.seq] : 0;
    b.item = item - base(b.first, b.seq);
    if (b.first < 0 || end < b.first || end > p.n_rows) return false;
    b.rows = end - b.first;
    if (b.past < 0 || b.past > p.capacity - b.rows) {
      if (b.rows > 0 && threadIdx.x == 0) raise_status(p.status, IKV_STATUS_POSITION);
      return false;
    }
  }
  b.n_blocks = (b.rows * G + BLOCK - 1) / BLOCK;
  return b.item >= 0 && b.item < b.n_blocks;  // (below 0: where row_start descends, if at all)
}

// Integer sum over the wave's lanes (DPP and lane swaps), in a scalar register: a
// workgroup that leaves on it leaves whole, for the compiler, too.
__device__ __forceinline__ int wave_sum_int(int x) {
  x += __builtin_amdgcn_mov_dpp(x, kDppXor1, 0xF, 0xF, false);
  x += __builtin_amdgcn_mov_dpp(x, kDppXor2, 0xF, 0xF, false);
  x += __builtin_amdgcn_mov_dpp(x, kDppHalfMirror, 0xF, 0xF, false);
  x += __builtin_amdgcn_mov_dpp(x, kDppMirror, 0xF, 0xF, false);
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = static_cast<int>(a[0] + a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return __builtin_amdgcn_readfirstlane(static_cast<int>(b[0] + b[1]));
}

// Of a sequence's blocks, those whose last row sees at least L tiles of `tile` keys:
// its last ones.
__host__ __device__ constexpr int blocks_of_tiles(int rows, int past, int G, int block, int tile, int L) {
  const int blocks = (rows * G + block - 1) / block;
  const int unseen = tile * (L - 1) - past;  // tokens before the first that sees so many keys
  if (unseen <= 0) return blocks;
  return unseen >= rows ? 0 : blocks - unseen * G / block;
}

// packed_block with the blocks of all sequences (up to kLaneSeqs) in the order of
// their tiles of TILE keys, the longest first, so that a launch of more blocks
// than fit the card does not end on a long one. The number of blocks of at least
// L tiles is a sum over the sequences, each a division; the L of item's block is
// found by bisection, about 1 us.
template <int BLOCK, int TILE>
__device__ __forceinline__ bool packed_block_longest(const PackedSeqs &p, int G, int item, PackedBlock &b) {
  check_row_start(p.row_start, p.n_seq, p.n_rows, p.status);
  const int lane = threadIdx.x & 63;
  const LaneSeq mine(p);
  const int first = mine.first, rows = mine.rows, past = mine.past;
  const int blocks = (rows * G + BLOCK - 1) / BLOCK;
  auto at_least = [&](int L) { return blocks_of_tiles(rows, past, G, BLOCK, TILE, L); };
  if (item >= wave_sum_int(blocks)) return false;
  int lo = 1, hi = 1;  // wave_sum_int(at_least(lo)) > item
  const int most = rows > 0 ? (past + rows + TILE - 1) / TILE : 0;
  while (__builtin_amdgcn_ballot_w64(most > hi) != 0) hi *= 2;
  ++hi;  // more tiles than any block has
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (wave_sum_int(at_least(mid)) > item)
      lo = mid;
    else
      hi = mid;
  }
  const int longer = at_least(lo + 1), here = at_least(lo) - longer;
  int upto = here;  // blocks of lo tiles of this and the sequences before it
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int y = __shfl_up(upto, o, 64);
    if (lane >= o) upto += y;
  }
  const int rank = item - wave_sum_int(longer);
  b.seq = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > rank));
  b.first = __builtin_amdgcn_readlane(first, b.seq);
  b.rows = __builtin_amdgcn_readlane(rows, b.seq);
  b.past = __builtin_amdgcn_readlane(past, b.seq);
  b.n_blocks = __builtin_amdgcn_readlane(blocks, b.seq);
  b.item = __builtin_amdgcn_readlane(longer + rank - (upto - here), b.seq);
  return true;
}

}  // namespace ikv
