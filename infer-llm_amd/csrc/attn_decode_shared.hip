// attn_decode_shared.hip — one new token of each of several sequences where groups
// of sequences share their first blocks (ikv_attn_decode_shared_f32).
//
// A first launch takes the shared keys: the query heads of one KV head of all of a
// group's sequences are the rows of one product, so the keys are read once for a
// chunk of rows. A second one is the batched decode over each sequence's own keys
// (attn_decode_batch.hip), which joins the two at its end.
//
// The shared part has 4 D flops a key and row, on F32 matrix instructions
// (v_mfma_f32_32x32x2). Up to about 48 rows of a KV head the reads bound it, with
// more the matrix pipe.
//   * Shared blocks are whole, so no key is masked and no tile is short.
//   * A wave has 32 rows and takes tiles of 32 keys: S^T = K Q^T, O^T += V^T P^T. A
//     lane holds one row in both products, so weights stay where they are, and it
//     reads K as 16 bytes of a key's dims and V as D / 32 dims of a key, 64 matrix
//     instructions of 64 cycles for 64 registers each: nothing needs LDS. K of the
//     next tile is on its way during P V, its V during Q K^T.
//   * RB row blocks by 4 / RB key groups make a workgroup, one wave a SIMD.
//   * The (chunk, KV head) items' tiles are dealt to the workgroups in equal runs,
//     from the groups as they stand on the device; what a run has of an item goes to
//     the workspace.
// Measured (MI355X, us, traced), the shared part and the decode behind it: 48 sequences
// behind 16384 tokens, 32 heads of 128 over 8, 130 + 39 (the shared part 12.9 GF, 99
// TFLOP/s of the 151 of a large F32 product; with 127, of a workgroup's 113 on average 10
// were its start and 8 % the softmax and waits, the clock fell to 2.2 GHz, and the last
// workgroup was done 12 after the mean, one with parts of two items); 37 sequences in 3
// groups of 64-float heads 16.5 + 14.4: starts, joins and launches; unshared 46.9 and,
// the 48, 1002. The running sums of a row are a chain of additions over a wave's keys:
// the errors of the 48 are 6.5e-7 (2-norm), unshared 2.6e-7.
// Tried and not kept: two waves a SIMD (spilled; 140), two sums of S (the same).
#include "decode_shared.hpp"
#include "coherent.hpp"
#include "decode_runs.hpp"

#include <algorithm>
#include <type_traits>

namespace {

typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256, kWaves = 4;
constexpr int kRuns = 256;  // workgroups, one a compute unit: a run each
constexpr int BN = 32;      // keys of a tile, the unit of a run
constexpr float kRescale = 8.0f;  // log2 headroom before the running maximum is moved

struct Groups {
  const int32_t *start, *blocks;
  int n;
};

// A group as it stands: its first sequence, its sequences, its shared blocks (none
// where its sizes are out of range).
struct Group {
  int first, seqs, blocks;
};
__device__ __forceinline__ Group group_of(const ikv::BatchPages &b, const Groups &groups, int g) {
  const int first = groups.start[g], end = groups.start[g + 1], blocks = groups.blocks[g];
  if (first < 0 || end <= first || end > b.n_seq) return {0, 0, 0};
  return {first, end - first, blocks >= 0 && blocks <= b.stride ? blocks : 0};
}

// A sequence's keys and group (-1: none): by a thread.
struct Keys {
  int own, shared, group, row;  // row: its first of the group's
};
__device__ __forceinline__ Keys keys_of(const ikv::BatchPages &b, const Groups &groups, const int32_t *n_kv, int seq,
                                        int G) {
  Keys s{0, 0, -1, 0};
  const int n = n_kv[seq];
  bool found = groups.n == 0, bad = false;
  if (groups.n > 0) {
    int lo = 0, hi = groups.n;  // the last group that begins at or before seq is in [lo, hi)
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (groups.start[mid] <= seq)
        lo = mid;
      else
        hi = mid;
    }
    const Group g = group_of(b, groups, lo);
    found = g.seqs > 0 && g.first <= seq && seq < g.first + g.seqs;
    if (found) {
      s.group = lo;
      s.shared = g.blocks * b.bt;
      s.row = (seq - g.first) * G;
      bad = groups.blocks[lo] != g.blocks;
    }
  }
  if (found && n > s.shared && n <= b.capacity)
    s.own = n - s.shared;
  else
    bad |= n != 0;
  if (bad) ikv::raise_status(b.status, IKV_STATUS_POSITION);
  return s;
}

// The first of a group's sequences that has keys of its own, counted from its first
// one (-1: none), by a whole wave, where lane l has n_kv of sequence l of the group
// (of the last one, where there are fewer).
__device__ __forceinline__ int first_live(const ikv::BatchPages &b, const Group &g, const int32_t *n_kv, int n) {
  const int lane = threadIdx.x & 63, shared = g.blocks * b.bt;
  for (int s = 0;;) {
    const unsigned long long some = __builtin_amdgcn_ballot_w64(n > shared && n <= b.capacity);
    if (some) return s + __builtin_ctzll(some);
    s += 64;
    if (s >= g.seqs) return -1;
    n = n_kv[g.first + min(s + lane, g.seqs - 1)];
  }
}

// What the matrix kernel does not take, or is not worth its launch: the keys of each
// sequence, for a decode that reads all of them.
__global__ __launch_bounds__(kThreads) void shared_lengths_kernel(ikv::BatchPages b, Groups groups,
                                                                  const int32_t *n_kv, int32_t *keys) {
  ikv::check_row_start(groups.start, groups.n, b.n_seq, b.status);
  const int seq = blockIdx.x * kThreads + threadIdx.x;
  if (seq >= b.n_seq) return;
  const Keys s = keys_of(b, groups, n_kv, seq, 1);
  keys[seq] = s.own > 0 ? s.shared + s.own : 0;
}

struct Args {
  const float *q, *k, *v;
  const int32_t *n_kv;
  ikv::BatchPages b;
  Groups groups;
  int n_head_kv, G, dim;
  float scale_log2;
  ikv::SharedSeq *seqs;
  float *ml, *o;
  int slots;
};

// A place in the list of tiles: tile `tile` of `tiles` of item `item` of group g.
struct Place {
  int item, tile, tiles, items;
  Group g;
};

// The tiles of all groups' items, in the order (group, chunk, KV head, key), by a
// whole wave, 64 groups at a time.
template <int R>
struct Plan {
  using Units = unsigned long long;
  Units total, chunk;
  int g0;
  Group g;  // of this lane
  int tiles, items;
  Units upto;
  int item_upto;

  __device__ void look(const Args &a, int first, Units before, int items_before) {
    const int i = first + static_cast<int>(threadIdx.x & 63);
    g0 = first;
    g = i < a.groups.n ? group_of(a.b, a.groups, i) : Group{0, 0, 0};
    tiles = g.blocks * (a.b.bt / BN);
    items = tiles > 0 ? (g.seqs * a.G + R - 1) / R * a.n_head_kv : 0;
    upto = before + ikv::wave_prefix(static_cast<Units>(items) * tiles);
    item_upto = items_before + static_cast<int>(ikv::wave_prefix(items));
  }
  __device__ explicit Plan(const Args &a) {
    total = 0;
    for (int s = 0, n = 0; s < a.groups.n; s += 64) {
      look(a, s, total, n);
      total = ikv::lane_value(upto, 63);
      n = __builtin_amdgcn_readlane(item_upto, 63);
    }
    chunk = max((total + kRuns - 1) / kRuns, Units{kWaves});
  }
  // what the next launch has to know of a lane's sequence
  __device__ ikv::SharedSeq about(const Args &a, const Keys &k) {
    ikv::SharedSeq x{k.own, k.shared, k.row, 0, 0, chunk, 0, {}};
    Units before = 0;
    for (int s = 0, n = 0; s < a.groups.n; s += 64) {
      if (a.groups.n > 64) look(a, s, before, n);
      const int l = k.group - s;
      const bool here = l >= 0 && l < 64;
      const Units b = upto - static_cast<Units>(items) * tiles;
      const unsigned lo = __shfl(static_cast<unsigned>(b), l & 63, 64), hi = __shfl(static_cast<unsigned>(b >> 32), l & 63, 64);
      const int first = __shfl(item_upto - items, l & 63, 64), each = __shfl(tiles, l & 63, 64);
      if (here) {
        x.begin = static_cast<Units>(hi) << 32 | lo;
        x.item = first;
        x.tiles = each;
      }
      before = ikv::lane_value(upto, 63);
      n = __builtin_amdgcn_readlane(item_upto, 63);
    }
    return x;
  }
  // where unit u (< total) is; `first`: the item's place among all
  __device__ Place at(const Args &a, Units u, int &first) {
    if (a.groups.n > 64) {
      Units before = 0;
      int n = 0;
      for (int s = 0; s < a.groups.n; s += 64) {
        look(a, s, before, n);
        before = ikv::lane_value(upto, 63);
        n = __builtin_amdgcn_readlane(item_upto, 63);
        if (before > u) break;
      }
    }
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > u));
    Place p;
    p.g = {__builtin_amdgcn_readlane(g.first, l), __builtin_amdgcn_readlane(g.seqs, l),
           __builtin_amdgcn_readlane(g.blocks, l)};
    p.tiles = __builtin_amdgcn_readlane(tiles, l);
    p.items = __builtin_amdgcn_readlane(items, l);
    const Units r = u - (ikv::lane_value(upto, l) - static_cast<Units>(p.tiles) * p.items);
    if (r >> 32) {
      p.item = static_cast<int>(r / p.tiles);
      p.tile = static_cast<int>(r % p.tiles);
    } else {
      p.item = static_cast<int>(static_cast<unsigned>(r) / p.tiles);
      p.tile = static_cast<int>(static_cast<unsigned>(r) % p.tiles);
    }
    p.item = ikv::uniform(p.item);
    p.tile = ikv::uniform(p.tile);
    first = __builtin_amdgcn_readlane(item_upto, l) - p.items;
    return p;
  }
};

// The dims of lane m of 32: DT m + i, or, with 96, m + 32 i (three floats at 3 m
// would reach past a row of 80).
template <int DT>
__device__ __forceinline__ constexpr int dim_of(int m, int i) {
  return DT == 3 ? m + 32 * i : DT * m + i;
}
// Them at off[] of a row; one offset but for 96.
template <int DT>
__device__ __forceinline__ void load_dims(__amdgpu_buffer_rsrc_t r, const unsigned *off, unsigned row, float *d) {
  if constexpr (DT == 2) {
    const auto t = __builtin_bit_cast(floatx2, __builtin_amdgcn_raw_buffer_load_b64(r, off[0] + row, 0, 0));
    d[0] = t[0], d[1] = t[1];
  } else if constexpr (DT == 4) {
    const auto t = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(r, off[0] + row, 0, 0));
    d[0] = t[0], d[1] = t[1], d[2] = t[2], d[3] = t[3];
  } else {
#pragma unroll
    for (int i = 0; i < DT; ++i)
      d[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, off[i] + row, 0, 0));
  }
}

__device__ __forceinline__ float pair_max(float x) {  // lanes l and l ^ 32
  const float2 y = ikv::halves(x);
  return fmaxf(y.x, y.y);
}
__device__ __forceinline__ float pair_sum(float x) {
  const float2 y = ikv::halves(x);
  return y.x + y.y;
}

template <int DT, int RB>
__global__ __launch_bounds__(kThreads, 1) void shared_prefix_kernel(Args a) {
  constexpr int KG = kWaves / RB, R = 32 * RB, DP = 32 * DT, KJ = 4 * DT;
  __shared__ float s_x[kWaves * (16 * DT + 2) * 64];  // the waves' states
  __shared__ floatx4 s_q[RB][KJ][64];  // the query rows, scaled, as the lanes take them
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave / RB, rb = wave % RB;
  const int r32 = lane & 31, c2 = lane >> 5;
  const int stride = a.n_head_kv * a.dim;

  ikv::check_row_start(a.groups.start, a.groups.n, a.b.n_seq, a.b.status);
  Plan<R> plan(a);
  // (by whole waves, from the last workgroups on: in a small call they have no run)
  for (int s0 = (gridDim.x - 1 - blockIdx.x) * kThreads + 64 * wave; s0 < a.b.n_seq; s0 += gridDim.x * kThreads) {
    const int seq = min(s0 + lane, a.b.n_seq - 1);
    const ikv::SharedSeq x = plan.about(a, keys_of(a.b, a.groups, a.n_kv, seq, a.G));
    if (s0 + lane < a.b.n_seq) a.seqs[seq] = x;
  }

  // runs of one XCD next to each other: they read the same KV heads
  const int run = static_cast<int>(blockIdx.x % 8 * (kRuns / 8) + blockIdx.x / 8);
  unsigned long long u = plan.chunk * run;
  const unsigned long long end = min(plan.total, u + plan.chunk);
  // this lane's pieces of a tile's K rows, j 32 bytes further each, and its dims of the V rows
  constexpr unsigned kOut = 0x80000000u;
  const unsigned k_off = static_cast<unsigned>(r32 * stride + 4 * c2) * 4u;
  auto piece = [&](int j) { return j < KJ - 3 || 8 * j < a.dim; };  // whether there is a j
  unsigned v_off[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i)
    v_off[i] = dim_of<DT>(r32, i) < a.dim ? static_cast<unsigned>(4 * c2 * stride + dim_of<DT>(r32, i)) * 4u : kOut;

  while (u < end) {
    int item0;
    const Place p = plan.at(a, u, item0);
    const int last = static_cast<int>(min<unsigned long long>(p.tiles, p.tile + (end - u)));
    const int g = p.item % a.n_head_kv, row0 = p.item / a.n_head_kv * R;
    const int rows = p.g.seqs * a.G - row0;  // of the chunk, and those behind it
    const int row = row0 + 32 * rb + r32;
    const bool row_ok = row - row0 < rows;
    const bool busy = 32 * rb < rows;  // whether this wave has rows

    floatx16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = floatx16{};
    float m = -INFINITY, sum = 0.f;

    const int t0 = p.tile + kg;
    {
      // The blocks are those of the group's first sequence that has keys: an idle slot's
      // entries may be anything. The first slot's are loaded together with the lengths,
      // as it seldom is an idle one.
      const int32_t *table = a.b.tables + p.g.first * a.b.stride;
      int blk = t0 * BN / a.b.bt, in_blk = t0 * BN % a.b.bt, ent0 = 0, ent = 0;
      auto load_entries = [&]() {
        ent0 = blk;
        ent = table[min(blk + lane, p.g.blocks - 1)];
      };
      auto check_entries = [&]() {
        if (static_cast<unsigned>(ent) >= static_cast<unsigned>(a.b.n_blocks)) {
          ikv::raise_status(a.b.status, IKV_STATUS_BLOCK);
          ent = 0;
        }
      };
      load_entries();
      const int live = first_live(a.b, p.g, a.n_kv, a.n_kv[p.g.first + min(lane, p.g.seqs - 1)]);
      if (live < 0) {  // (nobody asks for the sums; by all waves alike)
        u += last - p.tile;
        continue;
      }
      if (live > 0) {
        table += live * a.b.stride;
        load_entries();
      }
      check_entries();
      constexpr int kMine = (KJ + KG - 1) / KG;  // of the rows' pieces: j = kg, kg + KG, ...
      floatx4 qr[kMine] = {};
      if (row_ok) {
        const int at = row % a.G;
        const float *const from =
            a.q + (static_cast<size_t>(p.g.first + row / a.G) * a.n_head_kv * a.G + g * a.G + at) * a.dim + 4 * c2;
#pragma unroll
        for (int i = 0; i < kMine; ++i)
          if (kg + KG * i < KJ && piece(kg + KG * i)) qr[i] = *reinterpret_cast<const floatx4 *>(from + 8 * (kg + KG * i));
      }
      auto next_row = [&]() -> long long {  // the tile's row of the pools, moved on to the next one
        const long long r = static_cast<long long>(__builtin_amdgcn_readlane(ent, blk - ent0)) * a.b.bt + in_blk;
        in_blk += KG * BN;
        while (in_blk >= a.b.bt) {
          in_blk -= a.b.bt;
          ++blk;
        }
        if (blk - ent0 >= 64) {
          load_entries();
          check_entries();
        }
        return r;
      };
      auto rsrc = [&](const float *base, long long r, int t) {  // (none of a tile behind the run)
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(base + r * stride + g * a.dim), 0,
                                                 busy && t < last ? ((BN - 1) * stride + a.dim) * 4 : 0, ikv::kBufWord3);
      };
      floatx4 kf[KJ];
      float vf[16][DT];
      auto load_k = [&](__amdgpu_buffer_rsrc_t x, int j) {
        kf[j] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(x, piece(j) ? k_off + 32 * j : kOut, 0, 0));
      };
      auto load_v = [&](__amdgpu_buffer_rsrc_t x, int e) {
        load_dims<DT>(x, v_off, static_cast<unsigned>((8 * (e >> 2) + (e & 3)) * stride * 4), vf[e]);
      };
      {
        const long long r = next_row();
        const auto rk = rsrc(a.k, r, t0), rv = rsrc(a.v, r, t0);
        // (in the order of the loop's: else its first product waits for what was loaded
        // last, here as there)
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          load_k(rk, j);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          load_v(rv, e);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int i = 0; i < kMine; ++i)
        if (kg + KG * i < KJ) s_q[rb][kg + KG * i][lane] = qr[i] * a.scale_log2;
      __syncthreads();
      for (int t = t0; busy && t < last; t += KG) {
        // (each piece of the next tile's as soon as this one's is in the product)
        const long long r = next_row();
        const auto rk = rsrc(a.k, r, t + KG), rv = rsrc(a.v, r, t + KG);
        floatx16 s{};
        floatx4 next = s_q[rb][0][lane];
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const floatx4 qf = next;
          if (j + 1 < KJ) next = s_q[rb][j + 1][lane];
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j][e], qf[e], s, 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          load_k(rk, j);
          __builtin_amdgcn_sched_barrier(0);
        }
        float mt = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mt = fmaxf(mt, s[e]);
        if (__builtin_amdgcn_ballot_w64(mt > m + kRescale) != 0) {
          const float top = fmaxf(m, pair_max(mt));
          const float f = ikv::weight(m, top);
          m = top;
          sum *= f;
#pragma unroll
          for (int i = 0; i < DT; ++i) o[i] *= f;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        // (a weight is formed behind the products of the one before it)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float w = ikv::fast_exp2(s[e] - ref);
          sum += w;
#pragma unroll
          for (int i = 0; i < DT; ++i) o[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[e][i], w, o[i], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          load_v(rv, e);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    sum = pair_sum(sum);
    // the key groups' states meet in LDS; a wave joins and stores every KG-th part of
    // its rows' dims
    constexpr int XW = 16 * DT + 2;
    {
      float *const x = s_x + (kg * RB + rb) * XW * 64 + lane;
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[(16 * i + e) * 64] = o[i][e];
      x[16 * DT * 64] = m;
      x[(16 * DT + 1) * 64] = sum;
    }
    __syncthreads();
    const int slot = item0 + p.item + run;
    if (row_ok && static_cast<unsigned>(slot) < static_cast<unsigned>(a.slots)) {  // (all of them, unless the groups overlap)
      const size_t at = static_cast<size_t>(slot) * R + 32 * rb + r32;
      float f[KG], top = -INFINITY, all = 0.f;
#pragma unroll
      for (int z = 0; z < KG; ++z) {
        f[z] = s_x[((z * RB + rb) * XW + 16 * DT) * 64 + lane];
        top = fmaxf(top, f[z]);
      }
#pragma unroll
      for (int z = 0; z < KG; ++z) {
        f[z] = ikv::weight(f[z], top);
        all = fmaf(f[z], s_x[((z * RB + rb) * XW + 16 * DT + 1) * 64 + lane], all);
      }
      if (kg == 0 && c2 == 0) *reinterpret_cast<float2 *>(a.ml + at * 2) = make_float2(top, all);
      // four of a lane's 16 DT values at a time: rows 8 q + 4 c2 .. + 3 of a product
      for (int z0 = kg; z0 < 4; z0 += KG) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v[DT] = {};
#pragma unroll
          for (int z = 0; z < KG; ++z)
#pragma unroll
            for (int i = 0; i < DT; ++i)
              v[i] = fmaf(f[z], s_x[((z * RB + rb) * XW + 16 * i + 4 * z0 + e) * 64 + lane], v[i]);
          const int mrow = 8 * z0 + 4 * c2 + e;
#pragma unroll
          for (int i = 0; i < DT; ++i) a.o[at * DP + dim_of<DT>(mrow, i)] = v[i];
        }
      }
    }
    __syncthreads();
    u += last - p.tile;
  }
}

// Whether the matrix kernel takes these operands.
bool on_matrices(int head_dim, std::initializer_list<const void *> operands) {
  if (head_dim % 8 != 0 || head_dim > 128) return false;
  for (const void *p : operands)
    if (!ikv::aligned16(p)) return false;
  return true;
}

// Whether all sequences' keys, as many as their tables hold, are so few that reading
// them for each sequence takes less than the launch for the shared ones, whose start
// and joins are some 15 us: 16 heads of 128 over 8, 6 sequences behind 1024 tokens (57
// MB of keys and values) 20.8 us and with the launch 25.4, 48 behind 128 (96 MB) 15.2 and
// 30.7; 6 behind 2048 (105 MB) 28.7 and 25.6, 2 behind 8192 (131 MB) 34.0 and 33.7. The
// host sees the tables' width, not the lengths: short contexts in wide tables take the
// launch.
constexpr int64_t kFewBytes = 96 << 20;
bool few_keys(const ikv::BatchPages &b, int n_head_kv, int head_dim) {
  return static_cast<int64_t>(b.n_seq) * b.capacity <= kFewBytes / (8 * n_head_kv * head_dim);
}

int dims_of(int head_dim) { return (head_dim + 31) / 32 * 32; }

// Row blocks of a workgroup, for the mean rows of a group.
int blocks_of(int64_t n_seq, int64_t n_groups, int G) { return n_seq * G <= 32 * n_groups ? 1 : 2; }

// Slots for the parts, in rows: the items' rows, each group's last chunk in part
// empty (R is at most twice a group's mean rows, or 32), and a run more of each.
constexpr int kMostRows = 64;
int64_t part_rows(int64_t n_seq, int64_t n_groups, int G, int n_head_kv) {
  return (3 * n_seq * G + 32 * n_groups + kMostRows) * n_head_kv + kRuns * kMostRows;
}

// The workspace behind that of the batched decode, in bytes.
struct Space {
  size_t seqs, ml, o, all;
  Space(int64_t n_seq, int64_t n_groups, int n_head, int n_head_kv, int head_dim) {
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    seqs = up(ikv_attn_decode_batch_workspace_bytes(n_head, n_head_kv, head_dim));
    if (head_dim % 8 != 0 || head_dim > 128) {  // the lengths alone
      all = seqs + static_cast<size_t>(n_seq) * sizeof(int32_t);
      return;
    }
    const size_t rows = static_cast<size_t>(part_rows(n_seq, n_groups, n_head / n_head_kv, n_head_kv));
    ml = up(seqs + n_seq * sizeof(ikv::SharedSeq));
    o = up(ml + rows * 2 * sizeof(float));
    all = o + rows * dims_of(head_dim) * sizeof(float);
  }
};

}  // namespace

extern "C" size_t ikv_attn_decode_shared_workspace_bytes(int64_t n_seq, int64_t n_groups, int n_head, int n_head_kv,
                                                         int head_dim) {
  if (ikv_attn_decode_batch_workspace_bytes(n_head, n_head_kv, head_dim) == 0 || n_seq < 0 || n_seq > ikv::kMaxSeqs ||
      n_groups < 0 || n_groups > ikv::kMaxSeqs || n_head > (1 << 29) / std::max<int64_t>(n_seq, 1))
    return 0;
  return Space(n_seq, n_groups, n_head, n_head_kv, head_dim).all;
}

extern "C" int ikv_attn_decode_shared_f32(const float *q, float *k_pool, float *v_pool, const ikv_kv_batch *batch,
                                          const int32_t *group_start, const int32_t *shared_blocks, int64_t n_groups,
                                          const int32_t *n_kv, const float *k_new, const float *v_new, float *out,
                                          int n_head, int n_head_kv, int head_dim, float scale, void *workspace,
                                          size_t workspace_bytes, void *stream) {
  Args a;
  if (const int rc = ikv::batch_arg(batch, a.b)) return rc;
  if (n_groups < 0 || n_head <= 0 || n_head_kv <= 0 || n_head % n_head_kv != 0 || head_dim <= 0) return -EINVAL;
  if (head_dim > 512) return -ENOTSUP;
  if (n_groups > ikv::kMaxSeqs) return -EOVERFLOW;
  const int64_t n_seq = a.b.n_seq;
  if (n_seq == 0) return 0;
  if (!q || !k_pool || !v_pool || !n_kv || !out || (k_new == nullptr) != (v_new == nullptr)) return -EINVAL;
  if (n_groups > 0 && (!group_start || !shared_blocks)) return -EINVAL;
  // a tile's rows are one buffer range; a sequence's heads and all rows index in int
  if (n_head_kv > INT_MAX / (64 * 4) / head_dim || n_head > INT_MAX / head_dim || n_head > (1 << 29) / n_seq)
    return -EOVERFLOW;
  if (!workspace || !ikv::aligned16(workspace) ||
      workspace_bytes < ikv_attn_decode_shared_workspace_bytes(n_seq, n_groups, n_head, n_head_kv, head_dim))
    return -EINVAL;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Space at(n_seq, n_groups, n_head, n_head_kv, head_dim);
  char *const space = static_cast<char *>(workspace);
  a.groups = {group_start, shared_blocks, static_cast<int>(n_groups)};
  if (n_groups == 0 || few_keys(a.b, n_head_kv, head_dim) ||
      !on_matrices(head_dim, {q, k_pool, v_pool, k_new, v_new, out})) {
    int32_t *const keys = reinterpret_cast<int32_t *>(space + at.seqs);
    shared_lengths_kernel<<<(a.b.n_seq + kThreads - 1) / kThreads, kThreads, 0, s>>>(a.b, a.groups, n_kv, keys);
    return ikv_attn_decode_batch_f32(q, k_pool, v_pool, batch, keys, k_new, v_new, out, n_head, n_head_kv, head_dim,
                                     scale, workspace, at.seqs, stream);
  }
  if (!(scale > 0.0f)) scale = 1.0f / sqrtf(static_cast<float>(head_dim));
  a.q = q;
  a.k = k_pool;
  a.v = v_pool;
  a.n_kv = n_kv;
  a.n_head_kv = n_head_kv;
  a.G = n_head / n_head_kv;
  a.dim = head_dim;
  a.scale_log2 = scale * ikv::kLog2e;
  a.seqs = reinterpret_cast<ikv::SharedSeq *>(space + at.seqs);
  a.ml = reinterpret_cast<float *>(space + at.ml);
  a.o = reinterpret_cast<float *>(space + at.o);
  const int rb = blocks_of(n_seq, n_groups, a.G);
  a.slots = static_cast<int>(part_rows(n_seq, n_groups, a.G, n_head_kv) / (32 * rb));
  auto launch = [&](auto dt) {
    if (rb == 1)
      shared_prefix_kernel<dt.value, 1><<<kRuns, kThreads, 0, s>>>(a);
    else
      shared_prefix_kernel<dt.value, 2><<<kRuns, kThreads, 0, s>>>(a);
  };
  const int dims = dims_of(head_dim);
  if (dims == 32)
    launch(std::integral_constant<int, 1>{});
  else if (dims == 64)
    launch(std::integral_constant<int, 2>{});
  else if (dims == 96)
    launch(std::integral_constant<int, 3>{});
  else
    launch(std::integral_constant<int, 4>{});
  if (const int rc = ikv::launch_status()) return rc;
  const ikv::SharedParts parts{a.seqs, a.ml, a.o, 32 * rb, dims, a.slots, n_head_kv};
  return ikv::decode_behind_shared(q, k_pool, v_pool, a.b, k_new, v_new, out, n_head, n_head_kv, head_dim, scale,
                                   workspace, parts, s);
}
