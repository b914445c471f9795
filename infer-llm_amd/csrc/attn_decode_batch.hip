// attn_decode_batch.hip — one new token of each of several sequences over a
// paged KV cache (ikv_attn_decode_batch_f32): GQA attention over contexts of
// different lengths, the new rows' append fused.
//
// HBM bounds it: every K and V row is read once and takes 4 G flops a float.
//
//   * The work is cut into units of KT keys of one KV head of one sequence, in
//     the order (sequence, KV head, keys), and these into runs of equal length,
//     from n_kv as it stands on the device: each workgroup adds up the lengths
//     itself. There are as many runs as workgroups, or, where that makes them
//     longer than 16 units, up to four times as many: a workgroup that has done
//     its own takes the next one that is left (with equal shares the last
//     workgroup was done 13 % after the average one).
//   * A run may end inside a (sequence, head): the workgroup then leaves the
//     maximum, sum and weighted values of its part in the workspace (at most
//     two parts a run, so the workspace depends on no length) and counts
//     itself; the one that comes last joins the parts in their order. Nothing
//     waits. A (sequence, head) of few units stays with the run that holds its first
//     one (Plan::kept): joining takes longer than reading that much.
//   * LPK lanes hold a key row, NV 16-byte pieces each, so a wave loads 64 / LPK
//     keys at once; the scores need only the sum over LPK lanes, and each group
//     of LPK lanes has a running maximum and sums of its own, which meet when
//     the run leaves the head. The maximum moves only when a score exceeds it
//     by 2^8.
//   * A sequence's next 64 block table entries are held one per lane; the query
//     rows and the new token's stay in LDS (in registers the four heads of a KV
//     head of 128 spilled).
// Measured (MI355X, us): 48 contexts of up to 16384 tokens, 32 heads of 128 over 8,
// 2.4 GB: 371, 6.6 TB/s; 37 of up to 5003, 12 heads of 64 over 4, 128 MB: 31, of
// which 1 to the first load, 5 to join and for the last workgroup to be done; 3 of
// up to 150 and an idle slot, 16 heads of 128: 10, three units one after the other.
// Query groups of more than 8 read the keys once per 8 heads, each time from behind
// the L2 (FETCH_SIZE of 16 heads 1.9 times that of 8). Groups of 8 and more are far
// from what the reads take: a wave on a SIMD, whose vector instructions are issued in
// 44-49 % of its cycles and which waits in 34-38 %. 32 contexts of up to 5448, 40 MB, 6
// at 6.6 TB/s: 8 heads of 80 over 1 37, 16 over 1 43; of 128, 64 MB, 10: 16 over 1 54,
// 32 over 1 76. Heads of over 128 dims, the same contexts: 8 of 200 over 4, 402 MB, 80
// (61 at that rate), of 256 88 (78), 8 of 512 over 2 102 (78); loads of 4 bytes: 16 of
// 65 over 8, 262 MB, 157 (40).
#include "batch.hpp"
#include "coherent.hpp"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kCUs = 256;       // MI355X compute units
constexpr int kWaves = 4;       // of a workgroup
// Workgroups of a launch: as many as are on the card at once. With 8 query heads
// and more than 64 dims, whose registers leave room for one on a CU, 512 were two
// rounds: 16 heads of 80 over 1, 64 contexts of 380 tokens 33 us, with 256 20; 32 of
// up to 5448 59 and 53.
constexpr int groups_of(int nv, int gq) { return gq > 4 && nv > 2 ? kCUs : 2 * kCUs; }
constexpr int kRuns = 8 * kCUs;  // most runs of units
constexpr int kRunUnits = 16;        // units of a run where there are more runs than workgroups
constexpr float kRescale = 8.0f;  // log2 headroom before the running maximum is moved
constexpr int kMaxDim = 512;
constexpr int kWhole = 3;  // units of a (sequence, head) that are not split anywhere
// Cache policy of a load: rows of the pools are read once (non-temporal: 48 long
// contexts of the 8B heads 410 -> 373 us).
constexpr std::integral_constant<int, 0> kKept{};
constexpr std::integral_constant<int, 2> kOnce{};
constexpr int kAhead = 2;  // keys of a lane group loaded at once

struct Args {
  const float *q;
  float *k, *v;
  const float *k_new, *v_new;
  float *out;
  const int32_t *n_kv;
  ikv::BatchPages b;
  int n_head_kv, G, dim;
  int passes;  // a KV head's query heads are taken GQ at a time
  float scale_log2;
  float *part;
};

// Keys of a sequence; 0 for an idle slot and for a length that is out of range.
__device__ __forceinline__ int keys_of(const Args &a, int seq) {
  const int n = a.n_kv[seq];
  return n > 0 && n <= a.b.capacity ? n : 0;
}

__device__ __forceinline__ unsigned long long wave_prefix(unsigned long long x) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const unsigned long long y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  return x;
}

// x of lane l (the same for the whole wave), in scalar registers.
__device__ __forceinline__ unsigned long long lane_value(unsigned long long x, int l) {
  const unsigned lo = __builtin_amdgcn_readlane(static_cast<unsigned>(x), l);
  const unsigned hi = __builtin_amdgcn_readlane(static_cast<unsigned>(x >> 32), l);
  return static_cast<unsigned long long>(hi) << 32 | lo;
}

// A place in the list of units: unit `tile` of `tiles` of head pass `item`.
struct Place {
  int seq, keys, tiles, item, tile;
};

template <int KT, int GROUPS>
struct Plan {
  using Units = unsigned long long;
  Units total, chunk;  // all units, those of a run
  int runs, whole;
  unsigned items;  // head passes of a sequence
  // the sequence s0 + lane of 64: its keys, and the units up to its end
  int s0, keys;
  Units upto;

  __device__ static int tiles_of(int keys) { return (keys + KT - 1) / KT; }

  __device__ void look(const Args &a, int first, Units before) {
    const int s = first + static_cast<int>(threadIdx.x & 63);
    s0 = first;
    keys = s < a.b.n_seq ? keys_of(a, s) : 0;
    upto = before + wave_prefix(static_cast<Units>(tiles_of(keys)) * items);
  }

  __device__ Plan(const Args &a) : items(a.n_head_kv * a.passes) {
    total = 0;
    for (int s = 0; s < a.b.n_seq; s += 64) {
      look(a, s, total);
      total = lane_value(upto, 63);
    }
    runs = static_cast<int>(min(max(total / kRunUnits, static_cast<Units>(GROUPS)), static_cast<Units>(kRuns)));
    chunk = (total + runs - 1) / runs;
    if (chunk == 0) chunk = 1;
    whole = chunk > 1 ? static_cast<int>(min(chunk, static_cast<Units>(4))) + 3 : kWhole;
  }

  // whether a (sequence, head) of so many units stays with one run: up to kWhole, and
  // up to three more than a run has where those are two or more and it is no whole
  // number of them (a run of two parts then has two starts and two joins): 16 heads
  // of 128 over 8, 16 contexts of 300 tokens 18.2 -> 13.0 us, 24 of 380, two whole
  // runs each, 18.8 split and 22.5 not; of 200, runs of one unit, 9.8 and 11.3; over
  // ragged lengths between 10 % more and as much less.
  __device__ bool kept(int tiles) const {
    return tiles <= kWhole || (tiles <= whole && static_cast<unsigned>(tiles) % static_cast<unsigned>(chunk) != 0);
  }

  // where unit u (< total) is
  __device__ Place at(const Args &a, Units u) {
    if (a.b.n_seq > 64) {
      Units before = 0;
      for (int s = 0; s < a.b.n_seq; s += 64) {
        look(a, s, before);
        before = lane_value(upto, 63);
        if (before > u) break;
      }
    }
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > u));
    Place p;
    p.seq = s0 + l;
    p.keys = __builtin_amdgcn_readlane(keys, l);
    p.tiles = tiles_of(p.keys);
    const Units r = u - (lane_value(upto, l) - static_cast<Units>(p.tiles) * items);
    if (r >> 32) {
      p.item = static_cast<int>(r / p.tiles);
      p.tile = static_cast<int>(r % p.tiles);
    } else {
      p.item = static_cast<int>(static_cast<unsigned>(r) / p.tiles);
      p.tile = static_cast<int>(static_cast<unsigned>(r) % p.tiles);
    }
    p.item = __builtin_amdgcn_readfirstlane(p.item);
    p.tile = __builtin_amdgcn_readfirstlane(p.tile);
    return p;
  }

  // the first unit of the next head pass
  __device__ void next(const Args &a, Place &p) {
    p.tile = 0;
    if (++p.item < static_cast<int>(items)) return;
    p.item = 0;
    const int lane = threadIdx.x & 63;
    for (int first = s0;; first += 64) {
      if (first != s0) {
        if (first >= a.b.n_seq) return;  // (behind the last sequence: nobody goes on)
        look(a, first, 0);               // (upto is not asked again)
      }
      const unsigned long long some = __builtin_amdgcn_ballot_w64(keys > 0 && first + lane > p.seq);
      if (some) {
        const int l = __builtin_ctzll(some);
        p.seq = first + l;
        p.keys = __builtin_amdgcn_readlane(keys, l);
        p.tiles = tiles_of(p.keys);
        return;
      }
    }
  }
};

template <int LPK>
__device__ __forceinline__ float lanes_sum(float x) {  // over a key's lanes
  x += ikv::dpp<ikv::kDppXor1>(x);
  x += ikv::dpp<ikv::kDppXor2>(x);
  x += ikv::dpp<ikv::kDppHalfMirror>(x);
  if constexpr (LPK >= 16) x += ikv::dpp<ikv::kDppMirror>(x);
  if constexpr (LPK >= 32) {
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(b[0]) + __uint_as_float(b[1]);
  }
  return x;
}

constexpr int kDppRor8 = 0x128;  // lane i <-> i ^ 8 within 16 lanes

// f over the lanes that hold the same dims of the wave's keys
template <int LPK, class F>
__device__ __forceinline__ float across_keys(float x, F &&f) {
  if constexpr (LPK <= 8) x = f(x, ikv::dpp<kDppRor8>(x));
  if constexpr (LPK <= 16) {
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(b[0]), __uint_as_float(b[1]));
  }
  const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(c[0]), __uint_as_float(c[1]));
}

__device__ __forceinline__ float weight(float m, float top) {  // of sums kept at maximum m
  return m == -INFINITY ? 0.f : ikv::fast_exp2(m - top);
}

// The workspace: a counter a run (of the parts of the head pass that begins in it
// and goes on behind it) and one of the runs that were fetched, then (maximum,
// sum) of each part's heads and their values. Part 2 r is run r's of a head pass
// that began before it, 2 r + 1 of one that goes on behind it. Stored and read at agent scope, as
// the parts come from several XCDs.
constexpr size_t kCounterBytes = sizeof(int) * (kRuns + 64);
template <int GQ, int DP>
struct Parts {
  int *counters;  // [kRuns], then the fetched runs'
  float *ml, *o;
  __device__ explicit Parts(float *p)
      : counters(reinterpret_cast<int *>(p)), ml(p + kCounterBytes / sizeof(float)),
        o(ml + static_cast<size_t>(kRuns) * 2 * GQ * 2) {}
  __device__ float *ml_of(int part, int h) const { return ml + (static_cast<size_t>(part) * GQ + h) * 2; }
  __device__ float *o_of(int part, int h) const { return o + (static_cast<size_t>(part) * GQ + h) * DP; }
};

__device__ __forceinline__ float2 load2(const float *p) {
  const unsigned long long x = __hip_atomic_load(reinterpret_cast<const unsigned long long *>(p),
                                                 __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float(static_cast<unsigned>(x)), __uint_as_float(static_cast<unsigned>(x >> 32)));
}

template <int LPK, int NV, int GQ, bool VEC>
__global__ __launch_bounds__(kWaves * 64, GQ <= 4 ? 2 : 1) void decode_batch_kernel(Args a) {
  constexpr int KPW = 64 / LPK;               // keys that a wave loads at once
  constexpr int KT = kWaves * kAhead * KPW;   // keys of a unit
  constexpr int DP = LPK * NV * 4;            // dims held
  static_assert(64 % KT == 0, "a unit stays within a block");
  __shared__ float s_m[kWaves][GQ], s_l[kWaves][GQ];
  __shared__ __attribute__((aligned(16))) float s_o[kWaves][GQ][DP];
  __shared__ float4 s_q[GQ][NV][LPK];  // the query rows, scaled
  __shared__ float4 s_new[2][NV][LPK];  // the new token's K and V row
  __shared__ int s_last;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane % LPK, grp = lane / LPK;
  const int n_head = a.n_head_kv * a.G;
  const int stride = a.n_head_kv * a.dim;  // floats of a token row

  // slots without keys: a zero row, and the flag where the length is no length
  // (from the last workgroups on: in a small call they have nothing else to do)
  for (int s = gridDim.x - 1 - blockIdx.x; s < a.b.n_seq; s += gridDim.x) {
    if (keys_of(a, s) > 0) continue;
    if (a.n_kv[s] != 0 && threadIdx.x == 0) ikv::raise_status(a.b.status, IKV_STATUS_POSITION);
    float *o = a.out + static_cast<size_t>(s) * n_head * a.dim;
    for (int d = threadIdx.x; d < n_head * a.dim; d += kWaves * 64) o[d] = 0.f;
  }

  constexpr int kGroups = groups_of(NV, GQ);
  Plan<KT, kGroups> plan(a);
  const Parts<GQ, DP> parts(a.part);
  unsigned off[NV];  // of this lane's pieces in a row; out of range past head_dim
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int d = 4 * (l + LPK * n);
    off[n] = d < a.dim ? static_cast<unsigned>(d) * 4 : 0x80000000u;
  }
  // piece n of the row at `at`
  auto load = [&]<int POLICY>(__amdgpu_buffer_rsrc_t r, unsigned at, int n, std::integral_constant<int, POLICY>) -> float4 {
    if constexpr (VEC) {
      return __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(r, at + off[n], 0, POLICY));
    } else {
      const int d = 4 * (l + LPK * n);
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
                                             r, d + e < a.dim ? at + (d + e) * 4u : 0x80000000u, 0, POLICY));
      return make_float4(x[0], x[1], x[2], x[3]);
    }
  };
  auto whole_row = [&](const float *row) {  // a row of head_dim floats on its own
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(row), 0, a.dim * 4, ikv::kBufWord3);
  };
  auto store = [&](float *row, int n, float4 x) {
    const int d = 4 * (l + LPK * n);
    if constexpr (VEC) {
      if (d < a.dim) *reinterpret_cast<float4 *>(row + d) = x;
    } else {
      const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < a.dim) row[d + e] = y[e];
    }
  };

  int run = blockIdx.x;
  unsigned long long u = plan.chunk * run, end = min(plan.total, u + plan.chunk);
  Place p{};
  if (u < end) p = plan.at(a, u);
  for (;;) {
    if (u >= end) {
      // the next run that nobody has: the first come, first served, so that no
      // workgroup is left with more than a run at the end. Every workgroup fetches
      // until there is none, runs times in all; the last fetch clears the counter.
      if (plan.runs <= kGroups) return;
      if (threadIdx.x == 0) {
        int *const fetched = parts.counters + kRuns;
        const int before = __hip_atomic_fetch_add(fetched, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (before == plan.runs - 1) __hip_atomic_store(fetched, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = before;
      }
      __syncthreads();
      run = kGroups + __builtin_amdgcn_readfirstlane(s_last);
      __syncthreads();
      if (run >= plan.runs) return;
      u = plan.chunk * run;
      end = min(plan.total, u + plan.chunk);
      if (u < end) p = plan.at(a, u);
      continue;
    }
    // the run's part of one (sequence, KV head, pass): tiles [p.tile, last)
    if (plan.kept(p.tiles) && p.tile > 0) {  // (with the run that holds its first unit)
      u += p.tiles - p.tile;
      plan.next(a, p);
      continue;
    }
    const int last =
        plan.kept(p.tiles) ? p.tiles : static_cast<int>(min<unsigned long long>(p.tiles, p.tile + (end - u)));
    const int g = p.item / a.passes, h0 = p.item % a.passes * GQ;
    const int heads = min(GQ, a.G - h0);
    const ikv::Pages pg = ikv::pages_of(a.b, p.seq);
    const size_t head0 = static_cast<size_t>(p.seq) * n_head + g * a.G + h0;
    float4 o[GQ][NV];
    float m[GQ], sum[GQ];
#pragma unroll
    for (int h = 0; h < GQ; ++h) {
      m[h] = -INFINITY;
      sum[h] = 0.f;
#pragma unroll
      for (int n = 0; n < NV; ++n) o[h][n] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // the query rows, a head a wave (to LDS once the first keys are on their way)
    constexpr int kHeads = (GQ + kWaves - 1) / kWaves;
    float4 qr[kHeads][NV];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const int h = min(wave + kWaves * i, heads - 1);
#pragma unroll
      for (int n = 0; n < NV; ++n) qr[i][n] = load(whole_row(a.q + (head0 + h) * a.dim), 0, n, kKept);
    }
    // and, where the run has the last keys, the new rows by the last two waves
    const bool has_new = a.k_new != nullptr && last == p.tiles;
    float4 fresh[NV];
    if (has_new && wave >= kWaves - 2) {
      const float *row = (wave == kWaves - 2 ? a.k_new : a.v_new) + static_cast<size_t>(p.seq) * stride + g * a.dim;
#pragma unroll
      for (int n = 0; n < NV; ++n) fresh[n] = load(whole_row(row), 0, n, kKept);
    }
    // block table entries, 64 at a time, one per lane, checked as they are read
    const int last_blk = (p.keys - 1) / pg.bt;
    int blk = p.tile * KT / pg.bt, in_blk = p.tile * KT % pg.bt, ent0 = blk, ent = 0;
    auto entries = [&]() {
      ent0 = blk;
      ent = pg.table[min(blk + lane, last_blk)];
      if (static_cast<unsigned>(ent) >= static_cast<unsigned>(pg.n_blocks)) {
        ikv::raise_status(pg.status, IKV_STATUS_BLOCK);
        ent = -1;
      }
    };
    entries();
    float4 kr[kAhead][NV], vr[kAhead][NV];
    const int mine = wave * kAhead * KPW + grp;  // this lane's first key of a unit, then + KPW
    // row of the tile at (blk, in_blk), moved on to the next tile; ~row of
    // block 0's where the entry names no block
    auto next_row = [&]() -> long long {
      const int e = __builtin_amdgcn_readlane(ent, blk - ent0);
      const long long row = e < 0 ? ~static_cast<long long>(in_blk) : static_cast<long long>(e) * pg.bt + in_blk;
      in_blk += KT;
      if (in_blk == pg.bt) {
        in_blk = 0;
        if (++blk - ent0 >= 64) entries();
      }
      return row;
    };
    const int cached = p.keys - (a.k_new ? 1 : 0);  // keys that are read from the pools
    // (a tile behind the run: no memory is read)
    auto fetch = [&](const float *pool, long long row, int tile, float4 (&x)[kAhead][NV]) {
      const int rows = tile < last ? min(KT, cached - tile * KT) : 0;
      const auto r = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<float *>(pool + (row < 0 ? ~row : row) * stride + g * a.dim), 0,
          rows > 0 ? ((rows - 1) * stride + a.dim) * 4 : 0, ikv::kBufWord3);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int n = 0; n < NV; ++n)
          x[i][n] = load(r, static_cast<unsigned>(mine + KPW * i) * stride * 4u, n, kOnce);
    };
    // this lane's scores of N rows of pieces with each head
    auto scores = [&]<int N>(const float4 (&x)[N][NV], float (&s)[N][GQ]) {
#pragma unroll
      for (int h = 0; h < GQ; ++h) {
        float y[N] = {};
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          const float4 w = s_q[h][n][l];
#pragma unroll
          for (int i = 0; i < N; ++i) y[i] += ikv::dot4(w, x[i][n]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) s[i][h] = lanes_sum<LPK>(y[i]);
      }
    };
    auto raise = [&]<int N>(const float (&s)[N][GQ]) {  // the maxima to these scores', if need be
      bool move = false;
#pragma unroll
      for (int h = 0; h < GQ; ++h)
#pragma unroll
        for (int i = 0; i < N; ++i) move |= s[i][h] > m[h] + kRescale;
      if (__builtin_amdgcn_ballot_w64(move) == 0) return;
#pragma unroll
      for (int h = 0; h < GQ; ++h) {
        float top = m[h];
#pragma unroll
        for (int i = 0; i < N; ++i) top = fmaxf(top, s[i][h]);
        const float f = weight(m[h], top);
        m[h] = top;
        sum[h] *= f;
#pragma unroll
        for (int n = 0; n < NV; ++n) o[h][n] = ikv::scale4(f, o[h][n]);
      }
    };
    auto add_values = [&]<int N>(const float (&s)[N][GQ], const float4 (&x)[N][NV]) {
#pragma unroll
      for (int h = 0; h < GQ; ++h) {
        const float ref = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float w = ikv::fast_exp2(s[i][h] - ref);
          sum[h] += w;
#pragma unroll
          for (int n = 0; n < NV; ++n) o[h][n] = ikv::fma4(w, x[i][n], o[h][n]);
        }
      }
    };

    long long row = next_row();
    fetch(a.k, row, p.tile, kr);
    fetch(a.v, row, p.tile, vr);
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (wave + kWaves * i < GQ && grp == 0) {
#pragma unroll
        for (int n = 0; n < NV; ++n) s_q[wave + kWaves * i][n][l] = ikv::scale4(a.scale_log2, qr[i][n]);
      }
    if (has_new && wave >= kWaves - 2 && grp == 0) {
#pragma unroll
      for (int n = 0; n < NV; ++n) s_new[wave - (kWaves - 2)][n][l] = fresh[n];
    }
    __syncthreads();
    for (int t = p.tile; t < last; ++t) {
      asm volatile("" ::: "memory");  // the query rows stay in LDS
      float s[kAhead][GQ];
      scores(kr, s);
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (t * KT + mine + KPW * i >= cached) {
#pragma unroll
          for (int h = 0; h < GQ; ++h) s[i][h] = -INFINITY;
        }
      const long long here = row;
      row = next_row();
      fetch(a.k, row, t + 1, kr);
      raise(s);
      add_values(s, vr);
      fetch(a.v, row, t + 1, vr);
      if (has_new && t + 1 == p.tiles) {
        // the new token, by the first wave's first lanes, and its place in the pools
        float4 kn[1][NV], vn[1][NV];
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          kn[0][n] = s_new[0][n][l];
          vn[0][n] = s_new[1][n][l];
        }
        float sn[1][GQ];
        scores(kn, sn);
        if (wave != 0 || grp != 0) {
#pragma unroll
          for (int h = 0; h < GQ; ++h) sn[0][h] = -INFINITY;
        }
        raise(sn);
        // (a weight of 0 would not silence what is not finite)
        if (wave == 0 && grp == 0) {
          add_values(sn, vn);
          if (here >= 0 && h0 == 0) {
            const long long to = (here + cached - t * KT) * stride + g * a.dim;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
              store(a.k + to, n, kn[0][n]);
              store(a.v + to, n, vn[0][n]);
            }
          }
        }
      }
    }

    // the lane groups and the waves meet
#pragma unroll
    for (int h = 0; h < GQ; ++h) {
      __builtin_amdgcn_sched_barrier(0);
      const float top = across_keys<LPK>(m[h], [](float x, float y) { return fmaxf(x, y); });
      const float f = weight(m[h], top);
      auto add = [](float x, float y) { return x + y; };
      const float all = across_keys<LPK>(sum[h] * f, add);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const float4 x = ikv::scale4(f, o[h][n]);
        const float4 y = make_float4(across_keys<LPK>(x.x, add), across_keys<LPK>(x.y, add),
                                     across_keys<LPK>(x.z, add), across_keys<LPK>(x.w, add));
        if (grp == 0) *reinterpret_cast<float4 *>(&s_o[wave][h][4 * (l + LPK * n)]) = y;
      }
      if (lane == 0) {
        s_m[wave][h] = top;
        s_l[wave][h] = all;
      }
    }
    __syncthreads();
    const bool whole = p.tile == 0 && last == p.tiles;
    const int part = 2 * run + (p.tile == 0 ? 1 : 0);
    for (int i = threadIdx.x; i < heads * DP / 2; i += kWaves * 64) {
      const int h = 2 * i / DP, d = 2 * i % DP;
      float top = s_m[0][h];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_m[w][h]);
      float all = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = weight(s_m[w][h], top);
        all = fmaf(f, s_l[w][h], all);
        x = fmaf(f, s_o[w][h][d], x);
        y = fmaf(f, s_o[w][h][d + 1], y);
      }
      if (whole) {
        float *const o = a.out + (head0 + h) * a.dim + d;
        if (d < a.dim) o[0] = x / all;
        if (d + 1 < a.dim) o[1] = y / all;
      } else {
        ikv::store2_agent(parts.o_of(part, h) + d, x, y);
        if (d == 0) ikv::store2_agent(parts.ml_of(part, h), top, all);
      }
    }
    if (!whole) {
      // this thread's stores have completed before the workgroup is counted
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      __builtin_amdgcn_s_waitcnt(0);
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      __syncthreads();
      // the head pass's first unit, its first run, its runs
      const unsigned long long begin = u - p.tile;
      const int w0 = static_cast<int>(begin / plan.chunk);
      const int n = static_cast<int>((begin + p.tiles - 1) / plan.chunk) - w0 + 1;
      if (threadIdx.x == 0) {
        int *const counter = parts.counters + w0;
        s_last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
        if (s_last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (s_last) {
        auto at = [&](int i) { return i == 0 ? 2 * w0 + 1 : 2 * (w0 + i); };
        for (int h = wave; h < heads; h += kWaves) {
          float top = -INFINITY;
          for (int i = lane; i < n; i += 64) top = fmaxf(top, load2(parts.ml_of(at(i), h)).x);
          top = ikv::wave_max(top);
          float all = 0.f;
          for (int i = lane; i < n; i += 64) {
            const float2 ml = load2(parts.ml_of(at(i), h));
            all = fmaf(weight(ml.x, top), ml.y, all);
          }
          all = ikv::wave_sum(all);
          if (lane == 0) {
            s_m[0][h] = top;
            s_l[0][h] = all;
          }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < heads * DP / 2; i += kWaves * 64) {
          const int h = 2 * i / DP, d = 2 * i % DP;
          if (d >= a.dim) continue;
          const float top = s_m[0][h], all = s_l[0][h];
          float x = 0.f, y = 0.f;
          constexpr int kParts = 8;  // loaded at once
          for (int j = 0; j < n; j += kParts) {
            float2 ml[kParts], v[kParts];
#pragma unroll
            for (int z = 0; z < kParts; ++z) {
              const int e = at(min(j + z, n - 1));
              ml[z] = load2(parts.ml_of(e, h));
              v[z] = load2(parts.o_of(e, h) + d);
            }
#pragma unroll
            for (int z = 0; z < kParts; ++z) {
              const float f = j + z < n ? weight(ml[z].x, top) : 0.f;
              if (j + z < n) {
                x = fmaf(f, v[z].x, x);
                y = fmaf(f, v[z].y, y);
              }
            }
          }
          float *const o = a.out + (head0 + h) * a.dim + d;
          o[0] = x / all;
          if (d + 1 < a.dim) o[1] = y / all;
        }
      }
    }
    __syncthreads();
    u += last - p.tile;
    plan.next(a, p);
  }
}

// The form of a shape: lanes per key and 16-byte pieces of a lane (head_dim up
// to 16 LPK NV / 4), query heads taken at once.
struct Form {
  int lpk, nv, gq;
};
Form form_of(int G, int dim) {
  Form f;
  f.lpk = dim <= 128 ? 8 : dim <= 256 ? 16 : 32;
  f.nv = dim <= 128 ? (dim + 31) / 32 : 4;
  f.gq = G <= 1 ? 1 : G <= 2 ? 2 : G <= 4 ? 4 : 8;
  return f;
}

template <int LPK, int NV, int GQ>
int launch(const Args &a, bool vec, hipStream_t s) {
  if (vec)
    decode_batch_kernel<LPK, NV, GQ, true><<<groups_of(NV, GQ), kWaves * 64, 0, s>>>(a);
  else
    decode_batch_kernel<LPK, NV, GQ, false><<<groups_of(NV, GQ), kWaves * 64, 0, s>>>(a);
  return ikv::launch_status();
}

}  // namespace

extern "C" size_t ikv_attn_decode_batch_workspace_bytes(int n_head, int n_head_kv, int head_dim) {
  if (n_head <= 0 || n_head_kv <= 0 || n_head % n_head_kv != 0 || head_dim <= 0 || head_dim > kMaxDim) return 0;
  const Form f = form_of(n_head / n_head_kv, head_dim);
  return kCounterBytes + static_cast<size_t>(kRuns) * 2 * f.gq * (f.lpk * f.nv * 4 + 2) * sizeof(float);
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
  const int G = n_head / n_head_kv;
  const Form f = form_of(G, head_dim);
  if (!(scale > 0.0f)) scale = 1.0f / sqrtf(static_cast<float>(head_dim));
  a.q = q;
  a.k = k_pool;
  a.v = v_pool;
  a.k_new = k_new;
  a.v_new = v_new;
  a.out = out;
  a.n_kv = n_kv;
  a.n_head_kv = n_head_kv;
  a.G = G;
  a.dim = head_dim;
  a.passes = (G + f.gq - 1) / f.gq;
  a.scale_log2 = scale * ikv::kLog2e;
  a.part = static_cast<float *>(workspace);
  bool vec = head_dim % 4 == 0;
  for (const void *x : {static_cast<const void *>(q), static_cast<const void *>(k_pool),
                        static_cast<const void *>(v_pool), static_cast<const void *>(k_new),
                        static_cast<const void *>(v_new)})
    vec = vec && ikv::aligned16(x);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define IKV_GQ(LPK, NV)                                 \
  switch (f.gq) {                                       \
    case 1: return launch<LPK, NV, 1>(a, vec, s);       \
    case 2: return launch<LPK, NV, 2>(a, vec, s);       \
    case 4: return launch<LPK, NV, 4>(a, vec, s);       \
    default: return launch<LPK, NV, 8>(a, vec, s);      \
  }
  if (f.lpk == 32) IKV_GQ(32, 4)
  if (f.lpk == 16) IKV_GQ(16, 4)
  if (f.nv == 4) IKV_GQ(8, 4)
  if (f.nv == 3) IKV_GQ(8, 3)
  if (f.nv == 2) IKV_GQ(8, 2)
  IKV_GQ(8, 1)
#undef IKV_GQ
}
