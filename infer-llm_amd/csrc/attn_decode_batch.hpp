// attn_decode_batch.hpp — one new token of each of several sequences over a paged KV
// cache: GQA attention over contexts of different lengths, the new rows' append fused.
// Of all of a sequence's keys (attn_decode_batch.hip) or of those behind the ones that
// it shares (attn_decode_own.hip).
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
#pragma once

#include "decode_runs.hpp"
#include "decode_shared.hpp"

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
constexpr int kRunUnits = 16;        // units of a run where there are more runs than workgroups
constexpr float kRescale = 8.0f;  // log2 headroom before the running maximum is moved
constexpr int kMaxDim = 512;
constexpr int kWhole = 3;  // units of a (sequence, head) that are not split anywhere
// The same behind shared keys, where most sequences have few units of their own and a
// (sequence, head) costs its start and its join, whatever it holds: runs of two units,
// taken as workgroups come free (48 sequences of up to 1500 keys of their own, 32 heads
// of 128, 52.6 -> 39.5 us; 37 of up to 511, heads of 64, 14.1, runs of one workgroup's
// share or of two; five units whole 15.6 there).
constexpr int kSharedUnits = 2, kSharedWhole = 4;
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

// With the first keys of each sequence attended to already (decode_shared.hpp): what
// is read here is behind them.
struct SharedArgs : Args {
  ikv::SharedParts shared;
};
__device__ __forceinline__ int keys_of(const SharedArgs &a, int seq) { return a.shared.seqs[seq].keys; }

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

template <int LPK, int NV, int GQ, bool VEC, class A>
__global__ __launch_bounds__(kWaves * 64, GQ <= 4 ? 2 : 1) void decode_batch_kernel(A a) {
  constexpr bool SHARED = std::is_same_v<A, SharedArgs>;
  constexpr int KPW = 64 / LPK;               // keys that a wave loads at once
  constexpr int KT = kWaves * kAhead * KPW;   // keys of a unit
  constexpr int DP = LPK * NV * 4;            // dims held
  static_assert(64 % KT == 0, "a unit stays within a block");
  __shared__ ikv::Meet<GQ, DP, kWaves> s_meet;
  __shared__ float4 s_q[GQ][NV][LPK];  // the query rows, scaled
  __shared__ float4 s_new[2][NV][LPK];  // the new token's K and V row
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane % LPK, grp = lane / LPK;
  const int n_head = a.n_head_kv * a.G;
  const int stride = a.n_head_kv * a.dim;  // floats of a token row

  // slots without keys: a zero row, and the flag where the length is no length
  // (from the last workgroups on: in a small call they have nothing else to do)
  for (int s = gridDim.x - 1 - blockIdx.x; s < a.b.n_seq; s += gridDim.x) {
    if (keys_of(a, s) > 0) continue;
    if constexpr (!SHARED)  // (there the launch before has flagged it)
      if (a.n_kv[s] != 0 && threadIdx.x == 0) ikv::raise_status(a.b.status, IKV_STATUS_POSITION);
    float *o = a.out + static_cast<size_t>(s) * n_head * a.dim;
    for (int d = threadIdx.x; d < n_head * a.dim; d += kWaves * 64) o[d] = 0.f;
  }

  constexpr int kGroups = groups_of(NV, GQ);
  ikv::Plan<A, KT, kGroups, SHARED ? kSharedUnits : kRunUnits, SHARED ? kSharedWhole : kWhole> plan(a);
  const ikv::Parts<GQ, DP> parts(a.part);
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
  ikv::Place p{};
  if (u < end) p = plan.at(a, u);
  for (;;) {
    if (u >= end) {
      run = ikv::next_run<kGroups>(plan, parts, s_meet);
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
    ikv::Pages pg = ikv::pages_of(a.b, p.seq);
    ikv::SharedSeq behind;
    if constexpr (SHARED) {
      behind = a.shared.seqs[p.seq];
      pg.table += behind.shared / pg.bt;
    }
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
        const float f = ikv::weight(m[h], top);
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
      const float f = ikv::weight(m[h], top);
      auto add = [](float x, float y) { return x + y; };
      const float all = across_keys<LPK>(sum[h] * f, add);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        const float4 x = ikv::scale4(f, o[h][n]);
        const float4 y = make_float4(across_keys<LPK>(x.x, add), across_keys<LPK>(x.y, add),
                                     across_keys<LPK>(x.z, add), across_keys<LPK>(x.w, add));
        if (grp == 0) *reinterpret_cast<float4 *>(&s_meet.o[wave][h][4 * (l + LPK * n)]) = y;
      }
      if (lane == 0) {
        s_meet.m[wave][h] = top;
        s_meet.l[wave][h] = all;
      }
    }
    __syncthreads();
    ikv::leave(s_meet, plan, parts, run, u, p, last, heads, a.dim, [&](int h, int d, float top, float all, float x, float y) {
      float *const o = a.out + (head0 + h) * a.dim + d;
      if constexpr (SHARED) {
        if (d >= a.dim) return;
        const ikv::SharedRow row(a.shared, behind, g, h0 + h);
        *reinterpret_cast<float2 *>(o) = ikv::join_shared(a.shared, row, d, top, all, x, y);
        return;
      }
      if (d < a.dim) o[0] = x / all;
      if (d + 1 < a.dim) o[1] = y / all;
    });
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
template <int LPK, int NV, int GQ>
int launch(const SharedArgs &a, bool, hipStream_t s) {
  decode_batch_kernel<LPK, NV, GQ, true><<<groups_of(NV, GQ), kWaves * 64, 0, s>>>(a);
  return ikv::launch_status();
}

template <int LPK, int NV, class A>
int launch_heads(const A &a, int gq, bool vec, hipStream_t s) {
  switch (gq) {
    case 1: return launch<LPK, NV, 1>(a, vec, s);
    case 2: return launch<LPK, NV, 2>(a, vec, s);
    case 4: return launch<LPK, NV, 4>(a, vec, s);
    default: return launch<LPK, NV, 8>(a, vec, s);
  }
}
// (up to 128 dims)
template <class A>
int launch_narrow(const A &a, const Form &f, bool vec, hipStream_t s) {
  if (f.nv == 4) return launch_heads<8, 4>(a, f.gq, vec, s);
  if (f.nv == 3) return launch_heads<8, 3>(a, f.gq, vec, s);
  if (f.nv == 2) return launch_heads<8, 2>(a, f.gq, vec, s);
  return launch_heads<8, 1>(a, f.gq, vec, s);
}

void set_args(Args &a, const float *q, float *k_pool, float *v_pool, const int32_t *n_kv, const float *k_new,
              const float *v_new, float *out, int n_head, int n_head_kv, int head_dim, float scale, void *workspace) {
  const int G = n_head / n_head_kv, gq = form_of(G, head_dim).gq;
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
  a.passes = (G + gq - 1) / gq;
  a.scale_log2 = scale * ikv::kLog2e;
  a.part = static_cast<float *>(workspace);
}

}  // namespace
