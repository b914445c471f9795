// decode_runs.hpp — one new token of each of several sequences: the contexts, cut
// into units of keys, as runs of equal length over the workgroups of a launch, and
// how the runs' parts of a (sequence, KV head) meet. What holds a unit's keys and
// forms its scores is the kernel's (attn_decode_batch.hip, attn_decode_q8.hip).
#pragma once

#include "batch.hpp"
#include "coherent.hpp"

#include <algorithm>

namespace ikv {

constexpr int kRuns = 8 * 256;  // most runs of units

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

// UNITS: of a run where there are more runs than workgroups (0: there never are);
// WHOLE: units of a (sequence, head) that are not split anywhere; LEAST: of a run, where
// a (sequence, head) has as many on average.
template <class Args, int KT, int GROUPS, int UNITS, int WHOLE, int LEAST = 1>
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
    runs = GROUPS;
    if constexpr (UNITS > 0)
      runs = static_cast<int>(min(max(total / UNITS, static_cast<Units>(GROUPS)), static_cast<Units>(kRuns)));
    chunk = (total + runs - 1) / runs;
    if (chunk == 0) chunk = 1;
    if constexpr (LEAST > 1)
      chunk = max(chunk, min(static_cast<Units>(LEAST), total / (static_cast<Units>(a.b.n_seq) * items)));
    whole = chunk > 1 ? static_cast<int>(min(chunk, static_cast<Units>(4))) + 3 : WHOLE;
  }

  // whether a (sequence, head) of so many units stays with one run: up to WHOLE, and
  // up to three more than a run has where those are two or more and it is no whole
  // number of them (a run of two parts then has two starts and two joins): 16 heads
  // of 128 over 8, 16 contexts of 300 tokens 18.2 -> 13.0 us, 24 of 380, two whole
  // runs each, 18.8 split and 22.5 not; of 200, runs of one unit, 9.8 and 11.3; over
  // ragged lengths between 10 % more and as much less.
  __device__ bool kept(int tiles) const {
    return tiles <= WHOLE || (tiles <= whole && static_cast<unsigned>(tiles) % static_cast<unsigned>(chunk) != 0);
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

__device__ __forceinline__ float weight(float m, float top) {  // of sums kept at maximum m
  return m == -INFINITY ? 0.f : ikv::fast_exp2(m - top);
}

// The workspace: a counter a run (of the parts of the head pass that begins in it
// and goes on behind it) and one of the runs that were fetched, then (maximum,
// sum) of each part's heads and their values. Part 2 r is run r's of a head pass
// that began before it, 2 r + 1 of one that goes on behind it. Stored and read at
// agent scope, as the parts come from several XCDs. RUNS: most runs of the kernel.
constexpr size_t kCounterBytes = sizeof(int) * (kRuns + 64);
template <int GQ, int DP, int RUNS = kRuns>
struct Parts {
  int *counters;  // [kRuns], then the fetched runs'
  float *ml, *o;
  __device__ explicit Parts(float *p)
      : counters(reinterpret_cast<int *>(p)), ml(p + kCounterBytes / sizeof(float)),
        o(ml + static_cast<size_t>(RUNS) * 2 * GQ * 2) {}
  __device__ float *ml_of(int part, int h) const { return ml + (static_cast<size_t>(part) * GQ + h) * 2; }
  __device__ float *o_of(int part, int h) const { return o + (static_cast<size_t>(part) * GQ + h) * DP; }
};

__device__ __forceinline__ float2 load2(const float *p) {
  const unsigned long long x = __hip_atomic_load(reinterpret_cast<const unsigned long long *>(p),
                                                 __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float(static_cast<unsigned>(x)), __uint_as_float(static_cast<unsigned>(x >> 32)));
}

inline size_t parts_bytes(int gq, int dims, int runs = kRuns) {
  return kCounterBytes + static_cast<size_t>(runs) * 2 * gq * (dims + 2) * sizeof(float);
}

// Where the waves of a workgroup meet: each wave's maxima, sums and weighted values.
template <int GQ, int DP, int WAVES>
struct Meet {
  float m[WAVES][GQ], l[WAVES][GQ];
  __attribute__((aligned(16))) float o[WAVES][GQ][DP];
  int last;
};

// The next run that nobody has, at least plan.runs where there is none: the first
// come, first served, so that no workgroup is left with more than a run at the end.
// Every workgroup fetches until there is none, runs times in all; the last fetch
// clears the counter.
template <int GROUPS, class Plan, int GQ, int DP, int WAVES>
__device__ __forceinline__ int next_run(const Plan &plan, const Parts<GQ, DP> &parts, Meet<GQ, DP, WAVES> &s) {
  if (plan.runs <= GROUPS) return plan.runs;
  if (threadIdx.x == 0) {
    int *const fetched = parts.counters + kRuns;
    const int before = __hip_atomic_fetch_add(fetched, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (before == plan.runs - 1) __hip_atomic_store(fetched, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s.last = before;
  }
  __syncthreads();
  const int run = GROUPS + __builtin_amdgcn_readfirstlane(s.last);
  __syncthreads();
  return run;
}

// What a run has of the head pass at p, tiles [p.tile, last) from unit u on, once
// every wave's state is in s (and a barrier behind that): write(head, dim, maximum,
// sum, value, the next dim's value), for every other dim, where that is all of it;
// else the part goes to the workspace, and the workgroup that is counted last joins
// the parts, in their order, and writes.
template <int GQ, int DP, int WAVES, int RUNS, class Plan, class F>
__device__ __forceinline__ void leave(Meet<GQ, DP, WAVES> &s, const Plan &plan, const Parts<GQ, DP, RUNS> &parts,
                                      int run, unsigned long long u, const Place &p, int last, int heads, int dim,
                                      F &&write) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool whole = p.tile == 0 && last == p.tiles;
  const int part = 2 * run + (p.tile == 0 ? 1 : 0);
  for (int i = threadIdx.x; i < heads * DP / 2; i += WAVES * 64) {
    const int h = 2 * i / DP, d = 2 * i % DP;
    float top = s.m[0][h];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, s.m[w][h]);
    float all = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = weight(s.m[w][h], top);
      all = fmaf(f, s.l[w][h], all);
      x = fmaf(f, s.o[w][h][d], x);
      y = fmaf(f, s.o[w][h][d + 1], y);
    }
    if (whole) {
      write(h, d, top, all, x, y);
    } else {
      store2_agent(parts.o_of(part, h) + d, x, y);
      if (d == 0) store2_agent(parts.ml_of(part, h), top, all);
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
      s.last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
      if (s.last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (s.last) {
      auto at = [&](int i) { return i == 0 ? 2 * w0 + 1 : 2 * (w0 + i); };
      for (int h = wave; h < heads; h += WAVES) {
        float top = -INFINITY;
        for (int i = lane; i < n; i += 64) top = fmaxf(top, load2(parts.ml_of(at(i), h)).x);
        top = wave_max(top);
        float all = 0.f;
        for (int i = lane; i < n; i += 64) {
          const float2 ml = load2(parts.ml_of(at(i), h));
          all = fmaf(weight(ml.x, top), ml.y, all);
        }
        all = wave_sum(all);
        if (lane == 0) {
          s.m[0][h] = top;
          s.l[0][h] = all;
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < heads * DP / 2; i += WAVES * 64) {
        const int h = 2 * i / DP, d = 2 * i % DP;
        if (d >= dim) continue;
        const float top = s.m[0][h], all = s.l[0][h];
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
        write(h, d, top, all, x, y);
      }
    }
  }
}

}  // namespace ikv
