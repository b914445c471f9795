// sample.hip — the next token of each row of logits from a given uniform number
// (ikv_sample_f32): temperature, top-k, top-p, min-p.
//
// With y_i = (x_i - max) / T and w_i = exp(y_i), in the order of descending x
// (ties by index): the first top_k tokens are kept, of them the shortest start
// whose mass reaches top_p of theirs, of it the tokens with y_i >= ln(min_p);
// all three keep a start of the order. The token is the first whose running
// mass exceeds u times the kept mass.
//
// A running mass next to a border decides a token, so masses are exact integers:
// w_i is computed in double and rounded once to a multiple of 2^-S, S so large
// that a row's sum stays below 2^63 (44 for 151936 tokens; a token lighter than
// 2^-45 of the heaviest weighs nothing). Sums of integers do not depend on their
// order, so histograms may be filled by atomics and results repeat bit for bit.
//
// The row is not sorted. Its tokens are put into 2048 bins by value, with each
// bin's mass and, where top_k asks, count; the bins' running sums say which bins
// hold the borders (nearly always one for each), the tokens of those are sorted
// and give the borders, and the token, exactly. Where they are too many for that
// (equal logits by the thousand, as a rule), the borders are found by radix
// selection in one workgroup instead: 11 bits of a value's place in the order a
// round, three rounds to one value, whose tokens weigh the same, so that what is
// left is a division.
//
// Measured (MI355X, us): one row of 151936 18-24 (three launches of 4, 7 and 13: each
// a chain of loads, sums over the workgroup and atomics of 1 us; the row itself is
// read in 0.1), 48 rows 46 (8, 16, 23: the weights in double, LDS atomics at 25
// cycles a wave, and the last workgroup's sums), 200 rows of 8191, each held in one
// workgroup's registers, 17. All logits equal, 151936 of them, with top_p: 410 (one
// workgroup goes over the row nine times), 48 such rows 640.
#include "../../include/ikv_model.h"
#include "ikv_common.hpp"

#include <algorithm>

namespace {

constexpr int kThreads = 512;
constexpr int kBits = 11, kBins = 1 << kBits;  // of a round

struct Args {
  const float *logits;
  const float *u, *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p;
  int n;
  int shift;  // S
  int32_t *token;
  float *logprob;
};

// 2^f for |f| <= 1/2 by its Taylor series, f ln2 <= 0.3466: the term left out
// is below 0.3466^13 / 13! = 2^-52.4.
__device__ double exp2_series(double f) {
  const double z = f * 0.69314718055994530942;
  double r = 1.0 / 479001600.0;
  r = fma(r, z, 1.0 / 39916800.0);
  r = fma(r, z, 1.0 / 3628800.0);
  r = fma(r, z, 1.0 / 362880.0);
  r = fma(r, z, 1.0 / 40320.0);
  r = fma(r, z, 1.0 / 5040.0);
  r = fma(r, z, 1.0 / 720.0);
  r = fma(r, z, 1.0 / 120.0);
  r = fma(r, z, 1.0 / 24.0);
  r = fma(r, z, 1.0 / 6.0);
  r = fma(r, z, 0.5);
  r = fma(r, z, 1.0);
  return fma(r, z, 1.0);
}

constexpr int kPowers = 64;

// 2^(j / 64) for j < 64, in LDS: 2^t is one of them, a power of two and 2^g with
// |g| <= 1/128, whose series needs five terms.
__device__ void fill_powers(double *powers) {
  const int j = threadIdx.x;
  if (j < kPowers / 2)
    powers[j] = exp2_series(j * (1.0 / kPowers));
  else if (j < kPowers)
    powers[j] = 2.0 * exp2_series(j * (1.0 / kPowers) - 1.0);
}

// A row as its workgroup sees it.
struct Row {
  const float *x;
  int n;
  float top;     // the largest logit
  double per_t;  // log2(e) / T
  double shift;  // S
  const double *powers;

  // w in multiples of 2^-S; the largest logit's is 2^S. The same bits wherever it
  // is inlined (the sums of one launch and the tokens of another have to agree),
  // so nothing is left to contraction. Without branches: the tokens of a thread
  // go through it side by side. The series' rest is below (ln2 / 128)^6 / 6! =
  // 2^-54.6.
  __device__ __forceinline__ unsigned long long weight(float v) const {
#pragma clang fp contract(off)
    const double t = (static_cast<double>(v) - static_cast<double>(top)) * per_t;
    const double moved = t + 0x1.8p46;  // a multiple of 1/64, its count in the low bits
    const double g = t - (moved - 0x1.8p46);
    const int k = static_cast<int>(__builtin_bit_cast(long long, moved));
    double r = fma(g, 1.3333558146428443e-3, 9.6181291076284772e-3);
    r = fma(r, g, 5.5504108664821580e-2);
    r = fma(r, g, 2.4022650695910072e-1);
    r = fma(r, g, 6.9314718055994531e-1);
    r = fma(r, g, 1.0);
    // times 2^(k / 64 + S), rounded to an integer: the bits of the sum with 2^52
    uint2 power = __builtin_bit_cast(uint2, powers[k & (kPowers - 1)]);
    power.y += static_cast<unsigned>((k >> 6) + static_cast<int>(shift)) << 20;
    const uint2 sum = __builtin_bit_cast(uint2, fma(r, __builtin_bit_cast(double, power), 0x1p52));
    const unsigned long long w = static_cast<unsigned long long>(sum.y & 0xfffffu) << 32 | sum.x;
    return t > -(shift + 2.0) ? w : 0;
  }
};

// Place of a logit in the order: smaller for larger ones, the same for -0 and 0.
__device__ __forceinline__ unsigned order_of(float v) {
  const unsigned b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? b : ~b & 0x7fffffffu;
}

// Inclusive prefix sums over the workgroup's threads, in thread order.
__device__ unsigned long long block_prefix(unsigned long long v, unsigned long long *s_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const unsigned long long y = __shfl_up(v, o, 64);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 63) s_wave[wave] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64 - 1; ++w) {  // (all read at once)
    const unsigned long long y = s_wave[w];
    if (w < wave) v += y;
  }
  return v;
}

// The tokens of a workgroup: x[begin, end), read anew at each pass, eight loads of
// a thread in flight.
struct Chunked {
  const float *x;
  int begin, end;
  // f(logit, index, g(logit)): g of eight tokens side by side, then f of each
  template <class G, class F>
  __device__ __forceinline__ void each(G &&g, F &&f) const {
    constexpr int kAhead = 8;
    for (int i = begin + static_cast<int>(threadIdx.x); i < end; i += kAhead * kThreads) {
      float v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) v[j] = i + j * kThreads < end ? x[i + j * kThreads] : 0.0f;
      decltype(g(0.0f)) y[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) y[j] = g(v[j]);
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (i + j * kThreads < end) f(v[j], i + j * kThreads, y[j]);
    }
  }
};

// Up to N * kThreads tokens, kept in registers.
template <int N>
struct Held {
  float v[N];
  int n;
  __device__ Held(const float *x, int n) : n(n) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = threadIdx.x + j * kThreads;
      v[j] = i < n ? x[i] : 0.0f;
    }
  }
  template <class G, class F>
  __device__ __forceinline__ void each(G &&g, F &&f) const {
#pragma unroll
    for (int j0 = 0; j0 < N; j0 += 8) {
      decltype(g(0.0f)) y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = g(v[j0 + j]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = threadIdx.x + (j0 + j) * kThreads;
        if (i < n) f(v[j0 + j], i, y[j]);
      }
    }
  }
};

__device__ __forceinline__ Chunked tokens_of(const Row &row) { return {row.x, 0, row.n}; }

// Tokens one by one for rows of equal logits by the thousand: a weight is computed
// where a logit differs from the thread's last one, and a thread's tokens of one
// bin that come one behind the other go there together (an atomic of 64 lanes at
// one address takes 64 turns). One row of 151936 equal ones 1650 to 410 us; for
// other rows it costs more than it gives (48 of them 49 to 59 us in fill_bins).
struct Run {
  unsigned long long *mass;
  unsigned *count;
  float x = NAN;
  unsigned long long each = 0;  // x's weight
  int bin = 0;
  unsigned n = 0;
  unsigned long long w = 0;
  __device__ __forceinline__ unsigned long long weight(const Row &row, float v) {
    if (v != x) {
      x = v;
      each = row.weight(v);
    }
    return each;
  }
  __device__ __forceinline__ void flush() {
    if (n == 0) return;
    atomicAdd(&mass[bin], w);
    atomicAdd(&count[bin], n);
  }
  __device__ __forceinline__ void add(const Row &row, int b, float v) {
    if (b != bin) {
      flush();
      bin = b;
      n = 0;
      w = 0;
    }
    ++n;
    w += weight(row, v);
  }
};

struct Shared {
  unsigned count[kBins];
  unsigned long long mass[kBins];
  unsigned long long wave[kThreads / 64];
  unsigned long long found[3];  // bin, count before it, mass before it
  float top[kThreads / 64];
  int bad;
};

// Where the border lies: tokens of one value, `equal` of them of `each` mass, and
// what comes before them.
struct Spot {
  unsigned order;
  unsigned long long count, mass;
  unsigned equal;
  unsigned long long each;
};

enum class Border { kCount, kMass };

// The first value at which the running count or mass reaches `border`; the last
// one where none does.
template <Border B>
__device__ Spot select(const Row &row, Shared &s, unsigned long long border) {
  Spot r{};
  int left = 32;  // bits of the order not yet fixed
  const int tid = threadIdx.x;
  for (int round = 0; round < 3; ++round) {
    const int bits = left < kBits ? left : kBits;
    for (int b = tid; b < kBins; b += kThreads) {
      s.count[b] = 0;
      s.mass[b] = 0;
    }
    if (tid == 0) s.found[0] = kBins;
    __syncthreads();
    Run run{s.mass, s.count};
    tokens_of(row).each([](float) { return 0; }, [&](float x, int, int) {
      const unsigned o = order_of(x);
      if (round > 0 && (o >> left) != r.order) return;
      run.add(row, static_cast<int>((o >> (left - bits)) & ((1u << bits) - 1)), x);
    });
    run.flush();
    __syncthreads();
    constexpr int kPer = kBins / kThreads;
    unsigned long long c = 0, m = 0;
    int last = -1;  // of this thread's bins that hold tokens
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int b = tid * kPer + j;
      c += s.count[b];
      m += s.mass[b];
      if (s.count[b]) last = b;
    }
    const unsigned long long first_c = r.count + block_prefix(c, s.wave) - c;
    const unsigned long long first_m = r.mass + block_prefix(m, s.wave) - m;
    unsigned long long upto_c = first_c, upto_m = first_m;
    for (int b = tid * kPer; b < (tid + 1) * kPer; ++b) {
      upto_c += s.count[b];
      upto_m += s.mass[b];
      if (s.count[b] && (B == Border::kCount ? upto_c : upto_m) >= border) {
        atomicMin(&s.found[0], static_cast<unsigned long long>(b));
        break;
      }
    }
    __syncthreads();
    if (s.found[0] == kBins) {  // none does: the last bin that holds tokens
      __syncthreads();
      if (tid == 0) s.found[0] = 0;
      __syncthreads();
      if (last >= 0) atomicMax(&s.found[0], static_cast<unsigned long long>(last));
      __syncthreads();
    }
    const int bin = static_cast<int>(s.found[0]);
    if (bin / kPer == tid) {
      upto_c = first_c, upto_m = first_m;
      for (int b = tid * kPer; b < bin; ++b) {
        upto_c += s.count[b];
        upto_m += s.mass[b];
      }
      s.found[1] = upto_c;
      s.found[2] = upto_m;
    }
    __syncthreads();
    r.count = s.found[1];
    r.mass = s.found[2];
    r.equal = s.count[bin];
    r.each = s.mass[bin];
    left -= bits;
    r.order = (r.order << bits) | static_cast<unsigned>(bin);
    __syncthreads();
  }
  r.each /= r.equal;
  return r;
}

// The fewest of a value's tokens with which the running mass reaches `border`.
__device__ __forceinline__ unsigned long long tokens_to(const Spot &b, unsigned long long border) {
  if (b.each == 0 || border <= b.mass) return 1;
  return min((border - b.mass + b.each - 1) / b.each, static_cast<unsigned long long>(b.equal));
}

// Sum of the weights of the tokens for which f holds.
template <class F>
__device__ unsigned long long mass_of(const Row &row, Shared &s, F &&f) {
  unsigned long long m = 0;
  Run run{};
  tokens_of(row).each([](float) { return 0; }, [&](float x, int, int) {
    if (f(x)) m += run.weight(row, x);
  });
  m = block_prefix(m, s.wave);
  __syncthreads();
  if (threadIdx.x == kThreads - 1) s.found[0] = m;
  __syncthreads();
  m = s.found[0];
  __syncthreads();
  return m;
}

// Index of the rank-th (from 1) token of a value, in index order: each wave counts
// those of its part of the row, and the wave that has it goes over its part again.
__device__ int index_of(const Row &row, Shared &s, unsigned order, unsigned long long rank) {
  constexpr int kWaves = kThreads / 64, kAhead = 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per = (row.n + kWaves - 1) / kWaves, begin = min(row.n, wave * per), end = min(row.n, begin + per);
  // f(index of lane 0's token, the lanes whose token it is) until it returns true
  auto scan = [&](auto &&f) {
    for (int i0 = begin; i0 < end; i0 += 64 * kAhead) {
      float v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) v[j] = i0 + j * 64 + lane < end ? row.x[i0 + j * 64 + lane] : 0.0f;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const bool is = i0 + j * 64 + lane < end && order_of(v[j]) == order;
        if (f(i0 + j * 64, __builtin_amdgcn_ballot_w64(is))) return;
      }
    }
  };
  unsigned long long own = 0;
  scan([&](int, unsigned long long is) {
    own += __popcll(is);
    return false;
  });
  if (lane == 0) s.wave[wave] = own;
  if (threadIdx.x == 0) s.found[0] = row.n - 1;
  __syncthreads();
  unsigned long long before = 0;
  for (int w = 0; w < wave; ++w) before += s.wave[w];
  if (before < rank && before + own >= rank) {
    scan([&](int i, unsigned long long is) {
      const unsigned long long upto = before + __popcll(is);
      if (upto < rank) {
        before = upto;
        return false;
      }
      const bool mine = (is >> lane & 1) && before + __popcll(is & ((2ull << lane) - 1)) == rank;
      if (mine) s.found[0] = i + lane;
      return true;
    });
  }
  __syncthreads();
  const int at = static_cast<int>(s.found[0]);
  __syncthreads();
  return at;
}

// A row's parameters.
struct Cuts {
  float t, p, low, u;
  int k;
  double floor;  // ln(min_p)

  __device__ Cuts(const Args &a, int r) {
    t = a.temperature ? a.temperature[r] : 1.0f;
    k = a.top_k ? a.top_k[r] : 0;
    p = a.top_p ? a.top_p[r] : 1.0f;
    low = a.min_p ? a.min_p[r] : 0.0f;
    u = a.u[r];
    floor = low > 0.0f ? log(static_cast<double>(low)) : 0.0;
  }
  __device__ bool bad() const { return !(t < INFINITY) || p != p || low != low || u != u; }
  __device__ bool passes(float x, float top) const {  // min_p
    return (static_cast<double>(x) - static_cast<double>(top)) / static_cast<double>(t) >= floor;
  }
};

// top_p of a mass, as the border that a running mass reaches: an integer, as it
// is (one at least, so that the first token does not fail it).
__device__ __forceinline__ unsigned long long share_of(unsigned long long mass, float p) {
  const double need = ceil(static_cast<double>(fmaxf(p, 0.0f)) * static_cast<double>(mass));
  return max(static_cast<unsigned long long>(need), 1ull);
}

// The drawn place in a mass; a running mass exceeds it where it reaches the next
// integer.
__device__ __forceinline__ unsigned long long drawn_of(unsigned long long mass, float u) {
  u = fminf(fmaxf(u, 0.0f), 0x1.fffffep-1f);
  return static_cast<unsigned long long>(static_cast<double>(u) * static_cast<double>(mass)) + 1;
}

__device__ void refuse(const Args &a, int r) {
  a.token[r] = -1;
  if (a.logprob) a.logprob[r] = __int_as_float(0x7fc00000);
}

__device__ void answer(const Args &a, int r, int token, float x, const Row &row, const Cuts &c,
                       unsigned long long kept) {
  a.token[r] = token;
  const double y = (static_cast<double>(x) - static_cast<double>(row.top)) / static_cast<double>(c.t);
  if (a.logprob)
    a.logprob[r] = static_cast<float>(y - log(ldexp(static_cast<double>(kept), -a.shift)));
}

// The whole of a row by radix selection.
__device__ void select_row(const Args &a, int r, const Row &row, const Cuts &c, Shared &s) {
  unsigned long long kept;
  if (c.k > 0 && c.k < a.n) {
    const Spot b = select<Border::kCount>(row, s, static_cast<unsigned long long>(c.k));
    kept = b.mass + (c.k - b.count) * b.each;
  } else {
    kept = mass_of(row, s, [](float) { return true; });
  }
  if (c.p < 1.0f) {
    const unsigned long long need = share_of(kept, c.p);
    const Spot b = select<Border::kMass>(row, s, need);
    kept = min(kept, b.mass + tokens_to(b, need) * b.each);
  }
  if (c.low > 0.0f) kept = min(kept, mass_of(row, s, [&](float x) { return c.passes(x, row.top); }));
  kept = max(kept, row.weight(row.top));
  const unsigned long long target = drawn_of(kept, c.u);
  const Spot b = select<Border::kMass>(row, s, target);
  const int at = index_of(row, s, b.order, tokens_to(b, target));
  if (threadIdx.x == 0) answer(a, r, at, row.x[at], row, c, kept);
}

// The bins of a row by value, the largest logits first: the window is what can
// weigh anything, or the row's range where that is smaller, in equal parts.
struct Window {
  float top, scale;
  __device__ Window(const Row &row, float low, float t) : top(row.top) {
    const float width = fminf(row.top - low, t * static_cast<float>((row.shift + 2.0) * 0.69314718055994530942));
    scale = width > 0.0f ? fminf(static_cast<float>(kBins) / width, 3.4e38f) : 0.0f;
  }
  // (monotone: a difference and a product, each rounded once)
  __device__ int bin(float x) const { return static_cast<int>(fminf((top - x) * scale, kBins - 1.0f)); }
};

constexpr int kList = 2048;  // tokens of a row that are looked at one by one
constexpr int kMaxChunks = 64;

// The bins that hold the borders (top_k's, top_p's, min_p's, the draw's; hi < lo:
// none). A border is known to a bin's mass before the ones ahead of it are looked
// at, so a range of bins may have to be: nearly always one.
struct Ranges {
  int lo[4], hi[4];
  unsigned long long total, before_m;  // all mass, and that before min_p's bins
  bool has_k;

  __device__ bool holds(int b) const {
    bool in = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) in |= b >= lo[j] && b <= hi[j];
    return in;
  }
};

// What a row's workgroups hand on: the largest and smallest finite logit of
// each chunk and the first index of the largest, the bins, the list.
struct Chunk {
  float top, low;
  int at, bad;
};
struct RowSpace {
  unsigned long long mass[kBins];
  unsigned long long list[kList];
  unsigned count[kBins];
  unsigned listed, arrived;
  Chunk chunk[kMaxChunks];
};

struct Lists {
  unsigned long long mass[kBins + 1];  // before each bin
  unsigned long long list[kList];      // (order, index) of a token
  unsigned count[kBins + 1];
  unsigned long long wave[kThreads / 64];
  unsigned long long kept_k, kept_p, kept_m;
  int spot[5];
  int n, last;
};

struct Extremes {
  float top[kThreads / 64], low[kThreads / 64];
  int at[kThreads / 64];
  int bad;
};

union Space {
  Shared select;
  Lists l;
};

// The largest logit, its first index, the smallest finite one.
template <class Tokens>
__device__ Chunk extremes(const Tokens &tokens, Extremes &l) {
  Chunk c{-INFINITY, INFINITY, INT_MAX, 0};
  auto take = [&](float v, int i, int) {
    c.bad |= !(v < INFINITY);
    if (v > c.top) c.top = v, c.at = i;
    if (v > -INFINITY) c.low = fminf(c.low, v);
  };
  tokens.each([](float) { return 0; }, take);
  const float top = ikv::wave_max(c.top);
  int at = c.top == top ? c.at : INT_MAX;
  for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
  const float low = -ikv::wave_max(-c.low);
  if (threadIdx.x == 0) l.bad = 0;
  __syncthreads();
  if (c.bad) l.bad = 1;  // benign race: every writer stores 1
  if ((threadIdx.x & 63) == 0) {
    l.top[threadIdx.x >> 6] = top;
    l.low[threadIdx.x >> 6] = low;
    l.at[threadIdx.x >> 6] = at;
  }
  __syncthreads();
  c = Chunk{-INFINITY, INFINITY, INT_MAX, l.bad};
  for (int w = 0; w < kThreads / 64; ++w) {
    if (l.top[w] > c.top || (l.top[w] == c.top && l.at[w] < c.at)) c.top = l.top[w], c.at = l.at[w];
    c.low = fminf(c.low, l.low[w]);
  }
  return c;
}

// Masses (and, for top_k, counts) of the tokens into l's bins. Tokens that weigh
// nothing are in none: they come last and move no border.
template <class Tokens>
__device__ void fill_bins(const Row &row, const Window &win, bool counts, const Tokens &tokens, Lists &l) {
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    l.mass[b] = 0;
    l.count[b] = 0;
  }
  __syncthreads();
  tokens.each([&](float x) { return row.weight(x); }, [&](float x, int, unsigned long long w) {
    if (w == 0) return;
    const int b = win.bin(x);
    atomicAdd(&l.mass[b], w);
    if (counts) atomicAdd(&l.count[b], 1u);
  });
  __syncthreads();
}

// l's bins to what comes before each, and the bins of the borders.
__device__ Ranges find_ranges(const Row &row, const Window &win, const Cuts &c, Lists &l) {
  constexpr int kPer = kBins / kThreads;
  unsigned long long m[kPer + 1], sum_m = 0;  // before this thread's bins, and behind the last
  unsigned n[kPer + 1], sum_n = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    sum_m += m[j + 1] = l.mass[threadIdx.x * kPer + j];
    sum_n += n[j + 1] = l.count[threadIdx.x * kPer + j];
  }
  m[0] = block_prefix(sum_m, l.wave) - sum_m;
  const bool counts = c.k > 0 && c.k < row.n;
  n[0] = counts ? static_cast<unsigned>(block_prefix(sum_n, l.wave)) - sum_n : 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    l.mass[threadIdx.x * kPer + j] = m[j];
    l.count[threadIdx.x * kPer + j] = n[j];
    m[j + 1] += m[j];
    n[j + 1] += n[j];
  }
  if (threadIdx.x == kThreads - 1) {
    l.mass[kBins] = m[kPer];
    l.count[kBins] = n[kPer];
  }
  if (threadIdx.x < 5) l.spot[threadIdx.x] = kBins - 1;
  __syncthreads();
  // the bin in which a running mass or count reaches a border, to l.spot
  auto find = [&](const auto *before, auto border, int to) {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (before[j] < border && before[j + 1] >= border) l.spot[to] = threadIdx.x * kPer + j;
  };
  Ranges r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.lo[j] = 1, r.hi[j] = 0;
  r.total = l.mass[kBins];
  unsigned long long least = r.total, most = r.total;  // of the kept mass
  r.has_k = counts && static_cast<unsigned>(c.k) < l.count[kBins];
  if (r.has_k) {
    find(n, static_cast<unsigned>(c.k), 0);
    __syncthreads();
    r.lo[0] = r.hi[0] = l.spot[0];
    least = l.mass[r.lo[0]];
    most = l.mass[r.lo[0] + 1];
  }
  if (c.p < 1.0f) {
    find(m, share_of(least, c.p), 1);
    find(m, share_of(most, c.p), 2);
    __syncthreads();
    r.lo[1] = l.spot[1];
    r.hi[1] = l.spot[2];
    least = min(least, l.mass[r.lo[1]]);
    most = min(most, l.mass[r.hi[1] + 1]);
  }
  r.before_m = 0;
  if (c.low > 0.0f) {
    const double move = static_cast<double>(c.t) * c.floor, at = row.top + move;
    const double slack = 1e-12 * (fabs(static_cast<double>(row.top)) + fabs(move));
    auto edge = [&](double x, float way) {
      const float f = static_cast<float>(x);
      return f < INFINITY && f > -INFINITY ? nextafterf(f, way) : f;
    };
    // (a min_p of more than 1 is past the largest logit, perhaps past all floats: a
    // window of no width would put that into its last bin)
    r.lo[2] = win.bin(fminf(edge(at + slack, INFINITY), row.top));
    r.hi[2] = win.bin(fminf(edge(at - slack, -INFINITY), row.top));
    r.before_m = l.mass[r.lo[2]];
    least = min(least, r.before_m);
    most = min(most, l.mass[r.hi[2] + 1]);
  }
  const unsigned long long heaviest = row.weight(row.top);
  find(m, drawn_of(max(least, heaviest), c.u), 3);
  find(m, drawn_of(max(most, heaviest), c.u), 4);
  __syncthreads();
  r.lo[3] = l.spot[3];
  r.hi[3] = l.spot[4];
  return r;
}

// The tokens of those bins into l's list (l.n may pass kList: then not all).
template <class Tokens>
__device__ void gather(const Row &row, const Window &win, const Ranges &rg, const Tokens &tokens, Lists &l) {
  if (threadIdx.x == 0) l.n = 0;
  __syncthreads();
  tokens.each([&](float x) { return rg.holds(win.bin(x)); }, [&](float x, int i, bool in) {
    if (!in || row.weight(x) == 0) return;
    const int at = atomicAdd(&l.n, 1);
    if (at < kList) l.list[at] = static_cast<unsigned long long>(order_of(x)) << 32 | static_cast<unsigned>(i);
  });
  __syncthreads();
}

// l's list by order, then index; no two entries are equal.
__device__ void sort_list(int n, Lists &l) {
  const int tid = threadIdx.x;
  if (n <= kThreads) {  // each entry's place is the number of smaller ones
    const unsigned long long mine = tid < n ? l.list[tid] : 0;
    int at = 0;
    if ((tid & ~63) < n) {
#pragma unroll 8
      for (int i = 0; i < n; ++i) at += l.list[i] < mine;
    }
    __syncthreads();
    if (tid < n) l.list[at] = mine;
    __syncthreads();
    return;
  }
  int size = 2 * kThreads;  // bitonic
  while (size < n) size *= 2;
  for (int i = n + tid; i < size; i += kThreads) l.list[i] = ~0ull;
  __syncthreads();
  for (int k = 2; k <= size; k *= 2) {
    for (int j = k / 2; j > 0; j /= 2) {
      for (int p = tid; p < size / 2; p += kThreads) {
        const int i = 2 * p - (p & (j - 1)), o = i + j;
        const unsigned long long x = l.list[i], y = l.list[o];
        if ((x > y) == ((i & k) == 0)) {
          l.list[i] = y;
          l.list[o] = x;
        }
      }
      __syncthreads();
    }
  }
}

// The token, from the bins' sums and the whole list (n <= kList tokens of it).
__device__ void resolve(const Args &a, int r, const Row &row, const Window &win, const Cuts &c, const Ranges &rg,
                        int n, Lists &l) {
  const int tid = threadIdx.x;
  if (tid == 0) {
    l.kept_k = rg.total;
    l.kept_p = ~0ull;
    l.kept_m = rg.before_m;
  }
  sort_list(n, l);
  // running masses and counts: a bin's tokens are all in the list, one behind
  // the other, so a token's are its bin's and those of the list since the bin's
  // first one. Each border has one token: no atomics (64-bit ones of a few
  // hundred lanes on one address took 20 us).
  constexpr int kPer = kList / kThreads;
  unsigned long long w[kPer], m[kPer], own = 0;  // a token's weight, the running mass with it
  float x[kPer];
  int bin[kPer];
  auto logit = [&](int i) {
    const unsigned o = static_cast<unsigned>(l.list[i] >> 32);
    return __uint_as_float((o & 0x80000000u) ? o : ~o & 0x7fffffffu);
  };
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = tid * kPer + j;
    w[j] = 0;
    if (i < n) {
      x[j] = logit(i);
      bin[j] = win.bin(x[j]);
      w[j] = row.weight(x[j]);
    }
    own += w[j];
  }
  unsigned long long run = block_prefix(own, l.wave) - own;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = tid * kPer + j;
    if (i < n && (i == 0 || win.bin(logit(i - 1)) != bin[j])) {  // the bin's first: nobody else's
      l.mass[bin[j]] -= run;
      l.count[bin[j]] -= static_cast<unsigned>(i);
    }
    run += w[j];
    m[j] = run;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = tid * kPer + j;
    if (i >= n) continue;
    m[j] += l.mass[bin[j]];
    if (rg.has_k && bin[j] == rg.lo[0] && l.count[bin[j]] + i + 1 == static_cast<unsigned>(c.k)) l.kept_k = m[j];
    if (c.low > 0.0f && c.passes(x[j], row.top) && (i + 1 == n || !c.passes(logit(i + 1), row.top)))
      l.kept_m = max(rg.before_m, m[j]);
  }
  __syncthreads();
  unsigned long long kept = l.kept_k;
  if (c.p < 1.0f) {
    const unsigned long long need = share_of(kept, c.p);
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (m[j] >= need && m[j] - w[j] < need && w[j] != 0) l.kept_p = m[j];
    __syncthreads();
    kept = min(kept, l.kept_p);
  }
  if (c.low > 0.0f) kept = min(kept, l.kept_m);
  kept = max(kept, row.weight(row.top));
  const unsigned long long target = drawn_of(kept, c.u);
#pragma unroll
  for (int j = 0; j < kPer; ++j)  // (a token that is not in the list weighs nothing)
    if (m[j] >= target && m[j] - w[j] < target && w[j] != 0)
      answer(a, r, static_cast<int>(static_cast<unsigned>(l.list[tid * kPer + j])), x[j], row, c, kept);
}

__device__ Row row_of(const Args &a, int r, const Cuts &c, float top, const double *powers) {
  return Row{a.logits + static_cast<size_t>(r) * a.n, a.n, top,
             1.4426950408889634074 / static_cast<double>(c.t), static_cast<double>(a.shift), powers};
}

// Whether a row needs no sums; its answer where `write`.
__device__ bool settled(const Args &a, int r, const Cuts &c, const Chunk &e, bool write) {
  if (e.bad || c.bad() || e.top == -INFINITY) {
    if (write) refuse(a, r);
    return true;
  }
  if (c.t <= 0.0f) {
    if (write) {
      a.token[r] = e.at;
      if (a.logprob) a.logprob[r] = 0.0f;
    }
    return true;
  }
  return false;
}

// A workgroup a row.
template <class Tokens>
__device__ void sample_row(const Args &a, int r, const Cuts &c, const Tokens &tokens, Space &s) {
  __shared__ Extremes x;
  __shared__ double powers[kPowers];
  fill_powers(powers);  // (a barrier follows)
  const Chunk e = extremes(tokens, x);
  if (settled(a, r, c, e, threadIdx.x == 0)) return;
  const Row row = row_of(a, r, c, e.top, powers);
  const Window win(row, e.low, c.t);
  fill_bins(row, win, c.k > 0 && c.k < a.n, tokens, s.l);
  const Ranges rg = find_ranges(row, win, c, s.l);
  gather(row, win, rg, tokens, s.l);
  const int n = s.l.n;
  if (n <= kList) {
    resolve(a, r, row, win, c, rg, n, s.l);
  } else {
    __syncthreads();
    select_row(a, r, row, c, s.select);
  }
}

constexpr int kHeld = 16;  // tokens of a thread that are kept in registers

__global__ __launch_bounds__(kThreads) void sample_held_kernel(Args a) {
  __shared__ Space s;
  const int r = blockIdx.x;
  const Held<kHeld> tokens(a.logits + static_cast<size_t>(r) * a.n, a.n);
  sample_row(a, r, Cuts(a, r), tokens, s);
}

__global__ __launch_bounds__(kThreads) void sample_row_kernel(Args a) {
  __shared__ Space s;
  const int r = blockIdx.x;
  sample_row(a, r, Cuts(a, r), Chunked{a.logits + static_cast<size_t>(r) * a.n, 0, a.n}, s);
}

// Several workgroups a row, in three launches. The first: each chunk's extremes,
// and the row's sums cleared.
__device__ __forceinline__ Chunked chunk_of(const Args &a) {
  const int per = (a.n + gridDim.x - 1) / gridDim.x;
  const int begin = min(a.n, static_cast<int>(blockIdx.x) * per);
  return Chunked{a.logits + static_cast<size_t>(blockIdx.y) * a.n, begin, min(a.n, begin + per)};
}

__global__ __launch_bounds__(kThreads) void sample_extremes_kernel(Args a, RowSpace *rows) {
  __shared__ Extremes l;
  const int r = blockIdx.y;
  RowSpace &w = rows[r];
  for (int b = blockIdx.x * kThreads + threadIdx.x; b < kBins; b += gridDim.x * kThreads) {
    w.mass[b] = 0;
    w.count[b] = 0;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) w.listed = w.arrived = 0;
  const Chunk e = extremes(chunk_of(a), l);
  if (threadIdx.x == 0) w.chunk[blockIdx.x] = e;
}

__device__ Chunk row_extremes(const RowSpace &w, int chunks) {
  const int lane = threadIdx.x & 63;
  const Chunk mine = lane < chunks ? w.chunk[lane] : Chunk{-INFINITY, INFINITY, INT_MAX, 0};
  Chunk e;
  e.top = ikv::wave_max(mine.top);
  e.low = -ikv::wave_max(-mine.low);
  e.bad = __builtin_amdgcn_ballot_w64(mine.bad != 0) != 0;
  const unsigned long long at = __builtin_amdgcn_ballot_w64(lane < chunks && mine.top == e.top);
  e.at = at ? __shfl(mine.at, __builtin_ctzll(at), 64) : 0;  // (a row of -inf has bits, too)
  return e;
}

// Whether this workgroup is the last of its row's to come here; what the others
// stored (agent scope) before they came is then there.
__device__ bool last_of_row(unsigned *counter, int *s_last) {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0);  // this thread's stores and atomics have completed
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
  if (threadIdx.x == 0)
    *s_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  __syncthreads();
  return *s_last != 0;
}

template <class T>
__device__ __forceinline__ T load_agent(const T *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The second: the bins.
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(Args a, RowSpace *rows) {
  __shared__ Lists l;
  __shared__ double powers[kPowers];
  fill_powers(powers);  // (a barrier follows)
  const int r = blockIdx.y;
  RowSpace &w = rows[r];
  const Cuts c(a, r);
  const Chunk e = row_extremes(w, gridDim.x);
  if (settled(a, r, c, e, blockIdx.x == 0 && threadIdx.x == 0)) return;
  const Row row = row_of(a, r, c, e.top, powers);
  const Window win(row, e.low, c.t);
  const bool counts = c.k > 0 && c.k < a.n;
  fill_bins(row, win, counts, chunk_of(a), l);
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    if (l.mass[b] == 0) continue;
    atomicAdd(&w.mass[b], l.mass[b]);
    if (counts) atomicAdd(&w.count[b], l.count[b]);
  }
}

// The third: the bins of the borders, by each workgroup for itself (by the one that
// came last with the bins, and read anew here: one row 28.4 us instead of 24.4), their
// tokens, and by the workgroup that comes last the answer.
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(Args a, RowSpace *rows) {
  __shared__ Space s;
  __shared__ double powers[kPowers];
  fill_powers(powers);  // (a barrier follows)
  Lists &l = s.l;
  const int r = blockIdx.y, tid = threadIdx.x;
  RowSpace &w = rows[r];
  const Cuts c(a, r);
  const Chunk e = row_extremes(w, gridDim.x);
  if (settled(a, r, c, e, false)) return;
  const Row row = row_of(a, r, c, e.top, powers);
  const Window win(row, e.low, c.t);
  for (int b = tid; b < kBins; b += kThreads) {
    l.mass[b] = w.mass[b];
    l.count[b] = w.count[b];
  }
  __syncthreads();
  const Ranges rg = find_ranges(row, win, c, l);
  gather(row, win, rg, chunk_of(a), l);
  if (tid == 0 && l.n > 0) l.last = static_cast<int>(atomicAdd(&w.listed, static_cast<unsigned>(l.n)));
  __syncthreads();
  const unsigned first = static_cast<unsigned>(l.last);
  for (int i = tid; i < min(l.n, kList); i += kThreads)
    if (first + i < kList)
      __hip_atomic_store(&w.list[first + i], l.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (!last_of_row(&w.arrived, &l.last)) return;
  const unsigned n = load_agent(&w.listed);
  if (n <= kList) {
    for (unsigned i = tid; i < n; i += kThreads) l.list[i] = load_agent(&w.list[i]);
    __syncthreads();
    resolve(a, r, row, win, c, rg, static_cast<int>(n), l);
  } else {
    __syncthreads();
    select_row(a, r, row, c, s.select);
  }
}

// Workgroups of a row: one up to 16384 tokens, or 32768 where there are 64 rows or
// more; else as many as bring all rows to kGroups, of 2048 tokens at least (one
// where there are many rows). One against several, in three launches (us): 1 row of
// 16385 22.5, 20.5, of 32768 33.5, 19.8; 16 rows of 16385 23.2, 22.7, of 24576 28.6,
// 23.7; 64 rows of 16385 23.3, 32.7, of 32768 34.7, 33.6, of 49152 47.0, 36.9; 200
// rows of 32768 35.6, 44.1, of 65536 67.9, 64.4. kGroups 256 and 1024: 48 rows of
// 151936 56.9 and 58.7 against 49.4; at most 32 workgroups: one row 29.8 against 28.0.
constexpr int kRowTokens = 16384, kRowsTokens = 32768, kManyRows = 64, kGroups = 512;
int chunks_of(int64_t n_rows, int64_t n_vocab) {
  if (n_vocab <= (n_rows < kManyRows ? kRowTokens : kRowsTokens)) return 1;
  const int64_t most = std::max<int64_t>(1, kGroups / n_rows);
  return static_cast<int>(std::min<int64_t>({most, (n_vocab + 2047) / 2048, kMaxChunks}));
}

}  // namespace

extern "C" size_t ikv_sample_workspace_bytes(int64_t n_rows, int64_t n_vocab) {
  if (n_rows <= 0 || n_vocab <= 0) return 0;
  // (enough for fewer rows, too, of which each has more workgroups)
  return n_vocab <= kRowTokens ? 256 : std::min<size_t>(n_rows, kGroups / 2) * sizeof(RowSpace);
}

extern "C" int ikv_sample_f32(const float *logits, const float *u, const float *temperature,
                              const int32_t *top_k, const float *top_p, const float *min_p, int64_t n_rows,
                              int64_t n_vocab, int32_t *token, float *logprob, void *workspace,
                              size_t workspace_bytes, void *stream) {
  if (n_rows < 0 || n_vocab < 1) return -EINVAL;
  if (n_rows == 0) return 0;
  if (!logits || !u || !token || !workspace || !ikv::aligned16(workspace)) return -EINVAL;
  if (n_vocab > (1 << 30) || n_rows > (1 << 21)) return -EOVERFLOW;
  if (workspace_bytes < ikv_sample_workspace_bytes(n_rows, n_vocab)) return -EINVAL;
  int bits = 0;  // of the count: a row's masses stay below 2^63
  while ((int64_t{1} << bits) < n_vocab) ++bits;
  const Args a{logits, u, temperature, top_k, top_p, min_p, static_cast<int>(n_vocab), std::min(62 - bits, 51),
               token, logprob};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int chunks = chunks_of(n_rows, n_vocab);
  if (chunks == 1) {
    // tokens in registers where they are many and each row has a CU: 200 rows of 8192
    // 15.8 us against 17.0, of 4096 15.0 against 13.7, 300 rows of 8192 28.9 against 21.1
    if (n_vocab > 4096 && n_vocab <= kHeld * kThreads && n_rows <= 256)
      sample_held_kernel<<<static_cast<unsigned>(n_rows), kThreads, 0, s>>>(a);
    else
      sample_row_kernel<<<static_cast<unsigned>(n_rows), kThreads, 0, s>>>(a);
  } else {
    auto *rows = static_cast<RowSpace *>(workspace);
    const dim3 grid(static_cast<unsigned>(chunks), static_cast<unsigned>(n_rows));
    sample_extremes_kernel<<<grid, kThreads, 0, s>>>(a, rows);
    sample_bins_kernel<<<grid, kThreads, 0, s>>>(a, rows);
    sample_pick_kernel<<<grid, kThreads, 0, s>>>(a, rows);
  }
  return ikv::launch_status();
}
