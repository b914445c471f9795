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
#include "../../include/ikv_model.h"
#include "ikv_common.hpp"

#include <algorithm>

namespace {

constexpr int kThreads = 1024;
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
__device__ __forceinline__ double exp2_series(double f) {
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

// A row as its workgroup sees it.
struct Row {
  const float *x;
  int n;
  float top;         // the largest logit
  double per_t;      // log2(e) / T
  double shift;      // S

  // w in multiples of 2^-S; the largest logit's is 2^S
  __device__ unsigned long long weight(float v) const {
    const double t = (static_cast<double>(v) - static_cast<double>(top)) * per_t;
    if (!(t > -(shift + 2.0))) return 0;
    const double whole = rint(t);
    // times 2^(whole + S), rounded to an integer: the bits of the sum with 2^52
    const long long power = static_cast<long long>(static_cast<int>(whole + shift) + 1023) << 52;
    const double sum = fma(exp2_series(t - whole), __builtin_bit_cast(double, power), 0x1p52);
    return __builtin_bit_cast(unsigned long long, sum) & 0xfffffffffffffull;
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
  for (int w = 0; w < wave; ++w) v += s_wave[w];
  return v;
}

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
    for (int i = tid; i < row.n; i += kThreads) {
      const unsigned o = order_of(row.x[i]);
      if (round > 0 && (o >> left) != r.order) continue;
      const unsigned b = (o >> (left - bits)) & ((1u << bits) - 1);
      atomicAdd(&s.count[b], 1u);
      const unsigned long long w = row.weight(row.x[i]);
      if (w) atomicAdd(&s.mass[b], w);
    }
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
  for (int i = threadIdx.x; i < row.n; i += kThreads)
    if (f(row.x[i])) m += row.weight(row.x[i]);
  m = block_prefix(m, s.wave);
  __syncthreads();
  if (threadIdx.x == kThreads - 1) s.found[0] = m;
  __syncthreads();
  m = s.found[0];
  __syncthreads();
  return m;
}

// Index of the rank-th (from 1) token of a value, in index order.
__device__ int index_of(const Row &row, Shared &s, unsigned order, unsigned long long rank) {
  unsigned long long before = 0;
  if (threadIdx.x == 0) s.found[0] = row.n - 1;
  for (int i0 = 0; i0 < row.n; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    const bool is = i < row.n && order_of(row.x[i]) == order;
    const unsigned long long upto = before + block_prefix(is ? 1 : 0, s.wave);
    if (is && upto == rank) s.found[0] = i;
    __syncthreads();
    if (threadIdx.x == kThreads - 1) s.found[1] = upto;
    __syncthreads();
    before = s.found[1];
    if (before >= rank) break;
  }
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

constexpr int kList = 4096;  // tokens of a row that are looked at one by one
constexpr int kMaxChunks = 64;

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
  unsigned long long kept_k, kept_p, kept_m, drawn;
  float top[kThreads / 64], low[kThreads / 64];
  int at[kThreads / 64];
  int bad, n, last;
};

union Space {
  Shared select;
  Lists l;
};

// f(x, index) over x[begin, end) by the workgroup, several loads in flight.
template <class F>
__device__ __forceinline__ void each_token(const float *x, int begin, int end, F &&f) {
  constexpr int kAhead = 4;
  int i = begin + threadIdx.x;
  for (; i + (kAhead - 1) * kThreads < end; i += kAhead * kThreads) {
    float v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) v[j] = x[i + j * kThreads];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) f(v[j], i + j * kThreads);
  }
  for (; i < end; i += kThreads) f(x[i], i);
}

// The largest logit of x[begin, end), its first index, the smallest finite one.
__device__ Chunk extremes(const float *x, int begin, int end, Lists &l) {
  Chunk c{-INFINITY, INFINITY, INT_MAX, 0};
  auto take = [&](float v, int i) {
    c.bad |= !(v < INFINITY);
    if (v > c.top) c.top = v, c.at = i;
    if (v > -INFINITY) c.low = fminf(c.low, v);
  };
  each_token(x, begin, end, take);
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

// Masses (and, for top_k, counts) of the tokens of x[begin, end) into l's bins.
// Tokens that weigh nothing are in none: they come last and move no border.
__device__ void fill_bins(const Row &row, const Window &win, bool counts, int begin, int end, Lists &l) {
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    l.mass[b] = 0;
    l.count[b] = 0;
  }
  __syncthreads();
  each_token(row.x, begin, end, [&](float x, int) {
    const unsigned long long w = row.weight(x);
    if (w == 0) return;
    const int b = win.bin(x);
    atomicAdd(&l.mass[b], w);
    if (counts) atomicAdd(&l.count[b], 1u);
  });
  __syncthreads();
}

// l's bins to what comes before each.
__device__ void sum_bins(Lists &l) {
  constexpr int kPer = kBins / kThreads;
  unsigned long long m[kPer], ms = 0;
  unsigned c[kPer], cs = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    ms += m[j] = l.mass[threadIdx.x * kPer + j];
    cs += c[j] = l.count[threadIdx.x * kPer + j];
  }
  unsigned long long bm = block_prefix(ms, l.wave) - ms;
  unsigned bc = static_cast<unsigned>(block_prefix(cs, l.wave)) - cs;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    l.mass[threadIdx.x * kPer + j] = bm;
    l.count[threadIdx.x * kPer + j] = bc;
    bm += m[j];
    bc += c[j];
  }
  if (threadIdx.x == kThreads - 1) {
    l.mass[kBins] = bm;
    l.count[kBins] = bc;
  }
  __syncthreads();
}

// The bins that hold the borders. A border is known to a bin's mass before the
// ones ahead of it are looked at, so a range of bins may have to be: nearly
// always one.
struct Ranges {
  int lo[4], hi[4];  // top_k, top_p, min_p, the draw; hi < lo: none
  unsigned long long total, before_m;
  bool has_k;

  template <class T>
  __device__ static int reaching(const T *before, T border) {  // the first bin at whose end it is reached
    int lo = 0, hi = kBins - 1;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (before[mid + 1] >= border)
        hi = mid;
      else
        lo = mid + 1;
    }
    return lo;
  }

  __device__ Ranges(const Row &row, const Window &win, const Cuts &c, const Lists &l) {
#pragma unroll
    for (int j = 0; j < 4; ++j) lo[j] = 1, hi[j] = 0;
    total = l.mass[kBins];
    unsigned long long least = total, most = total;  // of the kept mass
    has_k = c.k > 0 && static_cast<unsigned>(c.k) < l.count[kBins];
    if (has_k) {
      lo[0] = hi[0] = reaching(l.count, static_cast<unsigned>(c.k));
      least = l.mass[lo[0]];
      most = l.mass[lo[0] + 1];
    }
    if (c.p < 1.0f) {
      lo[1] = reaching(l.mass, share_of(least, c.p));
      hi[1] = reaching(l.mass, share_of(most, c.p));
      least = min(least, l.mass[lo[1]]);
      most = min(most, l.mass[hi[1] + 1]);
    }
    before_m = 0;
    if (c.low > 0.0f) {
      const double move = static_cast<double>(c.t) * c.floor, at = row.top + move;
      const double slack = 1e-12 * (fabs(static_cast<double>(row.top)) + fabs(move));
      auto edge = [&](double x, float way) {
        const float f = static_cast<float>(x);
        return f < INFINITY && f > -INFINITY ? nextafterf(f, way) : f;
      };
      lo[2] = max(win.bin(edge(at + slack, INFINITY)), 0);
      hi[2] = max(win.bin(edge(at - slack, -INFINITY)), 0);
      before_m = l.mass[lo[2]];
      least = min(least, before_m);
      most = min(most, l.mass[hi[2] + 1]);
    }
    const unsigned long long heaviest = row.weight(row.top);
    lo[3] = reaching(l.mass, drawn_of(max(least, heaviest), c.u));
    hi[3] = reaching(l.mass, drawn_of(max(most, heaviest), c.u));
  }

  __device__ bool holds(int b) const {
    bool in = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) in |= b >= lo[j] && b <= hi[j];
    return in;
  }
};

// The tokens of those bins into l's list (l.n may pass kList: then not all).
__device__ void gather(const Row &row, const Window &win, const Ranges &rg, int begin, int end, Lists &l) {
  if (threadIdx.x == 0) l.n = 0;
  __syncthreads();
  each_token(row.x, begin, end, [&](float x, int i) {
    if (!rg.holds(win.bin(x)) || row.weight(x) == 0) return;
    const int at = atomicAdd(&l.n, 1);
    if (at < kList) l.list[at] = static_cast<unsigned long long>(order_of(x)) << 32 | static_cast<unsigned>(i);
  });
  __syncthreads();
}

// The token, from the bins' sums and the whole list (n <= kList tokens of it).
__device__ void resolve(const Args &a, int r, const Row &row, const Window &win, const Cuts &c, const Ranges &rg,
                        int n, Lists &l) {
  const int tid = threadIdx.x;
  int size = 64;
  while (size < n) size *= 2;
  for (int i = n + tid; i < size; i += kThreads) l.list[i] = ~0ull;
  if (tid == 0) {
    l.kept_k = rg.total;
    l.kept_p = l.drawn = ~0ull;
    l.kept_m = rg.before_m;
  }
  __syncthreads();
  for (int k = 2; k <= size; k *= 2) {  // bitonic: by order, then index
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
  // running masses and counts: a bin's tokens are all in the list, one behind
  // the other, so a token's are its bin's and those of the list since the bin's
  // first one
  constexpr int kPer = kList / kThreads;
  unsigned long long m[kPer], own = 0;
  float x[kPer];
  int bin[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = tid * kPer + j;
    const unsigned o = i < n ? static_cast<unsigned>(l.list[i] >> 32) : 0u;
    x[j] = __uint_as_float((o & 0x80000000u) ? o : ~o & 0x7fffffffu);
    bin[j] = i < n ? win.bin(x[j]) : -1;
    own += m[j] = i < n ? row.weight(x[j]) : 0;
  }
  unsigned long long run = block_prefix(own, l.wave) - own;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = tid * kPer + j;
    bool first = i < n && i == 0;
    if (i < n && i > 0) {
      const unsigned o = static_cast<unsigned>(l.list[i - 1] >> 32);
      first = win.bin(__uint_as_float((o & 0x80000000u) ? o : ~o & 0x7fffffffu)) != bin[j];
    }
    if (first) {  // (one token of the bin: nobody else touches its sums)
      l.mass[bin[j]] -= run;
      l.count[bin[j]] -= static_cast<unsigned>(i);
    }
    run += m[j];
    m[j] = run;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = tid * kPer + j;
    if (i >= n) continue;
    m[j] += l.mass[bin[j]];
    if (rg.has_k && bin[j] == rg.lo[0] && l.count[bin[j]] + i + 1 == static_cast<unsigned>(c.k)) l.kept_k = m[j];
    if (c.low > 0.0f && c.passes(x[j], row.top)) atomicMax(&l.kept_m, m[j]);
  }
  __syncthreads();
  unsigned long long kept = l.kept_k;
  if (c.p < 1.0f) {
    const unsigned long long need = share_of(kept, c.p);
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (tid * kPer + j < n && m[j] >= need) atomicMin(&l.kept_p, m[j]);
    __syncthreads();
    kept = min(kept, l.kept_p);
  }
  if (c.low > 0.0f) kept = min(kept, l.kept_m);
  kept = max(kept, row.weight(row.top));
  const unsigned long long target = drawn_of(kept, c.u);
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (tid * kPer + j < n && m[j] >= target) atomicMin(&l.drawn, m[j]);
  __syncthreads();
  const unsigned long long drawn = l.drawn;
#pragma unroll
  for (int j = 0; j < kPer; ++j)  // (every token of the list weighs something: one has this running mass)
    if (tid * kPer + j < n && m[j] == drawn)
      answer(a, r, static_cast<int>(static_cast<unsigned>(l.list[tid * kPer + j])), x[j], row, c, kept);
}

__device__ Row row_of(const Args &a, int r, const Cuts &c, float top) {
  return Row{a.logits + static_cast<size_t>(r) * a.n, a.n, top,
             1.4426950408889634074 / static_cast<double>(c.t), static_cast<double>(a.shift)};
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
__global__ __launch_bounds__(kThreads) void sample_row_kernel(Args a) {
  __shared__ Space s;
  const int r = blockIdx.x;
  const Cuts c(a, r);
  const Chunk e = extremes(a.logits + static_cast<size_t>(r) * a.n, 0, a.n, s.l);
  if (settled(a, r, c, e, threadIdx.x == 0)) return;
  const Row row = row_of(a, r, c, e.top);
  const Window win(row, e.low, c.t);
  fill_bins(row, win, c.k > 0 && c.k < a.n, 0, a.n, s.l);
  sum_bins(s.l);
  const Ranges rg(row, win, c, s.l);
  gather(row, win, rg, 0, a.n, s.l);
  const int n = s.l.n;
  if (n <= kList) {
    resolve(a, r, row, win, c, rg, n, s.l);
  } else {
    __syncthreads();
    select_row(a, r, row, c, s.select);
  }
}

// Several workgroups a row, in three launches. The first: each chunk's extremes,
// and the row's sums cleared.
__device__ __forceinline__ void chunk_of(const Args &a, int &begin, int &end) {
  const int per = (a.n + gridDim.x - 1) / gridDim.x;
  begin = min(a.n, static_cast<int>(blockIdx.x) * per);
  end = min(a.n, begin + per);
}

__global__ __launch_bounds__(kThreads) void sample_extremes_kernel(Args a, RowSpace *rows) {
  __shared__ Lists l;
  const int r = blockIdx.y;
  RowSpace &w = rows[r];
  for (int b = blockIdx.x * kThreads + threadIdx.x; b < kBins; b += gridDim.x * kThreads) {
    w.mass[b] = 0;
    w.count[b] = 0;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) w.listed = w.arrived = 0;
  int begin, end;
  chunk_of(a, begin, end);
  const Chunk e = extremes(a.logits + static_cast<size_t>(r) * a.n, begin, end, l);
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

// The second: the bins.
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(Args a, RowSpace *rows) {
  __shared__ Lists l;
  const int r = blockIdx.y;
  RowSpace &w = rows[r];
  const Cuts c(a, r);
  const Chunk e = row_extremes(w, gridDim.x);
  if (settled(a, r, c, e, false)) return;
  const Row row = row_of(a, r, c, e.top);
  const Window win(row, e.low, c.t);
  int begin, end;
  chunk_of(a, begin, end);
  const bool counts = c.k > 0 && c.k < a.n;
  fill_bins(row, win, counts, begin, end, l);
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    if (l.mass[b] == 0) continue;
    atomicAdd(&w.mass[b], l.mass[b]);
    if (counts) atomicAdd(&w.count[b], l.count[b]);
  }
}

// The third: the borders' bins, their tokens, and, by the workgroup that comes
// last, the token.
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(Args a, RowSpace *rows) {
  __shared__ Space s;
  Lists &l = s.l;
  const int r = blockIdx.y, tid = threadIdx.x;
  RowSpace &w = rows[r];
  const Cuts c(a, r);
  const Chunk e = row_extremes(w, gridDim.x);
  if (settled(a, r, c, e, blockIdx.x == 0 && tid == 0)) return;
  const Row row = row_of(a, r, c, e.top);
  const Window win(row, e.low, c.t);
  for (int b = tid; b < kBins; b += kThreads) {
    l.mass[b] = w.mass[b];
    l.count[b] = w.count[b];
  }
  __syncthreads();
  sum_bins(l);
  const Ranges rg(row, win, c, l);
  int begin, end;
  chunk_of(a, begin, end);
  gather(row, win, rg, begin, end, l);
  if (tid == 0) l.last = static_cast<int>(atomicAdd(&w.listed, static_cast<unsigned>(l.n)));
  __syncthreads();
  const unsigned first = static_cast<unsigned>(l.last);
  for (int i = tid; i < min(l.n, kList); i += kThreads)
    if (first + i < kList)
      __hip_atomic_store(&w.list[first + i], l.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // the entries' stores have completed before the arrival
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_s_waitcnt(0);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __syncthreads();
  if (tid == 0)
    l.last = __hip_atomic_fetch_add(&w.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  __syncthreads();
  if (!l.last) return;
  const unsigned n = __hip_atomic_load(&w.listed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (n <= kList) {
    for (unsigned i = tid; i < n; i += kThreads)
      l.list[i] = __hip_atomic_load(&w.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    resolve(a, r, row, win, c, rg, static_cast<int>(n), l);
  } else {
    __syncthreads();
    select_row(a, r, row, c, s.select);
  }
}

// Workgroups of a row: one up to kRowTokens tokens, else as many as bring all
// rows to kGroups, of 2048 tokens at least (one where there are many rows).
constexpr int kRowTokens = 16384, kGroups = 1024;
int chunks_of(int64_t n_rows, int64_t n_vocab) {
  if (n_vocab <= kRowTokens) return 1;
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
