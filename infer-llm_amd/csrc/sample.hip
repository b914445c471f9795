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
// that a row's sum fits 64 bits (45 bits for 151936 tokens; a token lighter than
// 2^-46 of the heaviest weighs nothing). Sums of integers do not depend on their
// order, so histograms may be filled by atomics and results repeat bit for bit.
//
// Nothing is sorted. The place where a running count or mass crosses a border is
// found by radix selection: tokens are binned by the next 11 bits of their
// value's place in the order, bins are summed up to the border, and the bin that
// holds it is looked into again with the following bits; three rounds end at one
// value, whose tokens weigh the same, so what is left is a division. One
// workgroup takes a row.
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
    return static_cast<unsigned long long>(
        rint(ldexp(exp2_series(t - whole), static_cast<int>(whole + shift))));
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

__global__ __launch_bounds__(kThreads) void sample_kernel(Args a) {
  __shared__ Shared s;
  const int r = blockIdx.x, tid = threadIdx.x;
  Row row;
  row.x = a.logits + static_cast<size_t>(r) * a.n;
  row.n = a.n;
  const float t = a.temperature ? a.temperature[r] : 1.0f;
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.0f;
  const float low = a.min_p ? a.min_p[r] : 0.0f;
  float u = a.u[r];

  if (tid == 0) s.bad = 0;
  __syncthreads();
  float top = -INFINITY;
  bool bad = !(t < INFINITY) || p != p || low != low || u != u;
  for (int i = tid; i < a.n; i += kThreads) {
    const float x = row.x[i];
    bad |= !(x < INFINITY);
    top = fmaxf(top, x);
  }
  if (bad) s.bad = 1;  // benign race: every writer stores 1
  top = ikv::wave_max(top);
  if ((tid & 63) == 0) s.top[tid >> 6] = top;
  __syncthreads();
  for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, s.top[w]);
  if (s.bad || top == -INFINITY) {
    if (tid == 0) {
      a.token[r] = -1;
      if (a.logprob) a.logprob[r] = __int_as_float(0x7fc00000);
    }
    return;
  }
  if (t <= 0.0f) {
    const int at = index_of(row, s, order_of(top), 1);
    if (tid == 0) {
      a.token[r] = at;
      if (a.logprob) a.logprob[r] = 0.0f;
    }
    return;
  }
  u = fminf(fmaxf(u, 0.0f), 0x1.fffffep-1f);
  row.top = top;
  row.per_t = 1.4426950408889634074 / static_cast<double>(t);
  row.shift = a.shift;

  unsigned long long kept;
  if (k > 0 && k < a.n) {
    const Spot b = select<Border::kCount>(row, s, static_cast<unsigned long long>(k));
    kept = b.mass + (k - b.count) * b.each;
  } else {
    kept = mass_of(row, s, [](float) { return true; });
  }
  if (p < 1.0f) {
    // (a running mass is an integer: it reaches the border where it reaches the next one)
    const auto need = static_cast<unsigned long long>(ceil(static_cast<double>(fmaxf(p, 0.0f)) * static_cast<double>(kept)));
    const Spot b = select<Border::kMass>(row, s, need);
    kept = min(kept, b.mass + tokens_to(b, need) * b.each);
  }
  if (low > 0.0f) {
    const double floor = log(static_cast<double>(low));
    const unsigned long long m = mass_of(row, s, [&](float x) {
      return (static_cast<double>(x) - static_cast<double>(top)) / static_cast<double>(t) >= floor;
    });
    kept = min(kept, m);
  }
  const unsigned long long heaviest = row.weight(top);
  kept = max(kept, heaviest);
  const auto target = static_cast<unsigned long long>(static_cast<double>(u) * static_cast<double>(kept)) + 1;
  const Spot b = select<Border::kMass>(row, s, target);  // (exceeds: reaches the next integer)
  const int at = index_of(row, s, b.order, tokens_to(b, target));
  if (tid == 0) {
    a.token[r] = at;
    const double y = (static_cast<double>(row.x[at]) - static_cast<double>(top)) / static_cast<double>(t);
    if (a.logprob)
      a.logprob[r] = static_cast<float>(y - log(ldexp(static_cast<double>(kept), -a.shift)));
  }
}

}  // namespace

extern "C" size_t ikv_sample_workspace_bytes(int64_t n_rows, int64_t n_vocab) {
  if (n_rows <= 0 || n_vocab <= 0) return 0;
  return 256;
}

extern "C" int ikv_sample_f32(const float *logits, const float *u, const float *temperature,
                              const int32_t *top_k, const float *top_p, const float *min_p, int64_t n_rows,
                              int64_t n_vocab, int32_t *token, float *logprob, void *workspace,
                              size_t workspace_bytes, void *stream) {
  if (n_rows < 0 || n_vocab < 1) return -EINVAL;
  if (n_rows == 0) return 0;
  if (!logits || !u || !token || !workspace || !ikv::aligned16(workspace)) return -EINVAL;
  if (n_vocab > (1 << 30) || n_rows > INT_MAX) return -EOVERFLOW;
  if (workspace_bytes < ikv_sample_workspace_bytes(n_rows, n_vocab)) return -EINVAL;
  int bits = 0;  // of the count
  while ((int64_t{1} << bits) < n_vocab) ++bits;
  Args a{logits, u, temperature, top_k, top_p, min_p, static_cast<int>(n_vocab), std::min(63 - bits, 52),
         token, logprob};
  sample_kernel<<<static_cast<unsigned>(n_rows), kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  return ikv::launch_status();
}
