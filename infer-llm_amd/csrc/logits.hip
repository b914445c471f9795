// logits.hip — the logits of each row with penalties for the tokens of its history,
// biases and a mask of the tokens that a grammar allows (ikv_adjust_logits_f32),
// ahead of the samplers.
//
// Each logit is read once and written once: HBM bounds large calls. A workgroup
// takes a slice of a row's vocabulary and goes over the row's whole history and its
// biases; the slice's counts are in LDS, filled by integer atomics, whose order
// changes nothing: bit 31 a token of the prompt, the bits below how often it was
// generated, so a word is not 0 where the token was seen. Of biases that name one
// token the last counts: a maximum over their places in the list.
// Measured (MI355X, us): 48 rows of 151936 with histories of up to 6000, 59 MB, 18 (14
// without histories: each of a row's 38 workgroups reads all of its list, from behind
// the L2), one row with 1500 5.2. Slices of 4096 and 512 threads: of 2048 23 and 4.4, of
// 8192 23 and 5.9, 256 threads 27 and 6.2, 1024 23 and 4.6.
#include "../../include/ikv_model.h"
#include "ikv_common.hpp"

#include <algorithm>

namespace {

constexpr int kThreads = 512;
constexpr int kSlice = 4096;  // tokens of a workgroup
constexpr int kPer = kSlice / kThreads;
constexpr int kAhead = 4;  // tokens of a history that a thread loads at once
constexpr int64_t kMaxWorkgroups = (1 << 23) - 1;  // of 512 threads: 2^32 in a launch

struct Args {
  const float *logits;
  float *out;
  ikv_logit_rules r;
  int n_vocab, slices;
  int64_t mask_words;
  int *status;
};

template <bool VEC>
__global__ __launch_bounds__(kThreads) void adjust_logits_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) unsigned s_seen[kSlice];
  __shared__ __attribute__((aligned(16))) int s_bias[kSlice];  // place in the list, from 1
  const int64_t row = blockIdx.x / a.slices;
  const int first = blockIdx.x % a.slices * kSlice, n = min(kSlice, a.n_vocab - first);
  const int tid = threadIdx.x;
  auto length = [&](const int32_t *lengths, int64_t stride) -> int64_t {  // of the row's list
    const int64_t got = lengths ? lengths[row] : stride;
    if (got >= 0 && got <= stride) return got;
    if (first == 0 && tid == 0) ikv::raise_status(a.status, IKV_STATUS_POSITION);
    return 0;
  };
  const int64_t n_history = a.r.history ? length(a.r.n_history, a.r.history_stride) : 0;
  const int64_t n_bias = a.r.bias_tokens ? length(a.r.n_bias, a.r.bias_stride) : 0;
  const uint32_t *mask = nullptr;
  bool none = false;  // no token is allowed
  if (a.r.masks) {
    const int64_t which = a.r.mask_of ? a.r.mask_of[row] : 0;
    if (which >= a.r.n_masks) {
      none = true;
      if (first == 0 && tid == 0) ikv::raise_status(a.status, IKV_STATUS_POSITION);
    } else if (which >= 0) {
      mask = a.r.masks + which * a.mask_words + first / 32;
    }
  }
  const float repetition = a.r.repetition ? a.r.repetition[row] : 1.0f;
  const float presence = a.r.presence ? a.r.presence[row] : 0.0f;
  const float frequency = a.r.frequency ? a.r.frequency[row] : 0.0f;

  // this thread's logits and mask words, on their way while the lists are gone over
  constexpr int E = VEC ? 4 : 1;
  auto place = [&](int j) { return E * (tid + kThreads * (j / E)) + j % E; };
  const float *const x = a.logits + row * a.n_vocab + first;
  float *const y = a.out + row * a.n_vocab + first;
  float v[kPer];
  unsigned word[kPer / E];
#pragma unroll
  for (int j = 0; j < kPer; j += E) {
    const int i = place(j);
    word[j / E] = none ? 0u : ~0u;
    if (i >= n) continue;
    if constexpr (VEC) {
      const float4 z = *reinterpret_cast<const float4 *>(x + i);
      v[j] = z.x, v[j + 1] = z.y, v[j + 2] = z.z, v[j + 3] = z.w;
    } else {
      v[j] = x[i];
    }
    if (mask) word[j / E] = mask[i >> 5];
  }
  // f(token) of a list's tokens, several of a thread loaded at once; whether one is
  // none of the vocabulary
  auto each = [&](const int32_t *list, int64_t length, auto &&f) {
    bool bad = false;
    for (int64_t i0 = tid; i0 < length; i0 += kAhead * kThreads) {
      int token[kAhead];
#pragma unroll
      for (int z = 0; z < kAhead; ++z) token[z] = i0 + z * kThreads < length ? list[i0 + z * kThreads] : first;
#pragma unroll
      for (int z = 0; z < kAhead; ++z) {
        if (i0 + z * kThreads >= length) break;
        bad |= static_cast<unsigned>(token[z]) >= static_cast<unsigned>(a.n_vocab);
        const unsigned at = static_cast<unsigned>(token[z] - first);
        if (at < static_cast<unsigned>(n)) f(at, i0 + z * kThreads);
      }
    }
    if (bad && first == 0) ikv::raise_status(a.status, IKV_STATUS_TOKEN);
  };
  if (n_history > 0) {
    for (int i = 4 * tid; i < kSlice; i += 4 * kThreads) *reinterpret_cast<uint4 *>(s_seen + i) = uint4{};
    __syncthreads();
    const int64_t n_prompt = a.r.n_prompt ? a.r.n_prompt[row] : 0;
    each(a.r.history + row * a.r.history_stride, n_history, [&](unsigned at, int64_t i) {
      if (i < n_prompt)
        atomicOr(&s_seen[at], 0x80000000u);
      else
        atomicAdd(&s_seen[at], 1u);
    });
  }
  if (n_bias > 0) {
    for (int i = 4 * tid; i < kSlice; i += 4 * kThreads) *reinterpret_cast<int4 *>(s_bias + i) = int4{};
    __syncthreads();
    each(a.r.bias_tokens + row * a.r.bias_stride, n_bias,
         [&](unsigned at, int64_t i) { atomicMax(&s_bias[at], static_cast<int>(i + 1)); });
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kPer; j += E) {
    const int i = place(j);
    if (i >= n) continue;
    if (n_history > 0) {
      unsigned seen[E];
#pragma unroll
      for (int e = 0; e < E; ++e) seen[e] = s_seen[i + e];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (seen[e] == 0) continue;
        float z = v[j + e];
        z = z > 0.0f ? z / repetition : z * repetition;
        const unsigned count = seen[e] & 0x7fffffffu;
        if (count) z = z - frequency * static_cast<float>(count) - presence;
        v[j + e] = z;
      }
    }
    if (n_bias > 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int from = s_bias[i + e];
        if (from) v[j + e] += a.r.bias_values[row * a.r.bias_stride + from - 1];
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if ((word[j / E] >> ((i + e) & 31) & 1u) == 0) v[j + e] = -INFINITY;
    if constexpr (VEC)
      *reinterpret_cast<float4 *>(y + i) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    else
      y[i] = v[j];
  }
}

}  // namespace

extern "C" int ikv_adjust_logits_f32(const float *logits, float *out, const ikv_logit_rules *rules,
                                     int64_t n_rows, int64_t n_vocab, int32_t *status, void *stream) {
  if (!rules || n_rows < 0 || n_vocab <= 0) return -EINVAL;
  const ikv_logit_rules &r = *rules;
  if (r.history && r.history_stride < 0) return -EINVAL;
  if (r.bias_tokens && (r.bias_stride < 0 || !r.bias_values)) return -EINVAL;
  if (r.masks && r.n_masks <= 0) return -EINVAL;
  if (n_rows == 0) return 0;
  if (!logits || !out) return -EINVAL;
  constexpr int64_t kMost = int64_t{1} << 30;
  const int64_t slices = (n_vocab + kSlice - 1) / kSlice;
  if (n_vocab > kMost || n_rows > (1 << 21) || slices * n_rows > kMaxWorkgroups || (r.history && r.history_stride > kMost) ||
      (r.bias_tokens && r.bias_stride > kMost))
    return -EOVERFLOW;
  const Args a{logits, out, r, static_cast<int>(n_vocab), static_cast<int>(slices), (n_vocab + 31) / 32, status};
  const unsigned grid = static_cast<unsigned>(slices * n_rows);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (n_vocab % 4 == 0 && ikv::aligned16(logits) && ikv::aligned16(out))
    adjust_logits_kernel<true><<<grid, kThreads, 0, s>>>(a);
  else
    adjust_logits_kernel<false><<<grid, kThreads, 0, s>>>(a);
  return ikv::launch_status();
}
