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
#include "../../include/ikv_model.h"
#include "ikv_common.hpp"

#include <algorithm>

namespace {

constexpr int kThreads = 256;
constexpr int kSlice = 4096;  // tokens of a workgroup
constexpr int64_t kMaxWorkgroups = (1 << 24) - 1;  // of 256 threads: 2^32 in a launch

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
      mask = a.r.masks + which * a.mask_words;
    }
  }
  if (n_history > 0 || n_bias > 0) {
    for (int i = tid; i < kSlice; i += kThreads) {
      s_seen[i] = 0;
      s_bias[i] = 0;
    }
    __syncthreads();
    const int32_t *const history = a.r.history + row * a.r.history_stride;
    const int64_t n_prompt = a.r.n_prompt ? a.r.n_prompt[row] : 0;
    bool bad = false;
    for (int64_t i = tid; i < n_history; i += kThreads) {
      const int token = history[i], at = token - first;
      bad |= static_cast<unsigned>(token) >= static_cast<unsigned>(a.n_vocab);
      if (static_cast<unsigned>(at) >= static_cast<unsigned>(n)) continue;
      if (i < n_prompt)
        atomicOr(&s_seen[at], 0x80000000u);
      else
        atomicAdd(&s_seen[at], 1u);
    }
    const int32_t *const named = a.r.bias_tokens + row * a.r.bias_stride;
    for (int64_t i = tid; i < n_bias; i += kThreads) {
      const int token = named[i], at = token - first;
      bad |= static_cast<unsigned>(token) >= static_cast<unsigned>(a.n_vocab);
      if (static_cast<unsigned>(at) < static_cast<unsigned>(n)) atomicMax(&s_bias[at], static_cast<int>(i + 1));
    }
    if (bad && first == 0) ikv::raise_status(a.status, IKV_STATUS_TOKEN);
    __syncthreads();
  }
  const bool ruled = n_history > 0 || n_bias > 0;
  const float repetition = a.r.repetition ? a.r.repetition[row] : 1.0f;
  const float presence = a.r.presence ? a.r.presence[row] : 0.0f;
  const float frequency = a.r.frequency ? a.r.frequency[row] : 0.0f;
  const float *const x = a.logits + row * a.n_vocab + first;
  float *const y = a.out + row * a.n_vocab + first;
  auto adjusted = [&](float v, unsigned seen, int bias) {
    if (seen) {
      const unsigned count = seen & 0x7fffffffu;
      v = v > 0.0f ? v / repetition : v * repetition;
      if (count) v = v - frequency * static_cast<float>(count) - presence;
    }
    if (bias) v += a.r.bias_values[row * a.r.bias_stride + bias - 1];
    return v;
  };
  auto allowed = [&](unsigned word, int i) { return (word >> (i & 31) & 1u) != 0; };
  if constexpr (VEC) {
    for (int i = 4 * tid; i < n; i += 4 * kThreads) {
      float4 v = *reinterpret_cast<const float4 *>(x + i);
      if (ruled) {
        const uint4 seen = *reinterpret_cast<const uint4 *>(s_seen + i);
        const int4 bias = *reinterpret_cast<const int4 *>(s_bias + i);
        v.x = adjusted(v.x, seen.x, bias.x);
        v.y = adjusted(v.y, seen.y, bias.y);
        v.z = adjusted(v.z, seen.z, bias.z);
        v.w = adjusted(v.w, seen.w, bias.w);
      }
      const unsigned word = none ? 0u : mask ? mask[(first + i) >> 5] : ~0u;
      v.x = allowed(word, i) ? v.x : -INFINITY;
      v.y = allowed(word, i + 1) ? v.y : -INFINITY;
      v.z = allowed(word, i + 2) ? v.z : -INFINITY;
      v.w = allowed(word, i + 3) ? v.w : -INFINITY;
      *reinterpret_cast<float4 *>(y + i) = v;
    }
  } else {
    for (int i = tid; i < n; i += kThreads) {
      float v = x[i];
      if (ruled) v = adjusted(v, s_seen[i], s_bias[i]);
      const unsigned word = none ? 0u : mask ? mask[(first + i) >> 5] : ~0u;
      y[i] = allowed(word, i) ? v : -INFINITY;
    }
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
