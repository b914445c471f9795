// cache_q8.hpp — a paged KV cache of 8 bits an element (ikv_kv_q8) as the kernels
// see it, and the two formats of its codes.
//
// A block's rows lie head by head, [block][KV head][token of the block][head_dim],
// so what a workgroup reads of one head is contiguous, and its scales are, too. A
// row of head_dim values x has one scale: with top = max |x|,
//     int8  scale = top / 127, code = 127 x / top rounded to an integer,
//     e4m3  scale = top / 448, code = 448 x / top rounded to a float, then to e4m3,
// to the nearest, ties to even; a code stands for code * scale. The quotient is in
// 64 bits, so that a code next to a border is the definition's. A row with an
// element that is not finite has a NaN scale and zero codes.
#pragma once

#include "batch.hpp"

namespace ikv {

constexpr int kMaxDimQ8 = 256;

struct CacheQ8 {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  int n_head_kv, dim;
  bool e4m3;
};

// 0, or what is wrong with a cache (its pointers are looked at where there is work).
inline int cache_q8_arg(const ikv_kv_q8 *c, CacheQ8 &out) {
  if (!c || c->n_head_kv <= 0 || c->head_dim <= 0) return -EINVAL;
  if (c->format != IKV_Q8_INT8 && c->format != IKV_Q8_E4M3) return -EINVAL;
  if (c->head_dim % 16 != 0 || c->head_dim > kMaxDimQ8) return -ENOTSUP;
  if (c->n_head_kv > (1 << 23) / c->head_dim) return -EOVERFLOW;
  out.k = static_cast<uint8_t *>(c->k_codes);
  out.v = static_cast<uint8_t *>(c->v_codes);
  out.k_scale = c->k_scales;
  out.v_scale = c->v_scales;
  out.n_head_kv = c->n_head_kv;
  out.dim = c->head_dim;
  out.e4m3 = c->format == IKV_Q8_E4M3;
  return 0;
}
inline bool cache_q8_there(const CacheQ8 &c) {
  return c.k && c.v && c.k_scale && c.v_scale && aligned16(c.k) && aligned16(c.v) && aligned16(c.k_scale) &&
         aligned16(c.v_scale);
}

// The row of token `at` of block `blk` of a head: its scale's index, and its codes'
// over head_dim.
__device__ __forceinline__ int64_t row_q8(int blk, int n_head_kv, int g, int bt, int at) {
  return (static_cast<int64_t>(blk) * n_head_kv + g) * bt + at;
}

// A row's scale and its codes, from the bits of its largest |x|.
template <bool E4M3>
struct Quant {
  double top, inv;
  float scale;
  bool some;  // neither all zeros nor with an element that is not finite
  __device__ __forceinline__ explicit Quant(unsigned top_bits) {
    top = static_cast<double>(__uint_as_float(top_bits));
    // 1 / top from the hardware's estimate and two steps of Newton's
    inv = __builtin_amdgcn_rcp(top);
    inv = fma(inv, fma(-top, inv, 1.0), inv);
    inv = fma(inv, fma(-top, inv, 1.0), inv);
    some = top_bits - 1u < 0x7f7fffffu;
    scale = some ? static_cast<float>(top * (1.0 / (E4M3 ? 448.0 : 127.0))) : top_bits == 0 ? 0.0f : NAN;
  }
  // the quotient, its last bit by what the first one leaves (so exact ones are exact; the
  // signs are so that -0 stays -0)
  __device__ __forceinline__ double of(float v) const {
    const double a = static_cast<double>(v) * (E4M3 ? 448.0 : 127.0), q = a * inv;
    return fma(-fma(q, top, -a), inv, q);
  }
  // four codes, the first in the low byte
  __device__ __forceinline__ unsigned codes(const float4 x) const {
    unsigned w;
    if constexpr (E4M3) {
      auto y = [&](float v) { return static_cast<float>(of(v)); };
      w = __builtin_amdgcn_cvt_pk_fp8_f32(y(x.x), y(x.y), 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(y(x.z), y(x.w), w, true);
    } else {
      // (the sum with 1.5 2^52 is rounded to an integer, which its low bits then hold)
      auto y = [&](float v) { return static_cast<unsigned>(__builtin_bit_cast(unsigned long long, of(v) + 0x1.8p52)); };
      w = (y(x.x) & 0xffu) | (y(x.y) & 0xffu) << 8 | (y(x.z) & 0xffu) << 16 | y(x.w) << 24;
    }
    return some ? w : 0u;
  }
};

// The values of four codes, without their scale.
template <bool E4M3>
__device__ __forceinline__ float4 values_q8(unsigned w) {
  if constexpr (E4M3) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    return make_float4(a[0], a[1], b[0], b[1]);
  } else {
    auto y = [&](int i) { return static_cast<float>(static_cast<int>(w << (24 - 8 * i)) >> 24); };
    return make_float4(y(0), y(1), y(2), y(3));
  }
}

__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The largest over the 16, 32 or 64 lanes that hold a row (DPP and lane swaps).
template <int LANES>
__device__ __forceinline__ unsigned lanes_max(unsigned x) {
  auto with = [&](int other) { x = max(x, static_cast<unsigned>(other)); };
  with(__builtin_amdgcn_mov_dpp(static_cast<int>(x), kDppXor1, 0xF, 0xF, false));
  with(__builtin_amdgcn_mov_dpp(static_cast<int>(x), kDppXor2, 0xF, 0xF, false));
  with(__builtin_amdgcn_mov_dpp(static_cast<int>(x), kDppHalfMirror, 0xF, 0xF, false));
  with(__builtin_amdgcn_mov_dpp(static_cast<int>(x), kDppMirror, 0xF, 0xF, false));
  if constexpr (LANES >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(a[0], a[1]);
  }
  if constexpr (LANES >= 64) {
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = max(b[0], b[1]);
  }
  return x;
}

}  // namespace ikv
