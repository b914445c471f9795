// cache_q8.hip — K and V rows of several sequences' new tokens into a paged cache
// of 8 bits an element, and back as floats (ikv_append_packed_q8,
// ikv_read_packed_q8). The formats are in cache_q8.hpp.
//
// Each byte is read once and written once: HBM bounds both. A wave takes a packed
// row of all heads, finds its sequence (wave_find_last) and its block, and goes
// over the row's heads, a row of a head on 16, 32 or 64 lanes, four elements a
// lane, so that the largest magnitude is a maximum over those lanes and codes and
// floats move in whole lines.
// Measured (MI355X, us): 8190 rows of 8 heads of 128 written 22 (84 MB, 3.8 TB/s:
// the quotients in 64 bits, which leave 20 where they are a product instead), read back
// 16 (5.3 TB/s, the rate of a copy); 103356 rows read 199 (1.07 GB, 5.3 TB/s); 211 rows
// of 5 sequences written 5.6, 1398 read 6.1: a launch and four loads one after the other.
#include "cache_q8.hpp"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kRowWaves = 4;  // rows of a workgroup, one per wave

template <bool E4M3, int LANES>
__global__ __launch_bounds__(kRowWaves * 64) void append_q8_kernel(
    ikv::CacheQ8 c, const float *__restrict__ k_rows, const float *__restrict__ v_rows, ikv::BatchPages b,
    const int32_t *__restrict__ row_start, const int32_t *__restrict__ first_token, int64_t n_rows) {
  ikv::check_row_start(row_start, b.n_seq, n_rows, b.status);
  constexpr int kHeads = 64 / LANES;  // rows of heads that a wave holds
  constexpr int kAhead = 4;           // of them, loaded at once
  const int lane = threadIdx.x & 63, d = lane % LANES * 4, h = lane / LANES;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRowWaves;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kRowWaves + (threadIdx.x >> 6); i < n_rows; i += step) {
    const int seq = ikv::wave_find_last(b.n_seq, [&](int s) { return row_start[s] <= i; });
    if (seq < 0 || i >= row_start[seq + 1]) continue;  // a row of no sequence
    const int64_t t = (first_token ? first_token[seq] : 0) + (i - row_start[seq]);
    if (t < 0 || t >= b.capacity) {
      ikv::raise_status(b.status, IKV_STATUS_POSITION);
      continue;
    }
    const int in_table = static_cast<unsigned>(t) / static_cast<unsigned>(b.bt);
    const int at = static_cast<int>(t) - in_table * b.bt;
    const int blk = b.tables[seq * b.stride + in_table];
    if (static_cast<unsigned>(blk) >= static_cast<unsigned>(b.n_blocks)) {
      ikv::raise_status(b.status, IKV_STATUS_BLOCK);  // dropped: no block to write
      continue;
    }
    const float *const kr = k_rows + i * c.n_head_kv * c.dim, *const vr = v_rows + i * c.n_head_kv * c.dim;
    for (int g0 = 0; g0 < c.n_head_kv; g0 += kHeads * kAhead) {
      float4 x[2][kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int g = g0 + j * kHeads + h;
        const bool there = g < c.n_head_kv && d < c.dim;
        x[0][j] = there ? *reinterpret_cast<const float4 *>(kr + g * c.dim + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[1][j] = there ? *reinterpret_cast<const float4 *>(vr + g * c.dim + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int g = g0 + j * kHeads + h;
        if (g0 + j * kHeads >= c.n_head_kv) break;
        const int64_t row = ikv::row_q8(blk, c.n_head_kv, min(g, c.n_head_kv - 1), b.bt, at);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const float4 y = x[z][j];
          const unsigned top = ikv::lanes_max<LANES>(
              max(max(ikv::abs_bits(y.x), ikv::abs_bits(y.y)), max(ikv::abs_bits(y.z), ikv::abs_bits(y.w))));
          const ikv::Quant<E4M3> quant(top);
          const unsigned w = quant.codes(y);
          if (g >= c.n_head_kv || d >= c.dim) continue;
          *reinterpret_cast<unsigned *>((z == 0 ? c.k : c.v) + row * c.dim + d) = w;
          if (d == 0) (z == 0 ? c.k_scale : c.v_scale)[row] = quant.scale;
        }
      }
    }
  }
}

template <bool E4M3, int LANES>
__global__ __launch_bounds__(kRowWaves * 64) void read_q8_kernel(
    ikv::CacheQ8 c, float *__restrict__ k_rows, float *__restrict__ v_rows, ikv::BatchPages b,
    const int32_t *__restrict__ row_start, const int32_t *__restrict__ first_token,
    const int32_t *__restrict__ n_kv, int64_t n_rows) {
  ikv::check_row_start(row_start, b.n_seq, n_rows, b.status);
  constexpr int kHeads = 64 / LANES, kAhead = 4;
  const int lane = threadIdx.x & 63, d = lane % LANES * 4, h = lane / LANES;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRowWaves;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kRowWaves + (threadIdx.x >> 6); i < n_rows; i += step) {
    const int seq = ikv::wave_find_last(b.n_seq, [&](int s) { return row_start[s] <= i; });
    if (seq < 0 || i >= row_start[seq + 1]) continue;
    const int64_t t = (first_token ? first_token[seq] : 0) + (i - row_start[seq]);
    if (n_kv && t >= n_kv[seq]) continue;  // behind the sequence's last token
    if (t < 0 || t >= b.capacity) {
      ikv::raise_status(b.status, IKV_STATUS_POSITION);
      continue;
    }
    const int in_table = static_cast<unsigned>(t) / static_cast<unsigned>(b.bt);
    const int at = static_cast<int>(t) - in_table * b.bt;
    int blk = b.tables[seq * b.stride + in_table];
    if (static_cast<unsigned>(blk) >= static_cast<unsigned>(b.n_blocks)) {
      ikv::raise_status(b.status, IKV_STATUS_BLOCK);
      blk = 0;
    }
    float *const kr = k_rows + i * c.n_head_kv * c.dim, *const vr = v_rows + i * c.n_head_kv * c.dim;
    for (int g0 = 0; g0 < c.n_head_kv; g0 += kHeads * kAhead) {
      unsigned w[2][kAhead];
      float scale[2][kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int g = min(g0 + j * kHeads + h, c.n_head_kv - 1);
        const int64_t row = ikv::row_q8(blk, c.n_head_kv, g, b.bt, at);
        const int64_t from = row * c.dim + min(d, c.dim - 4);
        w[0][j] = *reinterpret_cast<const unsigned *>(c.k + from);
        w[1][j] = *reinterpret_cast<const unsigned *>(c.v + from);
        scale[0][j] = c.k_scale[row];
        scale[1][j] = c.v_scale[row];
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int g = g0 + j * kHeads + h;
        if (g >= c.n_head_kv || d >= c.dim) continue;
        *reinterpret_cast<float4 *>(kr + g * c.dim + d) = ikv::scale4(scale[0][j], ikv::values_q8<E4M3>(w[0][j]));
        *reinterpret_cast<float4 *>(vr + g * c.dim + d) = ikv::scale4(scale[1][j], ikv::values_q8<E4M3>(w[1][j]));
      }
    }
  }
}

// f(whether e4m3, lanes of a row) as constants
template <class F>
void with_form(const ikv::CacheQ8 &c, F &&f) {
  auto by_lanes = [&](auto e4m3) {
    if (c.dim <= 64)
      f(e4m3, std::integral_constant<int, 16>{});
    else if (c.dim <= 128)
      f(e4m3, std::integral_constant<int, 32>{});
    else
      f(e4m3, std::integral_constant<int, 64>{});
  };
  if (c.e4m3)
    by_lanes(std::true_type{});
  else
    by_lanes(std::false_type{});
}

// What the two entry points check alike; 1: nothing to do.
int rows_arg(const ikv_kv_q8 *cache, const ikv_kv_batch *batch, const float *k_rows, const float *v_rows,
             const int32_t *row_start, int64_t n_rows, ikv::CacheQ8 &c, ikv::BatchPages &b) {
  if (const int rc = ikv::batch_arg(batch, b)) return rc;
  if (const int rc = ikv::cache_q8_arg(cache, c)) return rc;
  if (n_rows < 0) return -EINVAL;
  if (n_rows == 0 || b.n_seq == 0) return 1;
  if (!ikv::cache_q8_there(c) || !k_rows || !v_rows || !row_start || !ikv::aligned16(k_rows) ||
      !ikv::aligned16(v_rows))
    return -EINVAL;
  return n_rows > INT_MAX ? -EOVERFLOW : 0;
}

unsigned grid_of(int64_t n_rows) {
  return static_cast<unsigned>(std::min<int64_t>((n_rows + kRowWaves - 1) / kRowWaves, 65536));
}

}  // namespace

extern "C" int ikv_append_packed_q8(const ikv_kv_q8 *cache, const float *k_rows, const float *v_rows,
                                    const ikv_kv_batch *batch, const int32_t *row_start,
                                    const int32_t *first_token, int64_t n_rows, void *stream) {
  ikv::CacheQ8 c;
  ikv::BatchPages b;
  if (const int rc = rows_arg(cache, batch, k_rows, v_rows, row_start, n_rows, c, b)) return rc < 0 ? rc : 0;
  with_form(c, [&](auto e4m3, auto lanes) {
    append_q8_kernel<e4m3.value, lanes.value><<<grid_of(n_rows), kRowWaves * 64, 0, static_cast<hipStream_t>(stream)>>>(
        c, k_rows, v_rows, b, row_start, first_token, n_rows);
  });
  return ikv::launch_status();
}

extern "C" int ikv_read_packed_q8(const ikv_kv_q8 *cache, float *k_rows, float *v_rows,
                                  const ikv_kv_batch *batch, const int32_t *row_start,
                                  const int32_t *first_token, const int32_t *n_kv, int64_t n_rows,
                                  void *stream) {
  ikv::CacheQ8 c;
  ikv::BatchPages b;
  if (const int rc = rows_arg(cache, batch, k_rows, v_rows, row_start, n_rows, c, b)) return rc < 0 ? rc : 0;
  with_form(c, [&](auto e4m3, auto lanes) {
    read_q8_kernel<e4m3.value, lanes.value><<<grid_of(n_rows), kRowWaves * 64, 0, static_cast<hipStream_t>(stream)>>>(
        c, k_rows, v_rows, b, row_start, first_token, n_kv, n_rows);
  });
  return ikv::launch_status();
}
