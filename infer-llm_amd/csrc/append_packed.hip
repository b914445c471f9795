// append_packed.hip — the K and V rows of several sequences' new tokens into
// their pages, one launch (ikv_append_packed_f32).
//
// A copy: each byte is read once and written once, so HBM bounds it. A wave
// takes a packed row of K and the same one of V: its sequence is found once by
// the whole wave (wave_find_last), its block is one table entry, and the lanes
// copy the two rows in 16-byte pieces. 8190 rows of 8 heads of 128 into 24
// sequences, 134 MB: 28 us with the rows in memory, 4.8 TB/s, the rate of a
// large copy; 211 rows into 5: 3.8 us, a launch and three loads one after the
// other. Non-temporal loads and stores: 26.6 us against 22.8 where the rows are
// still in the last cache, as they are behind the projection that made them.
#include "batch.hpp"

namespace {

constexpr int kRowWaves = 4;  // rows of a workgroup, one per wave

template <class Piece>
__global__ __launch_bounds__(kRowWaves * 64) void append_packed_kernel(
    Piece *__restrict__ k_pool, Piece *__restrict__ v_pool, const Piece *__restrict__ k_rows,
    const Piece *__restrict__ v_rows, ikv::BatchPages b, const int32_t *__restrict__ row_start,
    const int32_t *__restrict__ first_token, int64_t n_rows, int64_t per_row) {
  ikv::check_row_start(row_start, b.n_seq, n_rows, b.status);
  const int lane = threadIdx.x & 63;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRowWaves;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kRowWaves + (threadIdx.x >> 6); i < n_rows; i += step) {
    const int seq = ikv::wave_find_last(b.n_seq, [&](int s) { return row_start[s] <= i; });
    if (seq < 0 || i >= row_start[seq + 1]) continue;  // a row of no sequence
    const int64_t t = (first_token ? first_token[seq] : 0) + (i - row_start[seq]);
    if (t < 0 || t >= b.capacity) {
      ikv::raise_status(b.status, IKV_STATUS_POSITION);
      continue;
    }
    const int blk = b.tables[seq * b.stride + t / b.bt];
    if (static_cast<unsigned>(blk) >= static_cast<unsigned>(b.n_blocks)) {
      ikv::raise_status(b.status, IKV_STATUS_BLOCK);  // dropped: no block to write
      continue;
    }
    const int64_t to = (static_cast<int64_t>(blk) * b.bt + t % b.bt) * per_row, from = i * per_row;
    for (int64_t c = lane; c < per_row; c += 64) {
      const Piece x = k_rows[from + c], y = v_rows[from + c];
      k_pool[to + c] = x;
      v_pool[to + c] = y;
    }
  }
}

}  // namespace

extern "C" int ikv_append_packed_f32(void *k_pool, void *v_pool, const void *k_rows, const void *v_rows,
                                     const ikv_kv_batch *batch, const int32_t *row_start,
                                     const int32_t *first_token, int64_t n_rows, size_t row_bytes,
                                     void *stream) {
  ikv::BatchPages b;
  if (const int rc = ikv::batch_arg(batch, b)) return rc;
  if (n_rows < 0 || row_bytes % 4 != 0) return -EINVAL;
  if (n_rows == 0 || row_bytes == 0 || b.n_seq == 0) return 0;
  if (!k_pool || !v_pool || !k_rows || !v_rows || !row_start) return -EINVAL;
  if (n_rows > INT_MAX || row_bytes > static_cast<size_t>(INT64_MAX) / INT_MAX) return -EOVERFLOW;
  uintptr_t any = row_bytes;
  for (const void *p : {static_cast<const void *>(k_pool), static_cast<const void *>(v_pool), k_rows, v_rows})
    any |= reinterpret_cast<uintptr_t>(p);
  if (any % 4 != 0) return -EINVAL;
  const int64_t wgs = (n_rows + kRowWaves - 1) / kRowWaves;
  const unsigned grid = static_cast<unsigned>(wgs < 65536 ? wgs : 65536);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto piece) {
    using Piece = decltype(piece);
    append_packed_kernel<Piece><<<grid, kRowWaves * 64, 0, s>>>(
        static_cast<Piece *>(k_pool), static_cast<Piece *>(v_pool), static_cast<const Piece *>(k_rows),
        static_cast<const Piece *>(v_rows), b, row_start, first_token, n_rows,
        static_cast<int64_t>(row_bytes / sizeof(Piece)));
  };
  if (any % 16 == 0)
    launch(uint4{});
  else
    launch(uint32_t{});
  return ikv::launch_status();
}
