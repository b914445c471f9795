// attn_decode_q8.hip — one new token of each of several sequences over a paged cache
// of 8 bits an element (ikv_attn_decode_batch_q8), the new rows' append fused.
//
// The codes of a KV head are read once, so HBM bounds it as long as what is done
// with a byte keeps up. At G query heads a byte takes 4 G flops and its conversion;
// on the vector pipe that is more than the reads leave time for from G = 4 on, so
// both products are on the matrix pipe. An int8 or e4m3 code is a bf16 number as it
// stands; queries and weights are three bf16 pieces that add up to the float
// (bf16x3.hpp), so the products are exact and the sums F32.
//
//   * The runs of units of decode_runs.hpp, a unit of 64 keys, each wave of a
//     workgroup taking whole units: nothing is shared until the waves meet.
//   * S^T = K Q^T: 16 keys by 16 query heads of one KV head, of which G are there,
//     a step of 32 dims. O^T += V^T P^T: 16 dims by 16 heads, a step of 32 keys.
//     A lane holds one head in both, so weights go from the softmax into the second
//     product in place, and its maximum and sum are the lane's own.
//   * The key's K scale multiplies its scores, its V scale its weights.
//   * A lane reads its K codes 16 bytes at a time and its V codes, 8 keys by 4 W
//     dims, a key at a time; V's transpose is the choice of registers when two
//     converted codes are packed. The registers of half a unit's codes are loaded
//     again, with the next unit's, as soon as the half is in the products (48 long
//     contexts 122 -> 113 us).
// Measured (MI355X, us): 48 contexts of up to 16384 tokens, 32 heads of 128 over 8, 554
// MB: 105, 5.3 TB/s, with the append 4 more; of up to 110000, 5 GB: 763, 6.6 TB/s; as
// much in e4m3. The first in F32, 2.4 GB: 371. 37 of up to 5003, 12 heads of 64 over 4,
// 33 MB: 19, with the append 20.5, most of it the start (lengths, tables, first codes),
// two units one behind the other in a wave and the join; three of up to 52 and an idle
// slot 8 by the trace, one unit each. Neither pipe bounds the 554 MB: matrix
// instructions are issued in 19 % of the cycles, vector ones in 36 %; 23 % of the waves'
// time is waits for memory, 43 % for a place to issue.
#include "cache_q8.hpp"
#include "bf16x3.hpp"
#include "decode_runs.hpp"

#include <type_traits>

namespace {

using namespace ikv::pieces;

constexpr int kWaves = 4;  // of a workgroup
constexpr int KT = 64;     // keys of a unit
// One run a workgroup, however many units (decode_runs.hpp). 48 contexts of 32 heads of
// 128 over 8, equal shares against runs of 64 units, taken as workgroups come free: 39000
// units 118 and 130 us, 57000 162 and 179, 113000 304 and 320, 297000 770 and 785; heads
// of 64, 33000 units 57 and 75; of 256, 21000 160 and 198. (As many whole rounds of equal
// runs: 133, 183, 322, 782, 70 and 161.)
constexpr int kRunUnits = 0, kWhole = 8;
// Fewest units of a run of long contexts: the workgroup that joins a context's parts
// reads all of them, and they grow with the query heads. 16 heads of 80 over 1: 2
// contexts of 16000 tokens 116 us in runs of one unit, 33 of eight, 15 of up to 13800 53
// and 33; but 16 heads of 128 over 8, 16 contexts of up to 1500, 19.4 and 22.4.
constexpr int least_of(int gq) { return gq / 2; }
// Cache policy of the values' loads: non-temporal, as each line is read once (48 long
// contexts 115 -> 108.5 us; 110 with the keys' too, of which two loads read a line; both
// before a workgroup had one run).
constexpr int kOnce = 2;
constexpr float kRescale = 8.0f;  // log2 headroom before the running maximum is moved
constexpr int groups_of(int w) { return w > 2 ? 256 : 512; }

struct Args {
  const float *q;
  ikv::CacheQ8 c;
  const float *k_new, *v_new;
  float *out;
  const int32_t *n_kv;
  ikv::BatchPages b;
  int n_head_kv, G;
  int passes;  // a KV head's query heads are taken GQ at a time
  float scale_log2;
  float *part;
};

// Keys of a sequence; 0 for an idle slot and for a length that is out of range.
__device__ __forceinline__ int keys_of(const Args &a, int seq) {
  const int n = a.n_kv[seq];
  return n > 0 && n <= a.b.capacity ? n : 0;
}

// The high halfs of two floats that are bf16 numbers.
__device__ __forceinline__ unsigned pack2(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// 8 codes as they lie.
template <bool E4M3>
__device__ __forceinline__ bf16x8 bf16_of(uint2 w) {
  const float4 a = ikv::values_q8<E4M3>(w.x), b = ikv::values_q8<E4M3>(w.y);
  return __builtin_bit_cast(bf16x8, uintx4{pack2(a.x, a.y), pack2(a.z, a.w), pack2(b.x, b.y), pack2(b.z, b.w)});
}

// A wave-wide value over the lanes that hold one head.
template <class F>
__device__ __forceinline__ float quarters(float x, F &&f) {
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = f(__uint_as_float(b[0]), __uint_as_float(b[1]));
  const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(c[0]), __uint_as_float(c[1]));
}

template <int W, int GQ, bool E4M3>
__global__ __launch_bounds__(kWaves * 64, W > 2 ? 1 : 2) void decode_q8_kernel(Args a) {
  constexpr int DP = 64 * W;  // dims held
  constexpr int DB = 4 * W;   // of V, of a lane
  __shared__ ikv::Meet<GQ, DP, kWaves> s_meet;
  constexpr int kSteps = 2 * W;  // of 32 dims (a lane's 8: 16 (quad + 4 w) + 8 z)
  __shared__ __attribute__((aligned(16))) uint8_t s_new[2][DP];  // the new token's codes
  __shared__ bf16x8 s_q[kSteps][3][64];  // the query rows' pieces, as the lanes take them
  __shared__ __attribute__((aligned(16))) float s_scale[kWaves][2][KT];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int n_head = a.n_head_kv * a.G, dim = a.c.dim;

  // slots without keys: a zero row, and the flag where the length is no length
  for (int s = gridDim.x - 1 - blockIdx.x; s < a.b.n_seq; s += gridDim.x) {
    if (keys_of(a, s) > 0) continue;
    if (a.n_kv[s] != 0 && threadIdx.x == 0) ikv::raise_status(a.b.status, IKV_STATUS_POSITION);
    float *o = a.out + static_cast<size_t>(s) * n_head * dim;
    for (int d = threadIdx.x; d < n_head * dim; d += kWaves * 64) o[d] = 0.f;
  }

  constexpr int kGroups = groups_of(W);
  ikv::Plan<Args, KT, kGroups, kRunUnits, kWhole, least_of(GQ)> plan(a);
  const ikv::Parts<GQ, DP, kGroups> parts(a.part);
  // this lane's bytes of a unit's rows: of K row 32 (T / 2) + 8 (col / 4) + 4 (T % 2)
  // + col % 4 of tile T (so that the two tiles of a product with V leave lane quarter
  // quad the scores of keys 8 quad .. + 7), of V rows 32 u + 8 quad + i
  constexpr unsigned kOut = 0x80000000u;
  unsigned k_off[W];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int d = 16 * (quad + 4 * w);
    k_off[w] = d < dim ? static_cast<unsigned>((8 * (col >> 2) + (col & 3)) * dim + d) : kOut;
  }
  const unsigned v_off = DB * col < dim ? static_cast<unsigned>(8 * quad * dim + DB * col) : kOut;

  const int run = blockIdx.x;
  unsigned long long u = plan.chunk * run;
  const unsigned long long end = min(plan.total, u + plan.chunk);
  ikv::Place p{};
  if (u < end) p = plan.at(a, u);
  while (u < end) {
    if (plan.kept(p.tiles) && p.tile > 0) {  // (with the run that holds its first unit)
      u += p.tiles - p.tile;
      plan.next(a, p);
      continue;
    }
    const int last =
        plan.kept(p.tiles) ? p.tiles : static_cast<int>(min<unsigned long long>(p.tiles, p.tile + (end - u)));
    const int g = p.item / a.passes, h0 = p.item % a.passes * GQ;
    const int heads = min(GQ, a.G - h0);
    const ikv::Pages pg = ikv::pages_of(a.b, p.seq);
    const size_t head0 = static_cast<size_t>(p.seq) * n_head + g * a.G + h0;

    floatx4 o[DB];
#pragma unroll
    for (int j = 0; j < DB; ++j) o[j] = floatx4{};
    float m = -INFINITY, sum = 0.f;

    // block table entries, 64 at a time, one per lane, checked as they are read
    const int last_blk = (p.keys - 1) / pg.bt;
    // this wave's units, t0, t0 + kWaves, ..., those of its number in the whole list: each
    // wave has as many of a run as any other, or one more
    const int t0 = p.tile + ((wave - static_cast<int>(u)) & (kWaves - 1));
    int blk = t0 * KT / pg.bt, in_blk = t0 * KT % pg.bt, ent0 = blk, ent = 0;
    auto entries = [&]() {
      ent0 = blk;
      ent = pg.table[min(blk + lane, last_blk)];
      if (static_cast<unsigned>(ent) >= static_cast<unsigned>(pg.n_blocks)) {
        ikv::raise_status(pg.status, IKV_STATUS_BLOCK);
        ent = -1;
      }
    };
    const bool has_new = a.k_new != nullptr && last == p.tiles;
    const int cached = p.keys - (a.k_new ? 1 : 0);  // keys that are read from the cache
    // this head's first row of the unit at (blk, in_blk), moved on to the next one;
    // ~row of block 0's where the entry names no block
    auto next_row = [&]() -> int64_t {
      const int e = __builtin_amdgcn_readlane(ent, blk - ent0);
      const int64_t row = ikv::row_q8(max(e, 0), a.n_head_kv, g, pg.bt, in_blk);
      in_blk = ikv::uniform(in_blk + kWaves * KT);
      while (in_blk >= pg.bt) {
        in_blk -= pg.bt;
        ++blk;
      }
      if (blk - ent0 >= 64) entries();
      return ikv::uniform(e < 0 ? ~row : row);
    };
    uint4 kr[4][W];
    unsigned vr[2][8][W];
    float ks, vs;  // of key `lane`
    auto rsrc = [&](const void *base, int64_t byte, int bytes) {
      return __builtin_amdgcn_make_buffer_rsrc(static_cast<uint8_t *>(const_cast<void *>(base)) + byte, 0, bytes,
                                               ikv::kBufWord3);
    };
    // A unit's resources: codes and scales; of a unit behind the run no memory is read.
    // The row part of an offset is not checked against the size: rows behind the last
    // token are read (they are in the block) and masked.
    struct Unit {
      __amdgpu_buffer_rsrc_t k, v, ks, vs;
    };
    auto unit_at = [&](int64_t row, int t) {
      const int rows = ikv::uniform(t < last ? max(0, min(KT, cached - t * KT)) : 0);
      row = row < 0 ? ~row : row;
      return Unit{rsrc(a.c.k, row * dim, rows * dim), rsrc(a.c.v, row * dim, rows * dim),
                  rsrc(a.c.k_scale, row * 4, rows * 4), rsrc(a.c.v_scale, row * 4, rows * 4)};
    };
    auto fetch_k = [&](const Unit &r, int h) {  // the keys 32 h .. + 31
#pragma unroll
      for (int T = 2 * h; T < 2 * h + 2; ++T)
#pragma unroll
        for (int w = 0; w < W; ++w)
          kr[T][w] = __builtin_bit_cast(
              uint4, __builtin_amdgcn_raw_buffer_load_b128(r.k, k_off[w], (32 * h + 4 * (T & 1)) * dim, 0));
    };
    auto fetch_v = [&](const Unit &r, int h) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = (32 * h + i) * dim;
        if constexpr (W == 1) {
          vr[h][i][0] = __builtin_amdgcn_raw_buffer_load_b32(r.v, v_off, at, kOnce);
        } else if constexpr (W == 2) {
          const auto x = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(r.v, v_off, at, kOnce));
          vr[h][i][0] = x.x, vr[h][i][1] = x.y;
        } else {
          const auto x = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r.v, v_off, at, kOnce));
          vr[h][i][0] = x.x, vr[h][i][1] = x.y, vr[h][i][2] = x.z, vr[h][i][3] = x.w;
        }
      }
    };
    auto fetch_scales = [&](const Unit &r) {
      ks = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r.ks, 4 * lane, 0, 0));
      vs = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r.vs, 4 * lane, 0, 0));
    };

    entries();
    // the query rows, a step a wave
    floatx4 qr[(kSteps + kWaves - 1) / kWaves][2] = {};
#pragma unroll
    for (int i = 0; i < (kSteps + kWaves - 1) / kWaves; ++i) {
      const int step = wave + kWaves * i, d = 16 * (quad + 4 * (step >> 1)) + 8 * (step & 1);
      const float *const row = a.q + (head0 + min(col, heads - 1)) * dim;
      if (step < kSteps && col < heads && d < dim) {
        qr[i][0] = *reinterpret_cast<const floatx4 *>(row + d);
        qr[i][1] = *reinterpret_cast<const floatx4 *>(row + d + 4);
      }
    }
    // the new token: its codes and scales, by the wave that has the last unit
    float new_scale[2] = {0.f, 0.f};
    const bool mine = has_new && t0 < last && (p.tiles - 1 - t0) % kWaves == 0;
    float4 new_row[2] = {};
    if (mine && 4 * lane < dim) {
      const size_t at = (static_cast<size_t>(p.seq) * a.n_head_kv + g) * dim + 4 * lane;
      new_row[0] = *reinterpret_cast<const float4 *>(a.k_new + at);
      new_row[1] = *reinterpret_cast<const float4 *>(a.v_new + at);
    }
    {
      const Unit r = unit_at(next_row(), t0);
      fetch_scales(r);
      fetch_k(r, 0);
      fetch_k(r, 1);
      fetch_v(r, 0);
      fetch_v(r, 1);
    }
#pragma unroll
    for (int i = 0; i < (kSteps + kWaves - 1) / kWaves; ++i) {
      const int step = wave + kWaves * i;
      if (step >= kSteps) break;
      unsigned none = 0;
      const Pieces x = split8<false>(qr[i][0] * a.scale_log2, qr[i][1] * a.scale_log2, none);
#pragma unroll
      for (int z = 0; z < 3; ++z) s_q[step][z][lane] = x.p[z];
    }
    if (mine) {
      unsigned codes[2];
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const float4 x = new_row[z];
        const ikv::Quant<E4M3> quant(ikv::lanes_max<64>(
            max(max(ikv::abs_bits(x.x), ikv::abs_bits(x.y)), max(ikv::abs_bits(x.z), ikv::abs_bits(x.w)))));
        new_scale[z] = quant.scale;
        codes[z] = quant.codes(x);
        if (4 * lane < DP) *reinterpret_cast<unsigned *>(&s_new[z][4 * lane]) = codes[z];
      }
      const int e = pg.table[last_blk];
      if (h0 == 0 && static_cast<unsigned>(e) < static_cast<unsigned>(pg.n_blocks)) {
        const int64_t to = ikv::row_q8(e, a.n_head_kv, g, pg.bt, (p.keys - 1) % pg.bt);
        if (4 * lane < dim) {
          *reinterpret_cast<unsigned *>(a.c.k + to * dim + 4 * lane) = codes[0];
          *reinterpret_cast<unsigned *>(a.c.v + to * dim + 4 * lane) = codes[1];
        }
        if (lane == 0) {
          a.c.k_scale[to] = new_scale[0];
          a.c.v_scale[to] = new_scale[1];
        }
      }
    }
    __syncthreads();
    for (int t = t0; t < last; t += kWaves) {
        const bool fresh = mine && t == p.tiles - 1;
        const int at = cached - t * KT;  // the new token's place in the unit
        if (fresh) {
#pragma unroll
          for (int T = 0; T < 4; ++T)
#pragma unroll
            for (int w = 0; w < W; ++w)
              if (32 * (T >> 1) + 8 * (col >> 2) + 4 * (T & 1) + (col & 3) == at)
                kr[T][w] = *reinterpret_cast<const uint4 *>(&s_new[0][16 * (quad + 4 * w)]);
#pragma unroll
          for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (32 * z + 8 * quad + i == at) {
#pragma unroll
                for (int w = 0; w < W; ++w)
                  vr[z][i][w] = *reinterpret_cast<const unsigned *>(&s_new[1][DB * col + 4 * w]);
              }
          if (lane == at) {
            ks = new_scale[0];
            vs = new_scale[1];
          }
        }
        s_scale[wave][0][lane] = ks;
        s_scale[wave][1][lane] = vs;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        auto scales = [&](int z, int T) {  // of this lane's keys of tile T
          return *reinterpret_cast<const floatx4 *>(&s_scale[wave][z][32 * (T >> 1) + 8 * quad + 4 * (T & 1)]);
        };
        // scores of keys 32 (T / 2) + 8 quad + 4 (T % 2) + e with this lane's head
        // each half of the codes is loaded again as soon as it is in the products
        const Unit r = unit_at(next_row(), t + kWaves);
        fetch_scales(r);
        floatx4 s[4] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int step = 0; step < kSteps; ++step) {
            bf16x8 qp[3];
#pragma unroll
            for (int i = 0; i < 3; ++i) qp[i] = s_q[step][i][lane];
#pragma unroll
            for (int T = 2 * h; T < 2 * h + 2; ++T) {
              const uint4 y = kr[T][step / 2];
              const bf16x8 x = bf16_of<E4M3>(step % 2 == 0 ? make_uint2(y.x, y.y) : make_uint2(y.z, y.w));
#pragma unroll
              for (int i = 2; i >= 0; --i) s[T] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, qp[i], s[T], 0, 0, 0);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
          fetch_k(r, h);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int T = 0; T < 4; ++T) s[T] *= scales(0, T);
        const int keys = p.keys - t * KT;
        if (keys < KT) {
#pragma unroll
          for (int T = 0; T < 4; ++T)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (32 * (T >> 1) + 8 * quad + 4 * (T & 1) + e >= keys) s[T][e] = -INFINITY;
          // (a weight of 0 would not silence a NaN)
#pragma unroll
          for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (32 * z + 8 * quad + i >= keys) {
#pragma unroll
                for (int w = 0; w < W; ++w) vr[z][i][w] = 0;
              }
        }
        float mt = s[0][0];
#pragma unroll
        for (int T = 0; T < 4; ++T)
#pragma unroll
          for (int e = 0; e < 4; ++e) mt = fmaxf(mt, s[T][e]);
        if (__builtin_amdgcn_ballot_w64(mt > m + kRescale) != 0) {
          const float top = fmaxf(m, quarters(mt, [](float x, float y) { return fmaxf(x, y); }));
          const float f = ikv::weight(m, top);
          m = top;
          sum *= f;
#pragma unroll
          for (int j = 0; j < DB; ++j) o[j] *= f;
        }
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          floatx4 x[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const floatx4 scale = scales(1, 2 * z + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w = ikv::fast_exp2(s[2 * z + i][e] - ref);
              sum += w;
              x[i][e] = w * scale[e];
            }
          }
          unsigned none = 0;
          const Pieces pw = split8<false>(x[0], x[1], none);
#pragma unroll
          for (int w = 0; w < W; ++w) {
            float4 y[8];  // dims DB col + 4 w .. + 3 of keys 32 z + 8 quad ..
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = ikv::values_q8<E4M3>(vr[z][i][w]);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              auto at_d = [&](int i) { return d == 0 ? y[i].x : d == 1 ? y[i].y : d == 2 ? y[i].z : y[i].w; };
              const bf16x8 v = __builtin_bit_cast(
                  bf16x8, uintx4{pack2(at_d(0), at_d(1)), pack2(at_d(2), at_d(3)), pack2(at_d(4), at_d(5)),
                                 pack2(at_d(6), at_d(7))});
#pragma unroll
              for (int i = 2; i >= 0; --i)
                o[4 * w + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pw.p[i], o[4 * w + d], 0, 0, 0);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
          fetch_v(r, z);
          __builtin_amdgcn_sched_barrier(0);
        }
    }

    // the waves meet: this lane has dims DB (4 quad + e) + j of its head
    sum = quarters(sum, [](float x, float y) { return x + y; });
    if (col < heads) {
      if (quad == 0) {
        s_meet.m[wave][col] = m;
        s_meet.l[wave][col] = sum;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int w = 0; w < W; ++w)
          *reinterpret_cast<float4 *>(&s_meet.o[wave][col][DB * (4 * quad + e) + 4 * w]) =
              make_float4(o[4 * w][e], o[4 * w + 1][e], o[4 * w + 2][e], o[4 * w + 3][e]);
    }
    __syncthreads();
    ikv::leave(s_meet, plan, parts, run, u, p, last, heads, dim, [&](int h, int d, float, float all, float x, float y) {
      if (d < dim) *reinterpret_cast<float2 *>(a.out + (head0 + h) * dim + d) = make_float2(x / all, y / all);
    });
    __syncthreads();
    u += last - p.tile;
    plan.next(a, p);
  }
}

// The form of a shape: 64 dims at a time, query heads taken at once.
int wide_of(int dim) { return dim <= 64 ? 1 : dim <= 128 ? 2 : 4; }
int heads_of(int G) { return G <= 4 ? 4 : G <= 8 ? 8 : 16; }

}  // namespace

extern "C" size_t ikv_attn_decode_batch_q8_workspace_bytes(int n_head, int n_head_kv, int head_dim) {
  if (n_head <= 0 || n_head_kv <= 0 || n_head % n_head_kv != 0 || head_dim <= 0 || head_dim % 16 != 0 ||
      head_dim > ikv::kMaxDimQ8)
    return 0;
  const int w = wide_of(head_dim);
  return ikv::parts_bytes(heads_of(n_head / n_head_kv), 64 * w, groups_of(w));
}

extern "C" int ikv_attn_decode_batch_q8(const float *q, const ikv_kv_q8 *cache, const ikv_kv_batch *batch,
                                        const int32_t *n_kv, const float *k_new, const float *v_new, float *out,
                                        int n_head, float scale, void *workspace, size_t workspace_bytes,
                                        void *stream) {
  Args a;
  if (const int rc = ikv::batch_arg(batch, a.b)) return rc;
  if (const int rc = ikv::cache_q8_arg(cache, a.c)) return rc;
  const int n_head_kv = a.c.n_head_kv, dim = a.c.dim;
  if (n_head <= 0 || n_head % n_head_kv != 0) return -EINVAL;
  if (a.b.n_seq == 0) return 0;
  if (!q || !ikv::cache_q8_there(a.c) || !n_kv || !out || (k_new == nullptr) != (v_new == nullptr)) return -EINVAL;
  for (const void *x : {static_cast<const void *>(q), static_cast<const void *>(k_new),
                        static_cast<const void *>(v_new), static_cast<const void *>(out), static_cast<const void *>(workspace)})
    if (!ikv::aligned16(x)) return -EINVAL;
  if (!workspace || workspace_bytes < ikv_attn_decode_batch_q8_workspace_bytes(n_head, n_head_kv, dim)) return -EINVAL;
  if (n_head > INT_MAX / dim) return -EOVERFLOW;  // a sequence's heads index in int
  if (!(scale > 0.0f)) scale = 1.0f / sqrtf(static_cast<float>(dim));
  a.q = q;
  a.k_new = k_new;
  a.v_new = v_new;
  a.out = out;
  a.n_kv = n_kv;
  a.n_head_kv = n_head_kv;
  a.G = n_head / n_head_kv;
  const int gq = heads_of(a.G), w = wide_of(dim);
  a.passes = (a.G + gq - 1) / gq;
  a.scale_log2 = scale * ikv::kLog2e;
  a.part = static_cast<float *>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto wc, auto gc) {
    constexpr int W = wc.value, GQ = gc.value;
    if (a.c.e4m3)
      decode_q8_kernel<W, GQ, true><<<groups_of(W), kWaves * 64, 0, s>>>(a);
    else
      decode_q8_kernel<W, GQ, false><<<groups_of(W), kWaves * 64, 0, s>>>(a);
  };
  auto by_heads = [&](auto wc) {
    if (gq == 4)
      launch(wc, std::integral_constant<int, 4>{});
    else if (gq == 8)
      launch(wc, std::integral_constant<int, 8>{});
    else
      launch(wc, std::integral_constant<int, 16>{});
  };
  if (w == 1)
    by_heads(std::integral_constant<int, 1>{});
  else if (w == 2)
    by_heads(std::integral_constant<int, 2>{});
  else
    by_heads(std::integral_constant<int, 4>{});
  return ikv::launch_status();
}
