// partition_kernels.hpp -- the products of ragged groups of queries with the paged rows of their partitions (include/rsgpu_rows.h) on
// gfx950.  Included by one source file for each type of queries, partition_{f32,f16,bf16}.hip, which compile side by side.
#pragma once
#include <type_traits>

#include "rows_device.hpp"

namespace rsgpu {
namespace {

// ---- products with a partition's rows --------------------------------------------------------------------------------------
//
// p[m][j] = sum_k q[m][k] c[j][k] s[j][k / block].  The codes are integers or e4m3 values that a 16-bit float holds exactly, so the
// matrix cores multiply codes with queries, and a block's sum is multiplied by its scale in fp32: no operand is rounded.
// fp32 operands go in as three bf16 each, exactly.

template <int Q>
__device__ __forceinline__ f32x16 mfma(u4 a, u4 b, f32x16 c) {
  if constexpr (Q == F16) {
    half8 x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
  } else {
    bf16x8 x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
  }
}

template <int Q>
__device__ __forceinline__ f32x4 mfma16(u4 a, u4 b, f32x4 c) {
  if constexpr (Q == F16) {
    half8 x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
  } else {
    bf16x8 x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
  }
}

__device__ __forceinline__ uint32_t upper2(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }
__device__ __forceinline__ float low_bf16(uint32_t two) { return __uint_as_float(two << 16); }
__device__ __forceinline__ float high_bf16(uint32_t two) { return __uint_as_float(two & 0xffff0000u); }

// what is left of x behind the nearest bf16 (`hi`, which is cut off instead where the nearest is an infinity and x is not)
__device__ __forceinline__ float behind(float x, float &hi) {
  const float a = __builtin_fabsf(x);
  if (a >= 0x1.ffp127f) hi = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  return a == __builtin_inff() ? 0.0f : x - hi;
}

// Eight fp32 -> eight bf16 in each of three planes, x = hi + mid + lo exactly: hi and mid are rounded to the nearest, so that mid is at
// most 2^-8 of x's binade and lo 2^-17, of either sign.  (Cut off, as upper halves are, they are twice that and all of x's sign: what the
// products leave out came to 2^-21 of a product, and to 2^-24 of every sum of products of one sign.)  An infinity is hi alone.
__device__ __forceinline__ void planes8(const float (&v)[8], u4 (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t near = narrow2<BF16>(v[2 * i], v[2 * i + 1]);
    float a = low_bf16(near), b = high_bf16(near);
    const float ra = behind(v[2 * i], a), rb = behind(v[2 * i + 1], b);
    const uint32_t mid = narrow2<BF16>(ra, rb);
    p[0][i] = upper2(__float_as_uint(a), __float_as_uint(b));
    p[1][i] = mid;
    p[2][i] = upper2(__float_as_uint(ra - low_bf16(mid)), __float_as_uint(rb - high_bf16(mid)));
  }
}

// bf16 and fp32 queries reach 2^128, and codes are summed before they meet their scale: 65 536 elements times codes of up to 448 would
// leave fp32 where the score, of rows of thousandths, does not.  So one side goes in by SHRUNK, exactly, and the score is multiplied by
// what that was when its scales are in it: no sum overflows unless the score's own sums do.  (fp16 queries times codes stay below
// 2^41.)  It costs what of a query's elements lies below 2^-107, or of a score below 2^-119.  Which side: codes where their conversion
// does it for nothing (E4M3) or where rows are converted no more often than queries (many queries: 1 - 4 % of the time), else queries,
// once a partition (8 x 700 INT8 rows of 768, fp32 queries: queries 8.3 us as without, codes 8.8).
constexpr float SHRUNK = 0x1p-26f;
enum { BY_NOTHING = 0, BY_CODES = 1, BY_QUERIES = 2 };
template <int FMT, int Q, bool MANY>
constexpr int SHRINK = FMT == NATIVE || Q == F16 ? BY_NOTHING : FMT == E4M3 || MANY ? BY_CODES : BY_QUERIES;

// eight codes -> eight 16-bit floats, STEP for a code of 1 (INT4 with bf16: by sixteenths if not by SHRUNK)
template <int FMT, int Q, int BY>
constexpr float STEP = BY == BY_CODES ? SHRUNK : FMT == INT4 && Q != F16 ? 0.0625f : 1.0f;
// what a sum of products is multiplied by
template <int FMT, int Q, int BY>
constexpr float UNIT = 1.0f / STEP<FMT, Q, BY> / (BY == BY_QUERIES ? SHRUNK : 1.0f);

__device__ __forceinline__ uint32_t minus2(uint32_t x, float y) {
  half2v h;
  __builtin_memcpy(&h, &x, 4);
  h -= half2v{(_Float16)y, (_Float16)y};
  __builtin_memcpy(&x, &h, 4);
  return x;
}

template <int FMT, int Q, int BY>
__device__ __forceinline__ u4 widen8(uint32_t w0, uint32_t w1) {
  constexpr float ONE = STEP<FMT, Q, BY>;
  u4 r;
  if constexpr (FMT == E4M3) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int w = (int)(i < 2 ? w0 : w1);
      if constexpr (Q == F16) {
        const half2v h = i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
        uint32_t x;
        __builtin_memcpy(&x, &h, 4);
        r[i] = x;
      } else {
        const bf16x2 h = i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, ONE, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, ONE, false);
        uint32_t x;
        __builtin_memcpy(&x, &h, 4);
        r[i] = x;
      }
    }
  } else if constexpr (Q == F16) {
    // an fp16 number in [1024, 2048) has its integer in the low bits: 1024 + (code + bias), and the bias goes off exactly
    if constexpr (FMT == INT8) {
      const uint32_t a = w0 ^ 0x80808080u, b = w1 ^ 0x80808080u;
      r = u4{minus2(__builtin_amdgcn_perm(0x64646464u, a, 0x04010400u), 1152.0f), minus2(__builtin_amdgcn_perm(0x64646464u, a, 0x04030402u), 1152.0f),
             minus2(__builtin_amdgcn_perm(0x64646464u, b, 0x04010400u), 1152.0f), minus2(__builtin_amdgcn_perm(0x64646464u, b, 0x04030402u), 1152.0f)};
    } else {
      const uint32_t t = w0 ^ 0x88888888u, even = t & 0x0f0f0f0fu, odd = t >> 4 & 0x0f0f0f0fu;
#pragma unroll
      for (int i = 0; i < 4; i++) r[i] = minus2(__builtin_amdgcn_perm(odd, even, 0x0c040c00u + 0x00010001u * i) | 0x64006400u, 1032.0f);
    }
  } else {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if constexpr (FMT == INT8) f[i] = (float)(int8_t)((i < 4 ? w0 : w1) >> (8 * (i % 4)));
      else f[i] = __builtin_amdgcn_cvt_off_f32_i4((int)(w0 >> (4 * i)));   // the low four bits, two's complement, by 16
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      uint32_t two = upper2(__float_as_uint(f[2 * i]), __float_as_uint(f[2 * i + 1]));
      if constexpr (BY == BY_CODES) {   // off the exponents; 0 (+0: it comes from an integer) stays 0 by saturation
        constexpr uint16_t by = (FMT == INT4 ? 22 : 26) << 7;
        two = __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(__builtin_bit_cast(ushort2v, two), ushort2v{by, by}));
      }
      r[i] = two;
    }
  }
  return r;
}

// queries [lo, lo + m) and rows of partition g
__device__ __forceinline__ void partition(const PartitionArgs &a, uint32_t g, uint32_t &lo, uint32_t &m, uint32_t &n) {
  const int32_t from = cut(a.query_offsets[g], (int32_t)a.n_queries), to = cut(a.query_offsets[g + 1], (int32_t)a.n_queries);
  lo = (uint32_t)from;
  m = to > from ? (uint32_t)(to - from) : 0;
  n = (uint32_t)cut(a.row_counts[g], (int32_t)a.most_rows);
}

__device__ __noinline__ float plain_product(const float *row, const float *query, uint32_t dim) {
  float p = 0.0f;
  for (uint32_t k = 0; k < dim; k++) p = __builtin_fmaf(query[k], row[k], p);
  return p;
}

// A workgroup's run of tiles, and where its first one is: the partition, that partition's queries and rows, the tile's number in it
struct Place {
  uint32_t g, lo, m, n, left;
};
struct Run {
  uint64_t tiles;
  uint32_t stride;
  Place at;
};
struct RunShared {
  uint64_t wave_sums[16];
  Place at;
};
// The offsets and counts are on the device, so every workgroup sums the partitions' tiles itself, takes its even part of them, and
// looks where that begins.  A thread has a few neighbouring partitions; from COARSE a thread on, 64 neighbours are a wavefront's lanes,
// so that a load is of whole lines, and the place is looked for 512 partitions at a time (256 queries in 10 000 / 100 000 partitions of
// 128 x 128: 41 -> 28 / 338 -> 189 us; at 1000, four a thread, lanes that are neighbours took 9.6 us for 8.6).
// TOGETHER: an eighth of the tiles, one after the other, is for the workgroups b, b + 8, ... that share a die's L2, and they go through
// it side by side.
constexpr uint32_t DIES = 8, COARSE = 8;
template <int THREADS, bool TOGETHER>
__device__ __forceinline__ Run find_run(const PartitionArgs &a, uint32_t tq, uint32_t tr, RunShared &shared) {
  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), per = (a.n_partitions + THREADS - 1) / THREADS;
  // this lane's partitions: begin, begin + step, ...
  const uint32_t step = per < COARSE ? 1 : 64, begin = per < COARSE ? threadIdx.x * per : wave * 64 * per + lane;
  uint32_t lo, m, n;
  const auto tiles_of = [&](uint32_t g) {
    partition(a, g < a.n_partitions ? g : a.n_partitions - 1, lo, m, n);
    return g < a.n_partitions ? (m + tq - 1) / tq * ((n + tr - 1) / tr) : 0;
  };
  const auto up_to_lane = [&](uint64_t own) {
#pragma unroll
    for (int k = 1; k < 64; k *= 2) {
      const uint64_t v = __shfl_up((unsigned long long)own, k, 64);
      if (lane >= (uint32_t)k) own += v;
    }
    return own;
  };
  uint64_t own = 0;   // (offsets that rise and fall can name more tiles than 32 bits count)
#pragma unroll 4
  for (uint32_t i = 0; i < per; i++) own += tiles_of(begin + i * step);
  uint64_t up_to = up_to_lane(own);
  if (lane == 63) shared.wave_sums[wave] = up_to;
  __syncthreads();
  uint64_t total = 0, before = 0, after = 0;
#pragma unroll
  for (uint32_t w = 0; w < THREADS / 64; w++) {
    if (w == wave) before = total;
    total += shared.wave_sums[w];
    if (w == wave) after = total;
  }
  Run run;
  uint64_t first;
  if (TOGETHER) {
    const uint64_t die = blockIdx.x % DIES, from = total * die / DIES, to = total * (die + 1) / DIES;
    run.stride = gridDim.x / DIES;   // a multiple of the dies
    first = from + blockIdx.x / DIES;
    run.tiles = first < to ? (to - first + run.stride - 1) / run.stride : 0;
  } else {
    run.stride = 1;
    first = total * blockIdx.x / gridDim.x;
    run.tiles = total * (blockIdx.x + 1) / gridDim.x - first;
  }
  if (run.tiles == 0) return run;
  if (before <= first && first < after) {
    uint64_t left = first - before;
    uint32_t g = begin;
    if (per >= COARSE) {
      const auto behind_these = [&]() {   // or the place is among the partitions that `own` has summed
        const uint64_t all = __shfl((unsigned long long)up_to, 63, 64);
        if (left < all) return false;
        left -= all;
        return true;
      };
      for (;; g += COARSE * 64) {
        own = 0;
#pragma unroll
        for (uint32_t k = 0; k < COARSE; k++) own += tiles_of(g + k * 64);
        up_to = up_to_lane(own);
        if (!behind_these()) break;
      }
      for (;; g += 64) {
        own = tiles_of(g);
        up_to = up_to_lane(own);
        if (!behind_these()) break;
      }
    }
    if (up_to - own <= left && left < up_to) {
      left -= up_to - own;
      for (;; g++) {   // (more than once where neighbours are a lane's)
        const uint32_t tiles = tiles_of(g);
        if (left < tiles) break;
        left -= tiles;
      }
      shared.at = Place{g, lo, m, n, (uint32_t)left};
    }
  }
  __syncthreads();
  run.at.g = __builtin_amdgcn_readfirstlane(shared.at.g);
  run.at.lo = __builtin_amdgcn_readfirstlane(shared.at.lo);
  run.at.m = __builtin_amdgcn_readfirstlane(shared.at.m);
  run.at.n = __builtin_amdgcn_readfirstlane(shared.at.n);
  run.at.left = __builtin_amdgcn_readfirstlane(shared.at.left);
  return run;
}

// two bf16 in a dword by SHRUNK
__device__ __forceinline__ uint32_t shrink2(uint32_t w) {
  return upper2(__float_as_uint(__uint_as_float(w << 16) * SHRUNK), __float_as_uint(__uint_as_float(w & 0xffff0000u) * SHRUNK));
}

// eight elements of a query as 16-bit fragments (an fp32 query: three planes)
template <int Q, int BY>
__device__ __forceinline__ void stage8(const PartitionArgs &a, uint32_t query, uint32_t at, u4 (&w)[Q == F32 ? 3 : 1]) {
  const uint8_t *src = static_cast<const uint8_t *>(a.queries) + (size_t)query * a.stride * elem_size<Q>;
  if constexpr (Q == F32) {
    float v[8];
    load8<F32>(src, at, at < a.c.dim ? a.c.dim - at : 0, v);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] *= BY == BY_QUERIES ? SHRUNK : 1.0f;
    planes8(v, w);
  } else if (at + 8 <= a.c.dim) {
    const u4 x = *reinterpret_cast<const u4_any *>(src + at * 2);
    w[0] = BY == BY_QUERIES ? u4{shrink2(x[0]), shrink2(x[1]), shrink2(x[2]), shrink2(x[3])} : x;
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      uint32_t x = 0;
      if (at + 2 * i < a.c.dim) x = reinterpret_cast<const uint16_t *>(src)[at + 2 * i];
      if (at + 2 * i + 1 < a.c.dim) x |= (uint32_t)reinterpret_cast<const uint16_t *>(src)[at + 2 * i + 1] << 16;
      w[0][i] = BY == BY_QUERIES ? shrink2(x) : x;
    }
  }
}

// the same where all lanes ask for one partition: scalar loads
typedef const __attribute__((address_space(4))) int32_t *scalar_i32;
__device__ __forceinline__ void partition_of_all(const PartitionArgs &a, uint32_t g, uint32_t &lo, uint32_t &m, uint32_t &n) {
  const scalar_i32 offsets = (scalar_i32)(uintptr_t)a.query_offsets, counts = (scalar_i32)(uintptr_t)a.row_counts;
  const int32_t from = cut(offsets[g], (int32_t)a.n_queries), to = cut(offsets[g + 1], (int32_t)a.n_queries);
  lo = (uint32_t)from;
  m = to > from ? (uint32_t)(to - from) : 0;
  n = (uint32_t)cut(counts[g], (int32_t)a.most_rows);
}

// the next partition that has queries and rows; there is one, and it is the same for all lanes
__device__ __forceinline__ uint32_t next_asked(const PartitionArgs &a, uint32_t g) {
  for (g += threadIdx.x % 64;; g += 64) {
    uint32_t lo, m = 0, n = 0;
    if (g < a.n_partitions) partition(a, g, lo, m, n);
    const uint64_t asked = __builtin_amdgcn_ballot_w64(m && n);
    if (asked) return __builtin_amdgcn_readfirstlane(g) + __builtin_ctzll(asked);
  }
}

// W neighbouring elements of a row, as a lane takes them from LDS
template <int FMT, int Q, int W, int BY>
struct Piece {
  static constexpr int BYTES = FMT == NATIVE ? W * elem_size<Q> : FMT == INT4 ? W / 2 : W;
  static constexpr int PLANES = FMT == NATIVE && Q == F32 ? 3 : 1;
  uint32_t raw[BYTES / 4];

  // elements 8 f .. 8 f + 7
  __device__ __forceinline__ void fragment(int f, u4 (&out)[PLANES]) const {
    if constexpr (FMT == NATIVE && Q == F32) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = __uint_as_float(raw[i]);
      planes8(v, out);
    } else if constexpr (FMT == NATIVE) {
      out[0] = u4{raw[0], raw[1], raw[2], raw[3]};
    } else if constexpr (FMT == INT4) {
      out[0] = widen8<INT4, Q, BY>(raw[f], 0);
    } else {
      out[0] = widen8<FMT, Q, BY>(raw[2 * f], raw[2 * f + 1]);
    }
  }
};

// Few queries a partition: the rows' bytes are what it takes.  A workgroup has a run of tiles of 16 QT queries x 16 S rows a wavefront;
// the queries of a partition are put into LDS once for all its tiles (in parts of KP stages if the rows are longer than that).
// A wavefront takes its rows in stages of 4 KiB, 16 S rows x 256 / S bytes: four loads of 16 neighbouring bytes a lane, whole lines of
// the rows, one stage in registers under way (across tiles too) while the one before is multiplied.  (Loads in the shape of the matrix
// instruction's operand touch 16 lines each and cost the same whatever they bring: 2.4 TB/s with 8 bytes a lane, 4.6 with 16.)  A stage
// passes through 4 KiB of LDS that the wavefront has to itself, so nothing but the order of its own instructions guards it, and comes
// back as operands; the sixteen-byte chunks of a row change places with its number, so that neither side meets a bank twice.
// ONCE: the rows are read past the caches' keeping (a batch of 256 over 64 partitions: 57 us for 63; with three query tiles a
// partition, which read the rows three times, 170 for 134).
// 256 queries, 64 partitions x 5461 rows of 768: INT8 with fp16 queries, a scale each 128, 55 us (5.1 TB/s); bf16 rows as they are 94
// (5.8); x 32 768 rows: INT8 299 (5.7), with fp32 queries 303, INT4 177 (5.0); fp32 rows x 8192 267 (6.1).
// Every part of the loop is in the code once: a small call is mostly the first pass of its instructions through the caches.
template <int FMT, int Q, int W, int QT, int S, int WAVES, bool ONCE>
__global__ __launch_bounds__(64 * WAVES, 4) void partition_few_kernel(PartitionArgs a, FastDiv page) {
  constexpr int BY = SHRINK<FMT, Q, false>;
  typedef Piece<FMT, Q, W, BY> P;
  constexpr int QP = Q == F32 ? 3 : 1, FR = W / 8, TQ = 16 * QT, WR = 16 * S, TR = WR * WAVES;
  constexpr int CS = 16 / S;                                  // chunks of a row in a stage
  constexpr int SP = CS * 16 / (4 * P::BYTES);                // steps of 4 W elements in a stage
  constexpr int QS = FMT == NATIVE ? 0 : (SP + 3) / 4;        // scale loads a stage and row group: a lane's quarter has every fourth
  constexpr int KP = (Q == F32 ? 24 : 32) / (SP * FR);        // stages of queries in LDS at a time: 72 or 32 QT KiB
  static_assert(SP >= 1 && KP >= 1, "");
  __shared__ u4 staged[KP * SP * FR * QP * QT * 64];
  __shared__ u4 passing[WAVES][256];
  __shared__ RunShared run_shared;

  const uint32_t tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), col = lane % 16, quarter = lane / 16;
  const Run run = find_run<64 * WAVES, false>(a, TQ, TR, run_shared);
  if (run.tiles == 0) return;
  Place at = run.at;
  const uint32_t chunks = a.c.row_bytes / 16, stages = (chunks + CS - 1) / CS;
  // blocks are one step or two, or the row
  const uint32_t block_shift = a.c.block >= a.c.dim ? 31 : a.c.block / (4 * W) >= 2 ? 1 : 0;
  const float gone = a.form == RSGPU_SCORES_DISTANCE ? __builtin_inff() : -__builtin_inff();

  struct Tile {
    uint32_t g, query_tile, q0, q_end, n, j0;   // j0: the first row of this wavefront
  };
  // slot of row j in page `id`; one that is not there is read from slot 0 and not used
  const auto slot_of = [&](uint32_t j, int32_t id, bool &there) {
    const uint64_t slot = (uint64_t)(uint32_t)id * page.d + (j - page.div(j) * page.d);
    there = id >= 0 && slot < a.c.capacity;
    return (uint64_t)(uint32_t)(there ? slot : 0);
  };

  // Three tiles: `now` is multiplied, `held` is in registers or LDS (its rows in `source`), the pages of `coming` are looked up.
  // Chunk i of a lane is of row i * 64 / CS + lane / CS of the wavefront.
  constexpr uint32_t ROWS_A_LOAD = 64 / CS;
  const uint32_t my_row = lane / CS;
  Tile now = {}, held = {}, coming = {};
  uint32_t there = 0, held_there = 0;             // which of the rows 16 k + col are there
  int32_t id[4], col_id[S];
  const uint8_t *source[4];
  const float *scale_source[S];
  u4 chunk[4];
  float next_scale[S][QS ? QS : 1], scale[S][QS ? QS : 1];
  u4 *const mine = passing[wave];
  f32x4 acc[S][QT];
#pragma unroll
  for (int k = 0; k < S; k++)
#pragma unroll
    for (int t = 0; t < QT; t++) acc[k][t] = f32x4{0, 0, 0, 0};
  uint32_t staged_g = ~0u, staged_q = 0, staged_p = 0;   // whose queries are in LDS, from which stage on
  uint64_t taken = 0;
  uint32_t use_stage = 0, load_stage = stages;           // stages: on to the next tile before the next load
  const int64_t rounds = (int64_t)run.tiles * stages;

  for (int64_t round = -2; round < rounds; round++) {
    if (load_stage == stages) {
      // the tile whose pages are known is loaded from now on (behind the run's last tile: that one again)
      load_stage = 0;
      held = coming;
      held_there = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        bool is;
        const uint64_t slot = slot_of(held.j0 + i * ROWS_A_LOAD + my_row, round == -2 ? -1 : id[i], is);
        source[i] = a.c.codes + slot * a.c.row_bytes;
      }
#pragma unroll
      for (int k = 0; k < S; k++) {
        bool is;
        const uint64_t slot = slot_of(held.j0 + k * 16 + col, round == -2 ? -1 : col_id[k], is);
        held_there |= is ? 1u << k : 0;
        scale_source[k] = a.c.scales + slot * a.c.nb;
      }
      if (taken < run.tiles) {
        uint32_t row_tiles = (at.n + TR - 1) / TR;
        while (at.left >= (at.m + TQ - 1) / TQ * row_tiles) {   // behind this partition's last tile
          at.g++;
          at.left = 0;
          partition_of_all(a, at.g, at.lo, at.m, at.n);
          if (!at.m || !at.n) {
            at.g = next_asked(a, at.g);
            partition_of_all(a, at.g, at.lo, at.m, at.n);
          }
          row_tiles = (at.n + TR - 1) / TR;
        }
        const uint32_t query_tile = at.left / row_tiles;
        coming = Tile{at.g, query_tile, at.lo + query_tile * TQ, at.lo + at.m, at.n, (at.left - query_tile * row_tiles) * TR + wave * WR};
        at.left++;
        taken++;
      }
      // page of row j (of a row behind the partition's last: of its first, whose scores are not written)
      const int32_t *pages = a.pages + (size_t)coming.g * a.max_pages;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint32_t j = coming.j0 + i * ROWS_A_LOAD + my_row;
        id[i] = pages[j < coming.n ? page.div(j) : 0];
      }
#pragma unroll
      for (int k = 0; k < S; k++) {
        const uint32_t j = coming.j0 + k * 16 + col;
        col_id[k] = pages[j < coming.n ? page.div(j) : 0];
      }
      if (round == -2) {
        load_stage = stages;
        continue;
      }
    }

    // a stage under way
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t row = i * ROWS_A_LOAD + my_row, c = load_stage * CS + (lane % CS ^ (CS == 4 ? row >> 1 & 3 : row & (CS - 1)));
      const u4 *p = reinterpret_cast<const u4 *>(source[i] + (c < chunks ? c : chunks - 1) * 16);
      chunk[i] = ONCE ? __builtin_nontemporal_load(p) : *p;
    }
#pragma unroll
    for (int k = 0; k < S; k++)
#pragma unroll
      for (int q = 0; q < QS; q++) {
        const uint32_t b = ((load_stage * SP) >> block_shift) + q * 4 + quarter;
        next_scale[k][q] = scale_source[k][b < a.c.nb ? b : a.c.nb - 1];
      }
    load_stage++;

    if (round >= 0) {
      // the one in LDS multiplied
      const u4 *queries = staged + use_stage % KP * (SP * FR * QP * QT * 64) + lane;
      const uint32_t first_block = (use_stage * SP) >> block_shift;
      P piece[SP][S];
#pragma unroll
      for (int st = 0; st < SP; st++)
#pragma unroll
        for (int k = 0; k < S; k++) {
          const uint32_t row = k * 16 + col, bytes = st * 4 * P::BYTES + quarter * P::BYTES, turn = CS == 4 ? row >> 1 & 3 : row & (CS - 1);
#pragma unroll
          for (int e = 0; e < (P::BYTES + 15) / 16; e++) {
            const uint8_t *p = reinterpret_cast<const uint8_t *>(mine + row * CS + ((bytes / 16 + e) ^ turn)) + bytes % 16;
            if constexpr (P::BYTES == 4) {
              piece[st][k].raw[0] = *reinterpret_cast<const uint32_t *>(p);
            } else if constexpr (P::BYTES == 8) {
              const u2 w = *reinterpret_cast<const u2 *>(p);
              piece[st][k].raw[0] = w[0];
              piece[st][k].raw[1] = w[1];
            } else {
              const u4 w = *reinterpret_cast<const u4 *>(p);
#pragma unroll
              for (int i = 0; i < 4; i++) piece[st][k].raw[4 * e + i] = w[i];
            }
          }
        }
#pragma unroll
      for (int st = 0; st < SP; st++) {
        f32x4 part[S][QT];
#pragma unroll
        for (int k = 0; k < S; k++)
#pragma unroll
          for (int t = 0; t < QT; t++) part[k][t] = FMT == NATIVE ? acc[k][t] : f32x4{0, 0, 0, 0};
#pragma unroll
        for (int f = 0; f < FR; f++) {
          u4 q[QT][QP];
#pragma unroll
          for (int t = 0; t < QT; t++)
#pragma unroll
            for (int p = 0; p < QP; p++) q[t][p] = queries[(((st * FR + f) * QP + p) * QT + t) * 64];
#pragma unroll
          for (int k = 0; k < S; k++) {
            u4 b[P::PLANES];
            piece[st][k].fragment(f, b);
            if (FMT == NATIVE) {   // behind the row's end its last chunk comes again: an infinity there would meet a zero
              const bool in = (use_stage * SP + st) * 4 * W + quarter * W < a.c.row_bytes / elem_size<Q>;
#pragma unroll
              for (int c = 0; c < P::PLANES; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) b[c][e] = in ? b[c][e] : 0;
            }
#pragma unroll
            for (int p = QP - 1; p >= 0; p--)   // the smallest first
#pragma unroll
              for (int c = P::PLANES - 1; c >= 0; c--)
#pragma unroll
                for (int t = 0; t < QT; t++)
                  if (p + c < 3) part[k][t] = mfma16<Q>(q[t][p], b[c], part[k][t]);   // left out: no more than 2^-24 of the product
          }
        }
        // a step's sum, times the scale of the block that it is in (no branch for the block's end: the steps overlap)
        const uint32_t block = ((use_stage * SP + st) >> block_shift) - first_block;
#pragma unroll
        for (int k = 0; k < S; k++) {
          if (FMT == NATIVE) {
#pragma unroll
            for (int t = 0; t < QT; t++) acc[k][t] = part[k][t];
          } else {
            float v = scale[k][0];
#pragma unroll
            for (int q = 1; q < QS; q++) v = block / 4 == (uint32_t)q ? scale[k][q] : v;
            v = __uint_as_float(__builtin_amdgcn_ds_bpermute((block % 4 * 16 + col) * 4, __float_as_uint(v)));
#pragma unroll
            for (int t = 0; t < QT; t++)
#pragma unroll
              for (int r = 0; r < 4; r++) acc[k][t][r] = __builtin_fmaf(v, part[k][t][r], acc[k][t][r]);
          }
        }
      }
      use_stage++;
    }

    // the queries that the next stage meets, if they are not in LDS yet; they and the stage under way come together
    const bool turned = round < 0 || use_stage == stages;
    const uint32_t meets_g = turned ? held.g : now.g, meets_q = turned ? held.query_tile : now.query_tile, p0 = turned ? 0 : use_stage / KP * KP;
    if ((staged_g != meets_g || staged_q != meets_q || staged_p != p0) && round + 1 < rounds) {
      const uint32_t q0 = turned ? held.q0 : now.q0, q_end = turned ? held.q_end : now.q_end;
      __syncthreads();
      const uint32_t np = stages - p0 < KP ? stages - p0 : KP, asked = q_end - q0 < TQ ? q_end - q0 : TQ;
      const uint32_t shift = asked > 16 ? 5 : asked > 8 ? 4 : asked > 4 ? 3 : asked > 2 ? 2 : asked > 1 ? 1 : 0;
      for (uint32_t i = tid; i < np * (SP * FR * 4) << shift; i += 64 * WAVES) {
        const uint32_t q = i & ((1u << shift) - 1), e = i >> shift, f = e % FR, h = e / FR % 4, st = e / (4 * FR);
        if (q >= asked) continue;   // what is in LDS behind them is multiplied and not used
        u4 w[QP];
        stage8<Q, BY>(a, q0 + q, (p0 * SP + st) * (4 * W) + h * W + f * 8, w);
#pragma unroll
        for (int p = 0; p < QP; p++) staged[(((st * FR + f) * QP + p) * QT + q / 16) * 64 + h * 16 + q % 16] = w[p];
      }
      __syncthreads();
      staged_g = meets_g;
      staged_q = meets_q;
      staged_p = p0;
    }

    // the stage under way into LDS, behind the reads of the one before it
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 4; i++) mine[i * 64 + lane] = chunk[i];
#pragma unroll
    for (int k = 0; k < S; k++)
#pragma unroll
      for (int q = 0; q < QS; q++) scale[k][q] = next_scale[k][q];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();

    if (use_stage == stages) {
#pragma unroll
      for (int k = 0; k < S; k++) {
        const uint32_t j = now.j0 + k * 16 + col;
        if (j < now.n) {
#pragma unroll
          for (int e = 0; e < 4 * QT; e++) {
            const uint32_t q = now.q0 + e / 4 * 16 + quarter * 4 + e % 4;
            if (q < now.q_end) {
              float p = acc[k][e / 4][e % 4] * UNIT<FMT, Q, BY>;
              if constexpr (FMT == NATIVE && Q == F32) {
                // an infinity meets the other side's planes, some of them 0, and two hi that were rounded up may pass the type's end: the
                // sum is taken again, element by element
                if (!__builtin_isfinite(p) && (there >> k & 1)) {
                  bool is;
                  const uint64_t slot = slot_of(j, a.pages[(size_t)now.g * a.max_pages + page.div(j)], is);
                  p = plain_product(reinterpret_cast<const float *>(a.c.codes + slot * a.c.row_bytes), static_cast<const float *>(a.queries) + q * a.stride, a.c.dim);
                }
              }
              if (a.form == RSGPU_SCORES_DISTANCE) p = 1.0f - p;
              a.scores[(size_t)q * a.ld + j] = there >> k & 1 ? p : gone;
            }
          }
        }
#pragma unroll
        for (int t = 0; t < QT; t++) acc[k][t] = f32x4{0, 0, 0, 0};
      }
      use_stage = 0;
    }
    if (use_stage == 0) {
      now = held;
      there = held_there;
    }
  }
}

// Many queries a partition: the matrix cores' work.  A workgroup has a run of tiles of 128 queries x TR = 128 or 256 rows, a wavefront 64 x 64
// or 128 x 64 of each; both sides go through LDS as operands of the 32 x 32 x 16 product, the rows' codes widened once on the way
// there.  A stage is 64 elements (32 where both sides are fp32) in two halves: one half is multiplied, the next is in the other half of
// LDS, and the two behind it are on their way in registers, of this tile or the next one's; with one on its way every half waited for
// memory.  In LDS an operand's 32 rows change places with the number of its eight elements, so that neither side meets a bank twice.  A
// block's products are summed by themselves and multiplied by the row's scale at every FLUSH elements (0: rows that have one scale or
// none, at the end).
// 16 partitions x 512 queries x 4096 bf16 rows of 768: 75 us, 0.69 PFLOP/s.  Rows of 64 elements, almost nothing but the scores' way
// to memory (134 MB), take 35; the next 704 elements 40 (1.17 PFLOP/s), 768 more 48 (1.08; a large matrix product of the library 1.27).
// Stores and loads are counted in one order, so the next tile's rows are waited for behind this one's scores.  Workgroups begun at
// different times, four columns a lane's store, a tile's scores kept in registers for the next tile's products to hide: no faster.
template <int FMT, int Q, int FLUSH, int TR>
__global__ __launch_bounds__(256, 2) void partition_many_kernel(PartitionArgs a, FastDiv page) {
  constexpr int TQ = 128, X = TR / 64, Y = 2, KC = FMT == NATIVE && Q == F32 ? 16 : 32, QP = Q == F32 ? 3 : 1, RP = FMT == NATIVE && Q == F32 ? 3 : 1;
  constexpr int C8 = KC / 8;                                                 // eights of a half
  constexpr int PIECE = FMT == NATIVE ? 8 : FMT == INT4 ? 32 : 16;           // elements of a row that a thread loads together
  constexpr int PIECE_BYTES = FMT == NATIVE ? 8 * elem_size<Q> : 16, PU = PIECE_BYTES / 16;
  constexpr int NP = KC / PIECE, RT = (TR * NP + 255) / 256;                  // pieces of a row in a half, of a thread
  constexpr int QN = TQ * C8 / 256;                                          // eights of the queries in a half, of a thread
  constexpr int BY = SHRINK<FMT, Q, true>;
  typedef Piece<FMT, Q, PIECE, BY> P;
  __shared__ u4 q_lds[2][KC / 16 * QP * TQ * 2], r_lds[2][KC / 16 * RP * TR * 2];
  __shared__ float s_lds[2][TR];
  __shared__ RunShared run_shared;

  const uint32_t tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), col = lane % 32, half_wave = lane / 32;
  const Run run = find_run<256, true>(a, TQ, TR, run_shared);
  if (run.tiles == 0) return;
  const uint32_t padded = rows_padded(a.c.dim), stages = (padded + 2 * KC - 1) / (2 * KC);
  const float gone = a.form == RSGPU_SCORES_DISTANCE ? __builtin_inff() : -__builtin_inff();
  const auto slot_of = [&](uint32_t j, int32_t id, bool &there) {
    const uint64_t slot = (uint64_t)(uint32_t)id * page.d + (j - page.div(j) * page.d);
    there = id >= 0 && slot < a.c.capacity;
    return (uint64_t)(uint32_t)(there ? slot : 0);   // one that is not there is read from slot 0 and not used
  };
  // the place of eight elements (number c of the half) of row r in an operand of plane p
  const auto place = [](uint32_t rows, uint32_t c, uint32_t planes, uint32_t p, uint32_t r) {
    return ((c / 2 * planes + p) * (rows / 32) + r / 32) * 64 + c % 2 * 32 + (r % 32 ^ c * (8 / C8));
  };
  struct Tile {
    uint32_t g, q0, q_end, n, j0;
  };
  const auto take = [&](Place &at) {
    uint32_t query_tiles = (at.m + TQ - 1) / TQ, tiles = query_tiles * ((at.n + TR - 1) / TR);
    while (at.left >= tiles) {   // behind this partition's last tile
      at.g++;
      at.left -= tiles;
      partition_of_all(a, at.g, at.lo, at.m, at.n);
      if (!at.m || !at.n) {
        at.g = next_asked(a, at.g);
        partition_of_all(a, at.g, at.lo, at.m, at.n);
      }
      query_tiles = (at.m + TQ - 1) / TQ;
      tiles = query_tiles * ((at.n + TR - 1) / TR);
    }
    const uint32_t row_tile = at.left / query_tiles;
    const Tile t = {at.g, at.lo + (at.left - row_tile * query_tiles) * TQ, at.lo + at.m, at.n, row_tile * TR};
    at.left += run.stride;
    return t;
  };
  // page of row j (of a row behind the partition's last: of its first, whose scores are not written)
  const auto page_of = [&](const Tile &t, uint32_t j) { return a.pages[(size_t)t.g * a.max_pages + (j < t.n ? page.div(j) : 0)]; };

  // ---- the loads: `loading` is the tile they are at, the pages of `coming` are looked up.  Piece i of a thread is of row
  // (i * 256 + tid) / NP, eight i of query (i * 256 + tid) / C8; its scale is row tid % TR's
  Place load_at = run.at;
  uint64_t loads_taken = 1;
  uint32_t load_stage = 0;
  Tile loading = {}, coming = take(load_at);
  int32_t id[RT], scale_id;
  const uint8_t *source[RT], *queries[QN];
  const float *scale_source;
  const auto look_up = [&]() {
#pragma unroll
    for (int i = 0; i < RT; i++) id[i] = page_of(coming, coming.j0 + (i * 256 + tid) / NP % TR);
    if (FMT != NATIVE) scale_id = page_of(coming, coming.j0 + tid % TR);
  };
  // on to the tile whose pages are known (behind the run's last tile: that one again)
  const auto next_tile = [&]() {
    loading = coming;
    bool is;
#pragma unroll
    for (int i = 0; i < RT; i++) source[i] = a.c.codes + slot_of(loading.j0 + (i * 256 + tid) / NP % TR, id[i], is) * a.c.row_bytes;
    if (FMT != NATIVE) scale_source = a.c.scales + slot_of(loading.j0 + tid % TR, scale_id, is) * a.c.nb;
#pragma unroll
    for (int i = 0; i < QN; i++) {
      const uint32_t q = loading.q0 + (i * 256 + tid) / C8;   // of a query behind the partition's last: the last's, not used
      queries[i] = static_cast<const uint8_t *>(a.queries) + (size_t)(q < loading.q_end ? q : loading.q_end - 1) * a.stride * elem_size<Q>;
    }
    if (loads_taken < run.tiles) {
      coming = take(load_at);
      loads_taken++;
    }
    look_up();
  };
  u4 row_held[2][RT][PU];
  Raw8<Q> query_held[2][QN];
  float scale_held[2];
  uint32_t held_base[2];
  const auto load = [&](auto which) {
    constexpr int H = decltype(which)::value;
    const uint32_t base = held_base[H] = (load_stage * 2 + H) * KC, e = base + tid % NP * PIECE;
#pragma unroll
    for (int i = 0; i < RT; i++) {
      const u4 *p = reinterpret_cast<const u4 *>(source[i] + (e < padded ? e : 0) / PIECE * PIECE_BYTES);
#pragma unroll
      for (int u = 0; u < PU; u++) row_held[H][i][u] = p[u];
    }
    if (FMT != NATIVE && (FLUSH || H == 1)) {
      const uint32_t b = base / a.c.block;
      scale_held[H] = scale_source[b < a.c.nb ? b : a.c.nb - 1];
    }
    // an eight that the query's end cuts is loaded from where it is whole, and moved below (rows of less than eight elements do not
    // come here)
    const uint32_t at = base + tid % C8 * 8;
#pragma unroll
    for (int i = 0; i < QN; i++) query_held[H][i].load_whole(queries[i], at + 8 <= a.c.dim ? at : a.c.dim - 8);
    if (H == 1 && ++load_stage == stages) {
      load_stage = 0;
      next_tile();
    }
  };
  // a half in registers into its half of LDS, which nobody has read since the last barrier
  const auto put = [&](auto which) {
    constexpr int H = decltype(which)::value;
    const uint32_t base = held_base[H];
    if (base + KC > a.c.dim) {   // the row's end is in it or before it: zeros behind it
      const uint32_t at = base + tid % C8 * 8, by = at - (at + 8 <= a.c.dim ? at : a.c.dim - 8);
#pragma unroll
      for (int i = 0; i < QN; i++) {
        if (by >= 8) query_held[H][i].zero();
        else query_held[H][i].drop(by);
      }
      if (FMT == NATIVE) {
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
          for (int k = 0; k < 4 * PU; k++) row_held[H][i][k / 4][k % 4] = base + tid % NP * PIECE < padded ? row_held[H][i][k / 4][k % 4] : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < QN; i++) {
      u4 w[QP];
      if constexpr (Q == F32) {
        float v[8];
        query_held[H][i].floats(v);
        planes8(v, w);
      } else {
        w[0] = query_held[H][i].w[0];
      }
#pragma unroll
      for (int p = 0; p < QP; p++) q_lds[H][place(TQ, tid % C8, QP, p, (i * 256 + tid) / C8)] = w[p];
    }
#pragma unroll
    for (int i = 0; i < RT; i++) {
      if (TR * NP < 256 && tid >= (uint32_t)(TR * NP)) break;
      P piece;
#pragma unroll
      for (int k = 0; k < PIECE_BYTES / 4; k++) piece.raw[k] = row_held[H][i][k / 4][k % 4];
#pragma unroll
      for (int f = 0; f < PIECE / 8; f++) {
        u4 w[RP];
        piece.fragment(f, w);
#pragma unroll
        for (int p = 0; p < RP; p++) r_lds[H][place(TR, tid % NP * (PIECE / 8) + f, RP, p, (i * 256 + tid) / NP)] = w[p];
      }
    }
    if (FMT != NATIVE && (FLUSH || H == 1) && tid < TR) s_lds[H][tid] = scale_held[H];
  };

  // ---- the products
  const uint32_t wave_q = X == 2 ? wave / 2 * 64 : 0, wave_r = X == 2 ? wave % 2 * 64 : wave * 64;
  f32x16 acc[X][Y], part[X][Y];
  float row_scale[Y];
#pragma unroll
  for (int x = 0; x < X; x++)
#pragma unroll
    for (int y = 0; y < Y; y++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[x][y][r] = 0.0f;
  const auto multiply = [&](auto which) {
    constexpr int H = decltype(which)::value;
    constexpr bool FRESH = FLUSH && (H == 0 || FLUSH == KC);   // a block's sums begin
    f32x16(&sum)[X][Y] = FLUSH ? part : acc;
#pragma unroll
    for (int k = 0; k < KC / 16; k++) {
      u4 q[X][QP], r[Y][RP];
#pragma unroll
      for (int y = 0; y < Y; y++)
#pragma unroll
        for (int p = 0; p < RP; p++) r[y][p] = r_lds[H][place(TR, 2 * k + half_wave, RP, p, wave_r + y * 32 + col)];
#pragma unroll
      for (int x = 0; x < X; x++)
#pragma unroll
        for (int p = 0; p < QP; p++) q[x][p] = q_lds[H][place(TQ, 2 * k + half_wave, QP, p, wave_q + x * 32 + col)];
#pragma unroll
      for (int p = QP - 1; p >= 0; p--)   // the smallest first
#pragma unroll
        for (int c = RP - 1; c >= 0; c--)
          if (p + c < 3) {   // left out: no more than 2^-24 of the product
#pragma unroll
            for (int x = 0; x < X; x++)
#pragma unroll
              for (int y = 0; y < Y; y++) {
                const f32x16 none = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
                sum[x][y] = mfma<Q>(q[x][p], r[y][c], FRESH && k == 0 && p == QP - 1 ? none : sum[x][y]);   // (one plane of rows there)
              }
          }
    }
    if (FMT != NATIVE && !FLUSH && H == 1) {   // here, where nobody writes them
#pragma unroll
      for (int y = 0; y < Y; y++) row_scale[y] = s_lds[1][wave_r + y * 32 + col];
    }
    if (FLUSH && (H == 1 || FLUSH == KC)) {
#pragma unroll
      for (int y = 0; y < Y; y++) {
        const float scale = s_lds[H][wave_r + y * 32 + col];
#pragma unroll
        for (int x = 0; x < X; x++)
#pragma unroll
          for (int r = 0; r < 16; r++) acc[x][y][r] = __builtin_fmaf(scale, part[x][y][r], acc[x][y][r]);
      }
      if (FLUSH == KC) {   // here and not with the next half's, whose sums take part's registers
#pragma unroll
        for (int x = 0; x < X; x++)
#pragma unroll
          for (int y = 0; y < Y; y++) asm volatile("" : "+v"(acc[x][y]));
      }
    }
  };

  // ---- the scores, an eighth of a wavefront's at a time
  const auto write = [&](auto which, const Tile &t, uint32_t there, const auto &sums) {
    constexpr int W = decltype(which)::value, x = W / 4, y = W / 2 % 2, R = W % 2 * 8;
    const uint32_t j = t.j0 + wave_r + y * 32 + col;
    float *at = a.scores + j;
    if (j >= t.n) return;
#pragma unroll
    for (int r = R; r < R + 8; r++) {
      const uint32_t q = t.q0 + wave_q + x * 32 + 8 * (r / 4) + 4 * half_wave + r % 4;
      if (q >= t.q_end) continue;
      float p = sums[x][y][r];
      if (FMT != NATIVE && !FLUSH) p *= row_scale[y];
      p *= UNIT<FMT, Q, BY>;
      if constexpr (FMT == NATIVE && Q == F32) {
        // as above: the sum is taken again, element by element
        if (!__builtin_isfinite(p) && (there >> y & 1)) {
          bool is;
          const uint64_t slot = slot_of(j, page_of(t, j), is);
          p = plain_product(reinterpret_cast<const float *>(a.c.codes + slot * a.c.row_bytes), static_cast<const float *>(a.queries) + q * a.stride, a.c.dim);
        }
      }
      if (a.form == RSGPU_SCORES_DISTANCE) p = 1.0f - p;
      __builtin_nontemporal_store(there >> y & 1 ? p : gone, at + (uint64_t)q * a.ld);   // (kept in the caches, rows of 1536 took 139 us for 106)
    }
  };
  const std::integral_constant<int, 0> first_half;
  const std::integral_constant<int, 1> second_half;
  look_up();
  next_tile();
  load(first_half);
  load(second_half);
  Place use_at = run.at;
  Tile now = take(use_at);
  int32_t col_id[2];
#pragma unroll
  for (int y = 0; y < Y; y++) col_id[y] = page_of(now, now.j0 + wave_r + y * 32 + col);
  put(first_half);
  load(first_half);
  __syncthreads();
  uint32_t use_stage = 0;
  uint64_t used = 0;
  for (;;) {
    multiply(first_half);
    put(second_half);
    load(second_half);
    __syncthreads();
    multiply(second_half);
    put(first_half);
    load(first_half);
    __syncthreads();
    if (++use_stage < stages) continue;

    uint32_t there = 0;
#pragma unroll
    for (int y = 0; y < Y; y++) {
      bool is;
      slot_of(now.j0 + wave_r + y * 32 + col, col_id[y], is);
      there |= is ? 1u << y : 0;
    }
    write(std::integral_constant<int, 0>(), now, there, acc);
    write(std::integral_constant<int, 1>(), now, there, acc);
    write(std::integral_constant<int, 2>(), now, there, acc);
    write(std::integral_constant<int, 3>(), now, there, acc);
    write(std::integral_constant<int, 4>(), now, there, acc);
    write(std::integral_constant<int, 5>(), now, there, acc);
    write(std::integral_constant<int, 6>(), now, there, acc);
    write(std::integral_constant<int, 7>(), now, there, acc);
    if constexpr (X == 4) {
      write(std::integral_constant<int, 8>(), now, there, acc);
      write(std::integral_constant<int, 9>(), now, there, acc);
      write(std::integral_constant<int, 10>(), now, there, acc);
      write(std::integral_constant<int, 11>(), now, there, acc);
      write(std::integral_constant<int, 12>(), now, there, acc);
      write(std::integral_constant<int, 13>(), now, there, acc);
      write(std::integral_constant<int, 14>(), now, there, acc);
      write(std::integral_constant<int, 15>(), now, there, acc);
    }
#pragma unroll
    for (int x = 0; x < X; x++)
#pragma unroll
      for (int y = 0; y < Y; y++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[x][y][r] = 0.0f;
    if (++used == run.tiles) break;
    use_stage = 0;
    now = take(use_at);
#pragma unroll
    for (int y = 0; y < Y; y++) col_id[y] = page_of(now, now.j0 + wave_r + y * 32 + col);
  }
}

// workgroups of a kernel that the device holds at once: kernels that go round give each of them the same share
uint32_t resident(const void *kernel, uint32_t threads) {
  int device = 0, units = 0, each = 0;
  HIP_CHECK(hipGetDevice(&device));
  HIP_CHECK(hipDeviceGetAttribute(&units, hipDeviceAttributeMultiprocessorCount, device));
  HIP_CHECK(hipOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, (int)threads, 0));
  return (uint32_t)(units > 0 && each > 0 ? units * each : 256);
}

// Which kernel, by the queries of a partition on average: offsets and counts are on the device, and the host does not wait for them.
// Where the queries crowd on few of the partitions that are listed, tiles for fewer queries read those rows again for every 16 or 32
// (2000 queries for one of 400 partitions, 20 000 INT8 rows of 768: 358 us; that one listed alone: 93).
// 64 partitions x 5461 rows of 768, us; 20 / 40 / 60 queries:
//   int8 with fp16 queries    16 a tile 92 / 134 / -, 32 a tile 60 / 97 / -, the tiles of 128 107 / 115 / 126
//   bf16 as it is             160 / 340, 120 / 166, 134 / 149 / 168
//   int8 with fp32 queries    95 / 146, (no 32 a tile), 229 / 232 / 237
//   INT4 of 100 wide, 300 x 1000 (rows of 64 bytes)   27 / 35, 29 / 41, 45 / 47 / 51
constexpr uint32_t TWO_TILES = 13, MANY = 48, MANY_LATE = 80;   // late: fp32 queries, and rows of few chunks

// Tiles of 256 rows, for half the reads of the queries, where the sums of a tile are all that the registers hold (16-bit queries, rows of
// one scale or none) and there are as many tiles as the device holds at once.  16 partitions x 4096 rows of 768, 128 / 256 rows, us:
//   INT8, one scale, fp16 queries: 90 queries a partition (432 tiles at most) 21.8 / 25.2, 128 (512) 25.7 / 25.8, 512 (1280) 74 / 71
//   INT4, one scale, bf16 queries, 512: 81 / 66 (without SHRUNK: 1 - 2 % to either); bf16 rows as they are 68 / 66
// (Scaled at every 64 elements, as rows of more scales are, the 512 take 87 and 93.)
constexpr uint64_t MANY_TALL = 512;

// Workgroups of four waves where there are few tiles of theirs, every partition counted as long as the page table and the scores' rows
// allow (8 x 700 in a table for 70 000 takes the wide ones: 14.4 us): one's waves wait for each other while the queries are laid out,
// and four have less to wait for.  us with the wide ones / with four waves (int8 rows of 768, one query each):
//   fp32 queries: 8 x 700 (88 tiles) 14.4 / 8.3, 64 x 512 (512) 14.6 / 11.7, 64 x 1024 (1088) 15.4 / 19.3
//   fp16 queries: 8 x 700 8.5 / 7.3, 64 x 512 11.3 / 9.9, 64 x 1024 12.4 / 13.4
// rows of 64 bytes, whose tile is four times as long (INT4 of 100 wide): 300 x 1000 (1200) 20.4 / 17.4, 300 x 4000 36 / 38
constexpr uint64_t LITTLE = 1024, LITTLE_NARROW = 2048;

template <int FMT, int Q>
void scores_as(const PartitionArgs &a, hipStream_t s) {
  const FastDiv page(a.page_rows);
  const uint32_t asked = a.n_partitions < a.n_queries ? a.n_partitions : a.n_queries;   // partitions with queries, at most
  const uint32_t each = a.n_queries / a.n_partitions;
  const auto tiles = [&](uint32_t tq, uint32_t tr) {   // at most
    return ((uint64_t)a.n_queries / tq + asked) * ((a.most_rows + tr - 1) / tr);
  };
  // no more workgroups than there can be tiles, and no more than are resident at once
  const auto grid = [&](uint32_t tq, uint32_t tr, uint64_t resident) {
    const uint64_t n = tiles(tq, tr);
    return dim3((uint32_t)(n < resident ? n : resident));
  };
  // the rows' chunks of a stage: the number that leaves the fewest places empty, the largest of those
  const uint32_t chunks = a.c.row_bytes / 16;
  uint32_t cs = 16;
  constexpr bool widest = Q == F32;   // an fp32 step is eight chunks, and 64 rows of three planes do not fit into 128 registers
  for (uint32_t c : {8u, 4u})
    if (!(widest && c == 4) && (chunks + c - 1) / c * c < (chunks + cs - 1) / cs * cs) cs = c;
  if (each >= (Q == F32 || cs == 4 ? MANY_LATE : MANY) && a.c.dim >= 8) {
    const auto many = [&](auto kernel, uint32_t rows) {
      dim3 g = grid(128, rows, resident(reinterpret_cast<const void *>(kernel), 256));
      g.x = (g.x + DIES - 1) / DIES * DIES;
      launch(kernel, g, 256, s, a, page);
    };
    if (a.c.nb <= 1) {
      if constexpr (Q != F32) {
        if (tiles(128, 256) >= MANY_TALL) return many(partition_many_kernel<FMT, Q, 0, 256>, 256);
      }
      many(partition_many_kernel<FMT, Q, 0, 128>, 128);
    } else if constexpr (FMT != NATIVE) {
      if (a.c.block == 32) many(partition_many_kernel<FMT, Q, 32, 128>, 128);
      else many(partition_many_kernel<FMT, Q, 64, 128>, 128);
    }
    return;
  }
  const auto few = [&](auto w) {
    constexpr int W = decltype(w)::value, WAVES = Q == F32 ? 16 : 8;
    const auto go = [&](auto kernel, uint32_t tq, uint32_t tr, uint32_t waves) {
      launch(kernel, grid(tq, tr, resident(reinterpret_cast<const void *>(kernel), 64 * waves)), 64 * waves, s, a, page);
    };
    // at eight queries a partition hardly one has more than the sixteen of a tile, so that its rows are read once
    const auto sized = [&](auto waves, auto once) {
      constexpr int V = decltype(waves)::value;
      constexpr bool ONCE = decltype(once)::value;
      if (cs == 16) go(partition_few_kernel<FMT, Q, W, 1, 1, V, ONCE>, 16, 16 * V, V);
      else if (cs == 8) go(partition_few_kernel<FMT, Q, W, 1, 2, V, ONCE>, 16, 32 * V, V);
      else if constexpr (!widest) go(partition_few_kernel<FMT, Q, W, 1, 4, V, ONCE>, 16, 64 * V, V);
    };
    if (tiles(16, 256 / cs * 4) <= (cs == 4 ? LITTLE_NARROW : LITTLE)) return sized(std::integral_constant<int, 4>(), std::false_type());
    if (each <= 8) return sized(std::integral_constant<int, WAVES>(), std::true_type());
    if constexpr (Q != F32) {   // (three planes of 32 queries leave no room for whole rows)
      if (each >= TWO_TILES && cs != 4) {
        if (cs == 16) go(partition_few_kernel<FMT, Q, W, 2, 1, 16, false>, 32, 256, 16);
        else go(partition_few_kernel<FMT, Q, W, 2, 2, 16, false>, 32, 512, 16);
        return;
      }
    }
    sized(std::integral_constant<int, WAVES>(), std::false_type());
  };
  // a lane's piece of a row: as wide as four of them fit into a block
  if constexpr (FMT != NATIVE) {
    if (a.c.block != 32) return few(std::integral_constant<int, 16>());
  }
  few(std::integral_constant<int, 8>());
}

template <int Q>
void scores_from(const PartitionArgs &a, hipStream_t s) {
  switch (a.c.format) {
    case INT8: return scores_as<INT8, Q>(a, s);
    case E4M3: return scores_as<E4M3, Q>(a, s);
    case INT4: return scores_as<INT4, Q>(a, s);
    default: return scores_as<NATIVE, Q>(a, s);
  }
}

}  // namespace
}  // namespace rsgpu
