// rows_kernels.hip -- the row cache (include/rsgpu_rows.h) on gfx950: rows quantised into their slots and read back, and the rules on
// a batch's scores.  (The products with a partition's rows: partition_kernels.hpp.)
#include "rows_device.hpp"

namespace rsgpu {
namespace {

// ---- writing ---------------------------------------------------------------------------------------------------------------

// Pieces of a row that a thread of a workgroup has under way.  Writing (400 009 fp16 rows of 96 to INT4 / of 100 to INT8, in order, us): 1
// 25.0 / 27.2, 2 21.7 / 25.3, 4 23.8 / 26.1 (its registers leave five wavefronts a SIMD of eight).  Reading (fp16 rows of 768 from INT4 /
// fp32 ones from INT8): 2 102 / 99, 4 85 / 84, 8 89 / 84.
constexpr int WRITE_UNDER_WAY = 2, READ_UNDER_WAY = 4;

constexpr uint32_t SMALLEST = (127 - 100) << 23;   // 2^-100: below, a block is kept as zeros

// the scale of a block from the bits of its largest magnitude, and the factor its codes are found with (0: all codes are 0)
template <int FMT>
__device__ __forceinline__ void scale_of(uint32_t most, float &s, float &inv) {
  s = inv = 0.0f;
  if (most < SMALLEST) return;
  if (most >= 0x7f800000u) {
    s = __uint_as_float(0x7fc00000u);
    return;
  }
  if constexpr (FMT == E4M3) {
    // 2^e with e the smallest so that most <= 1.75 * 2^8 * 2^e
    const uint32_t e = (most >> 23) - 8 + ((most & 0x7fffffu) > 0x600000u ? 1u : 0u);
    s = __uint_as_float(e << 23);
    inv = __uint_as_float((254 - e) << 23);
  } else {
    s = __uint_as_float(most) / (FMT == INT8 ? 127.0f : 7.0f);
    inv = __builtin_amdgcn_rcpf(s);
  }
}

// x / s to the nearest integer, ties to even, as if divided exactly.  t is the answer or next to it; r = x - t s is exact (one fused
// step: |r| is at most about s and a multiple of the smaller ulp of x and s), so |r| against s / 2 says which.
__device__ __forceinline__ float settle(float x, float s, float t) {
  const float h = 0.5f * s;
  const float r = __builtin_fmaf(-t, s, x);
  const float a = __builtin_fabsf(r);
  const float next = t + (r > 0.0f ? 1.0f : -1.0f);
  const bool odd = ((int)t & 1) != 0;
  return a > h || (a == h && odd) ? next : t;
}

// fp32 numbers in [2^23, 2^24) have their integer in the low bits: x inv + 1.5 * 2^23 is rounded to one, in two's complement.  inv is
// off by an ulp or two, so the integer may be next to the right one where x / s is next to a border; x - t s (see settle) shows it.
template <int FMT>
__device__ __forceinline__ void encode8(const float (&v)[8], float s, float inv, uint32_t (&c)[2]) {
  c[0] = c[1] = 0;
  if (inv == 0.0f) return;   // nothing to keep, or a NaN: codes are 0
  if constexpr (FMT == E4M3) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      int w = 0;
      w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i] * inv, v[4 * i + 1] * inv, w, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2] * inv, v[4 * i + 3] * inv, w, true);
      c[i] = (uint32_t)w;
    }
  } else {
    constexpr float magic = 12582912.0f;
    float u[8], off = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      u[i] = __builtin_fmaf(v[i], inv, magic);
      off = __builtin_fmaxf(off, __builtin_fabsf(__builtin_fmaf(magic - u[i], s, v[i])));
    }
    if (off >= 0.5f * s) {
#pragma unroll
      for (int i = 0; i < 8; i++) u[i] = magic + settle(v[i], s, u[i] - magic);
    }
    uint32_t q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = __float_as_uint(u[i]);
    const auto bytes4 = [&](int i, int step) {   // the low bytes of q[i], q[i + step], ...
      return __builtin_amdgcn_perm(__builtin_amdgcn_perm(q[i + 3 * step], q[i + 2 * step], 0x0c0c0400u), __builtin_amdgcn_perm(q[i + step], q[i], 0x0c0c0400u), 0x05040100u);
    };
    if constexpr (FMT == INT8) {
      c[0] = bytes4(0, 1);
      c[1] = bytes4(4, 1);
    } else {
      c[0] = (bytes4(0, 2) & 0x0f0f0f0fu) | (bytes4(1, 2) << 4 & 0xf0f0f0f0u);
    }
  }
}

template <int FMT>
__device__ __forceinline__ void store_codes8(uint8_t *row, uint32_t chunk, const uint32_t (&c)[2]) {
  if constexpr (FMT == INT4) *reinterpret_cast<uint32_t *>(row + chunk * 4) = c[0];
  else *reinterpret_cast<u2 *>(row + chunk * 8) = u2{c[0], c[1]};
}

// the largest of a value in L neighbouring lanes, all of which are active: their neighbours by twos and fours, then halves mirrored
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t x) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
  return x > o ? x : o;
}
template <int L>
__device__ __forceinline__ uint32_t most_of_lanes(uint32_t x) {
  x = max_dpp<0xB1>(x);                      // quad_perm [1, 0, 3, 2]
  x = max_dpp<0x4E>(x);                      // quad_perm [2, 3, 0, 1]
  if (L >= 8) x = max_dpp<0x141>(x);         // row_half_mirror
  if (L >= 16) x = max_dpp<0x140>(x);        // row_mirror
#pragma unroll
  for (int k = 16; k < L; k *= 2) {
    const uint32_t o = __shfl_xor(x, k, 64);
    x = x > o ? x : o;
  }
  return x;
}

// Blocks of 8 L elements: L neighbouring lanes have a block, eight elements each, and find its largest magnitude among themselves, so a
// row is read once and neither LDS nor a second pass is needed.  The rows' bytes are what it takes.
// 262 144 bf16 rows of 768 to E4M3, a scale each 128, into slots in any order: 111 us, 5.5 TB/s (a copy of as much memory: 5.2); 50 021
// fp32 rows of 1000, 1003 apart, to INT8: 50 us, 5.0 TB/s; 400 009 fp16 rows of 100 to INT4: 28 us, 4.1 TB/s, where the arithmetic
// counts too (130 instructions for eight elements).  A single row: 2.4 us, an empty kernel's time.
template <int T, int FMT, int L>
__global__ __launch_bounds__(256) void row_write_kernel(RowCacheArgs c, const void *rows, uint32_t stride, const int64_t *slots, uint32_t n,
                                                        uint32_t rows_per_wg, FastDiv chunks) {
  constexpr int U = WRITE_UNDER_WAY;
  const uint32_t padded = rows_padded(c.dim);
  const uint64_t row_stride = (uint64_t)stride * elem_size<T>;
  for (uint64_t first = (uint64_t)blockIdx.x * rows_per_wg; first < n; first += (uint64_t)gridDim.x * rows_per_wg) {
    const uint32_t mine = n - first < rows_per_wg ? (uint32_t)(n - first) : rows_per_wg;
    const uint8_t *from = static_cast<const uint8_t *>(rows) + first * row_stride;
    for (uint32_t i0 = threadIdx.x; i0 < mine * chunks.d; i0 += 256 * U) {
      int64_t slot[U];
      uint32_t chunk[U], row[U];
      Raw8<T> raw[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t i = i0 + u * 256, r = chunks.div(i);
        const bool in = i < mine * chunks.d;
        chunk[u] = i - r * chunks.d;
        slot[u] = in ? slots[first + r] : -1;
        row[u] = r;
      }
#pragma unroll
      for (int u = 0; u < U; u++) {   // a row that is left out is not read
        const uint32_t at = chunk[u] * 8;
        const bool there = slot[u] >= 0 && (uint64_t)slot[u] < c.capacity;
        raw[u].load(from + (uint64_t)row[u] * row_stride, at, there && at < c.dim ? c.dim - at : 0, c.dim >= 4 && first + row[u] + 1 < n);   // (eight are at most two rows)
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        float v[8];
        const uint32_t at = chunk[u] * 8;
        raw[u].cut(at < c.dim ? c.dim - at : 0);
        raw[u].floats(v);
        const uint32_t most = most_of_lanes<L>(raw[u].most());
        float s, inv;
        scale_of<FMT>(most, s, inv);
        uint32_t code[2];
        encode8<FMT>(v, s, inv, code);
        if (slot[u] >= 0 && (uint64_t)slot[u] < c.capacity) {
          const uint32_t to = (uint32_t)slot[u];
          if (at < padded) store_codes8<FMT>(c.codes + (uint64_t)to * c.row_bytes, chunk[u], code);
          if (chunk[u] % L == 0) c.scales[(uint64_t)to * c.nb + chunk[u] / L] = s;
        }
      }
    }
  }
}

// One scale a row of more than 512 elements: a wavefront has a row, in C eights a lane, held in registers between the two passes (a
// million bf16 elements of 768-wide rows take 0.63 us; read twice 0.84).  C = 0, for rows that 32 registers do not hold, and the last
// row, behind which the memory may end: read a second time (from the caches) once the largest magnitude is known.
template <int T, int FMT, int C>
__global__ __launch_bounds__(256) void row_write_whole_kernel(RowCacheArgs c, const void *rows, uint32_t stride, const int64_t *slots, uint32_t n) {
  const uint32_t lane = threadIdx.x % 64, padded = rows_padded(c.dim);
  for (uint64_t r = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64; r < n; r += (uint64_t)gridDim.x * 4) {
    const int64_t slot = slots[r];
    if (slot < 0 || (uint64_t)slot >= c.capacity) continue;
    const uint8_t *row = static_cast<const uint8_t *>(rows) + r * ((uint64_t)stride * elem_size<T>);
    uint8_t *to = c.codes + (uint64_t)(uint32_t)slot * c.row_bytes;
    const bool more = r + 1 < n;   // the memory goes on behind this row
    float v[8], s, inv;
    uint32_t most = 0, code[2];
    if (C > 0 && more) {
      Raw8<T> raw[C ? C : 1];
#pragma unroll
      for (int k = 0; k < C; k++) {
        const uint32_t at = (k * 64 + lane) * 8;
        raw[k].zero();
        if (at < c.dim) raw[k].load_whole(row, at);
      }
#pragma unroll
      for (int k = 0; k < C; k++) {
        const uint32_t at = (k * 64 + lane) * 8;
        raw[k].cut(at < c.dim ? c.dim - at : 0);
        const uint32_t o = raw[k].most();
        most = most > o ? most : o;
      }
      most = most_of_lanes<64>(most);
      scale_of<FMT>(most, s, inv);
#pragma unroll
      for (int k = 0; k < C; k++) {
        const uint32_t at = (k * 64 + lane) * 8;
        raw[k].floats(v);
        encode8<FMT>(v, s, inv, code);
        if (at < padded) store_codes8<FMT>(to, at / 8, code);
      }
    } else {
      for (uint32_t at = lane * 8; at < c.dim; at += 512) {
        Raw8<T> raw;
        raw.load(row, at, c.dim - at);
        const uint32_t o = raw.most();
        most = most > o ? most : o;
      }
      most = most_of_lanes<64>(most);
      scale_of<FMT>(most, s, inv);
      for (uint32_t at = lane * 8; at < padded; at += 512) {
        load8<T>(row, at, at < c.dim ? c.dim - at : 0, v);
        encode8<FMT>(v, s, inv, code);
        store_codes8<FMT>(to, at / 8, code);
      }
    }
    if (lane == 0) c.scales[(uint32_t)slot] = s;
  }
}

// rows kept as they are: sixteen bytes a thread (400 009 bf16 rows of 128: 31.6 us, 6.6 TB/s)
template <int T>
__global__ __launch_bounds__(256) void row_copy_in_kernel(RowCacheArgs c, const void *rows, uint32_t stride, const int64_t *slots, uint32_t n,
                                                          uint32_t rows_per_wg, FastDiv chunks) {
  constexpr int E = 16 / elem_size<T>;
  for (uint64_t first = (uint64_t)blockIdx.x * rows_per_wg; first < n; first += (uint64_t)gridDim.x * rows_per_wg) {
    const uint32_t mine = n - first < rows_per_wg ? (uint32_t)(n - first) : rows_per_wg;
    for (uint32_t i = threadIdx.x; i < mine * chunks.d; i += 256) {
      const uint32_t r = chunks.div(i), chunk = i - r * chunks.d, at = chunk * E;
      const int64_t slot = slots[first + r];
      if (slot < 0 || (uint64_t)slot >= c.capacity) continue;
      const uint8_t *row = static_cast<const uint8_t *>(rows) + (size_t)(first + r) * stride * elem_size<T>;
      u4 w = {0, 0, 0, 0};
      if (at + E <= c.dim) {
        w = *reinterpret_cast<const u4_any *>(row + at * elem_size<T>);
      } else {
#pragma unroll
        for (int k = 0; k < E; k++)
          if (at + k < c.dim) {
            if constexpr (T == F32) w[k] = reinterpret_cast<const uint32_t *>(row)[at + k];
            else w[k / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(row)[at + k] << (16 * (k % 2));
          }
      }
      *reinterpret_cast<u4 *>(c.codes + (size_t)slot * c.row_bytes + chunk * 16) = w;
    }
  }
}

// ---- reading ---------------------------------------------------------------------------------------------------------------

// E neighbouring codes, as they are in memory
template <int FMT, int E>
__device__ __forceinline__ void load_codes(const uint8_t *row, uint32_t at, uint32_t (&w)[2]) {
  if constexpr (FMT == INT4) {
    if constexpr (E == 8) w[0] = *reinterpret_cast<const uint32_t *>(row + at / 2);
    else w[0] = *reinterpret_cast<const uint16_t *>(row + at / 2);
  } else {
    w[0] = *reinterpret_cast<const uint32_t *>(row + at);
    if constexpr (E == 8) w[1] = reinterpret_cast<const uint32_t *>(row + at)[1];
  }
}
template <int FMT, int E>
__device__ __forceinline__ void decode(const uint32_t (&w)[2], float (&v)[E]) {
#pragma unroll
  for (int i = 0; i < E; i++) {
    if constexpr (FMT == INT4) {
      v[i] = (float)((int32_t)(w[0] << (28 - 4 * i)) >> 28);
    } else if constexpr (FMT == INT8) {
      v[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4)));
    } else {
      switch (i % 4) {
        case 0: v[i] = __builtin_amdgcn_cvt_f32_fp8((int)w[i / 4], 0); break;
        case 1: v[i] = __builtin_amdgcn_cvt_f32_fp8((int)w[i / 4], 1); break;
        case 2: v[i] = __builtin_amdgcn_cvt_f32_fp8((int)w[i / 4], 2); break;
        default: v[i] = __builtin_amdgcn_cvt_f32_fp8((int)w[i / 4], 3); break;
      }
    }
  }
}

// Sixteen bytes of output a thread, neighbouring threads' next to each other: the output is most of the bytes, so its lines are written
// whole and the codes, half to an eighth as many bytes, are read in whatever pieces that makes.  Four of a thread under way hide
// slot -> codes -> output, three steps behind each other.  131 072 fp32 rows of 768 from INT8, slots in any order: 109 us, 4.7 TB/s.  Of
// narrow rows in any order the lines of codes and scales are read for a part of each: 400 009 fp16 rows of 100 from INT4 30 us, in
// order 22 us (5.2 TB/s).
template <int T, int FMT>
__global__ __launch_bounds__(256) void row_read_kernel(RowCacheArgs c, const int64_t *slots, uint32_t n, void *out, uint32_t stride,
                                                       uint32_t rows_per_wg, FastDiv chunks, FastDiv block) {
  constexpr int U = READ_UNDER_WAY, E = 16 / elem_size<T>;
  for (uint64_t first = (uint64_t)blockIdx.x * rows_per_wg; first < n; first += (uint64_t)gridDim.x * rows_per_wg) {
    const uint32_t mine = n - first < rows_per_wg ? (uint32_t)(n - first) : rows_per_wg, all = mine * chunks.d;
    const uint64_t row_stride = (uint64_t)stride * elem_size<T>;
    uint8_t *to = static_cast<uint8_t *>(out) + first * row_stride;
    for (uint32_t i0 = threadIdx.x; i0 < all; i0 += 256 * U) {
      uint32_t row[U], at[U], codes[U][2];
      int64_t slot[U];
      u4 as_is[U];
      float scale[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const uint32_t i = i0 + u * 256 < all ? i0 + u * 256 : i0;   // behind the end: the first again, not written
        row[u] = chunks.div(i);
        at[u] = (i - row[u] * chunks.d) * E;
        slot[u] = slots[first + row[u]];
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const bool there = slot[u] >= 0 && (uint64_t)slot[u] < c.capacity;
        const uint64_t from = there ? (uint32_t)slot[u] : 0;   // one that is not there is read from slot 0 and zeroed
        const uint8_t *p = c.codes + from * c.row_bytes;
        if constexpr (FMT == NATIVE) {
          as_is[u] = *reinterpret_cast<const u4 *>(p + at[u] * elem_size<T>);
          if (!there) as_is[u] = u4{0, 0, 0, 0};
        } else {
          load_codes<FMT, E>(p, at[u], codes[u]);
          scale[u] = c.scales[from * c.nb + block.div(at[u])];
          if (!there) codes[u][0] = codes[u][1] = 0;
          if (!there) scale[u] = 0.0f;
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (i0 + u * 256 >= all) break;
        u4 w;
        if constexpr (FMT == NATIVE) {
          w = as_is[u];
        } else {
          float v[E];
          decode<FMT, E>(codes[u], v);
#pragma unroll
          for (int k = 0; k < E; k++) v[k] *= scale[u];
          // a block whose codes reach past the type's range (a largest magnitude next to its end): nothing finite becomes infinite
          constexpr float most = T == F32 ? 3.40282347e38f : T == BF16 ? 3.38953139e38f : 65504.0f;
          if (scale[u] > most / (FMT == E4M3 ? 448.0f : FMT == INT8 ? 128.0f : 8.0f)) {
#pragma unroll
            for (int k = 0; k < E; k++) v[k] = __builtin_fabsf(v[k]) > most ? __builtin_copysignf(most, v[k]) : v[k];
          }
#pragma unroll
          for (int k = 0; k < 4; k++) {
            if constexpr (T == F32) w[k] = __float_as_uint(v[k]);
            else w[k] = narrow2<T>(v[2 * k], v[2 * k + 1]);
          }
        }
        uint8_t *dst = to + (uint64_t)row[u] * row_stride + at[u] * elem_size<T>;
        if (at[u] + E <= c.dim) {
          if constexpr (T == F32) *reinterpret_cast<u4_any4 *>(dst) = w;
          else *reinterpret_cast<u4_any *>(dst) = w;
        } else {
#pragma unroll
          for (int k = 0; k < E; k++)
            if (at[u] + k < c.dim) {
              if constexpr (T == F32) reinterpret_cast<uint32_t *>(dst)[k] = w[k];
              else reinterpret_cast<uint16_t *>(dst)[k] = (uint16_t)(w[k / 2] >> (16 * (k % 2)));
            }
        }
      }
    }
  }
}

// ---- rules on scores -------------------------------------------------------------------------------------------------------

constexpr uint32_t COLUMNS = 4096;   // columns of a workgroup, whose counts of a query's two lists are kept in LDS

// A workgroup finds in the lists what falls among its columns (sums and maxima of integers: the same in any order), then goes over
// them once: eight bytes a cell, whatever the rules are.  256 x 200 003 with all of them: 62 - 67 us, 6.1 - 6.6 TB/s (a copy of
// as much memory: 5.2).  4096 columns: their counts are 32 KiB of LDS, five workgroups a CU.  Each of a query's workgroups reads its
// lists whole: 16 queries x 1 000 000 columns take 23 us without a list, 28 with 1000 entries each, 69 with 10 000, 461 with 100 000.
__global__ __launch_bounds__(256) void adjust_scores_kernel(AdjustArgs a, uint32_t tiles, uint64_t work) {
  constexpr int PER = COLUMNS / 1024;
  __shared__ alignas(16) uint32_t times[COLUMNS];   // how often a column was shown
  __shared__ alignas(16) uint32_t boost[COLUMNS];   // 1 + the place in the list of a column's last boost, 0: none
  const uint32_t tid = threadIdx.x;
  for (uint64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const uint32_t m = (uint32_t)(w / tiles), c0 = (uint32_t)(w - (uint64_t)m * tiles) * COLUMNS;
    uint32_t n = a.n_columns;
    if (a.counts) n = (uint32_t)cut(a.counts[m], (int32_t)n);
    if (c0 >= n) continue;   // the same for the whole workgroup
    const uint32_t mine = n - c0 < COLUMNS ? n - c0 : COLUMNS;
    int32_t s0 = 0, s1 = 0, b0 = 0, b1 = 0;
    if (a.r.seen_offsets) {
      s0 = cut(a.r.seen_offsets[m], (int32_t)a.r.n_seen);
      s1 = cut(a.r.seen_offsets[m + 1], (int32_t)a.r.n_seen);
    }
    if (a.r.bias_offsets) {
      b0 = cut(a.r.bias_offsets[m], (int32_t)a.r.n_bias);
      b1 = cut(a.r.bias_offsets[m + 1], (int32_t)a.r.n_bias);
    }
    const bool lists = s1 > s0 || b1 > b0;
    if (lists) {
      __syncthreads();   // the last piece's counts have been read
      for (uint32_t i = tid; i < COLUMNS / 4; i += 256) reinterpret_cast<u4 *>(times)[i] = reinterpret_cast<u4 *>(boost)[i] = u4{0, 0, 0, 0};
      __syncthreads();
      for (uint32_t i = (uint32_t)s0 + tid; i < (uint32_t)s1; i += 256) {   // (a list may end at the last 31-bit number)
        const uint32_t c = (uint32_t)a.r.seen_ids[i] - c0;
        if (c < mine) atomicAdd(&times[c], 1u);
      }
      for (uint32_t i = (uint32_t)b0 + tid; i < (uint32_t)b1; i += 256) {
        const uint32_t c = (uint32_t)a.r.bias_ids[i] - c0;
        if (c < mine) atomicMax(&boost[c], i - (uint32_t)b0 + 1);
      }
      __syncthreads();
    }
    const bool distance = a.r.form == RSGPU_SCORES_DISTANCE;
    const float gone = distance ? __builtin_inff() : -__builtin_inff();
    const float rep = a.r.repetition ? a.r.repetition[m] : 1.0f;
    const float freq = a.r.frequency ? a.r.frequency[m] : 0.0f;
    const float pres = a.r.presence ? a.r.presence[m] : 0.0f;
    const uint32_t *mask = nullptr;
    if (a.r.mask) {
      const int64_t which = a.r.mask_rows ? a.r.mask_rows[m] : (int64_t)m;
      if (which >= 0 && (uint64_t)which < a.r.n_masks) mask = a.r.mask + (size_t)which * a.r.mask_words;
    }
    const float *in = a.in + (size_t)m * a.ld + c0;
    float *out = a.out + (size_t)m * a.ld + c0;
    // sixteen columns a thread, all loaded before the first is written (scores_out may be scores_in)
    f32x4 v[PER];
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const uint32_t i = (k * 256 + tid) * 4;
      if (i + 4 <= mine) {
        v[k] = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any *>(in + i));   // 63 us for 72
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) v[k][e] = i + e < mine ? in[i + e] : 0.0f;
      }
    }
    uint32_t allowed[PER];
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const uint32_t i = (k * 256 + tid) * 4;
      allowed[k] = mask && i < mine ? mask[(c0 + i) / 32] >> (c0 + i) % 32 : 15u;   // the four are in one word
    }
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const uint32_t i = (k * 256 + tid) * 4;
      if (lists) {
        const u4 n4 = *reinterpret_cast<const u4 *>(times + i), b4 = *reinterpret_cast<const u4 *>(boost + i);
        if (((n4[0] | n4[1]) | (n4[2] | n4[3])) | ((b4[0] | b4[1]) | (b4[2] | b4[3]))) {
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (n4[e] | b4[e]) {
              float p = distance ? 1.0f - v[k][e] : v[k][e];
              if (n4[e]) {
                p = p > 0.0f ? p / rep : p * rep;
                p -= __builtin_fmaf((float)n4[e], freq, pres);
              }
              if (b4[e]) p += a.r.bias_values[(uint32_t)b0 + b4[e] - 1];
              v[k][e] = distance ? 1.0f - p : p;
            }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; e++) v[k][e] = allowed[k] >> e & 1u ? v[k][e] : gone;
      if (i + 4 <= mine) {
        *reinterpret_cast<f32x4_any *>(out + i) = v[k];
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (i + e < mine) out[i + e] = v[k][e];
      }
    }
  }
}

// a grid holds fewer than 2^32 threads; kernels go round when there is more work
constexpr uint64_t MOST_WORKGROUPS = 1 << 20;
uint32_t workgroups(uint64_t work) { return (uint32_t)(work < MOST_WORKGROUPS ? work : MOST_WORKGROUPS); }

// rows of a workgroup so that it has about `most` chunks, with enough workgroups to fill the chip first
uint32_t rows_a_workgroup(uint32_t n, uint32_t chunks, uint32_t most) {
  uint32_t rows = (most + chunks - 1) / chunks;
  while (rows > 1 && (n + rows - 1) / rows < 2048) rows = (rows + 1) / 2;
  return rows;
}

template <int T, int FMT>
void write_as(const RowCacheArgs &c, const void *rows, uint32_t stride, const int64_t *slots, uint32_t n, hipStream_t s) {
  if (c.nb == 1 && c.dim > 512) {
    const dim3 grid(workgroups(((uint64_t)n + 3) / 4));
    if (c.dim <= 1024) launch(row_write_whole_kernel<T, FMT, 2>, grid, 256, s, c, rows, stride, slots, n);
    else if constexpr (T == F32) launch(row_write_whole_kernel<T, FMT, 0>, grid, 256, s, c, rows, stride, slots, n);
    else if (c.dim <= 2048) launch(row_write_whole_kernel<T, FMT, 4>, grid, 256, s, c, rows, stride, slots, n);
    else launch(row_write_whole_kernel<T, FMT, 0>, grid, 256, s, c, rows, stride, slots, n);
    return;
  }
  // the lanes of a block, or of a row that is one
  uint32_t lanes = 4;
  while (lanes * 8 < (c.nb == 1 ? rows_padded(c.dim) : c.block)) lanes *= 2;
  const uint32_t chunks = c.nb * lanes, per = rows_a_workgroup(n, chunks, 256 * WRITE_UNDER_WAY);
  const dim3 grid(workgroups(((uint64_t)n + per - 1) / per));
  const FastDiv d(chunks);
  switch (lanes) {
    case 4: launch(row_write_kernel<T, FMT, 4>, grid, 256, s, c, rows, stride, slots, n, per, d); break;
    case 8: launch(row_write_kernel<T, FMT, 8>, grid, 256, s, c, rows, stride, slots, n, per, d); break;
    case 16: launch(row_write_kernel<T, FMT, 16>, grid, 256, s, c, rows, stride, slots, n, per, d); break;
    case 32: launch(row_write_kernel<T, FMT, 32>, grid, 256, s, c, rows, stride, slots, n, per, d); break;
    default: launch(row_write_kernel<T, FMT, 64>, grid, 256, s, c, rows, stride, slots, n, per, d); break;
  }
}

template <int T>
void write_from(const RowCacheArgs &c, const void *rows, uint32_t stride, const int64_t *slots, uint32_t n, hipStream_t s) {
  switch (c.format) {
    case INT8: return write_as<T, INT8>(c, rows, stride, slots, n, s);
    case E4M3: return write_as<T, E4M3>(c, rows, stride, slots, n, s);
    case INT4: return write_as<T, INT4>(c, rows, stride, slots, n, s);
    default: {
      const uint32_t chunks = c.row_bytes / 16, per = rows_a_workgroup(n, chunks, 256 * WRITE_UNDER_WAY);
      launch(row_copy_in_kernel<T>, dim3(workgroups(((uint64_t)n + per - 1) / per)), 256, s, c, rows, stride, slots, n, per, FastDiv(chunks));
    }
  }
}

template <int T>
void read_to(const RowCacheArgs &c, const int64_t *slots, uint32_t n, void *out, uint32_t stride, hipStream_t s) {
  constexpr uint32_t E = 16 / elem_size<T>;
  const uint32_t chunks = (c.dim + E - 1) / E, per = rows_a_workgroup(n, chunks, 256 * READ_UNDER_WAY);
  const dim3 grid(workgroups(((uint64_t)n + per - 1) / per));
  const FastDiv d(chunks), b(c.block);
  switch (c.format) {
    case INT8: launch(row_read_kernel<T, INT8>, grid, 256, s, c, slots, n, out, stride, per, d, b); break;
    case E4M3: launch(row_read_kernel<T, E4M3>, grid, 256, s, c, slots, n, out, stride, per, d, b); break;
    case INT4: launch(row_read_kernel<T, INT4>, grid, 256, s, c, slots, n, out, stride, per, d, b); break;
    default: launch(row_read_kernel<T, NATIVE>, grid, 256, s, c, slots, n, out, stride, per, d, b); break;
  }
}


}  // namespace

void launch_row_write(const RowCacheArgs &c, const void *rows, uint32_t stride, const int64_t *slots, uint32_t n, hipStream_t s) {
  if (c.type == F32) write_from<F32>(c, rows, stride, slots, n, s);
  else if (c.type == F16) write_from<F16>(c, rows, stride, slots, n, s);
  else write_from<BF16>(c, rows, stride, slots, n, s);
}

void launch_row_read(const RowCacheArgs &c, const int64_t *slots, uint32_t n, void *out, uint32_t stride, hipStream_t s) {
  if (c.type == F32) read_to<F32>(c, slots, n, out, stride, s);
  else if (c.type == F16) read_to<F16>(c, slots, n, out, stride, s);
  else read_to<BF16>(c, slots, n, out, stride, s);
}

void launch_adjust_scores(const AdjustArgs &a, hipStream_t s) {
  const uint32_t tiles = (a.n_columns + COLUMNS - 1) / COLUMNS;
  const uint64_t work = (uint64_t)tiles * a.n_queries;
  launch(adjust_scores_kernel, dim3(workgroups(work)), 256, s, a, tiles, work);
}

}  // namespace rsgpu
