// rows_kernels.hip -- the row cache (include/rsgpu_rows.h) on gfx950: rows quantised into their slots and read back, the products
// of ragged groups of queries with the paged rows of their partitions, and the rules on a batch's scores.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "rows.hpp"

namespace rsgpu {
namespace {

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
// the caller's rows may begin at any element: gfx950 loads 16 bytes from any address its element type allows
typedef u4 u4_any __attribute__((aligned(2)));
typedef u4 u4_any4 __attribute__((aligned(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int F32 = VecSimType_FLOAT32, BF16 = VecSimType_BFLOAT16, F16 = VecSimType_FLOAT16;
constexpr int NATIVE = RSGPU_ROWS_NATIVE, INT8 = RSGPU_ROWS_INT8, E4M3 = RSGPU_ROWS_E4M3, INT4 = RSGPU_ROWS_INT4;

template <int T>
constexpr int elem_size = T == F32 ? 4 : 2;

// n / d for n, d < 2^31 without a division: m = ceil(2^(32 + l) / d), l = ceil(log2 d) (Granlund and Montgomery, 1994)
struct FastDiv {
  uint32_t d, m, l;
  explicit FastDiv(uint32_t div) : d(div), l(0) {
    while ((1ull << l) < d) l++;
    m = (uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return (uint32_t)(((uint64_t)__umulhi(n, m) + n) >> l);
  }
};

__device__ __forceinline__ float f16_to_f32(uint32_t low16) {
  const uint16_t h = (uint16_t)low16;
  _Float16 x;
  __builtin_memcpy(&x, &h, 2);
  return (float)x;
}

// eight elements as they are in memory; those from `valid` on are zeros.  They are read all the same where `more` says that the
// memory goes on behind them (another row follows)
template <int T>
struct Raw8 {
  u4 w[elem_size<T> / 2];

  __device__ __forceinline__ void load(const void *row, uint32_t at, uint32_t valid, bool more = false) {
    if (valid >= 8 || (more && valid)) {
      if constexpr (T == F32) {
        const u4_any4 *p = reinterpret_cast<const u4_any4 *>(static_cast<const float *>(row) + at);
        w[0] = p[0];
        w[1] = p[1];
      } else {
        w[0] = *reinterpret_cast<const u4_any *>(static_cast<const uint16_t *>(row) + at);
      }
      return;
    }
    zero();
    if (!valid) return;
#pragma unroll
    for (int i = 0; i < 8; i++)
      if ((uint32_t)i < valid) {
        if constexpr (T == F32) w[i / 4][i % 4] = static_cast<const uint32_t *>(row)[at + i];
        else w[0][i / 2] |= (uint32_t)static_cast<const uint16_t *>(row)[at + i] << (16 * (i % 2));
      }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)(elem_size<T> / 2); i++) w[i] = u4{0, 0, 0, 0};
  }
  // what was read behind the row's end is not of the row
  __device__ __forceinline__ void cut(uint32_t valid) {
    if (valid >= 8) return;
#pragma unroll
    for (int i = 0; i < 2 * (int)elem_size<T>; i++) {
      if constexpr (T == F32) w[i / 4][i % 4] = (uint32_t)i < valid ? w[i / 4][i % 4] : 0;
      else w[0][i] &= (uint32_t)(2 * i + 1) < valid ? 0xffffffffu : (uint32_t)(2 * i) < valid ? 0xffffu : 0;
    }
  }
  __device__ __forceinline__ void floats(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if constexpr (T == F32) v[i] = __uint_as_float(w[i / 4][i % 4]);
      else if constexpr (T == BF16) v[i] = __uint_as_float(i % 2 ? w[0][i / 2] & 0xffff0000u : w[0][i / 2] << 16);
      else v[i] = f16_to_f32(i % 2 ? w[0][i / 2] >> 16 : w[0][i / 2] & 0xffffu);
    }
  }
};

template <int T>
__device__ __forceinline__ void load8(const void *row, uint32_t at, uint32_t valid, float (&v)[8]) {
  Raw8<T> raw;
  raw.load(row, at, valid);
  raw.floats(v);
}

// ---- writing ---------------------------------------------------------------------------------------------------------------

// the bits of the largest magnitude: as integers, so that an infinity or a NaN is larger than every number
__device__ __forceinline__ uint32_t most8(const float (&v)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    a = a > b ? a : b;
  }
  return a;
}

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
    if constexpr (FMT == INT8) {
#pragma unroll
      for (int i = 0; i < 2; i++)
        c[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(q[4 * i + 3], q[4 * i + 2], 0x0c0c0400u), __builtin_amdgcn_perm(q[4 * i + 1], q[4 * i], 0x0c0c0400u), 0x05040100u);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) c[0] |= (q[i] & 15u) << (4 * i);
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

// blocks of 8 L elements: L neighbouring lanes have a block, eight elements each; a thread has several of them under way
template <int T, int FMT, int L>
__global__ __launch_bounds__(256) void row_write_kernel(RowCacheArgs c, const void *rows, uint32_t stride, const int64_t *slots, uint32_t n,
                                                        uint32_t rows_per_wg, FastDiv chunks) {
  constexpr int U = 4;
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
        raw[u].load(from + (uint64_t)row[u] * row_stride, at, there && at < c.dim ? c.dim - at : 0, first + row[u] + 1 < n);
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        float v[8];
        const uint32_t at = chunk[u] * 8;
        raw[u].cut(at < c.dim ? c.dim - at : 0);
        raw[u].floats(v);
        const uint32_t most = most_of_lanes<L>(most8(v));
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

// one scale a row: a wavefront has a row, and reads it again (from the caches) once its largest magnitude is known
template <int T, int FMT>
__global__ __launch_bounds__(256) void row_write_whole_kernel(RowCacheArgs c, const void *rows, uint32_t stride, const int64_t *slots, uint32_t n) {
  const uint32_t lane = threadIdx.x % 64;
  for (uint64_t r = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64; r < n; r += (uint64_t)gridDim.x * 4) {
    const int64_t slot = slots[r];
    if (slot < 0 || (uint64_t)slot >= c.capacity) continue;
    const void *row = static_cast<const uint8_t *>(rows) + (size_t)r * stride * elem_size<T>;
    const uint32_t padded = (c.dim + 31) / 32 * 32;
    float v[8];
    uint32_t most = 0;
    for (uint32_t at = lane * 8; at < c.dim; at += 512) {
      load8<T>(row, at, c.dim - at, v);
      const uint32_t o = most8(v);
      most = most > o ? most : o;
    }
    most = most_of_lanes<64>(most);
    float s, inv;
    scale_of<FMT>(most, s, inv);
    for (uint32_t at = lane * 8; at < padded; at += 512) {
      load8<T>(row, at, at < c.dim ? c.dim - at : 0, v);
      uint32_t code[2];
      encode8<FMT>(v, s, inv, code);
      store_codes8<FMT>(c.codes + (size_t)slot * c.row_bytes, at / 8, code);
    }
    if (lane == 0) c.scales[slot] = s;
  }
}

// rows kept as they are: sixteen bytes a thread
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

// two fp32 -> two 16-bit elements in a dword, nearest even
template <int T>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  uint32_t w;
  if constexpr (T == F16) {
    const half2v h = {(_Float16)a, (_Float16)b};
    __builtin_memcpy(&w, &h, 4);
  } else {
    const bf16x2 h = {(__bf16)a, (__bf16)b};
    __builtin_memcpy(&w, &h, 4);
  }
  return w;
}

// sixteen bytes of output a thread, neighbouring threads' next to each other; a thread has several under way
template <int T, int FMT>
__global__ __launch_bounds__(256) void row_read_kernel(RowCacheArgs c, const int64_t *slots, uint32_t n, void *out, uint32_t stride,
                                                       uint32_t rows_per_wg, FastDiv chunks, FastDiv block) {
  constexpr int U = 4, E = 16 / elem_size<T>;
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

// ---- products with a partition's rows --------------------------------------------------------------------------------------
//
// p[m][j] = sum_k q[m][k] c[j][k] s[j][k / block].  The codes are integers or e4m3 values that a 16-bit float holds exactly, so the
// matrix cores multiply codes with queries, and a block's sum is multiplied by its scale in fp32: no operand is rounded.
// fp32 operands go in as three bf16 each (8 + 8 + 8 bits of the significand, cut off exactly).

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

// x = hi + mid + lo, each a bf16 in the upper half of its dword.  An infinity or a NaN is hi alone.
__device__ __forceinline__ void split3(uint32_t x, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
  const bool special = (x & 0x7f800000u) == 0x7f800000u;
  hi = (x & 0xffff0000u) | (special && (x & 0xffffu) ? 0x400000u : 0);   // a NaN whose payload sits in the bits cut off stays one
  const float r = special ? 0.0f : __uint_as_float(x) - __uint_as_float(hi);
  mid = __float_as_uint(r) & 0xffff0000u;
  lo = __float_as_uint(r - __uint_as_float(mid));
}
__device__ __forceinline__ uint32_t upper2(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }

// eight fp32 -> eight bf16 in each of three planes
__device__ __forceinline__ void planes8(const float (&v)[8], u4 (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t a[3], b[3];
    split3(__float_as_uint(v[2 * i]), a[0], a[1], a[2]);
    split3(__float_as_uint(v[2 * i + 1]), b[0], b[1], b[2]);
#pragma unroll
    for (int k = 0; k < 3; k++) p[k][i] = upper2(a[k], b[k]);
  }
}

// eight codes -> eight 16-bit floats (INT4 with bf16: sixteenths of the codes, CODE_UNIT)
template <int FMT, int Q>
constexpr float CODE_UNIT = FMT == INT4 && Q != F16 ? 16.0f : 1.0f;

__device__ __forceinline__ uint32_t minus2(uint32_t x, float y) {
  half2v h;
  __builtin_memcpy(&h, &x, 4);
  h -= half2v{(_Float16)y, (_Float16)y};
  __builtin_memcpy(&x, &h, 4);
  return x;
}

template <int FMT, int Q>
__device__ __forceinline__ u4 widen8(uint32_t w0, uint32_t w1) {
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
        const bf16x2 h = i % 2 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
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
    for (int i = 0; i < 4; i++) r[i] = upper2(__float_as_uint(f[2 * i]), __float_as_uint(f[2 * i + 1]));
  }
  return r;
}

__device__ __forceinline__ int32_t cut(int32_t x, int32_t most) { return x < 0 ? 0 : x > most ? most : x; }

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
  uint32_t tiles, stride;
  Place at;
};
struct RunShared {
  uint32_t wave_sums[16];
  Place at;
};
// The offsets and counts are on the device, so every workgroup sums the partitions' tiles itself, a share of the partitions a
// thread, takes its even part of them, and the thread in whose share that begins says where.  TOGETHER: an eighth of the tiles, one
// after the other, is for the workgroups b, b + 8, ... that share a die's L2, and they go through it side by side.
constexpr uint32_t DIES = 8;
template <int THREADS, bool TOGETHER>
__device__ __forceinline__ Run find_run(const PartitionArgs &a, uint32_t tq, uint32_t tr, RunShared &shared) {
  const uint32_t tid = threadIdx.x, lane = tid % 64, per = (a.n_partitions + THREADS - 1) / THREADS;
  uint32_t own = 0;
  for (uint32_t i = 0; i < per; i++) {
    const uint32_t g = tid * per + i;
    if (g >= a.n_partitions) break;
    uint32_t lo, m, n;
    partition(a, g, lo, m, n);
    own += (m + tq - 1) / tq * ((n + tr - 1) / tr);
  }
  uint32_t sum = own;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) {
    const uint32_t v = __shfl_up(sum, k, 64);
    if (lane >= (uint32_t)k) sum += v;
  }
  if (lane == 63) shared.wave_sums[tid / 64] = sum;
  __syncthreads();
  uint32_t total = 0;
#pragma unroll
  for (uint32_t w = 0; w < THREADS / 64; w++) {
    const uint32_t v = shared.wave_sums[w];
    if (w < tid / 64) sum += v;
    total += v;
  }
  Run run;
  uint32_t first;
  if (TOGETHER) {
    const uint32_t die = blockIdx.x % DIES, from = (uint32_t)((uint64_t)total * die / DIES), to = (uint32_t)((uint64_t)total * (die + 1) / DIES);
    run.stride = gridDim.x / DIES;   // a multiple of the dies
    first = from + blockIdx.x / DIES;
    run.tiles = first < to ? (to - first + run.stride - 1) / run.stride : 0;
  } else {
    run.stride = 1;
    first = (uint32_t)((uint64_t)total * blockIdx.x / gridDim.x);
    run.tiles = (uint32_t)((uint64_t)total * (blockIdx.x + 1) / gridDim.x) - first;
  }
  if (run.tiles == 0) return run;
  if (sum - own <= first && first < sum) {
    Place p;
    p.left = first - (sum - own);
    for (p.g = tid * per;; p.g++) {
      partition(a, p.g, p.lo, p.m, p.n);
      const uint32_t tiles = (p.m + tq - 1) / tq * ((p.n + tr - 1) / tr);
      if (p.left < tiles) break;
      p.left -= tiles;
    }
    shared.at = p;
  }
  __syncthreads();
  run.at.g = __builtin_amdgcn_readfirstlane(shared.at.g);
  run.at.lo = __builtin_amdgcn_readfirstlane(shared.at.lo);
  run.at.m = __builtin_amdgcn_readfirstlane(shared.at.m);
  run.at.n = __builtin_amdgcn_readfirstlane(shared.at.n);
  run.at.left = __builtin_amdgcn_readfirstlane(shared.at.left);
  return run;
}

// eight elements of a query as 16-bit fragments (an fp32 query: three planes)
template <int Q>
__device__ __forceinline__ void stage8(const PartitionArgs &a, uint32_t query, uint32_t at, u4 (&w)[Q == F32 ? 3 : 1]) {
  const uint8_t *src = static_cast<const uint8_t *>(a.queries) + (size_t)query * a.stride * elem_size<Q>;
  if constexpr (Q == F32) {
    float v[8];
    load8<F32>(src, at, at < a.c.dim ? a.c.dim - at : 0, v);
    planes8(v, w);
  } else if (at + 8 <= a.c.dim) {
    w[0] = *reinterpret_cast<const u4_any *>(src + at * 2);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      uint32_t x = 0;
      if (at + 2 * i < a.c.dim) x = reinterpret_cast<const uint16_t *>(src)[at + 2 * i];
      if (at + 2 * i + 1 < a.c.dim) x |= (uint32_t)reinterpret_cast<const uint16_t *>(src)[at + 2 * i + 1] << 16;
      w[0][i] = x;
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

// W neighbouring elements of a row, as a lane takes them from LDS
template <int FMT, int Q, int W>
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
      out[0] = widen8<INT4, Q>(raw[f], 0);
    } else {
      out[0] = widen8<FMT, Q>(raw[2 * f], raw[2 * f + 1]);
    }
  }
};

// Few queries a partition: the rows' bytes are what it takes.  A workgroup has a run of tiles of 16 queries x 16 S rows a wavefront;
// the queries of a partition are put into LDS once for all its tiles (in parts of KP stages if the rows are longer than that).
// A wavefront takes its rows in stages of 4 KiB, 16 S rows x 256 / S bytes: four loads of 16 neighbouring bytes a lane, whole lines of
// the rows, one stage in registers under way (across tiles too) while the one before is multiplied.  (Loads in the shape of the matrix
// instruction's operand touch 16 lines each and cost the same whatever they bring: 2.4 TB/s with 8 bytes a lane, 4.6 with 16.)  A stage
// passes through 4 KiB of LDS that the wavefront has to itself, so nothing but the order of its own instructions guards it, and comes
// back as operands; the sixteen-byte chunks of a row change places with its number, so that neither side meets a bank twice.
// Every part of the loop is in the code once: a small call is mostly the first pass of its instructions through the caches.
template <int FMT, int Q, int W, int S, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 4) void partition_few_kernel(PartitionArgs a, FastDiv page) {
  typedef Piece<FMT, Q, W> P;
  constexpr int QP = Q == F32 ? 3 : 1, FR = W / 8, TQ = 16, WR = 16 * S, TR = WR * WAVES;
  constexpr int CS = 16 / S;                                  // chunks of a row in a stage
  constexpr int SP = CS * 16 / (4 * P::BYTES);                // steps of 4 W elements in a stage
  constexpr int QS = FMT == NATIVE ? 0 : (SP + 3) / 4;        // scale loads a stage and row group: a lane's quarter has every fourth
  constexpr int KP = (Q == F32 ? 24 : 32) / (SP * FR);        // stages of queries in LDS at a time: 72 or 32 KiB
  static_assert(SP >= 1 && KP >= 1, "");
  __shared__ u4 staged[KP * SP * FR * QP * 64];
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
  f32x4 acc[S];
#pragma unroll
  for (int k = 0; k < S; k++) acc[k] = f32x4{0, 0, 0, 0};
  uint32_t staged_g = ~0u, staged_q = 0, staged_p = 0;   // whose queries are in LDS, from which stage on
  uint32_t taken = 0;
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
      chunk[i] = *reinterpret_cast<const u4 *>(source[i] + (c < chunks ? c : chunks - 1) * 16);
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
      const u4 *queries = staged + use_stage % KP * (SP * FR * QP * 64) + lane;
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
        f32x4 part[S];
#pragma unroll
        for (int k = 0; k < S; k++) part[k] = FMT == NATIVE ? acc[k] : f32x4{0, 0, 0, 0};
#pragma unroll
        for (int f = 0; f < FR; f++) {
          u4 q[QP];
#pragma unroll
          for (int p = 0; p < QP; p++) q[p] = queries[((st * FR + f) * QP + p) * 64];
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
                if (p + c < 3) part[k] = mfma16<Q>(q[p], b[c], part[k]);   // the planes left out are below 2^-24 of the product
          }
        }
        // a step's sum, times the scale of the block that it is in (no branch for the block's end: the steps overlap)
        const uint32_t block = ((use_stage * SP + st) >> block_shift) - first_block;
#pragma unroll
        for (int k = 0; k < S; k++) {
          if (FMT == NATIVE) {
            acc[k] = part[k];
          } else {
            float v = scale[k][0];
#pragma unroll
            for (int q = 1; q < QS; q++) v = block / 4 == (uint32_t)q ? scale[k][q] : v;
            v = __uint_as_float(__builtin_amdgcn_ds_bpermute((block % 4 * 16 + col) * 4, __float_as_uint(v)));
#pragma unroll
            for (int r = 0; r < 4; r++) acc[k][r] = __builtin_fmaf(v, part[k][r], acc[k][r]);
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
      const uint32_t shift = asked > 8 ? 4 : asked > 4 ? 3 : asked > 2 ? 2 : asked > 1 ? 1 : 0;
      for (uint32_t i = tid; i < np * (SP * FR * 4) << shift; i += 64 * WAVES) {
        const uint32_t q = i & ((1u << shift) - 1), e = i >> shift, f = e % FR, h = e / FR % 4, st = e / (4 * FR);
        if (q >= asked) continue;   // what is in LDS behind them is multiplied and not used
        u4 w[QP];
        stage8<Q>(a, q0 + q, (p0 * SP + st) * (4 * W) + h * W + f * 8, w);
#pragma unroll
        for (int p = 0; p < QP; p++) staged[((st * FR + f) * QP + p) * 64 + h * 16 + q] = w[p];
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
          for (int r = 0; r < 4; r++) {
            const uint32_t q = now.q0 + quarter * 4 + r;
            if (q < now.q_end) {
              float p = acc[k][r] * CODE_UNIT<FMT, Q>;
              if constexpr (FMT == NATIVE && Q == F32) {
                // an infinity meets the other side's planes, some of them 0: the sum is taken again, element by element
                if (p != p && (there >> k & 1)) {
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
        acc[k] = f32x4{0, 0, 0, 0};
      }
      use_stage = 0;
    }
    if (use_stage == 0) {
      now = held;
      there = held_there;
    }
  }
}

// Many queries a partition: the matrix cores' work.  A workgroup has a run of tiles of 128 queries x 128 rows, a wavefront 64 x 64 of
// each; both sides go through LDS as operands of the 32 x 32 x 16 product, the rows' codes widened once on the way there.  A stage is
// 64 elements in two halves: one half is multiplied, the next is in the other half of LDS, and the two behind it are on their way in
// registers, of this tile or the next one's (with one on its way every half waited for memory: 132 us instead of the figure at the
// launch below).  In LDS an operand's 32 rows change places with the number of its eight elements, so that neither side meets a bank
// twice.  A block's products are summed by themselves and multiplied by the row's scale at every FLUSH elements.
// rows of a tile: 128 queries meet 256 rows where the sums of a tile are all that the registers hold
template <int FMT, int Q>
constexpr int MANY_ROWS = FMT == NATIVE && Q != F32 ? 256 : 128;
template <int FMT, int Q, int FLUSH>
__global__ __launch_bounds__(256, FMT == NATIVE && Q == F32 ? 1 : 2) void partition_many_kernel(PartitionArgs a, FastDiv page) {
  constexpr int TQ = 128, TR = MANY_ROWS<FMT, Q>, X = TR / 64, Y = 2, KC = 32, QP = Q == F32 ? 3 : 1, RP = FMT == NATIVE && Q == F32 ? 3 : 1;
  constexpr int C8 = KC / 8;                                                 // eights of a half
  constexpr int PIECE = FMT == NATIVE ? 8 : FMT == INT4 ? 32 : 16;           // elements of a row that a thread loads together
  constexpr int PIECE_BYTES = FMT == NATIVE ? 8 * elem_size<Q> : 16, PU = PIECE_BYTES / 16;
  constexpr int NP = KC / PIECE, RT = (TR * NP + 255) / 256;                  // pieces of a row in a half, of a thread
  constexpr int QU = Q == F32 ? 2 : 1, QN = TQ * C8 / 256;                    // 16 bytes of eight elements of a query, eights of a thread
  typedef Piece<FMT, Q, PIECE> P;
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
  uint32_t loads_taken = 1, load_stage = 0;
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
  u4 row_held[2][RT][PU], query_held[2][QN][QU];
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
    if (FMT != NATIVE) {
      const uint32_t b = base / a.c.block;
      scale_held[H] = scale_source[b < a.c.nb ? b : a.c.nb - 1];
    }
    // an eight that the query's end cuts is loaded from where it is whole, and moved below (rows of less than eight elements do not
    // come here)
    const uint32_t at = base + tid % C8 * 8;
#pragma unroll
    for (int i = 0; i < QN; i++) {
      const uint8_t *p = queries[i] + (size_t)(at + 8 <= a.c.dim ? at : a.c.dim - 8) * elem_size<Q>;
      if constexpr (Q == F32) {
        query_held[H][i][0] = reinterpret_cast<const u4_any4 *>(p)[0];
        query_held[H][i][1] = reinterpret_cast<const u4_any4 *>(p)[1];
      } else {
        query_held[H][i][0] = *reinterpret_cast<const u4_any *>(p);
      }
    }
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
        uint32_t v[4 * QU];
#pragma unroll
        for (int k = 0; k < 4 * QU; k++) v[k] = by < 8 ? query_held[H][i][k / 4][k % 4] : 0;
#pragma unroll
        for (int m = 4; m >= 1; m /= 2) {
          const bool move = by & m;
          const int d = m * elem_size<Q> / 4;
#pragma unroll
          for (int k = 0; k < 4 * QU; k++) {
            const uint32_t next = k + 1 < 4 * QU ? v[k + 1 < 4 * QU ? k + 1 : 0] : 0, far = d && k + d < 4 * QU ? v[k + d < 4 * QU ? k + d : 0] : 0;
            v[k] = move ? (d ? far : __builtin_amdgcn_alignbit(next, v[k], 16)) : v[k];
          }
        }
#pragma unroll
        for (int k = 0; k < 4 * QU; k++) query_held[H][i][k / 4][k % 4] = v[k];
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
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = __uint_as_float(query_held[H][i][k / 4][k % 4]);
        planes8(v, w);
      } else {
        w[0] = query_held[H][i][0];
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
    if (FMT != NATIVE && tid < TR) s_lds[H][tid] = scale_held[H];
  };

  // ---- the products
  const uint32_t wave_q = X == 2 ? wave / 2 * 64 : 0, wave_r = X == 2 ? wave % 2 * 64 : wave * 64;
  f32x16 acc[X][Y], part[X][Y];
#pragma unroll
  for (int x = 0; x < X; x++)
#pragma unroll
    for (int y = 0; y < Y; y++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[x][y][r] = 0.0f;
  const auto multiply = [&](auto which) {
    constexpr int H = decltype(which)::value;
    constexpr bool FRESH = FMT != NATIVE && (H == 0 || FLUSH == KC);   // a block's sums begin
    f32x16(&sum)[X][Y] = FMT == NATIVE ? acc : part;
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
          if (p + c < 3) {   // the planes left out are below 2^-24 of the product
#pragma unroll
            for (int x = 0; x < X; x++)
#pragma unroll
              for (int y = 0; y < Y; y++) {
                const f32x16 none = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
                sum[x][y] = mfma<Q>(q[x][p], r[y][c], FRESH && k == 0 && p == QP - 1 ? none : sum[x][y]);   // (one plane of rows there)
              }
          }
    }
    if (FMT != NATIVE && (H == 1 || FLUSH == KC)) {
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
      float p = sums[x][y][r] * CODE_UNIT<FMT, Q>;
      if constexpr (FMT == NATIVE && Q == F32) {
        // an infinity meets the other side's planes, some of them 0: the sum is taken again, element by element
        if (p != p && (there >> y & 1)) {
          bool is;
          const uint64_t slot = slot_of(j, page_of(t, j), is);
          p = plain_product(reinterpret_cast<const float *>(a.c.codes + slot * a.c.row_bytes), static_cast<const float *>(a.queries) + q * a.stride, a.c.dim);
        }
      }
      if (a.form == RSGPU_SCORES_DISTANCE) p = 1.0f - p;
      __builtin_nontemporal_store(there >> y & 1 ? p : gone, at + (uint64_t)q * a.ld);
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
  uint32_t use_stage = 0, used = 0;
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

// ---- rules on scores -------------------------------------------------------------------------------------------------------

constexpr uint32_t COLUMNS = 4096;   // columns of a workgroup, whose counts of a query's two lists are kept in LDS

// A workgroup finds in the lists what falls among its columns (sums and maxima of integers: the same in any order), then goes over
// them once.
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
      for (int32_t i = s0 + (int32_t)tid; i < s1; i += 256) {
        const uint32_t c = (uint32_t)a.r.seen_ids[i] - c0;
        if (c < mine) atomicAdd(&times[c], 1u);
      }
      for (int32_t i = b0 + (int32_t)tid; i < b1; i += 256) {
        const uint32_t c = (uint32_t)a.r.bias_ids[i] - c0;
        if (c < mine) atomicMax(&boost[c], (uint32_t)(i - b0) + 1);
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
        v[k] = *reinterpret_cast<const f32x4_any *>(in + i);
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
              if (b4[e]) p += a.r.bias_values[b0 + b4[e] - 1];
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

// rows of a workgroup so that it has a few chunks a thread, with enough workgroups to fill the chip first
uint32_t rows_a_workgroup(uint32_t n, uint32_t chunks) {
  uint32_t rows = (1024 + chunks - 1) / chunks;
  while (rows > 1 && (n + rows - 1) / rows < 2048) rows = (rows + 1) / 2;
  return rows;
}

template <int T, int FMT>
void write_as(const RowCacheArgs &c, const void *rows, uint32_t stride, const int64_t *slots, uint32_t n, hipStream_t s) {
  if (c.block != 32 && c.block != 64 && c.block != 128) {
    hipLaunchKernelGGL((row_write_whole_kernel<T, FMT>), dim3(workgroups(((uint64_t)n + 3) / 4)), dim3(256), 0, s, c, rows, stride, slots, n);
    return;
  }
  const uint32_t chunks = c.nb * (c.block / 8), per = rows_a_workgroup(n, chunks);
  const dim3 grid(workgroups(((uint64_t)n + per - 1) / per));
  const FastDiv d(chunks);
  if (c.block == 32) hipLaunchKernelGGL((row_write_kernel<T, FMT, 4>), grid, dim3(256), 0, s, c, rows, stride, slots, n, per, d);
  else if (c.block == 64) hipLaunchKernelGGL((row_write_kernel<T, FMT, 8>), grid, dim3(256), 0, s, c, rows, stride, slots, n, per, d);
  else hipLaunchKernelGGL((row_write_kernel<T, FMT, 16>), grid, dim3(256), 0, s, c, rows, stride, slots, n, per, d);
}

template <int T>
void write_from(const RowCacheArgs &c, const void *rows, uint32_t stride, const int64_t *slots, uint32_t n, hipStream_t s) {
  switch (c.format) {
    case INT8: return write_as<T, INT8>(c, rows, stride, slots, n, s);
    case E4M3: return write_as<T, E4M3>(c, rows, stride, slots, n, s);
    case INT4: return write_as<T, INT4>(c, rows, stride, slots, n, s);
    default: {
      const uint32_t chunks = c.row_bytes / 16, per = rows_a_workgroup(n, chunks);
      hipLaunchKernelGGL((row_copy_in_kernel<T>), dim3(workgroups(((uint64_t)n + per - 1) / per)), dim3(256), 0, s, c, rows, stride, slots, n, per, FastDiv(chunks));
    }
  }
}

template <int T>
void read_to(const RowCacheArgs &c, const int64_t *slots, uint32_t n, void *out, uint32_t stride, hipStream_t s) {
  constexpr uint32_t E = 16 / elem_size<T>;
  const uint32_t chunks = (c.dim + E - 1) / E, per = rows_a_workgroup(n, chunks);
  const dim3 grid(workgroups(((uint64_t)n + per - 1) / per));
  const FastDiv d(chunks), b(c.block);
  switch (c.format) {
    case INT8: hipLaunchKernelGGL((row_read_kernel<T, INT8>), grid, dim3(256), 0, s, c, slots, n, out, stride, per, d, b); break;
    case E4M3: hipLaunchKernelGGL((row_read_kernel<T, E4M3>), grid, dim3(256), 0, s, c, slots, n, out, stride, per, d, b); break;
    case INT4: hipLaunchKernelGGL((row_read_kernel<T, INT4>), grid, dim3(256), 0, s, c, slots, n, out, stride, per, d, b); break;
    default: hipLaunchKernelGGL((row_read_kernel<T, NATIVE>), grid, dim3(256), 0, s, c, slots, n, out, stride, per, d, b); break;
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

template <int FMT, int Q>
void scores_as(const PartitionArgs &a, hipStream_t s) {
  const FastDiv page(a.page_rows);
  const uint32_t asked = a.n_partitions < a.n_queries ? a.n_partitions : a.n_queries;   // partitions with queries, at most
  const uint32_t each = a.n_queries / a.n_partitions;
  // no more workgroups than there can be tiles, and no more than are resident at once
  const auto grid = [&](uint32_t tq, uint32_t tr, uint64_t resident) {
    const uint64_t tiles = ((uint64_t)a.n_queries / tq + asked) * ((a.most_rows + tr - 1) / tr);
    return dim3((uint32_t)(tiles < resident ? tiles : resident));
  };
  if (each >= 48 && a.c.dim >= 8) {
    const auto many = [&](auto kernel) {
      dim3 g = grid(128, MANY_ROWS<FMT, Q>, resident(reinterpret_cast<const void *>(kernel), 256));
      g.x = (g.x + DIES - 1) / DIES * DIES;
      hipLaunchKernelGGL(kernel, g, dim3(256), 0, s, a, page);
    };
    if constexpr (FMT == NATIVE) many(partition_many_kernel<FMT, Q, 64>);
    else if (a.c.block == 32) many(partition_many_kernel<FMT, Q, 32>);
    else many(partition_many_kernel<FMT, Q, 64>);
    return;
  }
  // the rows' chunks of a stage: the number that leaves the fewest places empty, the largest of those
  const uint32_t chunks = a.c.row_bytes / 16;
  uint32_t cs = 16;
  constexpr bool widest = Q == F32;   // an fp32 step is eight chunks, and 64 rows of three planes do not fit into 128 registers
  for (uint32_t c : {8u, 4u})
    if (!(widest && c == 4) && (chunks + c - 1) / c * c < (chunks + cs - 1) / cs * cs) cs = c;
  const auto few = [&](auto w) {
    constexpr int W = decltype(w)::value, WAVES = Q == F32 ? 16 : 8;
    const auto launch = [&](auto kernel, uint32_t tr) {
      hipLaunchKernelGGL(kernel, grid(16, tr, resident(reinterpret_cast<const void *>(kernel), 64 * WAVES)), dim3(64 * WAVES), 0, s, a, page);
    };
    if (cs == 16) launch(partition_few_kernel<FMT, Q, W, 1, WAVES>, 16 * WAVES);
    else if (cs == 8) launch(partition_few_kernel<FMT, Q, W, 2, WAVES>, 32 * WAVES);
    else if constexpr (!widest) launch(partition_few_kernel<FMT, Q, W, 4, WAVES>, 64 * WAVES);
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

void launch_row_write(const RowCacheArgs &c, const void *rows, uint32_t stride, const int64_t *slots, uint32_t n, hipStream_t s) {
  if (c.type == F32) write_from<F32>(c, rows, stride, slots, n, s);
  else if (c.type == F16) write_from<F16>(c, rows, stride, slots, n, s);
  else write_from<BF16>(c, rows, stride, slots, n, s);
  HIP_CHECK(hipGetLastError());
}

void launch_row_read(const RowCacheArgs &c, const int64_t *slots, uint32_t n, void *out, uint32_t stride, hipStream_t s) {
  if (c.type == F32) read_to<F32>(c, slots, n, out, stride, s);
  else if (c.type == F16) read_to<F16>(c, slots, n, out, stride, s);
  else read_to<BF16>(c, slots, n, out, stride, s);
  HIP_CHECK(hipGetLastError());
}

void launch_partition_scores(const PartitionArgs &a, hipStream_t s) {
  if (a.c.type == F32) scores_from<F32>(a, s);
  else if (a.c.type == F16) scores_from<F16>(a, s);
  else scores_from<BF16>(a, s);
  HIP_CHECK(hipGetLastError());
}

void launch_adjust_scores(const AdjustArgs &a, hipStream_t s) {
  const uint32_t tiles = (a.n_columns + COLUMNS - 1) / COLUMNS;
  const uint64_t work = (uint64_t)tiles * a.n_queries;
  hipLaunchKernelGGL(adjust_scores_kernel, dim3(workgroups(work)), dim3(256), 0, s, a, tiles, work);
  HIP_CHECK(hipGetLastError());
}

}  // namespace rsgpu
