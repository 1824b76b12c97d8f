// rows_device.hpp -- what the row cache's kernels share (rows_kernels.hip, partition_kernels.hpp).
#pragma once
#include <hip/hip_runtime.h>

#include <tuple>

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
typedef uint16_t ushort2v __attribute__((ext_vector_type(2)));
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

// Eight elements as they are in memory; those from `valid` on are zeros.  They are read all the same where `more` says that the
// memory goes on behind them (another row of at least four elements follows): see cut().
template <int T>
struct Raw8 {
  u4 w[elem_size<T> / 2];

  __device__ __forceinline__ void load_whole(const void *row, uint32_t at) {
    if constexpr (T == F32) {
      const u4_any4 *p = reinterpret_cast<const u4_any4 *>(static_cast<const float *>(row) + at);
      w[0] = p[0];
      w[1] = p[1];
    } else {
      w[0] = *reinterpret_cast<const u4_any *>(static_cast<const uint16_t *>(row) + at);
    }
  }
  __device__ __forceinline__ void load(const void *row, uint32_t at, uint32_t valid, bool more = false) {
    if (valid >= 8 || (more && valid)) {
      load_whole(row, at);
      return;
    }
    zero();
    if (!valid) return;
    if (at) {   // the row's last elements: the last eight, of which the first go
      load_whole(row, at + valid - 8);
      drop(8 - valid);
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
      if ((uint32_t)i < valid) {
        if constexpr (T == F32) w[i / 4][i % 4] = static_cast<const uint32_t *>(row)[i];
        else w[0][i / 2] |= (uint32_t)static_cast<const uint16_t *>(row)[i] << (16 * (i % 2));
      }
  }
  // the first `by` < 8 elements go, zeros follow
  __device__ __forceinline__ void drop(uint32_t by) {
    constexpr int N = 2 * elem_size<T>;
#pragma unroll
    for (int m = 4; m >= 1; m /= 2) {
      const bool move = by & m;
      constexpr int per = 4 / elem_size<T>;
      const int d = m / per;   // dwords; 0: half of one
#pragma unroll
      for (int k = 0; k < N; k++) {
        const uint32_t here = w[k / 4][k % 4], next = k + 1 < N ? w[(k + 1) / 4 % (N / 4)][(k + 1) % 4] : 0;
        const uint32_t far = k + d < N ? w[(k + d) / 4 % (N / 4)][(k + d) % 4] : 0;
        w[k / 4][k % 4] = move ? (d ? far : __builtin_amdgcn_alignbit(next, here, 16)) : here;
      }
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
  // the bits, as fp32, of the largest magnitude: as integers, so that an infinity or a NaN is larger than every number
  __device__ __forceinline__ uint32_t most() const {
    if constexpr (T == F32) {
      uint32_t a = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const uint32_t b = w[i / 4][i % 4] & 0x7fffffffu;
        a = a > b ? a : b;
      }
      return a;
    } else {   // two at a time
      ushort2v a = __builtin_bit_cast(ushort2v, w[0][0] & 0x7fff7fffu);
#pragma unroll
      for (int i = 1; i < 4; i++) a = __builtin_elementwise_max(a, __builtin_bit_cast(ushort2v, w[0][i] & 0x7fff7fffu));
      const uint32_t b = a[0] > a[1] ? a[0] : a[1];
      return T == BF16 ? b << 16 : __float_as_uint(f16_to_f32(b));
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

// A launch whose own error is what it returns: hipGetLastError() behind it would also hand over one that an earlier call of the caller's
// thread has left (an event asked before it was ready is one), for work that is already under way.
template <typename... P, typename... A>
void launch(void (*kernel)(P...), dim3 grid, uint32_t threads, hipStream_t s, const A &...args) {
  std::tuple<P...> held(args...);
  std::apply([&](P &...x) {
    void *at[] = {static_cast<void *>(&x)...};
    HIP_CHECK(hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, dim3(threads), at, 0, s));
  }, held);
}

// a count or an offset from the device, within its range
__device__ __forceinline__ int32_t cut(int32_t x, int32_t most) { return x < 0 ? 0 : x > most ? most : x; }

}  // namespace
}  // namespace rsgpu
