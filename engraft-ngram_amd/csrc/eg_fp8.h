// Blocks of 8-bit floating point: 128 values along a row share a scale 2^e (a byte, e + 127) and
// are e4m3 after the division by it.  Shared by the products (eg_fp8.hip) and the norm that writes
// its rows in this form (eg_norm.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include <initializer_list>

#include "eg_common.h"
#include "eg_overlap.h"

namespace eg {

constexpr int kFp8Block = 128;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Eight values of T at any address of its own alignment: unaligned 16-byte accesses are ordinary
// ones here, and rows of odd lengths start anywhere.
template <typename T>
struct Eight {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

// Eight values of a row from `p` on, of which `valid` exist (0 in the place of the others).
template <typename T>
__device__ inline void load8(const T* __restrict__ p, int valid, float (&v)[8]) {
  if (valid >= 8) {
    const typename Eight<T>::type x = *(const typename Eight<T>::type*)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? (float)p[i] : 0.0f;
  }
}

// A lane's eight values of a row of d, from column `at` on, in two steps, so that many loads are on their way before the first
// is waited for: their bytes, by a load without a branch (a lane past the row's end reads its first or last
// eight; rows of less than eight: one by one), and their values, zeros in the place of what does not
// exist.  RAGGED: d is no multiple of eight, and the lane at the end reads the row's last eight and moves them.
template <typename T>
struct Raw8 {
  i32x4 w[sizeof(T) / 2];
};

template <bool RAGGED, typename T>
__device__ inline Raw8<T> load_raw(const T* __restrict__ row, int at, int d) {
  typedef i32x4 unaligned __attribute__((aligned(2)));
  Raw8<T> r;
  if (RAGGED && d < 8) {
    T x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = row[min(at + i, d - 1)];
    __builtin_memcpy(&r, x, sizeof(r));
    return r;
  }
  const T* const p = row + (RAGGED ? min(at, d - 8) : at < d ? at : 0);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = ((const unaligned*)p)[i];
  return r;
}

template <bool RAGGED, typename T>
__device__ inline void values_of(Raw8<T> r, int at, int d, float (&v)[8]) {
  const int left = d - at;
  if (RAGGED && d >= 8) {
    const int by = left < 8 ? (8 - left) & 7 : 0;  // (all are zeros below where none is left)
    if constexpr (sizeof(T) == 2) {
      r.w[0] = __builtin_bit_cast(i32x4, __builtin_bit_cast(unsigned __int128, r.w[0]) >> (16 * by));
    } else {
#pragma unroll
      for (int step = 4; step > 0; step >>= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int from = i + step < 8 ? r.w[((i + step) & 7) >> 2][(i + step) & 3] : 0;
          r.w[i >> 2][i & 3] = by & step ? from : r.w[i >> 2][i & 3];
        }
    }
  }
  if constexpr (sizeof(T) == 2) {
    typedef T t8 __attribute__((ext_vector_type(8)));
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[0][i] = left > 0 ? r.w[0][i] : 0;
    const t8 x = __builtin_bit_cast(t8, r.w[0]);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = RAGGED && d < 8 && i >= left ? 0.0f : (float)x[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = left > (RAGGED && d < 8 ? i : 0) ? __int_as_float(r.w[i >> 2][i & 3]) : 0.0f;
  }
}

template <typename T>
__device__ inline void store8(T* __restrict__ p, int valid, const float (&v)[8]) {
  if (valid >= 8) {
    typename Eight<T>::type x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (T)v[i];
    *(typename Eight<T>::type*)p = x;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) p[i] = (T)v[i];
  }
}

// The bits of |x|'s largest finite value so far: what is not finite has no part in a block's scale.
__device__ inline uint32_t finite_max(uint32_t top, float x) {
  const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
  return a < 0x7f800000u && a > top ? a : top;
}

// The largest of 16 lanes (a DPP row), in all of them.
__device__ inline uint32_t row_max(uint32_t x) {
#define EG_ROW_MAX(ror)                                                                                   \
  {                                                                                                       \
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + (ror), 0xf, 0xf, false);  \
    x = y > x ? y : x;                                                                                    \
  }
  EG_ROW_MAX(8)
  EG_ROW_MAX(4)
  EG_ROW_MAX(2)
  EG_ROW_MAX(1)
#undef EG_ROW_MAX
  return x;
}

// The scale's byte of a block whose largest magnitude has the bits `top`: the least e >= -127 with
// max <= 448 2^e (448 = 1.75 2^8), 0 for a block of zeros.
__host__ __device__ inline int scale_byte(uint32_t top) {
  if (top == 0) return 127;
  const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < 0 ? 0 : e;
}

// 2^(127 - byte), what a block's values are multiplied by; the byte is at most 247.
__device__ inline float scale_inverse(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// 2^(byte - 127) (2^-127 is no normal number; 255 is NaN)
__device__ inline float scale_value(uint32_t byte) {
  return byte == 0 ? __uint_as_float(0x00400000u) : byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
}

// Four values to e4m3 bytes, each to the nearest, ties to even; what is not finite becomes NaN.
__device__ inline uint32_t to_e4m3(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

__device__ inline u32x2 quantize8(const float (&v)[8], float inv) {
  return u32x2{to_e4m3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
               to_e4m3(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)};
}

// A wavefront's part of a row: lane l holds values 8 l .. 8 l + 7 of 512 (four blocks of 16 lanes)
// that start at block 4 g of a row with `blocks` blocks; values past the row's end are 0.
__device__ inline void store_blocks(const float (&v)[8], uint8_t* __restrict__ q_row, uint8_t* __restrict__ scale_row,
                                    int g, int blocks, int lane) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
    top = a > top ? a : top;
  }
  top = row_max(top);
  if (__builtin_expect(top >= 0x7f800000u, 0)) {  // (the same in a block's 16 lanes)
    top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = finite_max(top, v[i]);
    top = row_max(top);
  }
  const int byte = scale_byte(top);
  const int block = 4 * g + (lane >> 4);
  if (block < blocks) *(u32x2*)(q_row + (int64_t)g * 512 + lane * 8) = quantize8(v, scale_inverse(byte));
  uint32_t packed = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) packed |= (uint32_t)__builtin_amdgcn_readlane(byte, 16 * i) << (8 * i);
  if (lane == 0) *(uint32_t*)(scale_row + 4 * g) = packed;  // 127 (a block of zeros) past the last block
}

inline int item_size(int32_t dtype) { return dtype == EG_DTYPE_F32 ? 4 : 2; }
inline bool known_dtype(int32_t dtype) { return dtype == EG_DTYPE_F32 || dtype == EG_DTYPE_BF16 || dtype == EG_DTYPE_F16; }

// f(a zero of the type)
template <typename F>
int with_type(int32_t dtype, const F& f) {
  switch (dtype) {
    case EG_DTYPE_F32: return f((float)0);
    case EG_DTYPE_BF16: return f((__bf16)0);
    default: return f((_Float16)0);
  }
}

// Validates rows x cols values with unit stride within a row.
inline int check_values(const void* x, int32_t dtype, int64_t rows, int64_t cols, int64_t row_stride, const char* what) {
  EG_CHECK_ARG(known_dtype(dtype), "%s: dtype=%d", what, dtype);
  EG_CHECK_ARG(x != nullptr || rows == 0, "%s: NULL", what);
  EG_CHECK_ARG((uintptr_t)x % item_size(dtype) == 0, "%s: misaligned", what);
  EG_CHECK_ARG(row_stride >= cols || rows <= 1, "%s: rows of %lld values are %lld apart", what, (long long)cols,
               (long long)row_stride);
  return EG_OK;
}

// Memory that a call reads or writes.
struct Area {
  Extent extent;
  const char* name;
};
inline Area values_area(const void* p, int32_t dtype, int64_t rows, int64_t cols, int64_t stride, const char* name) {
  return {Extent(p, rows, cols, stride, 1, item_size(dtype)), name};
}
inline Area bytes_area(const void* p, int64_t bytes, const char* name) { return {Extent(p, 1, p ? bytes : 0, bytes, 1, 1), name}; }
inline Area blocks_area(const eg_fp8_matrix& m, const char* name) {
  return {Extent(m.q, m.rows, (m.k + 127) / 128 * 128, m.stride, 1, 1), name};
}
inline Area scales_area(const eg_fp8_matrix& m, const char* name) {
  return {Extent(m.scales, (m.rows + m.block_rows - 1) / m.block_rows, (m.k + 511) / 512 * 4, m.scale_stride, 1, 1), name};
}

// Validates that what is written shares no memory with what is read, nor with one another.
inline int check_areas(const char* what, std::initializer_list<Area> written, std::initializer_list<Area> read) {
  for (const Area* w = written.begin(); w != written.end(); ++w) {
    for (const Area* x = w + 1; x != written.end(); ++x)
      EG_CHECK_ARG(!overlap(w->extent, x->extent), "%s: %s overlaps %s", what, w->name, x->name);
    for (const Area& x : read) EG_CHECK_ARG(!overlap(w->extent, x.extent), "%s: %s overlaps %s", what, w->name, x.name);
  }
  return EG_OK;
}

// Validates a matrix of blocks; `block_rows`: what its scales have to cover.
int check_fp8(const eg_fp8_matrix* m, int block_rows, const char* what);

}  // namespace eg
