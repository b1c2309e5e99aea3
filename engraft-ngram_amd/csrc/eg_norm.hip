// The residual's addition and the RMS norm of the sum, and their gradients.
//
//   h = x + residual (rounded to the residual's type: what is kept is what is normed)
//   r = 1 / sqrt(mean(h^2) + eps),   y = h r w       (y in 16 or 32 bits, or in blocks of 8)
//   d_h = d_residual + r (w d_y) - h r^3 / d sum(w d_y h),   d_w = sum over rows of d_y h r
//
// Bound by its bytes: every row is read once, held in registers between its sum and its output, and
// written once.  A row is w wavefronts' (1 to 16), of which each holds CH pieces of 512 values, eight
// consecutive ones a lane: a piece is four blocks of the 8-bit output, whose largest values are found
// within 16 lanes.  A lane's eight squares are added in 32 bits (in 64 where they leave its range), the lanes' sums and r in 64
// (r's error is in all of a row's values), and a value next to a border between two e4m3 numbers is 64 bits: it rounds as the
// exact one does (of 3.5 million values none or one otherwise, 2 or 3 in 32 bits).  One piece a wavefront up to d = 8192
// (d = 2560: five wavefronts a row): a wavefront a row of 2560 held five, and its registers left four wavefronts a SIMD, or
// spilled; 61 us for 8,188 rows of bf16.  Longer rows hold two or three pieces a wavefront of 1,024 threads' 128 registers: the
// forward's ragged kernels and all of the gradient's spill there.
#include <algorithm>

#include "eg_fp8.h"

namespace eg {
namespace {

struct Value {
  const void* p;
  int32_t dtype;
};

__device__ inline void store8_any(void* p, int32_t dtype, int64_t at, int valid, const float (&x)[8]) {
  if (dtype == EG_DTYPE_F32)
    store8((float*)p + at, valid, x);
  else if (dtype == EG_DTYPE_BF16)
    store8((__bf16*)p + at, valid, x);
  else
    store8((_Float16*)p + at, valid, x);
}

__device__ inline float wave_sum(float x) {
#define EG_ROW_ADD(ror) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + (ror), 0xf, 0xf, false));
  EG_ROW_ADD(8)
  EG_ROW_ADD(4)
  EG_ROW_ADD(2)
  EG_ROW_ADD(1)
#undef EG_ROW_ADD
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

__device__ inline double wave_sum(double x) {
#define EG_ROW_ADD(ror)                                                                                                           \
  {                                                                                                                               \
    const u32x2 b = __builtin_bit_cast(u32x2, x);                                                                                 \
    x += __builtin_bit_cast(double, u32x2{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)b[0], 0x120 + (ror), 0xf, 0xf, false),     \
                                          (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b[1], 0x120 + (ror), 0xf, 0xf, false)});   \
  }
  EG_ROW_ADD(8)
  EG_ROW_ADD(4)
  EG_ROW_ADD(2)
  EG_ROW_ADD(1)
#undef EG_ROW_ADD
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// The sum over a row's W wavefronts; `part`: W values for each row of the workgroup, of the buffer that
// this call's parity names (one barrier a call: the next one uses the other buffer).
template <typename T>
__device__ inline T row_sum(T x, int w, int row_of_block, int wave_of_row, T* part) {
  x = wave_sum(x);
  if (w == 1) return x;
  if ((threadIdx.x & 63) == 0) part[row_of_block * w + wave_of_row] = x;
  __syncthreads();
  T s = 0;
#pragma unroll 2
  for (int i = 0; i < w; ++i) s += part[row_of_block * w + i];
  return s;
}

// 1 / sqrt(a) to about 2^-50: the instruction's approximation and two steps towards it
__device__ inline double inverse_root(double a) {
  const double first = __builtin_amdgcn_rsq(a);
  double r = first;
#pragma unroll
  for (int i = 0; i < 2; ++i) r *= 1.5 - 0.5 * a * r * r;
  return r == r ? r : first;  // 0 and infinity, whose steps are NaN
}

// v g r as floats for the rounding to 8 bits, which round there as the exact products do.  e4m3 values and scales turn at floats
// with 19 low bits of zeros; 32-bit products are off by 3 units of 2^-24, at most 3 last places, and those within 4
// of such a float (1.7e-5 of all) are taken again in 64 bits, and beside it if that is where they round to (from more than
// 2^-48 away, the products' own error).  `wide`: all in 64 bits, where r is no normal 32-bit number.  All of them in 64 bits: 40 us for 8,188 rows of 2560 bf16, 30 so.
__device__ inline void normed8(const float (&v)[8], const float (&g)[8], double r, bool wide, float (&y)[8]) {
  const float rf = (float)r;
  bool near = wide;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = v[i] * rf * g[i];
    near |= ((__float_as_uint(y[i]) + 4) & 0x7ffffu) <= 8 && y[i] != 0.0f;
  }
  if (__builtin_expect(near, 0)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x = v[i], w = g[i];
      asm volatile("" : "+v"(x), "+v"(w));  // one value after the other: eight at once take the registers of two wavefronts
      const double a = (double)x * (double)w * r;
      const uint32_t bits = __float_as_uint((float)a);
      const double d = fabs((double)(float)a);
      const bool aside = (bits & 0x7ffffu) == 0 && fabs(d - fabs(a)) > d * 0x1p-48;
      y[i] = __uint_as_float(!aside ? bits : d < fabs(a) ? bits + 1 : bits - 1);
      asm volatile("" : "+v"(y[i]));
    }
  }
}

// Whether a mean of squares that were added in 32 bits (eight of them) may be far off: infinite (or NaN), or below 2^-120,
// where the squares' own roundings, up to 2^-150 each, reach 2^-30 of it.  From its sign and exponent.
__device__ inline bool leaves_32(double mean) {
  return __builtin_bit_cast(u32x2, mean)[1] - ((1023u - 120u) << 20) >= (0x7ffu - (1023u - 120u)) << 20;
}

struct NormArgs {
  Value x, residual;
  const float* weight;        // NULL: 1
  int64_t x_stride, r_stride;
  int64_t rows;
  int d, w;                   // w: wavefronts a row
  float eps;
  double inv_d;
  void* h;
  int64_t h_stride;
  void* y;
  int32_t y_dtype;            // < 0: blocks
  int64_t y_stride;
  uint8_t* scales;
  int64_t scale_stride;
  float* rstd;
};

// T's rounding, as fp32
template <typename T>
__device__ inline float rounded(float x) {
  return (float)(T)x;
}

// R void: no residual (h is x, and not written).
template <typename X, typename R, int CH, bool RAGGED>
__global__ __launch_bounds__(1024) void norm_kernel(const NormArgs a) {
  __shared__ double part[2][16];
  constexpr bool ADD = !std::is_same<R, void>::value;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slot = wave / a.w, w = wave - slot * a.w, rows_here = (blockDim.x >> 6) / a.w;
  const bool weighted = a.weight != nullptr;
  int at[CH], left[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    at[c] = (c * a.w + w) * 512 + lane * 8;
    left[c] = RAGGED ? a.d - at[c] : at[c] < a.d ? 8 : 0;
  }
  const int blocks = (a.d + 127) >> 7;
  int parity = 0;
  for (int64_t first = (int64_t)blockIdx.x * rows_here; first < a.rows; first += (int64_t)gridDim.x * rows_here) {
    const bool live = first + slot < a.rows;
    const int64_t row = live ? first + slot : a.rows - 1;
    float v[CH][8];
    const X* const x = (const X*)a.x.p + row * a.x_stride;
    Raw8<X> raw_x[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) raw_x[c] = load_raw<RAGGED>(x, at[c], a.d);
    if constexpr (ADD) {
      const R* const res = (const R*)a.residual.p + row * a.r_stride;
      Raw8<R> raw_r[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c) raw_r[c] = load_raw<RAGGED>(res, at[c], a.d);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float r[8];
        values_of<RAGGED, X>(raw_x[c], at[c], a.d, v[c]);
        values_of<RAGGED, R>(raw_r[c], at[c], a.d, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = rounded<R>(v[c][i] + r[i]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c) values_of<RAGGED, X>(raw_x[c], at[c], a.d, v[c]);
    }
    // the weights' loads (from L2) take the registers that the row's bytes had, and the time of its sum
    Raw8<float> raw_g[CH];
    if (weighted) {
#pragma unroll
      for (int c = 0; c < CH; ++c) raw_g[c] = load_raw<RAGGED>(a.weight, at[c], a.d);
    }
    double s = 0.0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float part8[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) part8[i] = v[c][i] * v[c][i] + v[c][i + 4] * v[c][i + 4];
      s += (double)((part8[0] + part8[1]) + (part8[2] + part8[3]));
    }
    s = row_sum(s, a.w, slot, w, part[parity]);
    const double eps = (double)a.eps;
    double mean = fma(s, a.inv_d, eps);
    // Such a row's squares are added again in 64 bits; the other rows keep their sums.  Where two rows share a workgroup's barrier
    // (of two wavefronts each), every wavefront finds out the same of both, from the same sums.  The look costs 1 to 3 %.
    const bool wide = __builtin_amdgcn_readfirstlane((int)leaves_32(mean)) != 0;
    bool again = wide;
    if (CH == 1 && a.w == 2) {
      const double* const other = part[parity] + 2 - 2 * slot;
      again |= leaves_32(fma(other[0] + other[1], a.inv_d, eps));
    }
    parity ^= 1;
    if (__builtin_expect(__builtin_amdgcn_readfirstlane((int)again) != 0, 0)) {
      s = 0.0;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float x = v[c][i];
          asm volatile("" : "+v"(x));
          s += (double)x * (double)x;
        }
      s = row_sum(s, a.w, slot, w, part[parity]);
      parity ^= 1;
      if (wide) mean = fma(s, a.inv_d, eps);
    }
    const double root = inverse_root(mean);
    const float rstd = (float)root;
    if (!live) continue;
    if (a.rstd != nullptr && w == 0 && lane == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if constexpr (ADD) store8((R*)a.h + row * a.h_stride + at[c], left[c], v[c]);
      float y[8], g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = 1.0f;
      if (weighted) values_of<RAGGED, float>(raw_g[c], at[c], a.d, g);
      if (a.y_dtype >= 0 && !wide) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = v[c][i] * rstd * g[i];
      } else {
        normed8(v[c], g, root, wide, y);
      }
      if (a.y_dtype >= 0) {
        store8_any(a.y, a.y_dtype, row * a.y_stride + at[c], left[c], y);
      } else {
        const int piece = c * a.w + w;
        if (piece * 4 < blocks)
          store_blocks(y, (uint8_t*)a.y + row * a.y_stride, a.scales + row * a.scale_stride, piece, blocks, lane);
      }
    }
  }
}

struct GradArgs {
  Value d_y, h, d_res;          // d_res.p NULL: none
  const float* weight;          // NULL: 1
  int64_t dy_stride, h_stride, dr_stride;
  const float* rstd;
  int64_t rows;
  int d, w;
  void* d_x;
  int32_t dx_dtype;
  int64_t dx_stride;
  void* d_x2;                   // the same in a second type (NULL: not wanted)
  int32_t dx2_dtype;
  int64_t dx2_stride;
  float* partial;               // [gridDim][d] sums of the weight's gradient; NULL: not wanted
};

// D: d_y's type; T: h's (and d_res's).
template <typename D, typename T, int CH, bool RAGGED>
__global__ __launch_bounds__(1024) void norm_grad_kernel(const GradArgs a) {
  __shared__ float part[2][16];
  extern __shared__ float sums[];  // [d]: a workgroup's share of the weight's gradient, with several rows in flight
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slot = wave / a.w, w = wave - slot * a.w, rows_here = (blockDim.x >> 6) / a.w;
  const bool weighted = a.weight != nullptr;
  int at[CH], left[CH];
  float d_w[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    at[c] = (c * a.w + w) * 512 + lane * 8;
    left[c] = a.d - at[c];
#pragma unroll
    for (int i = 0; i < 8; ++i) d_w[c][i] = 0.0f;
  }
  const float inv_d = 1.0f / (float)a.d;
  int parity = 0;
  for (int64_t first = (int64_t)blockIdx.x * rows_here; first < a.rows; first += (int64_t)gridDim.x * rows_here) {
    const bool live = first + slot < a.rows;
    const int64_t row = live ? first + slot : a.rows - 1;
    float p[CH][8], u[CH][8];
    const D* const d_y = (const D*)a.d_y.p + row * a.dy_stride;
    const T* const h = (const T*)a.h.p + row * a.h_stride;
    const T* const d_res = (const T*)a.d_res.p + row * a.dr_stride;
    const float rstd = a.rstd[row];
    Raw8<D> raw_p[CH];
    Raw8<T> raw_u[CH], raw_r[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) raw_p[c] = load_raw<RAGGED>(d_y, at[c], a.d);
#pragma unroll
    for (int c = 0; c < CH; ++c) raw_u[c] = load_raw<RAGGED>(h, at[c], a.d);
    Raw8<float> raw_g[CH];
    if (weighted) {
#pragma unroll
      for (int c = 0; c < CH; ++c) raw_g[c] = load_raw<RAGGED>(a.weight, at[c], a.d);
    }
    if (a.d_res.p != nullptr) {
#pragma unroll
      for (int c = 0; c < CH; ++c) raw_r[c] = load_raw<RAGGED>(d_res, at[c], a.d);
    }
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      values_of<RAGGED, D>(raw_p[c], at[c], a.d, p[c]);
      values_of<RAGGED, T>(raw_u[c], at[c], a.d, u[c]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        u[c][i] *= rstd;
        d_w[c][i] = live ? d_w[c][i] + p[c][i] * u[c][i] : d_w[c][i];
      }
      if (weighted) {
        float g[8];
        values_of<RAGGED, float>(raw_g[c], at[c], a.d, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) p[c][i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) s += p[c][i] * u[c][i];
    }
    s = row_sum(s, a.w, slot, w, part[parity]) * inv_d;
    parity ^= 1;
    if (!live) continue;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = 0.0f;
      if (a.d_res.p != nullptr) values_of<RAGGED, T>(raw_r[c], at[c], a.d, o);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] += rstd * (p[c][i] - u[c][i] * s);
      store8_any(a.d_x, a.dx_dtype, row * a.dx_stride + at[c], left[c], o);
      if (a.d_x2 != nullptr) store8_any(a.d_x2, a.dx2_dtype, row * a.dx2_stride + at[c], left[c], o);
    }
  }
  if (a.partial == nullptr) return;
  // the workgroup's rows in flight, in order
  for (int k = 0; k < rows_here; ++k) {
    if (slot == k) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left[c]) {
            if (k > 0) d_w[c][i] += sums[at[c] + i];
            if (k + 1 < rows_here) sums[at[c] + i] = d_w[c][i];
          }
      if (k + 1 == rows_here) {
#pragma unroll
        for (int c = 0; c < CH; ++c) store8(a.partial + (int64_t)blockIdx.x * a.d + at[c], left[c], d_w[c]);
      }
    }
    if (k + 1 < rows_here) __syncthreads();
  }
}

// d_w: the workgroups' partial sums, in order: 64 columns a workgroup, whose wavefronts take every 16th of them.
__global__ __launch_bounds__(1024) void weight_grad_kernel(const float* __restrict__ partial, int count, int d, float* __restrict__ d_w) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  float x = 0.0f;
  if (c < d) {
#pragma unroll 8
    for (int i = wave; i < count; i += 16) x += partial[(int64_t)i * d + c];
  }
  s[wave][lane] = x;
  __syncthreads();
  if (wave == 0 && c < d) {
    x = s[0][lane];
#pragma unroll
    for (int i = 1; i < 16; ++i) x += s[i][lane];
    d_w[c] = x;
  }
}

constexpr int64_t kMaxWidth = 40 * 512;

// Wavefronts a row, and pieces a wavefront holds.
struct Split {
  int w, ch;
};
Split split_of(int64_t d) {
  const int pieces = (int)((d + 511) / 512), ch = (pieces + 15) / 16;
  return {(pieces + ch - 1) / ch, ch};
}

// f(the kernel's pieces a wavefront as a constant)
template <typename F>
int with_pieces(int ch, const F& f) {
  if (ch == 1) return f(std::integral_constant<int, 1>{});
  if (ch == 2) return f(std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 3>{});
}

// Rows that a workgroup has in flight, and workgroups: all rows' of the forward; of the gradient two of up to 16 wavefronts a CU,
// since every one adds a row of partial sums of the weight's.
int rows_at_once(int w, int wavefronts) { return w > wavefronts ? 1 : wavefronts / w; }
int64_t grad_groups(int64_t rows, int w) {
  const int at_once = rows_at_once(w, 16);
  return std::min<int64_t>((rows + at_once - 1) / at_once, 512);
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" {

int eg_add_rms_norm(const eg_norm* o, void* h, int64_t h_stride, void* y, int32_t y_dtype, int64_t y_stride,
                    const eg_fp8_matrix* y8, float* rstd, void* stream) {
  EG_CHECK_ARG(o != nullptr, "add_rms_norm: NULL");
  EG_CHECK_ARG(o->rows >= 0 && o->d >= 1, "add_rms_norm: %lld rows of %lld", (long long)o->rows, (long long)o->d);
  if (o->d > kMaxWidth) return set_error(EG_ERR_UNSUPPORTED, "add_rms_norm: rows of %lld values, at most %lld", (long long)o->d, (long long)kMaxWidth);
  EG_CHECK_ARG(o->eps >= 0.0f, "add_rms_norm: eps=%g", (double)o->eps);
  if (const int rc = check_values(o->x, o->x_dtype, o->rows, o->d, o->x_stride, "add_rms_norm: x"); rc != EG_OK) return rc;
  if (o->residual != nullptr) {
    if (const int rc = check_values(o->residual, o->r_dtype, o->rows, o->d, o->r_stride, "add_rms_norm: residual"); rc != EG_OK) return rc;
    EG_CHECK_ARG(o->r_dtype == o->x_dtype || o->r_dtype == EG_DTYPE_F32, "add_rms_norm: a residual of x's type or f32 expected");
    if (const int rc = check_values(h, o->r_dtype, o->rows, o->d, h_stride, "add_rms_norm: h"); rc != EG_OK) return rc;
  }
  EG_CHECK_ARG((uintptr_t)o->weight % 4 == 0, "add_rms_norm: misaligned weight");
  EG_CHECK_ARG((y != nullptr) != (y8 != nullptr) || o->rows == 0, "add_rms_norm: y or y8 expected");
  if (y8 != nullptr) {
    if (const int rc = check_fp8(y8, 1, "add_rms_norm: y8"); rc != EG_OK) return rc;
    EG_CHECK_ARG(y8->rows == o->rows && y8->k == o->d, "add_rms_norm: y8 is %lld x %lld for %lld rows of %lld", (long long)y8->rows,
                 (long long)y8->k, (long long)o->rows, (long long)o->d);
  } else {
    if (const int rc = check_values(y, y_dtype, o->rows, o->d, y_stride, "add_rms_norm: y"); rc != EG_OK) return rc;
  }
  EG_CHECK_ARG((uintptr_t)rstd % 4 == 0, "add_rms_norm: misaligned rstd");
  if (o->rows == 0) return EG_OK;
  const bool add = o->residual != nullptr;
  const Area none = bytes_area(nullptr, 0, ""), x_area = values_area(o->x, o->x_dtype, o->rows, o->d, o->x_stride, "x"),
             r_area = add ? values_area(o->residual, o->r_dtype, o->rows, o->d, o->r_stride, "the residual") : none,
             h_area = add ? values_area(h, o->r_dtype, o->rows, o->d, h_stride, "h") : none,
             y_area = y8 ? blocks_area(*y8, "y") : values_area(y, y_dtype, o->rows, o->d, y_stride, "y"),
             scales = y8 ? scales_area(*y8, "y's scales") : none, rstd_area = bytes_area(rstd, o->rows * 4, "rstd"),
             weight = bytes_area(o->weight, o->d * 4, "the weight");
  if (const int rc = check_areas("add_rms_norm", {y_area, scales, rstd_area}, {x_area, r_area, h_area, weight}); rc != EG_OK) return rc;
  // h in the place of x or of the residual: every value is read by the lane that writes it
  const bool on_x = h == o->x && h_stride == o->x_stride && o->x_dtype == o->r_dtype, on_r = h == o->residual && h_stride == o->r_stride;
  if (const int rc = check_areas("add_rms_norm", {h_area}, {on_r ? none : r_area, on_x ? none : x_area, weight}); rc != EG_OK) return rc;
  const Split s = split_of(o->d);
  const int at_once = rows_at_once(s.w, 4), threads = at_once * s.w * 64;
  const int64_t groups = std::min<int64_t>((o->rows + at_once - 1) / at_once, 1 << 20);
  const NormArgs a = {{o->x, o->x_dtype}, {o->residual, o->r_dtype}, o->weight, o->x_stride, o->r_stride, o->rows,
                      (int)o->d, s.w, o->eps, 1.0 / (double)o->d, h, h_stride, y8 ? y8->q : y, y8 ? -1 : y_dtype, y8 ? y8->stride : y_stride,
                      y8 ? y8->scales : nullptr, y8 ? y8->scale_stride : 0, rstd};
  auto launch = [&](auto x, auto r) {
    using X = decltype(x);
    using R = typename decltype(r)::type;
    return with_pieces(s.ch, [&](auto ch) {
      constexpr int CH = decltype(ch)::value;
      const auto kernel = o->d % 8 != 0 ? norm_kernel<X, R, CH, true> : norm_kernel<X, R, CH, false>;
      kernel<<<(unsigned)groups, threads, 0, (hipStream_t)stream>>>(a);
      return launch_status("norm_kernel");
    });
  };
  return with_type(o->x_dtype, [&](auto x) {
    if (o->residual == nullptr) return launch(x, std::common_type<void>{});
    if (o->r_dtype == o->x_dtype) return launch(x, std::common_type<decltype(x)>{});
    return launch(x, std::common_type<float>{});
  });
}

int64_t eg_add_rms_norm_grad_workspace_size(int64_t rows, int64_t d) {
  if (rows < 0 || d < 1 || d > kMaxWidth) return -1;
  return grad_groups(rows, split_of(d).w) * d * 4;
}

int eg_add_rms_norm_grad(const eg_norm_grad* o, void* d_x, int32_t dx_dtype, int64_t dx_stride, void* d_x2, int32_t dx2_dtype,
                         int64_t dx2_stride, float* d_weight, void* workspace, int64_t workspace_bytes, void* stream) {
  EG_CHECK_ARG(o != nullptr, "add_rms_norm_grad: NULL");
  EG_CHECK_ARG(o->rows >= 0 && o->d >= 1, "add_rms_norm_grad: %lld rows of %lld", (long long)o->rows, (long long)o->d);
  if (o->d > kMaxWidth)
    return set_error(EG_ERR_UNSUPPORTED, "add_rms_norm_grad: rows of %lld values, at most %lld", (long long)o->d, (long long)kMaxWidth);
  if (const int rc = check_values(o->d_y, o->dy_dtype, o->rows, o->d, o->dy_stride, "add_rms_norm_grad: d_y"); rc != EG_OK) return rc;
  if (const int rc = check_values(o->h, o->h_dtype, o->rows, o->d, o->h_stride, "add_rms_norm_grad: h"); rc != EG_OK) return rc;
  if (o->d_residual != nullptr)
    if (const int rc = check_values(o->d_residual, o->h_dtype, o->rows, o->d, o->dr_stride, "add_rms_norm_grad: d_residual"); rc != EG_OK) return rc;
  EG_CHECK_ARG((uintptr_t)o->weight % 4 == 0, "add_rms_norm_grad: misaligned weight");
  EG_CHECK_ARG(o->rstd != nullptr || o->rows == 0, "add_rms_norm_grad: NULL rstd");
  if (const int rc = check_values(d_x, dx_dtype, o->rows, o->d, dx_stride, "add_rms_norm_grad: d_x"); rc != EG_OK) return rc;
  if (d_x2 != nullptr)
    if (const int rc = check_values(d_x2, dx2_dtype, o->rows, o->d, dx2_stride, "add_rms_norm_grad: d_x2"); rc != EG_OK) return rc;
  EG_CHECK_ARG((uintptr_t)d_weight % 4 == 0, "add_rms_norm_grad: misaligned d_weight");
  const Split s = split_of(o->d);
  const int rows_here = rows_at_once(s.w, 16), threads = rows_here * s.w * 64;
  const int64_t groups = grad_groups(o->rows, s.w);
  if (d_weight != nullptr) {
    if (workspace_bytes < groups * o->d * 4)
      return set_error(EG_ERR_WORKSPACE, "add_rms_norm_grad needs %lld bytes of workspace, got %lld", (long long)(groups * o->d * 4),
                       (long long)workspace_bytes);
    EG_CHECK_ARG(groups == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0), "add_rms_norm_grad: the workspace must be 16-byte aligned");
  }
  const Area none = bytes_area(nullptr, 0, "");
  if (const int rc = check_areas("add_rms_norm_grad",
                                 {values_area(d_x, dx_dtype, o->rows, o->d, dx_stride, "d_x"),
                                  d_x2 ? values_area(d_x2, dx2_dtype, o->rows, o->d, dx2_stride, "d_x2") : none,
                                  bytes_area(d_weight, o->d * 4, "d_weight"),
                                  d_weight ? bytes_area(workspace, groups * o->d * 4, "the workspace") : none},
                                 {values_area(o->d_y, o->dy_dtype, o->rows, o->d, o->dy_stride, "d_y"),
                                  values_area(o->h, o->h_dtype, o->rows, o->d, o->h_stride, "h"),
                                  o->d_residual ? values_area(o->d_residual, o->h_dtype, o->rows, o->d, o->dr_stride, "d_residual") : none,
                                  bytes_area(o->weight, o->d * 4, "the weight"), bytes_area(o->rstd, o->rows * 4, "rstd")});
      rc != EG_OK)
    return rc;
  const GradArgs a = {{o->d_y, o->dy_dtype}, {o->h, o->h_dtype}, {o->d_residual, o->h_dtype}, o->weight, o->dy_stride,
                      o->h_stride, o->dr_stride, o->rstd, o->rows, (int)o->d, s.w, d_x, dx_dtype, dx_stride, d_x2, dx2_dtype, dx2_stride,
                      d_weight ? (float*)workspace : nullptr};
  if (o->rows > 0) {
    const int rc = with_type(o->dy_dtype, [&](auto dy) {
      return with_type(o->h_dtype, [&](auto t) {
        return with_pieces(s.ch, [&](auto ch) {
          using D = decltype(dy);
          using T = decltype(t);
          constexpr int CH = decltype(ch)::value;
          const auto kernel = o->d % 8 != 0 ? norm_grad_kernel<D, T, CH, true> : norm_grad_kernel<D, T, CH, false>;
          kernel<<<(unsigned)groups, threads, d_weight && rows_here > 1 ? o->d * 4 : 0, (hipStream_t)stream>>>(a);
          return launch_status("norm_grad_kernel");
        });
      });
    });
    if (rc != EG_OK) return rc;
  }
  if (d_weight != nullptr) {
    weight_grad_kernel<<<(unsigned)((o->d + 63) / 64), 1024, 0, (hipStream_t)stream>>>((const float*)workspace, (int)groups, (int)o->d, d_weight);
    return launch_status("weight_grad_kernel");
  }
  return EG_OK;
}

}  // extern "C"
