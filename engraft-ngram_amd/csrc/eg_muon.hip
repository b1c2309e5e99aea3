// A momentum step whose update is orthogonalised by Newton-Schulz products: the
// optimizer of the PLE block's projection weights (whose gradients ple_forward's
// backward gives; the reference's own descent trains table rows alone).
//
//   m = mu m + g,  u = g + mu m (nesterov) or m,  X = u / (|u|_F + eps),
//   `steps` times:  A = X X^T,  B = b A + c A^2,  X = a X + B X,
//   w = (1 - lr decay) w - lr scale X.
//
// X is taken with its shorter side as rows (an orthogonalised transpose is the
// transposed result), m x n with m <= n.  A and B are symmetric: only the tiles
// on and above the diagonal are computed, so an iteration costs
// m^2 n + m^3 + 2 m^2 n multiply-adds x 2 / 2.
//
// Arithmetic.  fp16 matrix cores, sums in fp32.  |X|_2 <= |X|_F <= 1 and the
// polynomial keeps the singular values below a bound the host follows from step
// to step, so every element of X, A and B has a known bound and one power of two
// an iteration puts it below 60,000: fp16's 11 bits (three more than bf16's at
// the same rate) over a range whose smallest normal is 2^-30 of that bound.  Two
// planes (PLANES 2: hi = rne(x), lo = rne(x - hi), 22 bits, products hi hi + hi lo
// + lo hi) keep fp32's accuracy (X within 1.2e-6 of float64's at 2560 x 2560, torch's fp32
// products 3.9e-6): what a step takes unless told otherwise.  One plane costs a third of the matrix
// work and leaves X within 1.1e-3, a rounding of 2^-12 at a time: less than half a unit of a bf16 X,
// but 1.3 % (10240 x 2560) to 4.6 % (64 x 256) of a step's bf16 weights then differ from the fp32
// update's, 0.01 % with two.  10240 x 2560: 1,366 us for 3,097.
//
// Layout.  An operand is kept fragment-major: 32 rows x 16 k are one 1 KB run
// (lane l holds row l % 32, k 8 (l / 32) .. + 7: one MFMA operand), [row block]
// [k / 16][plane].  A product needs X by rows (A = X X^T) and X^T by rows (B X =
// B (X^T)^T), so an iteration writes both; the MFMA's output registers hold
// four consecutive rows of a column, which is how X^T's runs are laid out, and X's
// go through LDS.  Rows and columns are padded with zeros to multiples of 64.
#include "eg_common.h"
#include "eg_lds.h"
#include "eg_overlap.h"

#include <math.h>

#include <algorithm>

namespace eg {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kRun = 1024;       // bytes of a fragment: 32 rows x 16 k of fp16
constexpr int kMaxBatch = 64;    // matrices a launch, at most

// Byte offset of fragment (row block, k / 16, plane) in an operand of k16 fragments a row block.
template <int PLANES>
__device__ inline int64_t run_at(int64_t row_block, int64_t k16s, int64_t k16, int plane) {
  return ((row_block * k16s + k16) * PLANES + plane) * kRun;
}

// ---- momentum, norm, planes -------------------------------------------------------------------

struct Strides {
  int64_t row, col;
};

struct Matrices {
  void* param[kMaxBatch];
  const void* grad[kMaxBatch];
  float* momentum[kMaxBatch];
};

template <typename F>
__device__ inline void by_type(int dtype, F&& f) {
  if (dtype == EG_DTYPE_F32) f(0.0f);
  else if (dtype == EG_DTYPE_BF16) f((__bf16)0.0f);
  else f((_Float16)0.0f);
}

// Four values of a row from column c on (zeros past the end).
template <typename T>
__device__ inline void load4(const T* row, Strides s, int64_t c, int64_t cols, float (&v)[4]) {
  struct __attribute__((packed, aligned(sizeof(T)))) Four {
    T x[4];
  };
  if (s.col == 1 && c + 4 <= cols) {
    const Four q = *(const Four*)(row + c);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (float)q.x[k];
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = c + k < cols ? (float)row[(c + k) * s.col] : 0.0f;
  }
}

struct UpdateArgs {
  int64_t rows, cols;
  Strides grad, momentum;
  int grad_dtype, has_momentum, nesterov;
  float mu;
  int tiles_c, tiles;  // 64 x 64 tiles along a row, and in all
  double* partials;    // [matrix][tile]: sums of u^2, in 64 bits: a square of 1e20 or 1e-23 has no place in fp32
};

// u of an element, from the gradient and the momentum after its update.
__device__ inline float update_of(const UpdateArgs& a, float g, float m) {
  if (!a.has_momentum) return g;
  return a.nesterov ? g + a.mu * m : m;
}

// A thread's part of a 64 x 64 tile: four columns from c on of the rows r0 + 16 i, i < 4.
struct TilePart {
  int64_t r0, c;
};
__device__ inline TilePart tile_part(const UpdateArgs& a, unsigned tile) {
  return {(int64_t)(tile / a.tiles_c) * 64 + threadIdx.x / 16, (int64_t)(tile % a.tiles_c) * 64 + threadIdx.x % 16 * 4};
}

// Grid (tiles, matrices): a 64 x 64 tile's momentum, and its part of |u|^2.  Bound by HBM: the
// gradient and the momentum read, the momentum written.
template <typename G>
__device__ inline double momentum_tile(const UpdateArgs& a, const G* grad, float* mom) {
  const TilePart p = tile_part(a, blockIdx.x);
  float g[4][4], m[4][4];
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = min(p.r0 + 16 * i, a.rows - 1);
    load4(grad + r * a.grad.row, a.grad, p.c, a.cols, g[i]);
    if (a.has_momentum) load4((const float*)mom + r * a.momentum.row, a.momentum, p.c, a.cols, m[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = p.r0 + 16 * i;
    if (r >= a.rows) continue;
    float now[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      now[k] = a.has_momentum ? a.mu * m[i][k] + g[i][k] : 0.0f;
      const double u = (double)update_of(a, g[i][k], now[k]);
      sum += u * u;
    }
    if (!a.has_momentum) continue;
    float* to = mom + r * a.momentum.row;
    struct __attribute__((packed, aligned(4))) Four {
      float x[4];
    };
    if (a.momentum.col == 1 && p.c + 4 <= a.cols) {
      *(Four*)(to + p.c) = {now[0], now[1], now[2], now[3]};
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (p.c + k < a.cols) to[(p.c + k) * a.momentum.col] = now[k];
    }
  }
  return sum;
}

__global__ __launch_bounds__(256) void muon_momentum_kernel(const UpdateArgs a, const Matrices mats) {
  __shared__ double red[4];
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double sum = 0.0;
  by_type(a.grad_dtype, [&](auto zero) {
    using G = decltype(zero);
    sum = momentum_tile(a, (const G*)mats.grad[b], mats.momentum[b]);
  });
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) red[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) a.partials[(int64_t)b * a.tiles + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// Grid (matrices): |u|^2 of matrices of many tiles, where every workgroup of the planes kernel would
// read them all.
__global__ __launch_bounds__(1024) void muon_norm_kernel(const double* partials, int tiles, double* squares) {
  __shared__ double red[16];
  const double* part = partials + (int64_t)blockIdx.x * tiles;
  double sum = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < tiles; i += 1024) sum += part[i];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 16; ++w) sum += red[w];
  squares[blockIdx.x] = sum;
}

struct PlanesArgs {
  UpdateArgs u;
  const double* squares;  // [matrix]: |u|^2; NULL: the partial sums' sum
  float eps, scale;     // x = u / (|u| + eps), kept times scale
  char *by_row, *by_col;  // fragments of u and of u^T
  int64_t batch_row, batch_col;  // bytes from one matrix to the next
  int64_t k16_row, k16_col;      // fragments along a row of u, of u^T
};

// scale / (|u| + eps) from |u|^2, finite also where both are tiny (zeros stay zeros).
__device__ inline float scale_of(double square, float scale, float eps) {
  const double s = (double)scale / (sqrt(square) + (double)eps);
  return s > 3.4e38 ? 3.4e38f : (float)s;  // NaN stays
}

// v's planes.  v is one fp32 value to the compiler: rounded to fp16 as part of the
// multiplication that made it (v_fma_mixlo_f16) in one place and by itself in the
// other, hi and the hi that lo is taken from differ at ties.
__device__ inline void split(float v, _Float16& hi, _Float16& lo) {
  asm("" : "+v"(v));
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

template <int PLANES>
__device__ inline void store_run(char* at, int lane, const float (&v)[8]) {
  f16x8 hi, lo;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    _Float16 h, l;
    split(v[i], h, l);
    hi[i] = h;
    lo[i] = l;
  }
  *(f16x8*)(at + lane * 16) = hi;
  if (PLANES == 2) *(f16x8*)(at + kRun + lane * 16) = lo;
}

// Grid (padded tiles, matrices): a 64 x 64 tile of x as fragments of both orders.  Bound by HBM: u's
// parts read again, both orders written; 26 M elements of bf16 gradient and fp32 momentum to one plane
// 44 us (262 MB, 5.9 TB/s), to two 62 (367 MB), the momentum kernel before it 50 us (262 MB, 5.3 TB/s).
template <int PLANES>
__global__ __launch_bounds__(256) void muon_planes_kernel(const PlanesArgs p, const Matrices mats) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const UpdateArgs& a = p.u;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = blockIdx.y;
  // the tiles the momentum kernel did last first: they are still cached
  const unsigned at_tile = gridDim.x - 1 - blockIdx.x;
  const int64_t tr = at_tile / a.tiles_c, tc = at_tile % a.tiles_c;
  if (p.squares == nullptr) {
    double sum = 0.0;
    const double* part = a.partials + (int64_t)b * a.tiles;
#pragma unroll 8
    for (int i = threadIdx.x; i < a.tiles; i += 256) sum += part[i];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) red[wave] = sum;
  }
  by_type(a.grad_dtype, [&](auto zero) {
    using G = decltype(zero);
    const G* grad = (const G*)mats.grad[b];
    const float* mom = mats.momentum[b];
    const TilePart at = tile_part(a, at_tile);
    float g[4][4], m[4][4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t r = min(at.r0 + 16 * i, a.rows - 1);
      load4(grad + r * a.grad.row, a.grad, at.c, a.cols, g[i]);
      if (a.has_momentum) load4(mom + r * a.momentum.row, a.momentum, at.c, a.cols, m[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        tile[threadIdx.x / 16 + 16 * i][threadIdx.x % 16 * 4 + k] =
            at.r0 + 16 * i < a.rows && at.c + k < a.cols ? update_of(a, g[i][k], m[i][k]) : 0.0f;
  });
  __syncthreads();
  const float s = scale_of(p.squares != nullptr ? p.squares[b] : red[0] + red[1] + red[2] + red[3], p.scale, p.eps);
  char* by_row = p.by_row + (int64_t)b * p.batch_row;
  char* by_col = p.by_col + (int64_t)b * p.batch_col;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int run = wave * 2 + q, blk = run >> 2, k = run & 3;  // row block and k / 16 within the tile
    const int row = blk * 32 + (lane & 31), col = k * 16 + 8 * (lane >> 5);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = tile[row][col + i] * s;
    store_run<PLANES>(by_row + run_at<PLANES>(tr * 2 + blk, p.k16_row, tc * 4 + k, 0), lane, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = tile[col + i][row] * s;
    store_run<PLANES>(by_col + run_at<PLANES>(tc * 2 + blk, p.k16_col, tr * 4 + k, 0), lane, v);
  }
}

// ---- the products -----------------------------------------------------------------------------

// What becomes of D = P Q^T:
//   kGram   alpha D, symmetric: its fragments (D^T's and, off the diagonal tiles, D's)
//   kPoly   alpha D + beta C with C symmetric: the same
//   kStep   alpha D + beta C: the fragments of it and of its transpose
//   kLast   o = alpha D + beta C: param = keep param - rate o
enum Epilogue { kGram, kPoly, kStep, kLast };

struct ProductArgs {
  const char *p, *q;          // operands, fragment-major
  int64_t batch_p, batch_q;   // bytes from one matrix to the next
  int p_blocks, q_blocks;     // row blocks of 32
  int k16;                    // K / 16
  int tiles_q;                // tiles along Q's rows (kStep, kLast); tiles a side (kGram, kPoly)
  const char* c;              // C^T by rows: [q block][p rows as k]
  int64_t batch_c;
  char *out_t, *out;          // D^T and D by rows (kStep: X^T, X; the symmetric ones: the same buffer)
  int64_t batch_out_t, batch_out;
  float alpha, beta;
  // kLast
  int64_t rows, cols;         // D's real size
  Strides param;
  int param_dtype, read_param;
  float keep, rate;
};

constexpr int kGroup = 8;  // row tiles that are walked together, column by column

// Workgroups are dealt to the 8 XCDs in turn; block b's tile is such that each XCD
// takes a contiguous run of tiles, whose panels its own L2 shares.
__device__ inline int xcd_order(int b, int n) {
  const int x = b % 8, k = b / 8, each = n / 8, more = n % 8;
  return x * each + min(x, more) + k;
}

// How a product's wavefronts finish: part w of the tile (its quarters, halves by rows, or all of it) is
// wavefront w's, SI x SJ blocks, and the others' sums of it come through LDS, kTurns at a time.
template <int T, int NW>
struct ProductShape {
  static constexpr int kParts = NW < 4 ? NW : 4;
  static constexpr int SI = kParts == 4 ? T / 2 : T / kParts, SJ = kParts == 4 ? T / 2 : T;
  static constexpr int kTurns = kParts * SI * SJ * 4096 * (NW - 1) > 163840 ? 2 : 1;  // SI / kTurns block rows each
  static constexpr int kSlot = SI / kTurns * SJ * 4096;                             // one wavefront's sums of one part
  static constexpr int kSums = kParts * (NW - 1) * kSlot;
  static constexpr int kBytes = kSums > kParts * 32 * 80 ? kSums : kParts * 32 * 80;
  static_assert(SI % kTurns == 0 && kSums <= 163840, "the sums fit");
};

// Grid (tiles, matrices): an output tile of T x T blocks of 32 x 32 a workgroup.  Its NW
// wavefronts each compute the whole tile over their share of K, fragments loaded
// straight into registers DEPTH k16 ahead (a fragment is 1 KB of consecutive memory):
// no LDS and no barrier until the wavefronts' sums are added at the end.  T 4 and NW 4 fill
// a SIMD's 512 registers (256 sums, 192 of fragments in flight) and read 43 bytes a cycle of MFMAs
// and CU with two planes, 64 with one.  Bound by the matrix cores: of 53 us for X X^T of 2560 x
// 2560 (two planes, 0.95 PFLOP/s of products) 41 are the loop, whose MFMAs alone take 36 at the 1.7 GHz
// the card keeps under them.  The same tiles through LDS (direct-to-LDS loads, a ring of 2 to 5 stages,
// fragments read half a step ahead) took 58 to 63 us: LDS reads and writes take as long as the
// MFMAs.  10240 x 2560: X X^T 174 us with two planes (1.2 PFLOP/s of products), 69 with one (1.0; through LDS 98).
template <int PLANES, int T, int NW, int DEPTH, Epilogue EPI>
__global__ __launch_bounds__(NW * 64, NW < 4 ? 1 : NW / 4) void muon_product_kernel(const ProductArgs a, const Matrices mats) {
  using Shape = ProductShape<T, NW>;
  constexpr int PARTS = Shape::kParts, SI = Shape::SI, SJ = Shape::SJ;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.y;
  int ti, tj;
  const int t = xcd_order(blockIdx.x, gridDim.x);
  if (EPI == kGram || EPI == kPoly) {  // tile t of the upper triangle, column by column
    tj = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while (tj * (tj + 1) / 2 > t) --tj;
    while ((tj + 1) * (tj + 2) / 2 <= t) ++tj;
    ti = t - tj * (tj + 1) / 2;
  } else {
    const int tiles_p = gridDim.x / a.tiles_q, group = t / (kGroup * a.tiles_q), first = group * kGroup;
    const int deep = min(kGroup, tiles_p - first), u = t - first * a.tiles_q;
    ti = first + u % deep;
    tj = u / deep;
  }
  const int i0 = ti * T, j0 = tj * T;  // first row blocks
  const int64_t block_bytes = (int64_t)a.k16 * PLANES * kRun;
  // blocks past the last re-read the last: their products only reach outputs that are not stored
  const char *ps[T], *qs[T];
#pragma unroll
  for (int i = 0; i < T; ++i) {
    ps[i] = a.p + b * a.batch_p + (int64_t)min(i0 + i, a.p_blocks - 1) * block_bytes;
    qs[i] = a.q + b * a.batch_q + (int64_t)min(j0 + i, a.q_blocks - 1) * block_bytes;
  }
  const int k_first = a.k16 * wave / NW, k_count = a.k16 * (wave + 1) / NW - k_first;

  f32x16 acc[T][T];
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  if (k_count > 0) {
    f16x8 pa[DEPTH][PLANES][T], qb[DEPTH][PLANES][T];
    const uint32_t lane16 = (uint32_t)lane * 16;
    auto load = [&](int f, int k) {
      const int64_t at = (int64_t)(k_first + min(k, k_count - 1)) * (PLANES * kRun);
#pragma unroll
      for (int x = 0; x < PLANES; ++x) {
#pragma unroll
        for (int i = 0; i < T; ++i) {
          pa[f][x][i] = *(const f16x8*)(ps[i] + at + lane16 + x * kRun);
          qb[f][x][i] = *(const f16x8*)(qs[i] + at + lane16 + x * kRun);
        }
      }
    };
    auto multiply = [&](int f) {
#pragma unroll
      for (int pass = PLANES == 2 ? 0 : 2; pass < 3; ++pass)  // lo hi, hi lo, hi hi
#pragma unroll
        for (int i = 0; i < T; ++i)
#pragma unroll
          for (int j = 0; j < T; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pa[f][pass == 0 ? PLANES - 1 : 0][i],
                                                               qb[f][pass == 1 ? PLANES - 1 : 0][j], acc[i][j], 0, 0, 0);
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(d, d);
    __builtin_amdgcn_sched_barrier(0);
    int k = 0;
    for (; k + DEPTH <= k_count; k += DEPTH) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        multiply(d);
        __builtin_amdgcn_sched_barrier(0);
        load(d, k + d + DEPTH);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d)
      if (k + d < k_count) multiply(d);
  }

  f32x16 sum[SI][SJ];
  auto part_i = [](int w) { return PARTS == 4 ? w / 2 * SI : w * SI; };
  auto part_j = [](int w) { return PARTS == 4 ? w % 2 * SJ : 0; };
#pragma unroll
  for (int w = 0; w < PARTS; ++w)
    if (wave == w) {
#pragma unroll
      for (int i = 0; i < SI; ++i)
#pragma unroll
        for (int j = 0; j < SJ; ++j) sum[i][j] = acc[part_i(w) + i][part_j(w) + j];
    }
  if (NW > 1) {
    constexpr int RI = SI / Shape::kTurns;
#pragma unroll
    for (int turn = 0; turn < Shape::kTurns; ++turn) {
      if (turn > 0) __syncthreads();
#pragma unroll
      for (int w = 0; w < PARTS; ++w) {
        if (wave == w) continue;
        char* at = lds + (w * (NW - 1) + (wave > w ? wave - 1 : wave)) * Shape::kSlot + lane * 16;
#pragma unroll
        for (int i = 0; i < RI; ++i)
#pragma unroll
          for (int j = 0; j < SJ; ++j) {
            const f32x16& v = acc[part_i(w) + turn * RI + i][part_j(w) + j];
#pragma unroll
            for (int g = 0; g < 4; ++g)
              *(f32x4*)(at + ((i * SJ + j) * 4 + g) * 1024) = f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
          }
      }
      __syncthreads();
      if (wave < PARTS)
#pragma unroll
        for (int i = 0; i < RI; ++i)
#pragma unroll
          for (int j = 0; j < SJ; ++j) {
            const char* at = lds + wave * (NW - 1) * Shape::kSlot + (i * SJ + j) * 4096 + lane * 16;
#pragma unroll
            for (int other = 0; other < NW - 1; ++other)
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const f32x4 v = *(const f32x4*)(at + other * Shape::kSlot + g * 1024);
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[turn * RI + i][j][4 * g + r] += v[r];
              }
          }
    }
  }
  if (NW > 1) __syncthreads();  // the transpose buffers are where sums were
  if (wave >= PARTS) return;
  const int bi0 = i0 + part_i(wave), bj0 = j0 + part_j(wave);

  // lane l of a 32 x 32 block holds column l % 32, rows 8 g + 4 (l / 32) + r
  constexpr int PITCH = 80;  // bytes of a row of 32 fp16 in the transpose buffer, 16-byte aligned
  char* turn = lds + wave * (32 * PITCH);
  const int col = lane & 31, half = lane >> 5;
  const int64_t p16 = (int64_t)a.p_blocks * 2, q16 = (int64_t)a.q_blocks * 2;  // k / 16 along D^T's and D's rows
  // all of C (and of the weights) is read before anything is stored: a load does not wait
  // for the stores before it
#pragma unroll
  for (int i = 0; i < SI; ++i)
#pragma unroll
    for (int j = 0; j < SJ; ++j) {
      const int bi = min(bi0 + i, a.p_blocks - 1), bj = min(bj0 + j, a.q_blocks - 1);
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[i][j][r] *= a.alpha;
      if (EPI == kGram) continue;
      const char* c = a.c + b * a.batch_c;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int64_t at = run_at<PLANES>(bj, p16, bi * 2 + (g >> 1), 0) + (col + 32 * (g & 1)) * 16 + 8 * half;
        const f16x4 hi = *(const f16x4*)(c + at);
        f16x4 lo = {0, 0, 0, 0};
        if (PLANES == 2) lo = *(const f16x4*)(c + at + kRun);
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[i][j][4 * g + r] += a.beta * ((float)hi[r] + (float)lo[r]);
      }
    }
  if (EPI == kLast) {
    by_type(a.param_dtype, [&](auto zero) {
      using W = decltype(zero);
      W* w = (W*)mats.param[b];
      auto place = [&](int i, int j, int r, int64_t& x, int64_t& y) {
        x = (int64_t)(bi0 + i) * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
        y = (int64_t)(bj0 + j) * 32 + col;
      };
      const float scale = a.read_param ? 1.0f : -a.rate;
      if (a.read_param) {
        W old[SI][SJ][16];
#pragma unroll
        for (int i = 0; i < SI; ++i)
#pragma unroll
          for (int j = 0; j < SJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              int64_t x, y;
              place(i, j, r, x, y);
              old[i][j][r] = w[min(x, a.rows - 1) * a.param.row + min(y, a.cols - 1) * a.param.col];
            }
#pragma unroll
        for (int i = 0; i < SI; ++i)
#pragma unroll
          for (int j = 0; j < SJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[i][j][r] = a.keep * (float)old[i][j][r] - a.rate * sum[i][j][r];
      }
#pragma unroll
      for (int i = 0; i < SI; ++i)
#pragma unroll
        for (int j = 0; j < SJ; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            int64_t x, y;
            place(i, j, r, x, y);
            if (x < a.rows && y < a.cols) w[x * a.param.row + y * a.param.col] = (W)(scale * sum[i][j][r]);
          }
    });
    return;
  }
#pragma unroll
  for (int i = 0; i < SI; ++i)
#pragma unroll
    for (int j = 0; j < SJ; ++j) {
      const int bi = bi0 + i, bj = bj0 + j;
      if (bi >= a.p_blocks || bj >= a.q_blocks) continue;
      _Float16 hi[16], lo[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) split(sum[i][j][r], hi[r], lo[r]);
      char* out_t = a.out_t + b * a.batch_out_t;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        char* at = out_t + run_at<PLANES>(bj, p16, bi * 2 + (g >> 1), 0) + (col + 32 * (g & 1)) * 16 + 8 * half;
        *(f16x4*)at = f16x4{hi[4 * g], hi[4 * g + 1], hi[4 * g + 2], hi[4 * g + 3]};
        if (PLANES == 2) *(f16x4*)(at + kRun) = f16x4{lo[4 * g], lo[4 * g + 1], lo[4 * g + 2], lo[4 * g + 3]};
      }
      if (EPI != kStep && ti == tj) continue;  // a diagonal tile's blocks cover its transpose
      char* out = a.out + b * a.batch_out;
#pragma unroll
      for (int x = 0; x < PLANES; ++x) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          *(_Float16*)(turn + (8 * (r >> 2) + 4 * half + (r & 3)) * PITCH + col * 2) = x == 0 ? hi[r] : lo[r];
        __builtin_amdgcn_wave_barrier();  // a wavefront's LDS operations are in order
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const f16x8 run = *(const f16x8*)(turn + col * PITCH + s * 32 + half * 16);
          *(f16x8*)(out + run_at<PLANES>(bi, q16, bj * 2 + s, x) + lane * 16) = run;
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
}

// ---- a matrix in one workgroup's LDS ------------------------------------------------------------

constexpr int kSmallWaves = 16;
constexpr int kSmallSteps = 32;
constexpr int kSmallBytes = 160 * 1024;

// run_at within LDS.
template <int PLANES>
__device__ inline int lds_run(int row_block, int k16s, int k16, int plane) {
  return ((row_block * k16s + k16) * PLANES + plane) * kRun;
}

// A matrix of which every element's offset fits 31 bits (the host sees to it).
struct Strides32 {
  int row, col;
};

// A step's factors: A = gram D; B = poly D + poly_c A; X = step D + step_c X.
struct Factors {
  float gram, poly, poly_c, step, step_c;
};

struct SmallArgs {
  int rows, cols;
  Strides32 grad, momentum, param;
  int grad_dtype, has_momentum, nesterov, param_dtype, read_param;
  float mu, eps, scale;
  int pr, pc;                  // rows and columns padded to 64
  int steps;
  float keep, rate;
  Factors f[kSmallSteps];
};

// Sum over k of a block's product, its operands in LDS: 32 rows of P (row block bp) by 32 of Q.
// TURNED adds the cross products in the other order: the transposed block's very sums.
template <int PLANES, bool TURNED>
__device__ inline f32x16 block_product(const char* p, int bp, const char* q, int bq, int k16s, int lane) {
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
  const char* pa = p + lds_run<PLANES>(bp, k16s, 0, 0) + lane * 16;
  const char* qa = q + lds_run<PLANES>(bq, k16s, 0, 0) + lane * 16;
  for (int k0 = 0; k0 < k16s; k0 += 4)  // K is padded to 64
#pragma unroll
    for (int k = k0; k < k0 + 4; ++k) {
      const f16x8 ph = *(const f16x8*)(pa + k * PLANES * kRun), qh = *(const f16x8*)(qa + k * PLANES * kRun);
      if (PLANES == 2) {
        const f16x8 pl = *(const f16x8*)(pa + (k * 2 + 1) * kRun), ql = *(const f16x8*)(qa + (k * 2 + 1) * kRun);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(TURNED ? ph : pl, TURNED ? ql : qh, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(TURNED ? pl : ph, TURNED ? qh : ql, acc, 0, 0, 0);
      }
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, qh, acc, 0, 0, 0);
    }
  return acc;
}

// A block's planes as its transpose's fragments hold them: 4 x 4 values a lane.
template <int PLANES>
struct BlockPlanes {
  f16x4 v[PLANES][4];
};

// alpha acc + beta C, C's transpose by rows at c (row block bq, k block bp).
template <int PLANES>
__device__ inline void add_c(f32x16& acc, float alpha, float beta, const char* c, int bp, int bq, int k16s, int lane) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const char* at = c + lds_run<PLANES>(bq, k16s, bp * 2 + (g >> 1), 0) + ((lane & 31) + 32 * (g & 1)) * 16 + 8 * (lane >> 5);
    const f16x4 hi = *(const f16x4*)at;
    f16x4 lo = {0, 0, 0, 0};
    if (PLANES == 2) lo = *(const f16x4*)(at + kRun);
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[4 * g + r] = alpha * acc[4 * g + r] + beta * ((float)hi[r] + (float)lo[r]);
  }
}

template <int PLANES>
__device__ inline BlockPlanes<PLANES> planes_of(const f32x16& v) {
  BlockPlanes<PLANES> o;
#pragma unroll
  for (int g = 0; g < 4; ++g)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      _Float16 hi, lo;
      split(v[4 * g + r], hi, lo);
      o.v[0][g][r] = hi;
      if (PLANES == 2) o.v[PLANES - 1][g][r] = lo;
    }
  return o;
}

// Into the transpose's rows at `to` (row block bq, k block bp).
template <int PLANES>
__device__ inline void store_planes(char* to, const BlockPlanes<PLANES>& o, int bp, int bq, int k16s, int lane) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    char* at = to + lds_run<PLANES>(bq, k16s, bp * 2 + (g >> 1), 0) + ((lane & 31) + 32 * (g & 1)) * 16 + 8 * (lane >> 5);
#pragma unroll
    for (int x = 0; x < PLANES; ++x) *(f16x4*)(at + x * kRun) = o.v[x][g];
  }
}

// Grid (matrices): the whole step of one matrix, in one launch where the products take 17: 16 bf16 matrices
// of 64 x 256 42.3 us with two planes, 28.9 with one (160 in 17 launches; 9 us of launch, loads and stores and
// 3.4 us a step, most of it the vector work on blocks between the products).  X, X^T, A and B stay in LDS as fragments; every
// block of a product is one wavefront's, X's and X^T's blocks both computed (B X and X^T B) rather
// than turned.  The two have to be the same values to the last bit, hence TURNED: a
// difference between X and X^T is not damped as X's own errors are, it grows by a step's a.
template <int PLANES>
__global__ __launch_bounds__(kSmallWaves * 64) void muon_small_kernel(const SmallArgs a, const Matrices mats) {
  constexpr int MAX_ELEMENTS = kSmallBytes / (4 * PLANES);       // of X, both orders
  constexpr int UNITS = (MAX_ELEMENTS / 512 + kSmallWaves - 1) / kSmallWaves;  // 8 x 64 elements
  constexpr int BLOCKS = (2 * MAX_ELEMENTS / 1024 + kSmallWaves - 1) / kSmallWaves;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, b = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool tall = a.rows > a.cols;
  const int m = tall ? a.pc : a.pr, n = tall ? a.pr : a.pc, m16 = m / 16, n16 = n / 16, mb = m / 32, nb = n / 32;
  char* x = lds;                                // X by rows: m x n
  char* xt = x + m * n * 2 * PLANES;            // X^T by rows
  char* gram = xt + m * n * 2 * PLANES;
  char* poly = gram + m * m * 2 * PLANES;
  double* red = (double*)gram;

  // momentum; a thread has 8 rows of a column in each of its units
  const int chunks = a.pc / 64, units = a.pr / 8 * chunks;
  float u[UNITS][8];
  double sum = 0.0;
  by_type(a.grad_dtype, [&](auto zero) {
    using G = decltype(zero);
    const G* grad = (const G*)mats.grad[b];
    float* mom = mats.momentum[b];
    G g[UNITS][8];
    float old[UNITS][8];
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int unit = min(wave + i * kSmallWaves, units - 1);
      const int r0 = unit / chunks * 8, c = min(unit % chunks * 64 + lane, a.cols - 1);
      const int gc = c * a.grad.col, mc = c * a.momentum.col;
#pragma unroll
      for (int r = 0; r < 8; ++r) g[i][r] = (grad + min(r0 + r, a.rows - 1) * a.grad.row)[gc];
      if (a.has_momentum) {
#pragma unroll
        for (int r = 0; r < 8; ++r) old[i][r] = (mom + min(r0 + r, a.rows - 1) * a.momentum.row)[mc];
      }
    }
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int unit = wave + i * kSmallWaves;
      if (unit >= units) break;
      const int r0 = unit / chunks * 8, c = unit % chunks * 64 + lane, mc = c * a.momentum.col;
#pragma unroll
      for (int r = 0; r < 8; ++r) u[i][r] = (float)g[i][r];
      if (a.has_momentum) {
        float now[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          now[r] = a.mu * old[i][r] + u[i][r];
          u[i][r] = a.nesterov ? u[i][r] + a.mu * now[r] : now[r];
        }
        if (c < a.cols) {
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (r0 + r < a.rows) (mom + (r0 + r) * a.momentum.row)[mc] = now[r];
        }
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        u[i][r] = r0 + r < a.rows && c < a.cols ? u[i][r] : 0.0f;
        sum += (double)u[i][r] * (double)u[i][r];
      }
    }
  });
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane == 0) red[wave] = sum;
  __syncthreads();
  double total = 0.0;
#pragma unroll
  for (int w = 0; w < kSmallWaves; ++w) total += red[w];
  const float s = scale_of(total, a.scale, a.eps);
  char* by_row = tall ? xt : x;
  char* by_col = tall ? x : xt;
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const int unit = wave + i * kSmallWaves;
    if (unit >= units) break;
    const int r0 = unit / chunks * 8, c = unit % chunks * 64 + lane;
    f16x8 hi, lo;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      _Float16 h, l;
      split(u[i][r] * s, h, l);
      hi[r] = h;
      lo[r] = l;
      char* at = by_row + lds_run<PLANES>((r0 + r) / 32, a.pc / 16, c / 16, 0) + ((r0 + r) % 32 + 32 * (c % 16 / 8)) * 16 + c % 8 * 2;
      *(_Float16*)at = h;
      if (PLANES == 2) *(_Float16*)(at + kRun) = l;
    }
    char* at = by_col + lds_run<PLANES>(c / 32, a.pr / 16, r0 / 16, 0) + (c % 32 + 32 * (r0 % 16 / 8)) * 16;
    *(f16x8*)at = hi;
    if (PLANES == 2) *(f16x8*)(at + kRun) = lo;
  }
  __syncthreads();

  for (int step = 0; step < a.steps; ++step) {
    const Factors f = a.f[step];
    for (int k = wave; k < mb * mb; k += kSmallWaves) {  // A = X X^T
      f32x16 acc = block_product<PLANES, false>(x, k / mb, x, k % mb, n16, lane);
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[r] *= f.gram;
      store_planes<PLANES>(gram, planes_of<PLANES>(acc), k / mb, k % mb, m16, lane);
    }
    __syncthreads();
    for (int k = wave; k < mb * mb; k += kSmallWaves) {  // B = b A + c A A
      f32x16 acc = block_product<PLANES, false>(gram, k / mb, gram, k % mb, m16, lane);
      add_c<PLANES>(acc, f.poly, f.poly_c, gram, k / mb, k % mb, m16, lane);
      store_planes<PLANES>(poly, planes_of<PLANES>(acc), k / mb, k % mb, m16, lane);
    }
    __syncthreads();
    if (step + 1 == a.steps) break;
    // X = a X + B X, and its transpose: blocks [0, mb nb) are X's, whose transpose goes to xt
    BlockPlanes<PLANES> out[BLOCKS];
    const int all = 2 * mb * nb;
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) {
      const int k = wave + i * kSmallWaves;
      if (k >= all) break;
      const bool turned = k >= mb * nb;
      const int e = turned ? k - mb * nb : k, bm = e / nb, bn = e % nb;
      f32x16 acc = turned ? block_product<PLANES, true>(xt, bn, poly, bm, m16, lane)
                          : block_product<PLANES, false>(poly, bm, xt, bn, m16, lane);
      if (turned)
        add_c<PLANES>(acc, f.step, f.step_c, x, bn, bm, n16, lane);
      else
        add_c<PLANES>(acc, f.step, f.step_c, xt, bm, bn, m16, lane);
      out[i] = planes_of<PLANES>(acc);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) {
      const int k = wave + i * kSmallWaves;
      if (k >= all) break;
      const bool turned = k >= mb * nb;
      const int e = turned ? k - mb * nb : k, bm = e / nb, bn = e % nb;
      if (turned)
        store_planes<PLANES>(x, out[i], bn, bm, n16, lane);
      else
        store_planes<PLANES>(xt, out[i], bm, bn, m16, lane);
    }
    __syncthreads();
  }

  // the last step's X goes to the weights, in the order whose lanes run along their rows
  const Factors f = a.f[a.steps - 1];
  for (int k = wave; k < mb * nb; k += kSmallWaves) {
    const int bm = k / nb, bn = k % nb;
    f32x16 acc = tall ? block_product<PLANES, true>(xt, bn, poly, bm, m16, lane) : block_product<PLANES, false>(poly, bm, xt, bn, m16, lane);
    if (tall)
      add_c<PLANES>(acc, f.step, f.step_c, x, bn, bm, n16, lane);
    else
      add_c<PLANES>(acc, f.step, f.step_c, xt, bm, bn, m16, lane);
    const int r0 = (tall ? bn : bm) * 32 + 4 * (lane >> 5), c = (tall ? bm : bn) * 32 + (lane & 31);
    by_type(a.param_dtype, [&](auto zero) {
      using W = decltype(zero);
      W* w = (W*)mats.param[b];
      const int cs = min(c, a.cols - 1) * a.param.col;
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[r] *= -a.rate;
      if (a.read_param) {
        W old[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) old[r] = w[min(r0 + 8 * (r >> 2) + (r & 3), a.rows - 1) * a.param.row + cs];
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] += a.keep * (float)old[r];
      }
      if (c < a.cols) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = r0 + 8 * (r >> 2) + (r & 3);
          if (row < a.rows) w[row * a.param.row + cs] = (W)acc[r];
        }
      }
    });
  }
}

// ---- host side --------------------------------------------------------------------------------

int64_t pad64(int64_t x) { return (x + 63) / 64 * 64; }

// The buffers of one matrix, m x n padded: X, two X^T, A, B.
struct Layout {
  int64_t m, n;          // padded, m <= n
  int64_t x, a;          // bytes of X (or X^T), of A (or B)
  int64_t tiles;         // 64 x 64 tiles of the padded matrix
  int64_t partials;      // bytes of all matrices' partial sums, and of their sums
  int64_t total;
};

Layout make_layout(int64_t rows, int64_t cols, int64_t count, int planes) {
  Layout l;
  l.m = pad64(std::min(rows, cols));
  l.n = pad64(std::max(rows, cols));
  l.x = l.m * l.n * 2 * planes;
  l.a = l.m * l.m * 2 * planes;
  l.tiles = (l.m / 64) * (l.n / 64);
  l.partials = (count * (l.tiles + 1) * 8 + 255) / 256 * 256;
  l.total = l.partials + count * (3 * l.x + 2 * l.a);
  return l;
}

// Workspace that a launch's matrices may take together; one alone takes what it needs.  Nothing is lost by it: 40 fp32
// matrices of 2560 x 2560 998 us each, 16 a launch (2.1 GB), 996 all in one (5.2 GB); 16 of 4096 x 4096 3,667 and 3,700.
constexpr int64_t kMaxWorkspace = int64_t{2} << 30;

// Matrices a launch.
int launch_count(int64_t rows, int64_t cols, int64_t count, int planes) {
  count = std::min<int64_t>(count, kMaxBatch);
  while (count > 1 && make_layout(rows, cols, count, planes).total > kMaxWorkspace) --count;
  return (int)count;
}

template <int PLANES, int T, int NW, int DEPTH, Epilogue EPI>
int launch_product_as(const ProductArgs& args, const Matrices& mats, int count, hipStream_t stream) {
  ProductArgs a = args;
  constexpr int bytes = ProductShape<T, NW>::kBytes;
  const int tp = (a.p_blocks + T - 1) / T, tq = (a.q_blocks + T - 1) / T;
  a.tiles_q = tq;
  const int tiles = EPI == kGram || EPI == kPoly ? tq * (tq + 1) / 2 : tp * tq;
  auto kernel = muon_product_kernel<PLANES, T, NW, DEPTH, EPI>;
  if (bytes > 65536) EG_CHECK_HIP(allow_lds((const void*)kernel, bytes));
  kernel<<<dim3((unsigned)tiles, (unsigned)count), NW * 64, bytes, stream>>>(a, mats);
  return launch_status("muon_product_kernel");
}

// The tile by the number of 128 x 128 ones, whose rounds over the 256 CUs (one a CU) cost what
// they cost however full they are:
//   few (kFewTiles): 64 x 64, four times the workgroups: a 1024 x 1024 fp32 step 174 us against 354, 1536 x
//     1536 420 against 468; 2048 x 2048 775 against 642;
//   one plane and four rounds' worth: a wavefront a tile with nothing to add up, since the sums of four
//     cost as much as a tile's products at K 2,560: 137 us a product of 1,600 tiles against 164
//     (two planes, 2,000 tiles: 470 against 442).
constexpr int kFewTiles = 128, kManyTiles = 1024;

template <int PLANES, Epilogue EPI>
int launch_product(const ProductArgs& a, const Matrices& mats, int count, hipStream_t stream) {
  const int64_t tp = (a.p_blocks + 3) / 4, tq = (a.q_blocks + 3) / 4;
  const int64_t tiles = count * (EPI == kGram || EPI == kPoly ? tq * (tq + 1) / 2 : tp * tq);
  if (tiles <= kFewTiles) return launch_product_as<PLANES, 2, 4, PLANES == 2 ? 4 : 6, EPI>(a, mats, count, stream);
  if (PLANES == 1 && EPI == kStep && tiles >= kManyTiles)
    return launch_product_as<PLANES, 4, 1, 6, EPI>(a, mats, count, stream);
  return launch_product_as<PLANES, 4, 4, PLANES == 2 ? 3 : 6, EPI>(a, mats, count, stream);
}

// Powers of two by which X, A and B of an iteration are kept, from the bound of X's
// singular values; false where the coefficients leave no finite ones.
struct Bounds {
  double sigma;         // X's singular values are at most this
  int x, gram, poly;    // exponents
};

int exponent_for(double bound) { return (int)floor(log2(60000.0 / std::max(bound, 1e-30))); }

constexpr double kMargin = 1.01;  // over what the bounds ignore: fp32 and fp16 roundings

Bounds bounds_of(double sigma, const float* k) {
  const double b = k[1], c = k[2], s2 = sigma * sigma;
  // |b y + c y^2| over [0, s2]: at the end, or where the slope b + 2 c y is zero
  double top = fabs(b * s2 + c * s2 * s2);
  const double y = c != 0.0 ? -b / (2.0 * c) : 0.0;
  if (y > 0.0 && y < s2) top = std::max(top, fabs(b * y + c * y * y));
  return {sigma, exponent_for(sigma), exponent_for(s2), exponent_for(kMargin * top)};
}

// The largest |a s + b s^3 + c s^5| over [0, sigma]: at the end, or where the slope, a quadratic
// a + 3 b y + 5 c y^2 of y = s^2, is zero.
double next_sigma(double sigma, const float* k) {
  const double a = k[0], b = k[1], c = k[2], s2 = sigma * sigma;
  double top = 0.0;
  auto at = [&](double y) {
    if (y > 0.0 && y <= s2) top = std::max(top, fabs(sqrt(y) * (a + y * (b + y * c))));
  };
  at(s2);
  if (c != 0.0) {
    const double d = 9.0 * b * b - 20.0 * a * c;
    if (d >= 0.0) {
      at((-3.0 * b + sqrt(d)) / (10.0 * c));
      at((-3.0 * b - sqrt(d)) / (10.0 * c));
    }
  } else if (b != 0.0) {
    at(-a / (3.0 * b));
  }
  return kMargin * top;
}

// Whether every element lies within 2^29 elements of the first.
bool near(const eg_muon* o, const int64_t* stride) {
  auto span = [](int64_t n, int64_t s) { return n == 1 ? 0.0 : (double)(n - 1) * fabs((double)s); };
  return span(o->rows, stride[0]) + span(o->cols, stride[1]) < (double)(1 << 29);
}

// Matrices of more 64 x 64 tiles have a launch for their norm: read by every workgroup, the partial sums are
// 8 bytes times the square of the tiles.  A step of one iteration, with the launch and without it: 4096 x 4096
// (4,096 tiles) 433 and 429 us, 10240 x 2560 395 and 404, 16384 x 4096 1,411 and 1,522, 16384 x 16384 20,960 and 22,780.
constexpr int64_t kOwnSumTiles = 4096;

// Bytes of LDS that X, X^T, A and B take.
int64_t small_bytes(const Layout& l) { return 2 * (l.x + l.a); }

template <int PLANES>
int run_small(const eg_muon* o, const Matrices& mats, int count, const Layout& l, hipStream_t stream) {
  SmallArgs a;
  a.rows = (int)o->rows;
  a.cols = (int)o->cols;
  a.grad = {(int)o->grad_stride[0], (int)o->grad_stride[1]};
  a.momentum = {(int)o->momentum_stride[0], (int)o->momentum_stride[1]};
  a.param = {(int)o->param_stride[0], (int)o->param_stride[1]};
  a.grad_dtype = o->grad_dtype;
  a.has_momentum = o->momenta != nullptr;
  a.nesterov = o->nesterov;
  a.param_dtype = o->param_dtype;
  a.read_param = o->keep != 0.0f;
  a.mu = o->momentum;
  a.eps = o->eps;
  a.pr = (int)pad64(o->rows);
  a.pc = (int)pad64(o->cols);
  a.steps = o->steps;
  a.keep = o->keep;
  a.rate = o->rate;
  Bounds bd = bounds_of(1.0, o->coefficients);
  a.scale = ldexpf(1.0f, bd.x);
  for (int s = 0; s < o->steps; ++s) {
    const float* k = o->coefficients + 3 * s;
    const bool last = s + 1 == o->steps;
    const Bounds nx = last ? bd : bounds_of(next_sigma(bd.sigma, k), k + 3);
    const int x = last ? 0 : nx.x;  // the last X is itself
    a.f[s] = {ldexpf(1.0f, bd.gram - 2 * bd.x), ldexpf(k[2], bd.poly - 2 * bd.gram), ldexpf(k[1], bd.poly - bd.gram),
              ldexpf(1.0f, x - bd.poly - bd.x), ldexpf(k[0], x - bd.x)};
    bd = nx;
  }
  const int bytes = (int)small_bytes(l);
  auto kernel = muon_small_kernel<PLANES>;
  EG_CHECK_HIP(allow_lds((const void*)kernel, kSmallBytes));
  kernel<<<dim3((unsigned)count), kSmallWaves * 64, bytes, stream>>>(a, mats);
  return launch_status("muon_small_kernel");
}

template <int PLANES>
int run_muon(const eg_muon* o, int first, int count, const Layout& l, char* ws, hipStream_t stream) {
  Matrices mats = {};
  for (int i = 0; i < count; ++i) {
    mats.param[i] = o->params[first + i];
    mats.grad[i] = o->grads[first + i];
    mats.momentum[i] = o->momenta != nullptr ? o->momenta[first + i] : nullptr;
  }
  const UpdateArgs update = {o->rows, o->cols, {o->grad_stride[0], o->grad_stride[1]},
                             {o->momentum_stride[0], o->momentum_stride[1]}, o->grad_dtype, o->momenta != nullptr,
                             o->nesterov, o->momentum, (int)(pad64(o->cols) / 64), (int)l.tiles, (double*)ws};
  if (small_bytes(l) <= kSmallBytes && o->steps <= kSmallSteps && near(o, o->param_stride) && near(o, o->grad_stride) &&
      near(o, o->momentum_stride))
    return run_small<PLANES>(o, mats, count, l, stream);
  const bool tall = o->rows > o->cols;
  char* base = ws + l.partials;
  char* x = base;
  char* xt[2] = {x + count * l.x, x + 2 * count * l.x};
  char* gram = x + 3 * count * l.x;
  char* poly = gram + count * l.a;
  const int m32 = (int)(l.m / 32), n32 = (int)(l.n / 32);
  const int m16 = (int)(l.m / 16), n16 = (int)(l.n / 16);
  Bounds bd = bounds_of(1.0, o->coefficients);

  PlanesArgs pa;
  pa.u = update;
  pa.eps = o->eps;
  pa.scale = ldexpf(1.0f, bd.x);
  pa.by_row = tall ? xt[0] : x;
  pa.by_col = tall ? x : xt[0];
  pa.batch_row = pa.batch_col = l.x;
  pa.k16_row = pad64(o->cols) / 16;
  pa.k16_col = pad64(o->rows) / 16;
  muon_momentum_kernel<<<dim3((unsigned)l.tiles, (unsigned)count), 256, 0, stream>>>(pa.u, mats);
  if (int rc = launch_status("muon_momentum_kernel"); rc != EG_OK) return rc;
  pa.squares = nullptr;
  if (l.tiles > kOwnSumTiles) {
    double* squares = (double*)ws + count * l.tiles;
    muon_norm_kernel<<<dim3((unsigned)count), 1024, 0, stream>>>((const double*)ws, (int)l.tiles, squares);
    if (int rc = launch_status("muon_norm_kernel"); rc != EG_OK) return rc;
    pa.squares = squares;
  }
  muon_planes_kernel<PLANES><<<dim3((unsigned)l.tiles, (unsigned)count), 256, 0, stream>>>(pa, mats);
  if (int rc = launch_status("muon_planes_kernel"); rc != EG_OK) return rc;

  for (int s = 0; s < o->steps; ++s) {
    const float* k = o->coefficients + 3 * s;
    const bool last = s + 1 == o->steps;
    char* xt_now = xt[s & 1];
    ProductArgs a = {};
    // A = X X^T
    a.p = a.q = x;
    a.batch_p = a.batch_q = l.x;
    a.p_blocks = a.q_blocks = m32;
    a.k16 = n16;
    a.out_t = a.out = gram;
    a.batch_out_t = a.batch_out = l.a;
    a.alpha = ldexpf(1.0f, bd.gram - 2 * bd.x);
    if (int rc = launch_product<PLANES, kGram>(a, mats, count, stream); rc != EG_OK) return rc;
    // B = b A + c A A
    a.p = a.q = a.c = gram;
    a.batch_p = a.batch_q = a.batch_c = l.a;
    a.k16 = m16;
    a.out_t = a.out = poly;
    a.alpha = ldexpf(k[2], bd.poly - 2 * bd.gram);
    a.beta = ldexpf(k[1], bd.poly - bd.gram);
    if (int rc = launch_product<PLANES, kPoly>(a, mats, count, stream); rc != EG_OK) return rc;
    // X = a X + B X
    if (!last) {
      const double sigma = next_sigma(bd.sigma, k);
      const Bounds nx = bounds_of(sigma, k + 3);
      a.p = poly;
      a.q = xt_now;
      a.batch_q = l.x;
      a.q_blocks = n32;
      a.c = xt_now;
      a.batch_c = l.x;
      a.out_t = xt[1 - (s & 1)];
      a.out = x;
      a.batch_out_t = a.batch_out = l.x;
      a.alpha = ldexpf(1.0f, nx.x - bd.poly - bd.x);
      a.beta = ldexpf(k[0], nx.x - bd.x);
      if (int rc = launch_product<PLANES, kStep>(a, mats, count, stream); rc != EG_OK) return rc;
      bd = nx;
    } else {
      // D is X, or X^T for a tall matrix: a lane's column runs along the matrix's rows
      a.p = tall ? xt_now : poly;
      a.q = tall ? poly : xt_now;
      a.batch_p = tall ? l.x : l.a;
      a.batch_q = tall ? l.a : l.x;
      a.p_blocks = tall ? n32 : m32;
      a.q_blocks = tall ? m32 : n32;
      a.c = tall ? x : xt_now;
      a.batch_c = l.x;
      a.alpha = ldexpf(1.0f, -bd.poly - bd.x);
      a.beta = ldexpf(k[0], -bd.x);
      a.rows = o->rows;
      a.cols = o->cols;
      a.param = {o->param_stride[0], o->param_stride[1]};
      a.param_dtype = o->param_dtype;
      a.read_param = o->keep != 0.0f;
      a.keep = o->keep;
      a.rate = o->rate;
      if (int rc = launch_product<PLANES, kLast>(a, mats, count, stream); rc != EG_OK) return rc;
    }
  }
  return EG_OK;
}

int check_muon(const eg_muon* o) {
  EG_CHECK_ARG(o != nullptr, "muon is NULL");
  EG_CHECK_ARG(o->rows >= 1 && o->cols >= 1 && o->rows <= (1 << 20) && o->cols <= (1 << 20),
               "a matrix of %lld x %lld: 1 to 2^20 rows and columns", (long long)o->rows, (long long)o->cols);
  EG_CHECK_ARG(o->count >= 0, "count=%d must not be negative", o->count);
  EG_CHECK_ARG(o->count == 0 || (o->params != nullptr && o->grads != nullptr), "params or grads is NULL");
  EG_CHECK_ARG(o->planes == 1 || o->planes == 2, "planes=%d must be 1 or 2", o->planes);
  for (const int d : {o->param_dtype, o->grad_dtype})
    EG_CHECK_ARG(d == EG_DTYPE_F32 || d == EG_DTYPE_BF16 || d == EG_DTYPE_F16, "dtype=%d must be f32, bf16 or f16", d);
  EG_CHECK_ARG(o->steps >= 1 && o->steps <= 100 && o->coefficients != nullptr, "steps=%d must be in [1, 100]", o->steps);
  EG_CHECK_ARG(o->eps > 0.0f && o->eps <= 1.0f, "eps=%g must be in (0, 1]", (double)o->eps);
  EG_CHECK_ARG(isfinite(o->keep) && isfinite(o->rate) && isfinite(o->momentum), "a factor is not finite");
  double sigma = 1.0;
  for (int s = 0; s < o->steps; ++s) {
    const float* k = o->coefficients + 3 * s;
    EG_CHECK_ARG(isfinite(k[0]) && isfinite(k[1]) && isfinite(k[2]) && sigma < 16.0 && sigma > 1.0 / 16.0,
                 "coefficients of step %d: singular values of up to %g (1/16 to 16 are kept)", s, sigma);
    sigma = next_sigma(sigma, k);
  }
  for (int i = 0; i < o->count; ++i)
    EG_CHECK_ARG(o->params[i] != nullptr && o->grads[i] != nullptr && (o->momenta == nullptr || o->momenta[i] != nullptr),
                 "matrix %d: a pointer is NULL", i);
  return EG_OK;
}

// What a launch writes lies apart from itself and from what its other workgroups read or write.
int check_apart(const eg_muon* o) {
  std::vector<Operand> all;
  all.reserve(3 * (size_t)o->count);
  const int64_t param = o->param_dtype == EG_DTYPE_F32 ? 4 : 2, grad = o->grad_dtype == EG_DTYPE_F32 ? 4 : 2;
  for (int i = 0; i < o->count; ++i) {
    all.push_back({Operand::kParam, (size_t)i, {o->params[i], o->rows, o->cols, o->param_stride[0], o->param_stride[1], param}});
    all.push_back({Operand::kGrad, (size_t)i, {o->grads[i], o->rows, o->cols, o->grad_stride[0], o->grad_stride[1], grad}});
    if (o->momenta != nullptr)
      all.push_back({Operand::kMomentum, (size_t)i,
                     {o->momenta[i], o->rows, o->cols, o->momentum_stride[0], o->momentum_stride[1], 4}});
  }
  const Operand *x, *y;
  if (!find_overlap(all, x, y)) return EG_OK;
  EG_CHECK_ARG(x != y, "%s of matrix %zu overlap themselves", name_of(x->kind), x->matrix);
  EG_CHECK_ARG(false, "%s of matrix %zu overlap %s of matrix %zu", name_of(x->kind), x->matrix, name_of(y->kind), y->matrix);
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" {

int64_t eg_muon_workspace_size(int64_t rows, int64_t cols, int32_t count, int32_t planes) {
  if (rows < 1 || cols < 1 || count < 0 || rows > (1 << 20) || cols > (1 << 20) || planes < 1 || planes > 2) return -1;
  return make_layout(rows, cols, launch_count(rows, cols, count, planes), planes).total;
}

int eg_muon_check(const eg_muon* muon) {
  if (int rc = check_muon(muon); rc != EG_OK) return rc;
  return check_apart(muon);
}

int eg_muon_step(const eg_muon* muon, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_muon(muon); rc != EG_OK) return rc;
  if (muon->count == 0) return EG_OK;
  const int64_t need = eg_muon_workspace_size(muon->rows, muon->cols, muon->count, muon->planes);
  if (workspace == nullptr || workspace_bytes < need)
    return set_error(EG_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                     (long long)need);
  EG_CHECK_ARG((uintptr_t)workspace % 256 == 0, "workspace must be 256-byte aligned");
  if (int rc = check_apart(muon); rc != EG_OK) return rc;
  const int most = launch_count(muon->rows, muon->cols, muon->count, muon->planes);
  for (int first = 0; first < muon->count; first += most) {
    const int count = std::min(muon->count - first, most);
    const Layout l = make_layout(muon->rows, muon->cols, count, muon->planes);
    const int rc = muon->planes == 2 ? run_muon<2>(muon, first, count, l, (char*)workspace, (hipStream_t)stream)
                                     : run_muon<1>(muon, first, count, l, (char*)workspace, (hipStream_t)stream);
    if (rc != EG_OK) return rc;
  }
  return EG_OK;
}

}  // extern "C"
