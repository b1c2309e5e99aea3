// Products of matrices in blocks of 8-bit floating point, the blocks themselves, and their values.
//
//   C[m, n] = sum_b 2^(ea[m, b] + eb[n / 128, b]) sum_{k in block b} qa[m, k] qb[n, k]
//
// Scales are powers of two because CDNA4's scaled MFMA takes them with its operands: a block costs no
// arithmetic outside the matrix cores, and a block's values are exact in bf16 (e4m3 has 4 significant
// bits).  What the fp8 matrix cores do not give is fp32 sums: they align eight products to the
// largest of the eight and drop what lies 2^-13 below it, before the fp32 addition (seen with
// 2^16 and 2^3, 2^2 among eight): at most 2^-10 of the products' magnitudes, 1.5e-5 of an output of normal
// values of any length, without a bias, and 4e-5 to 5e-5 where some columns are 20 times the others.  That
// is below the rounding of a bf16 (2^-8) or fp16 (2^-11; 2.1e-4 on the whole, 2.13e-4 with it) output; an fp32 output takes
// the bf16 matrix cores instead, at half the rate, on the same bytes: its products are exact and its sums fp32.
//
// The scaled MFMA's intrinsic is not convergent: where its result is used in a branch alone, the
// compiler may move it (with its operands' moves) into the branch, where the lanes that are off keep
// what their registers held.  Here its results are used again by the next step of a loop, which holds them outside.
#include "eg_fp8.h"

#include <algorithm>

#include "eg_lds.h"

namespace eg {
namespace {

constexpr int kXcds = 8, kCUs = 256;
constexpr int kGroupM = 8;  // row tiles a group: see grouped()

typedef __attribute__((address_space(3))) void lds_void;

// s_waitcnt vmcnt(N) and s_waitcnt lgkmcnt(0), each alone.
template <int N>
__device__ inline void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt field");
  __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8) | (N & 15) | ((N >> 4) << 14));
}
__device__ inline void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xf | (7 << 4) | (3 << 14)); }

// ---- blocks --------------------------------------------------------------------------------------

// A wavefront a row's 512 values (four blocks).
template <typename T>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, int64_t row_stride, int64_t units, int groups,
                                                       int k, int blocks, uint8_t* __restrict__ q, int64_t stride,
                                                       uint8_t* __restrict__ scales, int64_t scale_stride) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int64_t row = unit / groups;
  const int g = (int)(unit - row * groups);
  const int at = g * 512 + lane * 8;
  float v[8];
  load8(x + row * row_stride + at, k - at, v);
  store_blocks(v, q + row * stride, scales + row * scale_stride, g, blocks, lane);
}

// A workgroup a 128 x 128 block of a weight: the block's largest value, then its bytes by rows, and by
// columns through LDS (a dword of four rows a thread; rows of 132 bytes keep its columns in
// different banks).
template <typename T>
__global__ __launch_bounds__(256) void quantize_weight_kernel(const T* __restrict__ x, int64_t row_stride, int64_t col_stride,
                                                              int64_t rows, int64_t k, uint8_t* __restrict__ q, int64_t stride,
                                                              uint8_t* __restrict__ scales, int64_t scale_stride,
                                                              uint8_t* __restrict__ qt, int64_t t_stride,
                                                              uint8_t* __restrict__ t_scales, int64_t t_scale_stride) {
  __shared__ uint32_t part[4];
  __shared__ uint8_t tile[128][132];
  const int64_t r0 = (int64_t)blockIdx.y * 128, c0 = (int64_t)blockIdx.x * 128;
  const int tid = threadIdx.x;
  // lanes along whichever axis lies closer together
  const bool by_col = col_stride <= row_stride;
  float v[64];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const int e = i * 256 + tid;
    const int64_t r = r0 + (by_col ? e >> 7 : e & 127), c = c0 + (by_col ? e & 127 : e >> 7);
    v[i] = r < rows && c < k ? (float)(x[r * row_stride + c * col_stride]) : 0.0f;
    top = finite_max(top, v[i]);
  }
  top = row_max(top);
#pragma unroll
  for (int i = 16; i < 64; i <<= 1) {
    const uint32_t y = (uint32_t)__shfl_xor((int)top, i);
    top = y > top ? y : top;
  }
  if ((tid & 63) == 0) part[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) top = part[i] > top ? part[i] : top;
  const int byte = scale_byte(top);
  const float inv = scale_inverse(byte);
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const int e = i * 256 + tid;
    tile[by_col ? e >> 7 : e & 127][by_col ? e & 127 : e >> 7] = (uint8_t)to_e4m3(v[i] * inv, 0.0f, 0.0f, 0.0f);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int e = i * 256 + tid, r = e >> 5, c = (e & 31) * 4;
    if (r0 + r < rows)
      *(uint32_t*)(q + (r0 + r) * stride + c0 + c) = *(const uint32_t*)&tile[r][c];
  }
  if (qt != nullptr) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int e = i * 256 + tid, c = e >> 5, r = (e & 31) * 4;
      if (c0 + c < k)
        *(uint32_t*)(qt + (c0 + c) * t_stride + r0 + r) = (uint32_t)tile[r][c] | (uint32_t)tile[r + 1][c] << 8 |
                                                         (uint32_t)tile[r + 2][c] << 16 | (uint32_t)tile[r + 3][c] << 24;
    }
  }
  // its scale, and 1 in the places behind the last block up to a multiple of four
  const int bx = blockIdx.x, by = blockIdx.y;
  if (tid < 4 && (tid == 0 || bx == (int)gridDim.x - 1)) {
    if (tid == 0 || (bx & 3) + tid < 4) scales[by * scale_stride + bx + tid] = tid == 0 ? (uint8_t)byte : 127;
  }
  if (qt != nullptr && tid >= 64 && tid < 68 && (tid == 64 || by == (int)gridDim.y - 1)) {
    const int i = tid - 64;
    if (i == 0 || (by & 3) + i < 4) t_scales[bx * t_scale_stride + by + i] = i == 0 ? (uint8_t)byte : 127;
  }
}

// Eight values a thread.
template <typename T>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t* __restrict__ q, int64_t stride,
                                                         const uint8_t* __restrict__ scales, int64_t scale_stride, int shift,
                                                         int64_t rows, int k, T* __restrict__ out, int64_t out_stride) {
  const int per = (k + 7) >> 3;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / per;
  if (row >= rows) return;
  const int at = (int)(i - row * per) * 8;
  const u32x2 x = *(const u32x2*)(q + row * stride + at);
  const float s = scale_value(scales[(row >> shift) * scale_stride + (at >> 7)]);
  float v[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    v[4 * h + 0] = __builtin_amdgcn_cvt_f32_fp8((int)x[h], 0) * s;
    v[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8((int)x[h], 1) * s;
    v[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8((int)x[h], 2) * s;
    v[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8((int)x[h], 3) * s;
  }
  store8(out + row * out_stride + at, k - at, v);
}

// ---- products ------------------------------------------------------------------------------------

struct ProductArgs {
  const uint8_t* a;
  const uint8_t* a_scales;
  int64_t lda, lda_scales;
  const uint8_t* b[2];  // per column group
  const uint8_t* b_scales[2];
  int64_t ldb[2], ldb_scales[2];
  void* c[2];
  int64_t ldc[2];
  int64_t m, n[2];
  int blocks;  // of 128 along k
  int tiles_m, tiles_n0, tiles_n;
  // pieces along k of `per` blocks each, which write their sums piece_stride outputs apart
  int pieces, per;
  int64_t piece_stride;
  // the few-row kernel's unquantised A
  const void* x;
  int64_t ldx;
  int k;
};

__device__ inline i32x8 join(const i32x4 (&x)[2]) {
  return i32x8{x[0][0], x[0][1], x[0][2], x[0][3], x[1][0], x[1][1], x[1][2], x[1][3]};
}

constexpr int kFewBlocks = 5;  // blocks of k that a wavefront of the few-row kernel has in flight

// Eight e4m3 bytes times 2^e (`scale`: its float) as bf16, exactly.
__device__ inline bf16x8 widen8(int lo, int hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The float that the widening conversions take for a scale's byte: they read its exponent alone.
__device__ inline float byte_as_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Few rows: reading B bounds the product.  A wavefront 16 columns and every kw-th block of k, at most U of them
// in flight at once (all of its own up to U kw blocks); a workgroup kw wavefronts of each of cw column groups, whose sums
// are added in order through LDS.  A lane's weights are 32 consecutive bytes of a column's row: the
// 16 rows of 128 bytes that a load takes are whole lines, and go straight to registers.  B is the MFMA's first
// operand, so that a lane ends up with four consecutive columns of a row.  FUSED: A's blocks are taken
// here, into LDS (rows 16 bytes more than their blocks apart: 16 rows' chunks lie in different banks), while the
// first weights are on their way; every workgroup does it.
template <int G, bool FUSED, typename X, typename Out>
__global__ __launch_bounds__(1024) void few_rows_kernel(const ProductArgs p, int kw) {
  constexpr int U = kFewBlocks;
  constexpr bool EXACT = sizeof(Out) == 4;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), cw = (int)(blockDim.x >> 6) / kw;
  const int wk = wave % kw, wc = wave / kw;
  const int tiles = p.tiles_n0 + (int)((p.n[1] + 15) >> 4);
  const int tile = min((int)blockIdx.x * cw + wc, tiles - 1);  // the last workgroup's spare wavefronts repeat the last tile
  const int grp = tile < p.tiles_n0 ? 0 : 1;
  const int64_t n0 = (int64_t)(tile - (grp ? p.tiles_n0 : 0)) * 16, n = p.n[grp];
  const int64_t col = n0 + (lane & 15) < n ? n0 + (lane & 15) : n - 1;
  const uint8_t* const w = p.b[grp] + col * p.ldb[grp] + (lane >> 4) * 32;
  const uint8_t* const w_scales = p.b_scales[grp] + (n0 >> 7) * p.ldb_scales[grp];
  const int blocks = p.blocks;

  i32x4 wf[U][2];
  uint32_t ws[U];
  auto load_weights = [&](int kb0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = kb0 + u * kw < blocks ? kb0 + u * kw : blocks - 1;
      wf[u][0] = *(const i32x4*)(w + (int64_t)kb * 128);
      wf[u][1] = *(const i32x4*)(w + (int64_t)kb * 128 + 16);
      ws[u] = w_scales[kb];
    }
  };
  load_weights(wk);

  const int row_bytes = blocks * 128 + 16, scale_bytes = (blocks + 3) & ~3;
  uint8_t* const scales = lds + p.m * row_bytes;
  if constexpr (FUSED) {
    const int groups = scale_bytes >> 2, waves = kw * cw;
    for (int unit = wave; unit < (int)p.m * groups; unit += waves) {
      const int row = unit / groups, g = unit - row * groups, at = g * 512 + lane * 8;
      float v[8];
      load8((const X*)p.x + row * p.ldx + at, p.k - at, v);
      store_blocks(v, lds + row * row_bytes, scales + row * scale_bytes, g, blocks, lane);
    }
    __syncthreads();
  }

  // A's rows past the last one are the last one's: not stored
  int64_t row[G];
#pragma unroll
  for (int g = 0; g < G; ++g) row[g] = min((int64_t)(16 * g + (lane & 15)), p.m - 1);
  i32x4 xf[2][G][2];  // of a block and the next one
  uint32_t xs[2][G];
  auto load_rows = [&](int to, int kb) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint8_t* const q = FUSED ? lds + row[g] * row_bytes + kb * 128 + (lane >> 4) * 32
                                     : p.a + row[g] * p.lda + (int64_t)kb * 128 + (lane >> 4) * 32;
      xf[to][g][0] = *(const i32x4*)q;
      xf[to][g][1] = *(const i32x4*)(q + 16);
      xs[to][g] = FUSED ? scales[row[g] * scale_bytes + kb] : p.a_scales[row[g] * p.lda_scales + kb];
    }
  };

  f32x4 acc[G];
#pragma unroll
  for (int g = 0; g < G; ++g) acc[g] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int kb0 = wk; kb0 < blocks; kb0 += U * kw) {
    if (kb0 != wk) load_weights(kb0);
    load_rows(0, kb0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = kb0 + u * kw;
      if (kb < blocks) {
        if (u + 1 < U) load_rows((u + 1) & 1, kb + kw < blocks ? kb + kw : kb);
        if constexpr (EXACT) {
          const float s = byte_as_scale(ws[u]);
          bf16x8 wv[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) wv[i] = widen8(wf[u][i >> 1][2 * (i & 1)], wf[u][i >> 1][2 * (i & 1) + 1], s);
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const i32x4* const x = xf[u & 1][g];
            const float t = byte_as_scale(xs[u & 1][g]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[i], widen8(x[i >> 1][2 * (i & 1)], x[i >> 1][2 * (i & 1) + 1], t),
                                                               acc[g], 0, 0, 0);
          }
        } else {
#pragma unroll
          for (int g = 0; g < G; ++g)
            acc[g] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join(wf[u]), join(xf[u & 1][g]), acc[g], 0, 0, 0, (int)ws[u], 0,
                                                                      (int)xs[u & 1][g]);
        }
      }
    }
  }
  // the products are used outside of branches first
#pragma unroll
  for (int g = 0; g < G; ++g) asm volatile("" : "+v"(acc[g]));
  // the wavefronts' sums, in order; a lane: row lane % 16, columns 4 (lane / 16) .. + 3
  if constexpr (FUSED) __syncthreads();
  f32x4* const sums = (f32x4*)lds;
#pragma unroll
  for (int g = 0; g < G; ++g) sums[(wave * G + g) * 64 + lane] = acc[g];
  __syncthreads();
  if ((int)blockIdx.x * cw + wc >= tiles) return;
  for (int g = wk; g < G; g += kw) {
    f32x4 t = sums[(wc * kw * G + g) * 64 + lane];
    for (int i = 1; i < kw; ++i) t += sums[((wc * kw + i) * G + g) * 64 + lane];
    const int64_t r = 16 * g + (lane & 15);
    const int64_t c0 = n0 + 4 * (lane >> 4);
    if (r < p.m) {
      Out* const c = (Out*)p.c[grp] + r * p.ldc[grp] + c0;
      if (c0 + 4 <= n) {
        typedef Out o4 __attribute__((ext_vector_type(4), aligned(sizeof(Out))));
        *(o4*)c = o4{(Out)t[0], (Out)t[1], (Out)t[2], (Out)t[3]};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c0 + i < n) c[i] = (Out)t[i];
      }
    }
  }
}

// Logical tile -> (row tile, column tile): groups of kGroupM row tiles, each walked column tile by
// column tile, so that the tiles in flight share rows of both operands in L2.
__device__ inline void grouped(int logical, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int in_group = kGroupM * tiles_n;
  const int g = logical / in_group;
  const int first_m = g * kGroupM;
  const int gsize = (tiles_m - first_m) < kGroupM ? (tiles_m - first_m) : kGroupM;
  const int r = logical % in_group;
  tm = first_m + r % gsize;
  tn = r / gsize;
}

// Block b -> logical tile: block b runs on XCD b % 8, and each XCD takes a contiguous run of tiles.
__device__ inline int xcd_order(int b, int nb) {
  const int x = b % kXcds, i = b / kXcds;
  const int per = nb / kXcds, extra = nb % kXcds;
  return x * per + (x < extra ? x : extra) + i;
}

// Eight 16-bit outputs of a row from four registers of each of two groups: lanes below 32 hold columns 0..3
// of group a (and the lanes above them 4..7), and so of group b, 8 columns on.  The halves change places,
// so that a lane below 32 has a's eight columns and the one above it b's.
template <typename Out>
__device__ inline i32x4 pack_groups(const f32x16& v, int g) {
  typedef Out o4 __attribute__((ext_vector_type(4)));
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  const u2 a = __builtin_bit_cast(u2, o4{(Out)v[4 * g], (Out)v[4 * g + 1], (Out)v[4 * g + 2], (Out)v[4 * g + 3]});
  const u2 b = __builtin_bit_cast(u2, o4{(Out)v[4 * g + 4], (Out)v[4 * g + 5], (Out)v[4 * g + 6], (Out)v[4 * g + 7]});
  const u2 x = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
  const u2 y = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
  return i32x4{(int)x[0], (int)y[0], (int)x[1], (int)y[1]};
}

// A tile of BM x BN outputs, WM x WN wavefronts of 32 TI x 32 TJ.  A stage holds a block of k: A's BM
// rows and B's BN rows of 128 bytes, then a dword of each row's scales (the four blocks around this
// one).  The 16-byte chunk c of row r sits in slot c ^ ((r >> 1) & 7): the 16 lanes that a fragment
// read serves at a time (one chunk of 16 consecutive rows) then touch 16 different 16-byte
// banks.  A direct-to-LDS load fills 8 rows (1 KB).  Two stages.
//
// KH 2 (tiles of which one is in a CU, WN = 1): two such sets of wavefronts, each of which takes one half (64 k) of every block and
// all of its columns; their sums meet in LDS at the end.  There are two wavefronts a SIMD to fill each other's waits, no fragment of a half is
// read by more wavefronts than before, and four stages keep the loads of three blocks on their way: 2,047 x 2560 outputs of
// k 10,240 take 61 us in 128 x 160 tiles, 73 in one set that is PIPED (fp32 outputs 105 either way).  Reading the
// next block's fragments between the products as well gives nothing more.
//
// B's fragment is the MFMA's first operand, so that a lane's registers are consecutive columns of one row of C.
//
// PIPED (tiles of which two fit a CU): a block's two halves (64 k) are two sets of fragments; a set is read between
// the MFMAs of the other one.  In the middle of block kb, once every wavefront has read all of it (the barrier),
// the loads of block kb + 2 go out into its place, one at a time between the MFMAs of its second half.
// Otherwise (256-row tiles, 8 wavefronts, whose second set would not fit the registers) the loads of block kb + 1 go out
// at the start of block kb, and the two wavefronts of a SIMD fill each other's waits.
template <int BM, int BN, int WM, int WN, int KH, bool PIPED, bool EXACT, typename Out>
__global__ __launch_bounds__(WM * WN * KH * 64, WM * WN * KH / 4) void product_kernel(const ProductArgs p) {
  constexpr bool BY_ROW = sizeof(Out) == 2;
  constexpr int NW = WM * WN * KH, TI = BM / WM / 32, TJ = BN / WN / 32;
  constexpr int UNITS = (BM + BN) / 8;      // loads of 8 rows a stage
  constexpr int LPW = (UNITS + NW - 1) / NW, REST = UNITS % NW;  // of a wavefront; the last of those below REST alone
  constexpr int SPW = (BM + BN) / NW;       // rows whose scales a wavefront fetches, 64 a load
  constexpr int SL = (SPW + 63) / 64;
  constexpr int SCALES = (BM + BN) * 128;   // where a stage's scales are
  constexpr int STAGE = (BM + BN) * 132;
  constexpr int STAGES = KH == 2 ? 4 : 2;
  static_assert((BM / 8) % NW == 0 && (KH == 2 || REST == 0), "a wavefront's j-th load stays in one operand");
  static_assert(KH == 1 || (KH == 2 && !PIPED), "halves are not pipelined");
  static_assert(BM % (32 * WM) == 0 && BN % (32 * WN) == 0 && (BM + BN) % NW == 0, "whole fragments");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  const int tiles = p.tiles_m * p.tiles_n, piece = (int)blockIdx.x / tiles;
  grouped(xcd_order((int)blockIdx.x - piece * tiles, tiles), p.tiles_m, p.tiles_n, tm, tn);
  const int grp = tn < p.tiles_n0 ? 0 : 1;
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)(grp ? tn - p.tiles_n0 : tn) * BN;
  const int64_t n = p.n[grp];
  const int first = piece * p.per, blocks = min(p.per, p.blocks - first);  // this piece's

  // load j of a stage: 8 rows from row 8 (wave + NW j) of A's, then B's.  Rows past m or n read the last one:
  // their products only reach outputs that are not stored.
  uint32_t off[LPW];
#pragma unroll
  for (int j = 0; j < LPW; ++j) {
    const bool is_a = NW * j < BM / 8;
    const int row = 8 * (wave + NW * j) - (is_a ? 0 : BM) + (lane >> 3);
    const int64_t left = is_a ? p.m - m0 : n - n0;
    const int r = row < left ? row : (int)left - 1;
    off[j] = (uint32_t)r * (uint32_t)(is_a ? p.lda : p.ldb[grp]) + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
  }
  const uint8_t* const a0 = p.a + m0 * p.lda;
  const uint8_t* const b0 = p.b[grp] + n0 * p.ldb[grp];
  // this lane's rows of scales
  const uint8_t* scale_row[SL];
#pragma unroll
  for (int i = 0; i < SL; ++i) {
    const int e = wave * SPW + i * 64 + (i * 64 + lane < SPW ? lane : 0);
    const int64_t ra = m0 + e < p.m ? m0 + e : p.m - 1, rb = n0 + e - BM < n ? n0 + e - BM : n - 1;
    scale_row[i] = e < BM ? p.a_scales + ra * p.lda_scales : p.b_scales[grp] + (rb >> 7) * p.ldb_scales[grp];
  }
  auto load = [&](int kb, int j) {
    if (REST != 0 && j == LPW - 1 && wave >= REST) return;
    const uint8_t* base = (NW * j < BM / 8 ? a0 : b0) + (int64_t)(first + kb) * 128;
    __builtin_amdgcn_global_load_lds((const void*)(base + off[j]), (lds_void*)(lds + (kb & (STAGES - 1)) * STAGE + (wave + NW * j) * 1024), 16, 0, 0);
  };
  auto load_scales = [&](int kb) {
#pragma unroll
    for (int i = 0; i < SL; ++i)
      if (i * 64 + lane < SPW)
        __builtin_amdgcn_global_load_lds((const void*)(scale_row[i] + ((first + kb) & ~3)),
                                         (lds_void*)(lds + (kb & (STAGES - 1)) * STAGE + SCALES + (wave * SPW + i * 64) * 4), 4, 0, 0);
  };
  auto load_all = [&](int kb) {  // LPW + SL loads
    load_scales(kb);
#pragma unroll
    for (int j = 0; j < LPW; ++j) load(kb, j);
  };

  const int kh = KH == 2 ? wave / (WM * WN) : 0, wm = (wave - kh * WM * WN) / WN, wn = wave % WN;
  f32x16 acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  // a half's fragments, A's rows then B's: a lane holds 32 bytes (chunks 4 h + 2 (lane / 32) and the next) of row
  // lane % 32 of its 32
  constexpr int Q = TI + TJ, SETS = PIPED ? 2 : 1;
  i32x8 f[SETS][Q];
  uint32_t sc[Q], next_sc[Q];
  const int x = (lane >> 1) & 7;
  uint32_t at[2];  // of a lane's first chunk in its row, by half; the other one is 16 away
#pragma unroll
  for (int h = 0; h < 2; ++h) at[h] = (lane & 31) * 128 + ((((KH == 2 ? kh : h) * 4 + (lane >> 5) * 2) ^ x) << 4);
  auto row_of = [&](int q) { return q < TI ? (wm * TI + q) * 32 : BM + (wn * TJ + q - TI) * 32; };
  auto read = [&](int kb, int h, int q) {
    const uint8_t* const st = lds + (kb & (STAGES - 1)) * STAGE + row_of(q) * 128;
    const i32x4 lo = *(const i32x4*)(st + at[h]), hi = *(const i32x4*)(st + (at[h] ^ 16));
    f[SETS == 2 ? h : 0][q] = i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  // the dword of four blocks' scales; shifted to the block's own when it is used, so that a read between products is not waited for
  auto scales_at = [&](int kb, int q) {
    return *(const uint32_t*)(lds + (kb & (STAGES - 1)) * STAGE + SCALES + (row_of(q) + (lane & 31)) * 4);
  };
  auto take_scales = [&](int kb) {
#pragma unroll
    for (int q = 0; q < Q; ++q) sc[q] = next_sc[q] >> (((first + kb) & 3) * 8);
  };
  constexpr int QUARTERS = EXACT ? 4 : 1, PRODUCTS = TI * TJ, STEPS = QUARTERS * PRODUCTS;
  // a half's products, with `between(t)` after the t-th of STEPS
  auto half = [&](int h, auto between) {
    const int set = SETS == 2 ? h : 0;
#pragma unroll
    for (int s = 0; s < QUARTERS; ++s) {
      bf16x8 w[Q];
      if constexpr (EXACT) {
#pragma unroll
        for (int q = 0; q < Q; ++q) w[q] = widen8(f[set][q][2 * s], f[set][q][2 * s + 1], byte_as_scale(sc[q] & 255u));
      }
#pragma unroll
      for (int t = 0; t < PRODUCTS; ++t) {
        const int i = t / TJ, j = t % TJ, one = BY_ROW ? TI + j : i, two = BY_ROW ? i : TI + j;
        if constexpr (EXACT)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[one], w[two], acc[i][j], 0, 0, 0);
        else
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(f[set][one], f[set][two], acc[i][j], 0, 0, 0, (int)sc[one], 0,
                                                                      (int)sc[two]);
        between(s * PRODUCTS + t);
      }
    }
  };

  load_all(0);
  if constexpr (KH == 2) {
    if (blocks > 1) load_all(1);
    if (blocks > 2) load_all(2);
    constexpr int EACH = LPW + SL, LESS = EACH - (REST != 0 ? 1 : 0);
    for (int kb = 0; kb < blocks; ++kb) {
      // this wavefront's part of block kb is in LDS (those of the two behind it may be on their way) and its reads of block
      // kb - 1 are in registers; after the barrier, every wavefront's are
      if (kb + 2 < blocks) {
        if (wave < REST || REST == 0) wait_vm<2 * EACH>(); else wait_vm<2 * LESS>();
      } else if (kb + 1 < blocks) {
        if (wave < REST || REST == 0) wait_vm<EACH>(); else wait_vm<LESS>();
      } else {
        wait_vm<0>();
      }
      wait_lgkm0();
      __builtin_amdgcn_s_barrier();
      if (kb + 3 < blocks) load_all(kb + 3);
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        next_sc[q] = scales_at(kb, q);
        read(kb, 0, q);
      }
      take_scales(kb);
      half(0, [](int) {});
    }
  } else if constexpr (PIPED) {
    if (blocks > 1) {
      load_all(1);
      wait_vm<LPW + SL>();
    } else {
      wait_vm<0>();
    }
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      read(0, 0, q);
      next_sc[q] = scales_at(0, q);
    }
    take_scales(0);
    // a fragment's reads after each of the first products
    constexpr int PER = (Q + STEPS - 1) / STEPS;
    auto reads_at = [&](int t, auto one) {
#pragma unroll
      for (int q = t * PER; q < t * PER + PER; ++q)
        if (q < Q) one(q);
    };
    for (int kb = 0; kb + 1 < blocks; ++kb) {
      half(0, [&](int t) {
        __builtin_amdgcn_sched_barrier(0);
        reads_at(t, [&](int q) { read(kb, 1, q); });
        __builtin_amdgcn_sched_barrier(0);
      });
      // this wavefront's part of block kb + 1 is in LDS and its reads of block kb are in registers; after the
      // barrier, every wavefront's are
      wait_vm<0>();
      wait_lgkm0();
      __builtin_amdgcn_s_barrier();
      const bool more = kb + 2 < blocks;
      half(1, [&](int t) {
        __builtin_amdgcn_sched_barrier(0);
        reads_at(t, [&](int q) {
          read(kb + 1, 0, q);
          next_sc[q] = scales_at(kb + 1, q);
        });
        if (more) {
          if (t == 0) load_scales(kb + 2);
          if (t < LPW) load(kb + 2, t);
          if (t == STEPS - 1)
#pragma unroll
            for (int j = STEPS; j < LPW; ++j) load(kb + 2, j);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      take_scales(kb + 1);
    }
    half(0, [&](int t) { reads_at(t, [&](int q) { read(blocks - 1, 1, q); }); });
    half(1, [](int) {});
  } else {
    for (int kb = 0; kb < blocks; ++kb) {
      // this wavefront's part of block kb is in LDS and its reads of block kb - 1 are in registers; after the
      // barrier, every wavefront's are
      wait_vm<0>();
      wait_lgkm0();
      __builtin_amdgcn_s_barrier();
      if (kb + 1 < blocks) load_all(kb + 1);
#pragma unroll
      for (int q = 0; q < Q; ++q) next_sc[q] = scales_at(kb, q);
      take_scales(kb);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int q = 0; q < Q; ++q) read(kb, h, q);
        half(h, [](int) {});
      }
    }
  }
  // the last products are used outside the branches below
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) asm volatile("" : "+v"(acc[i][j]));

  // the halves' sums: each wavefront ends with those of a part of its columns
  constexpr int MINE = (TJ + 1) / 2;
  if constexpr (KH == 2) {
    static_assert(TI * TJ * WM * WN * 4096 <= STAGES * STAGE, "the halves' sums fit LDS");
    f32x4* const sums = (f32x4*)lds + (wave - kh * WM * WN) * (TI * TJ * 256) + lane;
    __syncthreads();  // every wavefront has read all of its last block
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j)
        if ((j < MINE) != (kh == 0))
#pragma unroll
          for (int r = 0; r < 4; ++r)
            sums[((i * TJ + j) * 4 + r) * 64] = f32x4{acc[i][j][4 * r], acc[i][j][4 * r + 1], acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]};
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j)
        if ((j < MINE) == (kh == 0))
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const f32x4 t = sums[((i * TJ + j) * 4 + r) * 64];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][4 * r + e] += t[e];
          }
  }

  Out* const c = (Out*)p.c[grp] + piece * p.piece_stride;
  const int64_t ldc = p.ldc[grp];
  if constexpr (BY_ROW) {
    // D: lane l holds row l % 32 of C's 32 x 32 and columns 8 (r / 4) + 4 (l / 32) + r % 4
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      const int64_t row = m0 + (wm * TI + i) * 32 + (lane & 31);
      if (row >= p.m) continue;
      Out* const c_row = c + row * ldc;
#pragma unroll
      for (int j = 0; j < TJ; ++j)
        if (KH == 1 || (j < MINE) == (kh == 0))
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
          typedef Out o8 __attribute__((ext_vector_type(8), aligned(2)));
          const o8 v = __builtin_bit_cast(o8, pack_groups<Out>(acc[i][j], g));
          const int64_t col = n0 + (wn * TJ + j) * 32 + 8 * g + 8 * (lane >> 5);
          if (col + 8 <= n) {
            *(o8*)(c_row + col) = v;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (col + e < n) c_row[col + e] = v[e];
          }
        }
    }
  } else {
    // D: lane l holds column l % 32 and rows 8 (r / 4) + 4 (l / 32) + r % 4: whole lines of a row
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        if (KH == 2 && (j < MINE) != (kh == 0)) continue;
        const int64_t col = n0 + (wn * TJ + j) * 32 + (lane & 31);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int64_t row = m0 + (wm * TI + i) * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
          if (row < p.m && col < n) c[row * ldc + col] = (Out)acc[i][j][r];
        }
      }
  }
}

// The pieces' sums, in order: eight outputs of a group's [m, n] (dense in the pieces) a thread.
template <typename Out>
__global__ __launch_bounds__(256) void piece_sum_kernel(const float* __restrict__ sums, int pieces, int64_t piece_stride, int64_t m,
                                                        int64_t n, Out* __restrict__ c, int64_t ldc) {
  const int64_t per = (n + 7) >> 3, i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / per, col = (i - row * per) * 8;
  if (row >= m) return;
  const int valid = (int)min(n - col, (int64_t)8);
  float v[8];
  load8(sums + row * n + col, valid, v);
  for (int q = 1; q < pieces; ++q) {
    float x[8];
    load8(sums + q * piece_stride + row * n + col, valid, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += x[e];
  }
  store8(c + row * ldc + col, valid, v);
}

// ---- host ----------------------------------------------------------------------------------------

// Rows of the few-row kernel.  With the rows' blocks, bf16 outputs: 32 rows of 2560 x 2560 take 8.9 us in it and 33 rows 14.4 in
// 64 x 64 tiles; 2560 x 640 9.0 and 14.7, 1000 x 1111 8.5 and 9.0.  Where outputs or k are long the tiles are ahead from about
// 25 rows on: 2560 x 10240 16.1 and 14.5 (24 rows 13.4), 10240 x 2560 21.1 and 15.9 (24 rows 18.7).
constexpr int kFewRows = 32;
constexpr int64_t kFusedBytes = 64 << 10;

template <int BM, int BN, int WM, int WN, int KH, bool PIPED, bool EXACT, typename Out>
int launch_tiles(ProductArgs p, hipStream_t st) {
  p.tiles_m = (int)((p.m + BM - 1) / BM);
  p.tiles_n0 = (int)((p.n[0] + BN - 1) / BN);
  p.tiles_n = p.tiles_n0 + (int)((p.n[1] + BN - 1) / BN);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  if (tiles > INT32_MAX) return set_error(EG_ERR_UNSUPPORTED, "fp8 product: %lld tiles", (long long)tiles);
  const auto kernel = product_kernel<BM, BN, WM, WN, KH, PIPED, EXACT, Out>;
  constexpr int bytes = (KH == 2 ? 4 : 2) * (BM + BN) * 132;
  EG_CHECK_HIP(allow_lds((const void*)kernel, bytes));
  kernel<<<(unsigned)(tiles * p.pieces), WM * WN * KH * 64, bytes, st>>>(p);
  return launch_status("product_kernel");
}

// What a tile costs, in the time that the fp8 (or, EXACT, the bf16) matrix cores take for a product at 256 x 256:
// `each` an output where all CUs are full (measured at 8192^3), `resident` tiles a CU at once.
struct Tile {
  int bm, bn, resident;
  float each, each_exact;
  bool halves;  // KH 2
};
constexpr Tile kTiles[] = {
    {256, 256, 1, 1.00f, 1.00f, false},  // fp8 437 us, bf16 816 us of 8192^3
    {256, 320, 1, 0.92f, 0.93f, false},  // 507 (205 tiles of 5/4, five rounds for four), 954
    {256, 192, 1, 1.05f, 1.00f, false},  // 503, 908
    {128, 128, 2, 1.17f, 1.09f, false},  // 514, 887
    {128, 160, 1, 1.43f, 1.37f, true},   // 623, 1080
    {64, 128, 3, 1.48f, 1.26f, false},   // 658, 1024
    {64, 64, 4, 1.94f, 1.49f, false},    // 858, 1209
    {64, 160, 1, 1.97f, 1.67f, true},    // 858, 1322
};

// The tile for m x (n0, n1) outputs of `blocks` blocks of k: the least time of the CU that gets the most tiles.  A block of a tile of
// four wavefronts of whole blocks that has its CU to itself takes 14,000 outputs' time (12,000 EXACT) and 0.95 (0.8) an output, its
// loads' latency; a halves' tile takes 138,000 (41,000) more, for its first loads and its sums' meeting: 1,024 x 2560 outputs of
// k 10,240 take 43.6 us (67.2) in 64 x 160 and 50.9 (75.7) in 64 x 64, of k 2560 14.9 and 14.0 (21.7 and 22.3).
template <bool EXACT>
int choose_tile(int64_t m, int64_t n0, int64_t n1, int blocks) {
  int best = 0;
  double least = 0;
  for (int i = 0; i < (int)(sizeof(kTiles) / sizeof(kTiles[0])); ++i) {
    const Tile& t = kTiles[i];
    const double area = (double)t.bm * t.bn, each = (EXACT ? t.each_exact : t.each) * area;
    const int64_t tiles = ((m + t.bm - 1) / t.bm) * ((n0 + t.bn - 1) / t.bn + (n1 + t.bn - 1) / t.bn);
    const int64_t a_cu = (tiles + kCUs - 1) / kCUs;
    const double alone = t.bm == 256 || t.halves ? 0.0 : EXACT ? 12000 + 0.8 * area : 14000 + 0.95 * area;
    const double once = t.halves ? (EXACT ? 41000.0 : 138000.0) / blocks : 0.0;
    auto cost = [&](int64_t count) { return count == 0 ? 0.0 : std::max(alone, count * each); };
    const double time = (a_cu / t.resident) * cost(t.resident) + cost(a_cu % t.resident) + a_cu * once;
    if (i == 0 || time < least) {
      best = i;
      least = time;
    }
  }
  return best;
}

// Pieces along k of a long product whose 64 x 64 tiles are few: as many as make three workgroups a CU, of at least 10 blocks
// each; their fp32 sums are added in order by a launch of its own.  bf16 outputs of 256 x 10240 x 2560 (160 tiles): 21 us
// in four pieces, 43 in one; 500 rows (320 tiles) 32 and 43; 256 x 2560 x 2560 13 in two, 9 in one.
int pieces_of(int64_t m, int64_t n0, int64_t n1, int blocks) {
  if (m <= kFewRows) return 1;
  const int64_t tiles = ((m + 63) / 64) * ((n0 + 63) / 64 + (n1 + 63) / 64);
  if (tiles == 0) return 1;
  const int pieces = blocks < 24 ? 1 : (int)std::min<int64_t>(3 * kCUs / tiles, blocks / 10);
  return std::max(1, pieces);
}

// Bytes of the pieces' sums.
int64_t piece_bytes(int64_t m, int64_t n0, int64_t n1, int64_t k) {
  const int pieces = pieces_of(m, n0, n1, (int)((k + 127) / 128));
  return pieces > 1 ? (int64_t)pieces * m * (n0 + n1) * 4 : 0;
}

template <bool EXACT, typename Out>
int launch_product(ProductArgs p, float* sums, hipStream_t st) {
  p.pieces = pieces_of(p.m, p.n[0], p.n[1], p.blocks);  // eg_fp8_product_tile tells of this plan
  p.per = (p.blocks + p.pieces - 1) / p.pieces;
  if (p.pieces > 1) {
    p.pieces = (p.blocks + p.per - 1) / p.per;  // none is empty
    ProductArgs to = p;
    to.piece_stride = p.m * (p.n[0] + p.n[1]);
    to.c[0] = sums;
    to.c[1] = sums + p.m * p.n[0];
    to.ldc[0] = p.n[0];
    to.ldc[1] = p.n[1];
    if (const int rc = launch_tiles<64, 64, 2, 2, 1, true, EXACT, float>(to, st); rc != EG_OK) return rc;
    for (int i = 0; i < 2; ++i) {
      if (p.n[i] == 0) continue;
      const int64_t groups = (p.m * ((p.n[i] + 7) / 8) + 255) / 256;
      piece_sum_kernel<Out><<<(unsigned)groups, 256, 0, st>>>((const float*)to.c[i], p.pieces, to.piece_stride, p.m, p.n[i], (Out*)p.c[i], p.ldc[i]);
      if (const int rc = launch_status("piece_sum_kernel"); rc != EG_OK) return rc;
    }
    return EG_OK;
  }
  switch (choose_tile<EXACT>(p.m, p.n[0], p.n[1], p.blocks)) {
    case 0: return launch_tiles<256, 256, 2, 4, 1, false, EXACT, Out>(p, st);
    case 1: return launch_tiles<256, 320, 4, 2, 1, false, EXACT, Out>(p, st);
    case 2: return launch_tiles<256, 192, 4, 2, 1, false, EXACT, Out>(p, st);
    case 3: return launch_tiles<128, 128, 2, 2, 1, true, EXACT, Out>(p, st);
    case 4: return launch_tiles<128, 160, 4, 1, 2, false, EXACT, Out>(p, st);
    case 5: return launch_tiles<64, 128, 2, 2, 1, true, EXACT, Out>(p, st);
    case 6: return launch_tiles<64, 64, 2, 2, 1, true, EXACT, Out>(p, st);
    default: return launch_tiles<64, 160, 2, 1, 2, false, EXACT, Out>(p, st);
  }
}

// How the few-row kernel is launched: kw wavefronts share a column group's blocks of k, so many that each has all of its
// blocks in flight at once; cw column groups a workgroup.  FUSED: at least four wavefronts, and as many
// column groups as leave 128 workgroups, for the rows' blocks that each of them takes.
struct FewPlan {
  int kw, cw;
};
FewPlan few_plan(int64_t m, int blocks, int64_t tiles, bool takes_blocks) {
  FewPlan f = {1, 1};
  while (f.kw < 16 && (blocks + f.kw - 1) / f.kw > kFewBlocks) f.kw *= 2;
  if (takes_blocks) {
    f.kw = std::max(f.kw, 4);
    while (m > 2 && f.kw * f.cw < 16 && tiles / (2 * f.cw) >= 128) f.cw *= 2;
  }
  return f;
}

// LDS of the rows' blocks, where the few-row kernel takes them itself.
int64_t fused_bytes(int64_t m, int64_t k) {
  const int64_t blocks = (k + 127) / 128;
  return m * (blocks * 128 + 16 + ((blocks + 3) & ~(int64_t)3));
}

// Whether it does: they fit, and a thread takes at most 64 values of them.  At 2560 x 10240, 24 rows (60 values a
// thread): 15.9 us, and 13.5 after a launch of 2.5 for the blocks; at 2560 x 2560, 4 rows (40): 6.6 and 4.4 + 2.5,
// 8 rows (80): 9.1 and 4.5 + 2.5.
bool fused(int64_t m, int64_t k, int64_t n0, int64_t n1) {
  if (m > kFewRows || fused_bytes(m, k) > kFusedBytes) return false;
  const int blocks = (int)((k + 127) / 128);
  const FewPlan f = few_plan(m, blocks, (n0 + 15) / 16 + (n1 + 15) / 16, true);
  return m * blocks * 128 <= 64 * 64 * f.kw * f.cw;
}

template <int G, bool FUSED, typename X>
int launch_few(ProductArgs p, int32_t dtype, hipStream_t st) {
  p.tiles_n0 = (int)((p.n[0] + 15) / 16);
  const int64_t tiles = p.tiles_n0 + (p.n[1] + 15) / 16;
  const FewPlan f = few_plan(p.m, p.blocks, tiles, FUSED);
  const int64_t a_bytes = FUSED ? fused_bytes(p.m, p.k) : 0, sums = (int64_t)f.kw * f.cw * G * 1024;
  return with_type(dtype, [&](auto out) {
    few_rows_kernel<G, FUSED, X, decltype(out)>
        <<<(unsigned)((tiles + f.cw - 1) / f.cw), f.kw * f.cw * 64, a_bytes > sums ? a_bytes : sums, st>>>(p, f.kw);
    return launch_status("few_rows_kernel");
  });
}

int check_product(const eg_fp8_matrix* b, const eg_fp8_matrix* b2, void* c, int64_t ldc, void* c2, int64_t ldc2,
                  int32_t dtype, int64_t m, int64_t k, ProductArgs* p) {
  EG_CHECK_ARG(known_dtype(dtype), "fp8 product: dtype=%d", dtype);
  if (const int rc = check_fp8(b, 128, "b"); rc != EG_OK) return rc;
  EG_CHECK_ARG(b->k == k, "fp8 product: a has k=%lld, b %lld", (long long)k, (long long)b->k);
  *p = ProductArgs{};
  const eg_fp8_matrix* const w[2] = {b, b2};
  void* const out[2] = {c, c2};
  const int64_t ld[2] = {ldc, ldc2};
  for (int i = 0; i < 2; ++i) {
    if (w[i] == nullptr) continue;
    if (i == 1) {
      if (const int rc = check_fp8(b2, 128, "b2"); rc != EG_OK) return rc;
      EG_CHECK_ARG(b2->k == k, "fp8 product: a has k=%lld, b2 %lld", (long long)k, (long long)b2->k);
    }
    EG_CHECK_ARG(ld[i] >= w[i]->rows, "fp8 product: rows of %lld outputs are %lld apart", (long long)w[i]->rows, (long long)ld[i]);
    EG_CHECK_ARG(out[i] != nullptr || m == 0 || w[i]->rows == 0, "fp8 product: NULL output");
    EG_CHECK_ARG((uintptr_t)out[i] % item_size(dtype) == 0, "fp8 product: misaligned output");
    p->b[i] = (const uint8_t*)w[i]->q;
    p->b_scales[i] = w[i]->scales;
    p->ldb[i] = w[i]->stride;
    p->ldb_scales[i] = w[i]->scale_stride;
    p->c[i] = out[i];
    p->ldc[i] = ld[i];
    p->n[i] = w[i]->rows;
  }
  p->m = m;
  p->k = (int)k;
  p->blocks = (int)((k + 127) / 128);
  if (p->n[0] == 0) {  // the second group alone
    p->b[0] = p->b[1];
    p->b_scales[0] = p->b_scales[1];
    p->ldb[0] = p->ldb[1];
    p->ldb_scales[0] = p->ldb_scales[1];
    p->c[0] = p->c[1];
    p->ldc[0] = p->ldc[1];
    p->n[0] = p->n[1];
    p->n[1] = 0;
  }
  return EG_OK;
}

// Validates that outputs and workspace share no memory with the weights, with A (its blocks and scales, or its values) or one another.
int check_product_areas(const ProductArgs& p, int32_t dtype, const eg_fp8_matrix& b, const eg_fp8_matrix* b2, const void* workspace,
                        int64_t workspace_bytes, const Area& a, const Area& a_scales, const char* what) {
  const eg_fp8_matrix none = {nullptr, nullptr, 0, 1, 0, 0, 128}, &second = b2 ? *b2 : none;
  return check_areas(what,
                     {values_area(p.c[0], dtype, p.m, p.n[0], p.ldc[0], "an output"),
                      values_area(p.c[1], dtype, p.m, p.n[1], p.ldc[1], "the second output"),
                      bytes_area(workspace, workspace_bytes, "the workspace")},
                     {a, a_scales, blocks_area(b, "b"), scales_area(b, "b's scales"), blocks_area(second, "b2"),
                      scales_area(second, "b2's scales")});
}

int run_product(const ProductArgs& p, int32_t dtype, float* sums, hipStream_t st) {
  if (p.m == 0 || p.n[0] == 0) return EG_OK;
  if (p.m <= 16) return launch_few<1, false, float>(p, dtype, st);
  if (p.m <= kFewRows) return launch_few<2, false, float>(p, dtype, st);
  switch (dtype) {
    case EG_DTYPE_F32: return launch_product<true, float>(p, sums, st);
    case EG_DTYPE_BF16: return launch_product<false, __bf16>(p, sums, st);
    default: return launch_product<false, _Float16>(p, sums, st);
  }
}

int check_workspace(const void* workspace, int64_t bytes, int64_t need, const char* what) {
  if (bytes < need)
    return set_error(EG_ERR_WORKSPACE, "%s needs %lld bytes of workspace, got %lld", what, (long long)need, (long long)bytes);
  EG_CHECK_ARG(need == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0), "%s: the workspace must be 16-byte aligned", what);
  return EG_OK;
}

// Bytes of A's blocks, a multiple of 16.
int64_t block_bytes(int64_t m, int64_t k) {
  const int64_t blocks = (k + 127) / 128;
  return (m * (blocks * 128 + (blocks + 3) / 4 * 4) + 15) / 16 * 16;
}

bool known_size(int64_t m, int64_t n, int64_t n2, int64_t k) {
  return m >= 0 && m < (1ll << 31) && n >= 0 && n < (1ll << 31) && n2 >= 0 && n2 < (1ll << 31) && k >= 1 && k <= (1 << 22);
}

}  // namespace

int check_fp8(const eg_fp8_matrix* m, int block_rows, const char* what) {
  EG_CHECK_ARG(m != nullptr, "%s: NULL matrix", what);
  EG_CHECK_ARG(m->block_rows == block_rows, "%s: a scale covers %d rows, %d expected", what, m->block_rows, block_rows);
  EG_CHECK_ARG(m->rows >= 0 && m->rows < (1ll << 31) && m->k >= 1 && m->k <= (1 << 22),
               "%s: %lld x %lld: rows in [0, 2^31) and k in [1, 2^22] expected", what, (long long)m->rows, (long long)m->k);
  const int64_t blocks = (m->k + 127) / 128;
  EG_CHECK_ARG(m->stride >= blocks * 128 && m->stride % 16 == 0 && m->stride <= (1 << 23),
               "%s: stride=%lld: a multiple of 16 from %lld to 2^23 expected", what, (long long)m->stride, (long long)(blocks * 128));
  EG_CHECK_ARG(m->scale_stride >= (blocks + 3) / 4 * 4 && m->scale_stride % 4 == 0 && m->scale_stride <= (1 << 23),
               "%s: scale_stride=%lld: a multiple of 4 from %lld to 2^23 expected", what, (long long)m->scale_stride,
               (long long)((blocks + 3) / 4 * 4));
  EG_CHECK_ARG(m->rows == 0 || (m->q != nullptr && m->scales != nullptr), "%s: NULL", what);
  EG_CHECK_ARG((uintptr_t)m->q % 16 == 0 && (uintptr_t)m->scales % 4 == 0,
               "%s: q must be 16-byte and scales 4-byte aligned", what);
  return EG_OK;
}

}  // namespace eg

using namespace eg;

extern "C" {

int eg_fp8_quantize(const void* x, int32_t dtype, int64_t row_stride, const eg_fp8_matrix* out, void* stream) {
  if (const int rc = check_fp8(out, 1, "fp8_quantize"); rc != EG_OK) return rc;
  if (const int rc = check_values(x, dtype, out->rows, out->k, row_stride, "fp8_quantize"); rc != EG_OK) return rc;
  if (out->rows == 0) return EG_OK;
  const int blocks = (int)((out->k + 127) / 128), groups = (blocks + 3) / 4;
  const int64_t units = out->rows * groups;
  EG_CHECK_ARG((units + 3) / 4 < (1 << 24), "fp8_quantize: %lld x %lld is too large", (long long)out->rows, (long long)out->k);
  if (const int rc = check_areas("fp8_quantize", {blocks_area(*out, "q"), scales_area(*out, "its scales")},
                                 {values_area(x, dtype, out->rows, out->k, row_stride, "the values")});
      rc != EG_OK)
    return rc;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    quantize_kernel<T><<<(unsigned)((units + 3) / 4), 256, 0, (hipStream_t)stream>>>(
        (const T*)x, row_stride, units, groups, (int)out->k, blocks, (uint8_t*)out->q, out->stride, out->scales, out->scale_stride);
    return launch_status("quantize_kernel");
  });
}

int eg_fp8_quantize_weight(const void* x, int32_t dtype, int64_t row_stride, int64_t col_stride, const eg_fp8_matrix* out,
                           const eg_fp8_matrix* out_t, void* stream) {
  if (const int rc = check_fp8(out, 128, "fp8_quantize_weight"); rc != EG_OK) return rc;
  EG_CHECK_ARG(known_dtype(dtype), "fp8_quantize_weight: dtype=%d", dtype);
  EG_CHECK_ARG(x != nullptr || out->rows == 0, "fp8_quantize_weight: NULL values");
  EG_CHECK_ARG((uintptr_t)x % item_size(dtype) == 0, "fp8_quantize_weight: misaligned values");
  if (out_t != nullptr && out->rows > 0) {
    if (const int rc = check_fp8(out_t, 128, "fp8_quantize_weight: the transpose"); rc != EG_OK) return rc;
    EG_CHECK_ARG(out_t->rows == out->k && out_t->k == out->rows, "fp8_quantize_weight: the transpose of %lld x %lld is %lld x %lld",
                 (long long)out->rows, (long long)out->k, (long long)out_t->rows, (long long)out_t->k);
  }
  if (out->rows == 0) return EG_OK;
  const int64_t by = (out->rows + 127) / 128;
  EG_CHECK_ARG(by <= 65535, "fp8_quantize_weight: %lld rows", (long long)out->rows);
  const eg_fp8_matrix none = {nullptr, nullptr, 0, 1, 0, 0, 128}, &transpose = out_t ? *out_t : none;
  if (const int rc = check_areas("fp8_quantize_weight",
                                 {blocks_area(*out, "q"), scales_area(*out, "its scales"), blocks_area(transpose, "the transpose"),
                                  scales_area(transpose, "the transpose's scales")},
                                 {{Extent(x, out->rows, out->k, row_stride, col_stride, item_size(dtype)), "the values"}});
      rc != EG_OK)
    return rc;
  const dim3 grid((unsigned)((out->k + 127) / 128), (unsigned)by);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    quantize_weight_kernel<T><<<grid, 256, 0, (hipStream_t)stream>>>(
        (const T*)x, row_stride, col_stride, out->rows, out->k, (uint8_t*)out->q, out->stride, out->scales, out->scale_stride,
        out_t ? (uint8_t*)out_t->q : nullptr, out_t ? out_t->stride : 0, out_t ? out_t->scales : nullptr,
        out_t ? out_t->scale_stride : 0);
    return launch_status("quantize_weight_kernel");
  });
}

int eg_fp8_dequantize(const eg_fp8_matrix* m, void* out, int32_t dtype, int64_t row_stride, void* stream) {
  EG_CHECK_ARG(m != nullptr, "fp8_dequantize: NULL matrix");
  if (const int rc = check_fp8(m, m->block_rows == 128 ? 128 : 1, "fp8_dequantize"); rc != EG_OK) return rc;
  if (const int rc = check_values(out, dtype, m->rows, m->k, row_stride, "fp8_dequantize"); rc != EG_OK) return rc;
  const int64_t count = m->rows * ((m->k + 7) / 8);
  if (count == 0) return EG_OK;
  EG_CHECK_ARG((count + 255) / 256 < (1 << 24), "fp8_dequantize: %lld x %lld is too large", (long long)m->rows, (long long)m->k);
  if (const int rc = check_areas("fp8_dequantize", {values_area(out, dtype, m->rows, m->k, row_stride, "the output")},
                                 {blocks_area(*m, "q"), scales_area(*m, "its scales")});
      rc != EG_OK)
    return rc;
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    dequantize_kernel<T><<<(unsigned)((count + 255) / 256), 256, 0, (hipStream_t)stream>>>(
        (const uint8_t*)m->q, m->stride, m->scales, m->scale_stride, m->block_rows == 128 ? 7 : 0, m->rows, (int)m->k, (T*)out, row_stride);
    return launch_status("dequantize_kernel");
  });
}

int64_t eg_fp8_product_workspace_size(int64_t m, int64_t n, int64_t n2, int64_t k) {
  return known_size(m, n, n2, k) ? piece_bytes(m, n, n2, k) : -1;
}

int64_t eg_fp8_product_tile(int64_t m, int64_t n, int64_t n2, int64_t k, int32_t dtype, int32_t* pieces) {
  if (!known_size(m, n, n2, k) || !known_dtype(dtype)) return -1;
  const int blocks = (int)((k + 127) / 128), cut = pieces_of(m, n, n2, blocks), per = (blocks + cut - 1) / cut;
  if (pieces != nullptr) *pieces = (blocks + per - 1) / per;
  if (m <= kFewRows || n + n2 == 0) return 0;
  if (cut > 1) return (int64_t)64 << 16 | 64;
  const Tile& t = kTiles[dtype == EG_DTYPE_F32 ? choose_tile<true>(m, n, n2, blocks) : choose_tile<false>(m, n, n2, blocks)];
  return (int64_t)t.bm << 16 | t.bn;
}

int eg_fp8_product(const eg_fp8_matrix* a, const eg_fp8_matrix* b, const eg_fp8_matrix* b2, void* c, int64_t ldc, void* c2,
                   int64_t ldc2, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const int rc = check_fp8(a, 1, "a"); rc != EG_OK) return rc;
  ProductArgs p;
  if (const int rc = check_product(b, b2, c, ldc, c2, ldc2, dtype, a->rows, a->k, &p); rc != EG_OK) return rc;
  const int64_t need = piece_bytes(p.m, p.n[0], p.n[1], p.k);
  if (const int rc = check_workspace(workspace, workspace_bytes, need, "fp8_product"); rc != EG_OK) return rc;
  if (const int rc = check_product_areas(p, dtype, *b, b2, workspace, need, blocks_area(*a, "a"), scales_area(*a, "a's scales"), "fp8_product");
      rc != EG_OK)
    return rc;
  p.a = (const uint8_t*)a->q;
  p.a_scales = a->scales;
  p.lda = a->stride;
  p.lda_scales = a->scale_stride;
  return run_product(p, dtype, (float*)workspace, (hipStream_t)stream);
}

int64_t eg_fp8_linear_workspace_size(int64_t m, int64_t n, int64_t n2, int64_t k) {
  if (!known_size(m, n, n2, k)) return -1;
  return fused(m, k, n, n2) ? 0 : block_bytes(m, k) + piece_bytes(m, n, n2, k);
}

int eg_fp8_linear(const void* x, int32_t x_dtype, int64_t m, int64_t x_stride, const eg_fp8_matrix* b, const eg_fp8_matrix* b2,
                  void* c, int64_t ldc, void* c2, int64_t ldc2, int32_t dtype, void* workspace, int64_t workspace_bytes,
                  void* stream) {
  EG_CHECK_ARG(b != nullptr, "fp8_linear: NULL matrix");
  ProductArgs p;
  EG_CHECK_ARG(m >= 0 && m < (1ll << 31), "fp8_linear: %lld rows", (long long)m);
  if (const int rc = check_product(b, b2, c, ldc, c2, ldc2, dtype, m, b->k, &p); rc != EG_OK) return rc;
  if (const int rc = check_values(x, x_dtype, m, b->k, x_stride, "fp8_linear"); rc != EG_OK) return rc;
  if (m == 0 || p.n[0] == 0) return EG_OK;
  const int64_t k = b->k, need = eg_fp8_linear_workspace_size(m, b->rows, b2 ? b2->rows : 0, k);
  if (const int rc = check_workspace(workspace, workspace_bytes, need, "fp8_linear"); rc != EG_OK) return rc;
  if (const int rc = check_product_areas(p, dtype, *b, b2, workspace, need, values_area(x, x_dtype, m, k, x_stride, "x"),
                                         bytes_area(nullptr, 0, ""), "fp8_linear");
      rc != EG_OK)
    return rc;
  if (fused(m, k, p.n[0], p.n[1])) {
    p.x = x;
    p.ldx = x_stride;
    return with_type(x_dtype, [&](auto t) {
      using X = decltype(t);
      return m <= 16 ? launch_few<1, true, X>(p, dtype, (hipStream_t)stream) : launch_few<2, true, X>(p, dtype, (hipStream_t)stream);
    });
  }
  const int64_t kp = (int64_t)p.blocks * 128;
  const eg_fp8_matrix a = {workspace, (uint8_t*)workspace + m * kp, m, k, kp, (p.blocks + 3) / 4 * 4, 1};
  if (const int rc = eg_fp8_quantize(x, x_dtype, x_stride, &a, stream); rc != EG_OK) return rc;
  p.a = (const uint8_t*)a.q;
  p.a_scales = a.scales;
  p.lda = a.stride;
  p.lda_scales = a.scale_stride;
  return run_product(p, dtype, (float*)((uint8_t*)workspace + block_bytes(m, k)), (hipStream_t)stream);
}

}  // extern "C"
