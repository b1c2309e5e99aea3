// Products of matrices in blocks of 8-bit floating point, the blocks themselves, and their values.
//
//   C[m, n] = sum_b 2^(ea[m, b] + eb[n / 128, b]) sum_{k in block b} qa[m, k] qb[n, k]
//
// Scales are powers of two because CDNA4's scaled MFMA takes them with its operands: a block costs no
// arithmetic outside the matrix cores, and a block's values are exact in bf16 (e4m3 has 4 significant
// bits).  What the fp8 matrix cores do not give is fp32 sums: they align eight products to the
// largest of the eight and drop what lies 2^-13 below it, before the fp32 addition (seen with
// 2^16 and 2^3, 2^2 among eight; 1.5e-5 of a product of normal values of any length, without a bias).  That
// is far below the rounding of a bf16 (2^-8) or fp16 (2^-11) output; an fp32 output takes the
// bf16 matrix cores instead, at half the rate, on the same bytes: its products are exact and its sums fp32.
//
// The scaled MFMA's intrinsic is not convergent: where its result is used in a branch alone, the
// compiler may move it (with its operands' moves) into the branch, where the lanes that are off keep
// what their registers held.  Here its results are used again by the next step of a loop, which holds them outside.
#include "eg_fp8.h"

#include "eg_lds.h"

namespace eg {
namespace {

constexpr int kXcds = 8;
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
  // the few-row kernel's unquantised A
  const void* x;
  int64_t ldx;
  int k;
};

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

// Few rows: reading B bounds the product.  A workgroup 16 columns, its wavefronts every KW-th block of k,
// their sums added in order through LDS.  A lane's weights are 32 consecutive bytes of a column's row: the
// 16 rows of 128 bytes that a load takes are whole lines, and go straight to registers.  B is the MFMA's first
// operand, so that a lane ends up with four consecutive columns of a row.  FUSED: A's blocks are taken
// here, into LDS, while the first weights are on their way (a few rows: every workgroup does it).
template <int G, bool FUSED, typename X, typename Out>
__global__ __launch_bounds__(1024) void few_rows_kernel(const ProductArgs p) {
  constexpr int U = 4;  // blocks of k in flight a wavefront
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kw = blockDim.x >> 6;
  const int grp = (int)blockIdx.x < p.tiles_n0 ? 0 : 1;
  const int64_t n0 = (int64_t)((int)blockIdx.x - (grp ? p.tiles_n0 : 0)) * 16, n = p.n[grp];
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
  load_weights(wave);

  const int kp = blocks * 128, sp = (blocks + 3) & ~3;
  if constexpr (FUSED) {
    const int groups = sp >> 2;
    for (int64_t unit = wave; unit < p.m * groups; unit += kw) {
      const int row = (int)(unit / groups), g = (int)(unit - (int64_t)row * groups), at = g * 512 + lane * 8;
      float v[8];
      load8((const X*)p.x + row * p.ldx + at, p.k - at, v);
      store_blocks(v, lds + row * kp, lds + p.m * kp + row * sp, g, blocks, lane);
    }
    __syncthreads();
  }

  f32x4 acc[G];
#pragma unroll
  for (int g = 0; g < G; ++g) acc[g] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int kb0 = wave; kb0 < blocks; kb0 += U * kw) {
    if (kb0 != wave) load_weights(kb0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = kb0 + u * kw;
      if (kb < blocks) {
        const float s = byte_as_scale(ws[u]);
        bf16x8 wv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) wv[i] = widen8(wf[u][i >> 1][2 * (i & 1)], wf[u][i >> 1][2 * (i & 1) + 1], s);
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int64_t row = 16 * g + (lane & 15);
          i32x4 xf[2] = {};
          uint32_t xs = 127;
          if (row < p.m) {
            if constexpr (FUSED) {
              const uint8_t* q = lds + row * kp + kb * 128 + (lane >> 4) * 32;
              xf[0] = *(const i32x4*)q;
              xf[1] = *(const i32x4*)(q + 16);
              xs = lds[p.m * kp + row * sp + kb];
            } else {
              const uint8_t* q = p.a + row * p.lda + (int64_t)kb * 128 + (lane >> 4) * 32;
              xf[0] = *(const i32x4*)q;
              xf[1] = *(const i32x4*)(q + 16);
              xs = p.a_scales[row * p.lda_scales + kb];
            }
          }
          const float t = byte_as_scale(xs);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                wv[i], widen8(xf[i >> 1][2 * (i & 1)], xf[i >> 1][2 * (i & 1) + 1], t), acc[g], 0, 0, 0);
        }
      }
    }
  }
  // the wavefronts' sums, in order; a lane: row lane % 16, columns 4 (lane / 16) .. + 3
  if constexpr (FUSED) __syncthreads();
  f32x4* const sums = (f32x4*)lds;
#pragma unroll
  for (int g = 0; g < G; ++g) sums[(wave * G + g) * 64 + lane] = acc[g];
  __syncthreads();
  for (int g = wave; g < G; g += kw) {
    f32x4 t = sums[g * 64 + lane];
    for (int i = 1; i < kw; ++i) t += sums[(i * G + g) * 64 + lane];
    const int64_t row = 16 * g + (lane & 15);
    const int64_t c0 = n0 + 4 * (lane >> 4);
    if (row < p.m) {
      Out* const c = (Out*)p.c[grp] + row * p.ldc[grp] + c0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c0 + i < n) c[i] = (Out)t[i];
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

// A tile of BM x BN outputs, WM x WN wavefronts of 32 TI x 32 TJ.  A stage holds a block of k: A's BM
// rows and B's BN rows of 128 bytes, then a dword of each row's scales (the four blocks around this
// one).  The 16-byte chunk c of row r sits in slot c ^ ((r >> 1) & 7): the 16 lanes that a fragment
// read serves at a time (one chunk of 16 consecutive rows) then touch 16 different 16-byte
// banks.  A direct-to-LDS load fills 8 rows (1 KB).
template <int BM, int BN, int WM, int WN, int STAGES, bool EXACT, typename Out>
__global__ __launch_bounds__(WM * WN * 64) void product_kernel(const ProductArgs p) {
  constexpr int NW = WM * WN, TI = BM / WM / 32, TJ = BN / WN / 32;
  constexpr int LPW = (BM + BN) / 8 / NW;   // loads a wavefront and stage
  constexpr int SPW = (BM + BN) / NW;       // rows whose scales a wavefront fetches
  constexpr int SCALES = (BM + BN) * 128;   // where a stage's scales are
  constexpr int STAGE = (BM + BN) * 132;
  static_assert((BM / 8) % NW == 0 && (BN / 8) % NW == 0 && SPW <= 64 && BM % SPW == 0, "a wavefront's loads stay in one operand");
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  grouped(xcd_order(blockIdx.x, p.tiles_m * p.tiles_n), p.tiles_m, p.tiles_n, tm, tn);
  const int grp = tn < p.tiles_n0 ? 0 : 1;
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)(grp ? tn - p.tiles_n0 : tn) * BN;
  const int64_t n = p.n[grp];
  const int blocks = p.blocks;

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
  // this lane's row of scales
  const uint8_t* scale_row;
  {
    const int e = wave * SPW + (lane < SPW ? lane : 0);
    if (wave * SPW < BM) {
      const int64_t r = m0 + e < p.m ? m0 + e : p.m - 1;
      scale_row = p.a_scales + r * p.lda_scales;
    } else {
      const int64_t r = n0 + e - BM < n ? n0 + e - BM : n - 1;
      scale_row = p.b_scales[grp] + (r >> 7) * p.ldb_scales[grp];
    }
  }
  auto issue = [&](int kb, int slot) {
    uint8_t* const st = lds + slot * STAGE;
#pragma unroll
    for (int j = 0; j < LPW; ++j) {
      const uint8_t* base = (NW * j < BM / 8 ? a0 : b0) + (int64_t)kb * 128;
      __builtin_amdgcn_global_load_lds((const void*)(base + off[j]), (lds_void*)(st + (wave + NW * j) * 1024), 16, 0, 0);
    }
    if (lane < SPW)
      __builtin_amdgcn_global_load_lds((const void*)(scale_row + (kb & ~3)), (lds_void*)(st + SCALES + wave * SPW * 4), 4, 0, 0);
  };

  const int wm = wave / WN, wn = wave % WN;
  f32x16 acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (s < blocks) issue(s, s);
  int slot = 0;
  for (int kb = 0; kb < blocks; ++kb) {
    // this wavefront's part of block kb is in LDS and its reads of block kb - 1 are in registers; after the barrier,
    // every wavefront's are
    if (kb + STAGES - 1 <= blocks)
      wait_vm<(STAGES - 2) * (LPW + 1)>();
    else
      wait_vm<0>();
    wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    if (kb + STAGES - 1 < blocks) issue(kb + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
    const uint8_t* const st = lds + slot * STAGE;
    const int shift = (kb & 3) * 8;
    uint32_t sa[TI], sb[TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i) sa[i] = *(const uint32_t*)(st + SCALES + ((wm * TI + i) * 32 + (lane & 31)) * 4) >> shift;
#pragma unroll
    for (int j = 0; j < TJ; ++j) sb[j] = *(const uint32_t*)(st + SCALES + (BM + (wn * TJ + j) * 32 + (lane & 31)) * 4) >> shift;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      i32x8 fa[TI], fb[TJ];
      auto fragment = [&](int row) {
        const int c = h * 4 + (lane >> 5) * 2, x = (row >> 1) & 7;
        const i32x4 lo = *(const i32x4*)(st + row * 128 + (c ^ x) * 16);
        const i32x4 hi = *(const i32x4*)(st + row * 128 + ((c + 1) ^ x) * 16);
        return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      };
#pragma unroll
      for (int i = 0; i < TI; ++i) fa[i] = fragment((wm * TI + i) * 32 + (lane & 31));
#pragma unroll
      for (int j = 0; j < TJ; ++j) fb[j] = fragment(BM + (wn * TJ + j) * 32 + (lane & 31));
      if constexpr (!EXACT) {
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
          for (int j = 0; j < TJ; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[i], fb[j], acc[i][j], 0, 0, 0, (int)sa[i], 0, (int)sb[j]);
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          bf16x8 wa[TI], wb[TJ];
#pragma unroll
          for (int i = 0; i < TI; ++i) wa[i] = widen8(fa[i][2 * s], fa[i][2 * s + 1], byte_as_scale(sa[i] & 255u));
#pragma unroll
          for (int j = 0; j < TJ; ++j) wb[j] = widen8(fb[j][2 * s], fb[j][2 * s + 1], byte_as_scale(sb[j] & 255u));
#pragma unroll
          for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wa[i], wb[j], acc[i][j], 0, 0, 0);
        }
      }
    }
    slot = slot + 1 == STAGES ? 0 : slot + 1;
  }
  // D: lane l holds column l % 32 and rows 8 (r / 4) + 4 (l / 32) + r % 4 of its 32 x 32
  Out* const c = (Out*)p.c[grp];
  const int64_t ldc = p.ldc[grp];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j) {
      const int64_t col = n0 + (wn * TJ + j) * 32 + (lane & 31);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t row = m0 + (wm * TI + i) * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
        if (row < p.m && col < n) c[row * ldc + col] = (Out)acc[i][j][r];
      }
    }
}

// ---- host ----------------------------------------------------------------------------------------

constexpr int kFewRows = 32;     // rows of the few-row kernel
constexpr int kFusedRows = 4;    // rows whose blocks it takes itself
constexpr int64_t kFusedBytes = 48 << 10;

template <int BM, int BN, int WM, int WN, int STAGES, bool EXACT, typename Out>
int launch_tiles(ProductArgs p, hipStream_t st) {
  p.tiles_m = (int)((p.m + BM - 1) / BM);
  p.tiles_n0 = (int)((p.n[0] + BN - 1) / BN);
  p.tiles_n = p.tiles_n0 + (int)((p.n[1] + BN - 1) / BN);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  if (tiles > INT32_MAX) return set_error(EG_ERR_UNSUPPORTED, "fp8 product: %lld tiles", (long long)tiles);
  const auto kernel = product_kernel<BM, BN, WM, WN, STAGES, EXACT, Out>;
  constexpr int bytes = STAGES * (BM + BN) * 132;
  EG_CHECK_HIP(allow_lds((const void*)kernel, bytes));
  kernel<<<(unsigned)tiles, WM * WN * 64, bytes, st>>>(p);
  return launch_status("product_kernel");
}

template <bool EXACT, typename Out>
int launch_product(const ProductArgs& p, hipStream_t st) {
  auto tiles = [&](int bm, int bn) { return ((p.m + bm - 1) / bm) * ((p.n[0] + bn - 1) / bn + (p.n[1] + bn - 1) / bn); };
  if (tiles(256, 256) >= 128) return launch_tiles<256, 256, 2, 4, 2, EXACT, Out>(p, st);
  if (tiles(128, 128) >= 256) return launch_tiles<128, 128, 2, 2, 2, EXACT, Out>(p, st);
  return launch_tiles<64, 64, 2, 2, 4, EXACT, Out>(p, st);
}

template <int G, bool FUSED, typename X>
int launch_few(ProductArgs p, int32_t dtype, hipStream_t st) {
  p.tiles_n0 = (int)((p.n[0] + 15) / 16);
  const int64_t tiles = p.tiles_n0 + (p.n[1] + 15) / 16;
  // wavefronts a workgroup: about four blocks of k each, so that all their loads are in flight at once
  const int kw = p.blocks <= 4 ? 1 : p.blocks <= 8 ? 2 : p.blocks <= 24 ? 4 : p.blocks <= 48 ? 8 : 16;
  const int64_t a_bytes = FUSED ? p.m * (p.blocks * 128 + ((p.blocks + 3) & ~3)) : 0;
  const int64_t bytes = a_bytes > kw * G * 1024 ? a_bytes : kw * G * 1024;
  return with_type(dtype, [&](auto out) {
    few_rows_kernel<G, FUSED, X, decltype(out)><<<(unsigned)tiles, kw * 64, bytes, st>>>(p);
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

int run_product(const ProductArgs& p, int32_t dtype, hipStream_t st) {
  if (p.m == 0 || p.n[0] == 0) return EG_OK;
  if (p.m <= 16) return launch_few<1, false, float>(p, dtype, st);
  if (p.m <= kFewRows) return launch_few<2, false, float>(p, dtype, st);
  switch (dtype) {
    case EG_DTYPE_F32: return launch_product<true, float>(p, st);
    case EG_DTYPE_BF16: return launch_product<false, __bf16>(p, st);
    default: return launch_product<false, _Float16>(p, st);
  }
}

bool fused(int64_t m, int64_t k) {
  const int64_t blocks = (k + 127) / 128;
  return m <= kFusedRows && m * (blocks * 128 + blocks + 3) <= kFusedBytes;
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
  EG_CHECK_ARG((units + 3) / 4 <= INT32_MAX, "fp8_quantize: %lld x %lld is too large", (long long)out->rows, (long long)out->k);
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
  EG_CHECK_ARG((count + 255) / 256 <= INT32_MAX, "fp8_dequantize: %lld x %lld is too large", (long long)m->rows, (long long)m->k);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    dequantize_kernel<T><<<(unsigned)((count + 255) / 256), 256, 0, (hipStream_t)stream>>>(
        (const uint8_t*)m->q, m->stride, m->scales, m->scale_stride, m->block_rows == 128 ? 7 : 0, m->rows, (int)m->k, (T*)out, row_stride);
    return launch_status("dequantize_kernel");
  });
}

int eg_fp8_product(const eg_fp8_matrix* a, const eg_fp8_matrix* b, const eg_fp8_matrix* b2, void* c, int64_t ldc, void* c2,
                   int64_t ldc2, int32_t dtype, void* stream) {
  if (const int rc = check_fp8(a, 1, "a"); rc != EG_OK) return rc;
  ProductArgs p;
  if (const int rc = check_product(b, b2, c, ldc, c2, ldc2, dtype, a->rows, a->k, &p); rc != EG_OK) return rc;
  p.a = (const uint8_t*)a->q;
  p.a_scales = a->scales;
  p.lda = a->stride;
  p.lda_scales = a->scale_stride;
  return run_product(p, dtype, (hipStream_t)stream);
}

int64_t eg_fp8_linear_workspace_size(int64_t m, int64_t k) {
  if (m < 0 || m >= (1ll << 31) || k < 1 || k > (1 << 22)) return -1;
  if (fused(m, k)) return 0;
  const int64_t blocks = (k + 127) / 128;
  return m * (blocks * 128 + (blocks + 3) / 4 * 4);
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
  if (fused(m, b->k)) {
    p.x = x;
    p.ldx = x_stride;
    return with_type(x_dtype, [&](auto t) {
      return launch_few<1, true, decltype(t)>(p, dtype, (hipStream_t)stream);
    });
  }
  const int64_t need = eg_fp8_linear_workspace_size(m, b->k);
  if (workspace_bytes < need)
    return set_error(EG_ERR_WORKSPACE, "fp8_linear needs %lld bytes of workspace, got %lld", (long long)need, (long long)workspace_bytes);
  EG_CHECK_ARG(workspace != nullptr && (uintptr_t)workspace % 16 == 0, "fp8_linear: the workspace must be 16-byte aligned");
  const int64_t kp = (int64_t)p.blocks * 128;
  const eg_fp8_matrix a = {workspace, (uint8_t*)workspace + m * kp, m, b->k, kp, (p.blocks + 3) / 4 * 4, 1};
  if (const int rc = eg_fp8_quantize(x, x_dtype, x_stride, &a, stream); rc != EG_OK) return rc;
  return eg_fp8_product(&a, b, b2, c, ldc, c2, ldc2, dtype, stream);
}

}  // extern "C"
