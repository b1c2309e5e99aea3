// Losses of next-token logits and the gradient of the logits: what a descent's
// d_out comes from (engraft/replica/distill.py:283-325 holds the reference's
// own loss, a torch expression over log_softmax).
//
// With z a row of n_vocab logits, c = log2(e) / temperature and M = max z,
//
//   S = sum_j 2^(c (z_j - M)),   lp = ln2 c (z_t - M) - ln S,
//   d_j = g ([j == t] - 2^(c (z_j - M)) / S) / temperature,   g = dL / d lp:
//
// a pass over the logits gives M and S of every row (row_stats_kernel, the running
// maximum and sum of each thread joined in a fixed order), then the rows' lp, the loss and
// every row's g are found (logprobs_finish, a thread a row; policy_finish and preference_finish,
// one workgroup over all rows), and a second pass reads the logits and writes d
// (logits_grad_kernel; policy_few_kernel and preference_few_kernel do the last two in one
// launch).  The differences z - M are taken
// before the multiplication by c, so a row of the type's lowest value gives a
// uniform softmax and -inf gives exact zeros.  A row whose target is negative is left
// out: its logits are not read (NaN there is harmless), its lp is 0 and its gradient
// zero.  A target beyond the vocabulary gives NaN (lp and gradient), never a
// read out of range.  A term whose coefficient is zero (kl_coef, label_smoothing) adds nothing,
// however large it is.
//
// Bound by HBM, 2,047 x 151,936 bf16 of which 30 % of the rows are left out: the statistics
// read 435 MB in 79 us (5.5 TB/s; a large copy moves 6.5), the gradient pass reads them
// again and writes 622 MB in 173 us (6.1 TB/s, the rows read last first, so that some are still
// in the Infinity Cache: first to last 205 us).  The policy loss, whose g needs its own row
// alone, does both in one workgroup a row and reads the logits once: 202 us for 1,057 MB.
// A thread keeps four 16-byte loads in flight (up to 20 where the row is held); 8 to 18 made no difference.
//
// A row's sum is fp32: a thread adds the terms of a chunk's group (16 or 32) in pairs, then the groups one by
// one (v / 32,768 of them for 16-bit logits in a workgroup of 1,024: 5 at 151,936).  Over 151,936 bf16 logits a
// log-probability is 7e-8 off (deviation; torch's fp32 form 6e-8) with a mean of -9e-8 at temperature 1, which is the
// rounding of c: its second half as one more multiplication a logit took the mean to -5e-9 and the
// policy loss from 207 to 213 us.  What one thread adds of a row (lp, ratio, KL, weights) and sums over rows
// and sequences are fp64; no floating atomics, so a call gives the same bits every time.
#include "eg_common.h"
#include "eg_overlap.h"

#include <algorithm>


namespace eg {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;

// 16 bytes at any element's alignment: rows of an odd vocabulary start anywhere
// (global accesses need no alignment beyond the element's on gfx950).
struct __attribute__((packed, aligned(2))) Chunk {
  uint32_t w[4];
};

typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));

// Past the caches: gradients, which nothing here reads again (written through them they push out the
// logits that the gradient pass reads a second time: 2,047 rows of 151,936 bf16, preference
// loss 268 us against 319), and logits that are read once.
__device__ inline Chunk stream_in(const void* p) {
  return __builtin_bit_cast(Chunk, __builtin_nontemporal_load((const u32x4u*)p));
}
__device__ inline void stream_out(void* p, const Chunk& c) {
  const u32x4u v = {c.w[0], c.w[1], c.w[2], c.w[3]};
  __builtin_nontemporal_store(v, (u32x4u*)p);
}

template <typename T>
struct Logit;  // values per chunk, chunk -> fp32, fp32 -> chunk

template <>
struct Logit<float> {
  static constexpr int kVec = 4;
  static __device__ inline void unpack(const Chunk& c, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __builtin_bit_cast(float, c.w[i]);
  }
  static __device__ inline Chunk pack(const float (&f)[4]) {
    Chunk c;
#pragma unroll
    for (int i = 0; i < 4; ++i) c.w[i] = __builtin_bit_cast(uint32_t, f[i]);
    return c;
  }
};

template <>
struct Logit<__bf16> {
  static constexpr int kVec = 8;
  static __device__ inline void unpack(const Chunk& c, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __builtin_bit_cast(float, c.w[i] << 16);
      f[2 * i + 1] = __builtin_bit_cast(float, c.w[i] & 0xffff0000u);
    }
  }
  static __device__ inline Chunk pack(const float (&f)[8]) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    Chunk c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const pair p = {(__bf16)f[2 * i], (__bf16)f[2 * i + 1]};
      c.w[i] = __builtin_bit_cast(uint32_t, p);
    }
    return c;
  }
};

template <>
struct Logit<_Float16> {
  static constexpr int kVec = 8;
  typedef _Float16 pair __attribute__((ext_vector_type(2)));
  static __device__ inline void unpack(const Chunk& c, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const pair p = __builtin_bit_cast(pair, c.w[i]);
      f[2 * i] = (float)p[0];
      f[2 * i + 1] = (float)p[1];
    }
  }
  static __device__ inline Chunk pack(const float (&f)[8]) {
    Chunk c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const pair p = {(_Float16)f[2 * i], (_Float16)f[2 * i + 1]};
      c.w[i] = __builtin_bit_cast(uint32_t, p);
    }
    return c;
  }
};

// What every kernel here knows of the rows.
struct Rows {
  const void* z;
  int64_t n, stride;  // rows, elements from one to the next
  const void* targets;
  int32_t v;
  int targets32;      // targets are int32, otherwise int64
  float c;            // log2(e) / temperature
  double inv_temp;
};

__device__ inline int64_t target_of(const Rows& r, int64_t i) {
  return r.targets32 ? (int64_t)((const int32_t*)r.targets)[i] : ((const int64_t*)r.targets)[i];
}

// The running maximum and sum of 2^(c (z - m)).
struct Stat {
  float m, s;
};

__device__ inline float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ inline Stat join(const Stat& a, const Stat& b, float c) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * pow2((a.m - m) * c) + b.s * pow2((b.m - m) * c)};
}

// The larger of three, NaNs dropped (they come back through the sum).
__device__ inline float max3(float a, float b, float x) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(x));
  return r;
}

template <typename T, int K>
__device__ inline void add_chunks(const Chunk (&q)[K], float c, Stat& st) {
  constexpr int VEC = Logit<T>::kVec;
  float f[K][VEC];
  float m = st.m;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    Logit<T>::unpack(q[k], f[k]);
#pragma unroll
    for (int i = 0; i < VEC; i += 2) m = max3(m, f[k][i], f[k][i + 1]);
  }
  // a chunk's terms by themselves first, in pairs: added to the row's largest one by one, each would lose
  // what is below that one's last place
  float s = st.s * pow2((st.m - m) * c);
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[k][i] = pow2((f[k][i] - m) * c);
#pragma unroll
    for (int o = VEC / 2; o >= 1; o /= 2)
#pragma unroll
      for (int i = 0; i < o; ++i) f[k][i] += f[k][i + o];
  }
#pragma unroll
  for (int o = K / 2; o >= 1; o /= 2)
#pragma unroll
    for (int k = 0; k < o; ++k) f[k][0] += f[k + o][0];
  st = {m, s + f[0][0]};
}

// A thread's statistics of elements [e0, e1) of a row, e0 a multiple of the chunk.
template <typename T, int THREADS>
__device__ inline Stat thread_stats(const T* row, int e0, int e1, float c, Stat st = {kLowest, 0.0f}) {
  constexpr int VEC = Logit<T>::kVec, K = 4;
  int e = e0 + (int)threadIdx.x * VEC;
  for (; e + (K - 1) * THREADS * VEC + VEC <= e1; e += K * THREADS * VEC) {
    Chunk q[K];
#pragma unroll
    for (int k = 0; k < K; ++k) q[k] = *(const Chunk*)(row + e + k * THREADS * VEC);
    add_chunks<T, K>(q, c, st);
  }
  for (; e + VEC <= e1; e += THREADS * VEC) {
    const Chunk q[1] = {*(const Chunk*)(row + e)};
    add_chunks<T, 1>(q, c, st);
  }
  for (; e < e1; ++e) {  // the one thread whose chunk passes the end
    const float f = (float)row[e];
    const float m = fmaxf(st.m, f);
    st = {m, st.s * pow2((st.m - m) * c) + pow2((f - m) * c)};
  }
  return st;
}

template <int THREADS>
__device__ inline Stat block_stats(Stat st, float c, Stat* red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) st = join(st, Stat{__shfl_xor(st.m, o), __shfl_xor(st.s, o)}, c);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) red[wave] = st;
  __syncthreads();
  st = red[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) st = join(st, red[w], c);
  return st;
}

// Elements [e0, e1) of part `p` of a row of v elements in `parts` parts.
__device__ inline void part_range(int v, int parts, int part_len, int p, int& e0, int& e1) {
  e0 = p * part_len;
  e1 = p + 1 == parts ? v : e0 + part_len;
}

// In 64 bits: a loss is a sum of terms that nearly cancel, and an fp32 lp's rounding (half a
// unit in the last place, 2^-21 at -10) would be most of its error.
__device__ inline double logprob_of(const Rows& r, float z_below_m, float s) {
  return (double)z_below_m * r.inv_temp - log((double)s);
}

// The same where every thread of a workgroup finds it, for the row's g: ln S to about 2^-23 absolute,
// fp32's, corrected once by S e^-y - 1.
__device__ inline double quick_logprob_of(const Rows& r, float z_below_m, float s) {
  const float y = logf(s);
  return (double)z_below_m * r.inv_temp - ((double)y + (double)fmaf(s, expf(-y), -1.0f));
}

// z_t - M, NaN for a target beyond the vocabulary.
template <typename T>
__device__ inline float z_below_m(const Rows& r, int64_t i, int64_t t, float m) {
  return t < r.v ? (float)((const T*)r.z)[i * r.stride + t] - m : __builtin_nanf("");
}

// A row that a workgroup did alone: its log-probability too, in either type.
struct WholeRow {
  float* lp;
  double* lp64;
};

// Grid (parts, rows): the statistics of a part of a row -> stats[row][part] (where kept).
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void row_stats_kernel(const Rows r, int parts, int part_len, Stat* stats,
                                                            const WholeRow whole) {
  __shared__ Stat red[THREADS / 64];
  const int64_t i = blockIdx.y + (int64_t)gridDim.y * blockIdx.z;
  if (i >= r.n) return;
  const int64_t t = target_of(r, i);
  if (t < 0) {
    if (threadIdx.x == 0 && whole.lp != nullptr) whole.lp[i] = 0.0f;
    if (threadIdx.x == 0 && whole.lp64 != nullptr) whole.lp64[i] = 0.0;
    return;
  }
  int e0, e1;
  part_range(r.v, parts, part_len, (int)blockIdx.x, e0, e1);
  Stat st = thread_stats<T, THREADS>((const T*)r.z + i * r.stride, e0, e1, r.c);
  st = block_stats<THREADS>(st, r.c, red);
  if (threadIdx.x != 0) return;
  if (stats != nullptr) stats[i * parts + blockIdx.x] = st;
  if (whole.lp != nullptr || whole.lp64 != nullptr) {
    const double lp = logprob_of(r, z_below_m<T>(r, i, t, st.m), st.s);
    if (whole.lp != nullptr) whole.lp[i] = (float)lp;
    if (whole.lp64 != nullptr) whole.lp64[i] = lp;
  }
}

// Segment of a row: a value outside [0, n) for none.
struct Segments {
  const void* ids;
  int64_t n;
  int ids32;
};

__device__ inline int64_t segment_of(const Segments& s, int64_t i) {
  return s.ids32 ? (int64_t)((const int32_t*)s.ids)[i] : ((const int64_t*)s.ids)[i];
}

// Elements [e0, e1) of a row that is left out.
template <typename T, int THREADS>
__device__ inline void write_zeros(T* out, int e0, int e1) {
  constexpr int VEC = Logit<T>::kVec;
  int e = e0 + (int)threadIdx.x * VEC;
  const Chunk zero = {{0, 0, 0, 0}};
  for (; e + VEC <= e1; e += THREADS * VEC) stream_out(out + e, zero);
  for (; e < e1; ++e) out[e] = (T)0.0f;
}

// What the gradient pass needs of a row: g (dL / d lp), M and 1 / S.
struct RowState {
  float g, m, inv_s;
};

// Elements [e0, e1) of g ([j == t] - 2^(c (z_j - m)) inv_s); f_t is z_t, read before anything
// is written (out may be the row itself).  The row's state is asked for once the first loads are on
// their way (by every thread: it may synchronise).
template <typename T, int THREADS, typename State>
__device__ inline void write_gradient(const T* row, T* out, int e0, int e1, int64_t t, float f_t, float c, State&& state) {
  constexpr int VEC = Logit<T>::kVec, K = 4, NEXT = THREADS * VEC;
  int e = e0 + (int)threadIdx.x * VEC;
  Chunk q[K];
  auto load = [&] {
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (e + j * NEXT + VEC <= e1) q[j] = *(const Chunk*)(row + e + j * NEXT);
  };
  load();
  const RowState st = state();
  const float m = st.m, k = -st.g * st.inv_s;
  auto value = [&](float f) { return k * pow2((f - m) * c); };
  auto store = [&](int at, const Chunk& chunk) {
    float f[VEC];
    Logit<T>::unpack(chunk, f);
#pragma unroll
    for (int x = 0; x < VEC; ++x) f[x] = value(f[x]);
    stream_out(out + at, Logit<T>::pack(f));
  };
  for (; e + (K - 1) * NEXT + VEC <= e1; load()) {
#pragma unroll
    for (int j = 0; j < K; ++j) store(e + j * NEXT, q[j]);
    e += K * NEXT;
  }
#pragma unroll
  for (int j = 0; j < K - 1; ++j)
    if (e + j * NEXT + VEC <= e1) store(e + j * NEXT, q[j]);
  // the row's incomplete chunk, by the thread whose turn it is
  const int whole = e0 + (e1 - e0) / VEC * VEC;
  if ((whole - e0) / VEC % THREADS == (int)threadIdx.x)
    for (int x = whole; x < e1; ++x) out[x] = (T)value((float)row[x]);
  // the target's element again, by the thread that wrote it
  if (t >= e0 && t < e1 && (int)((t - e0) / VEC) % THREADS == (int)threadIdx.x) out[t] = (T)(st.g + value(f_t));
}

// Grid (parts, rows): a part of a row's gradient; scale holds 1 / temperature.  g is the state's, or
// with d_seq that of the row's segment.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void logits_grad_kernel(const Rows r, int parts, int part_len,
                                                              const RowState* state, const Segments seg,
                                                              const float* d_seq, const float* upstream, float scale,
                                                              T* d, int64_t d_stride) {
  const int64_t i = r.n - 1 - (blockIdx.y + (int64_t)gridDim.y * blockIdx.z);  // the rows read last first
  if (i < 0) return;
  int e0, e1;
  part_range(r.v, parts, part_len, (int)blockIdx.x, e0, e1);
  const int64_t t = target_of(r, i);
  T* out = d + i * d_stride;
  if (t < 0) {
    write_zeros<T, THREADS>(out, e0, e1);
    return;
  }
  const T* row = (const T*)r.z + i * r.stride;
  const float f_t = t >= e0 && t < e1 ? (float)row[t] : 0.0f;
  if (row == out) __syncthreads();  // everyone has read f_t
  write_gradient<T, THREADS>(row, out, e0, e1, t, f_t, r.c, [&] {
    RowState st = state[i];
    if (d_seq != nullptr) {
      const int64_t s = segment_of(seg, i);
      st.g = s >= 0 && s < seg.n ? d_seq[s] : 0.0f;
    }
    st.g *= upstream != nullptr ? scale * *upstream : scale;
    return st;
  });
}

// ---- one workgroup over all rows ------------------------------------------------------------

constexpr int kFinish = 1024;
constexpr int64_t kFewRows = 256, kFewSegments = 2048;  // of the few-row kernels: a row a thread, segments in LDS

template <int THREADS>
__device__ inline double block_sum64(double x, double* red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < THREADS / 64; ++w) t += red[w];
  return t;
}

// A row's statistics joined over its parts, in order, eight loads at a time.
__device__ inline Stat row_stat(const Stat* stats, int64_t i, int parts, float c) {
  const Stat* at = stats + i * parts;
  Stat st = at[0];
  for (int p = 1; p < parts; p += 8) {
    Stat q[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = at[min(p + k, parts - 1)];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (p + k < parts) st = join(st, q[k], c);
  }
  return st;
}

template <typename T>
__global__ __launch_bounds__(256) void logprobs_finish(const Rows r, int parts, const Stat* stats, float* lp) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= r.n) return;
  const int64_t t = target_of(r, i);
  float x = 0.0f;
  if (t >= 0) {
    const Stat st = row_stat(stats, i, parts, r.c);
    x = (float)logprob_of(r, z_below_m<T>(r, i, t, st.m), st.s);
  }
  lp[i] = x;
}

struct Policy {
  const float* advantages;
  const float* old_lp;  // NULL: the policy's own (a ratio of 1)
  const float* ref_lp;  // NULL: no KL term
  Segments seg;         // mean over segments of the mean over their tokens
  int reduction;        // eg_reduction
  float clip_low, clip_high, kl_coef;
};

// r A and clamp(r) A.
template <typename Real>
struct Surrogate {
  Real free, held;
};

template <typename Real>
__device__ inline Surrogate<Real> surrogate(const Policy& p, Real ratio, Real advantage) {
  const Real lo = (Real)1 - (Real)p.clip_low, hi = (Real)1 + (Real)p.clip_high;
  const Real held = ratio < lo ? lo : ratio > hi ? hi : ratio;  // NaN stays
  return {ratio * advantage, held * advantage};
}

// dL / d lp of row i, of weight w: differences of log-probabilities in 64 bits, their exponentials in fp32
// (a gradient's terms do not cancel), few enough operations for every thread of a workgroup to do.
__device__ inline float policy_g(const Policy& p, int64_t i, double lp, float w) {
  const float ratio = p.old_lp != nullptr ? expf((float)(lp - (double)p.old_lp[i])) : (lp == lp ? 1.0f : (float)lp);
  const Surrogate<float> q = surrogate(p, ratio, p.advantages[i]);
  float g = q.free > q.held ? 0.0f : -q.free;  // NaN stays
  // a term of no weight may be infinite
  if (p.ref_lp != nullptr && p.kl_coef != 0.0f) g -= p.kl_coef * expm1f((float)((double)p.ref_lp[i] - lp));
  return w * g;
}

// What row i, of weight w, adds to the loss, the KL term and the clipped share, all in 64 bits.
__device__ inline void add_policy_terms(const Policy& p, int64_t i, double lp, double w, double (&sum)[3]) {
  const double ratio = p.old_lp != nullptr ? exp(lp - (double)p.old_lp[i]) : (lp == lp ? 1.0 : lp);
  const Surrogate<double> q = surrogate(p, ratio, (double)p.advantages[i]);
  double loss = q.free > q.held ? -q.held : -q.free;  // NaN stays
  if (p.ref_lp != nullptr) {
    const double diff = (double)p.ref_lp[i] - lp, up = expm1(diff);
    const double kl = up == (double)INFINITY ? up : up - diff;  // diff may be infinite too
    if (p.kl_coef != 0.0f) loss += (double)p.kl_coef * kl;
    sum[1] += w * kl;
  }
  sum[0] += w * loss;
  if (q.free > q.held) sum[2] += w;
}

// One workgroup: the weight of a row with a target, weights[segment] by segment, otherwise
// weights[0].  Counts are kept in the same place, the first half of a weight's.
template <int THREADS>
__device__ inline void policy_weights(const Rows& r, const Policy& p, double* weights) {
  __shared__ int total;
  const int tid = threadIdx.x, lane = tid & 63;
  int* counts = (int*)weights;
  const bool by_segment = p.reduction == EG_REDUCE_SEQUENCE;
  if (tid == 0) total = 0;
  if (by_segment)
    for (int64_t s = tid; s < p.seg.n; s += THREADS) counts[2 * s] = 0;
  __syncthreads();
  int some = 0;
  if (p.reduction == EG_REDUCE_TOKEN)
#pragma unroll 4
    for (int64_t i = tid; i < r.n; i += THREADS) some += target_of(r, i) >= 0;
  if (by_segment)
    for (int64_t i = tid; i < r.n; i += THREADS) {
      const bool in = target_of(r, i) >= 0;
      const int64_t s = segment_of(p.seg, i);
      // one addition for the rows of a wavefront that share a segment
      uint64_t left = __ballot(in && s >= 0 && s < p.seg.n);
      while (left != 0) {
        const int64_t one = __shfl(s, __ffsll((unsigned long long)left) - 1);
        const uint64_t same = __ballot(s == one) & left;
        if (lane == __ffsll((unsigned long long)same) - 1) atomicAdd(counts + 2 * one, __popcll(same));
        left &= ~same;
      }
    }
  __syncthreads();
  if (by_segment)
    for (int64_t s = tid; s < p.seg.n; s += THREADS) some += __hip_atomic_load(counts + 2 * s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) > 0;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) some += __shfl_xor(some, o);
  if (lane == 0) atomicAdd(&total, some);
  __syncthreads();
  const double all = p.reduction == EG_REDUCE_SUM ? 1.0 : 1.0 / (double)max(total, 1);
  if (!by_segment) {
    if (tid == 0) weights[0] = all;
  } else {
    for (int64_t s = tid; s < p.seg.n; s += THREADS) {
      const int c = __hip_atomic_load(counts + 2 * s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      weights[s] = all / (double)max(c, 1);
    }
  }
}

__device__ inline double weight_of(const Policy& p, int64_t i, const double* weights) {
  if (p.reduction != EG_REDUCE_SEQUENCE) return weights[0];
  const int64_t s = segment_of(p.seg, i);
  return s >= 0 && s < p.seg.n ? weights[s] : 0.0;
}

// The rows from tid on, THREADS apart within [i0, i1): lp, state and the thread's sums.  DONE: the
// gradient is written (perhaps over the logits), z_t - M is in the place of the state's g.
template <typename T, int THREADS, bool DONE>
__device__ inline void policy_rows(const Rows& r, const Policy& p, int64_t i0, int64_t i1, int parts,
                                   const Stat* stats, const double* weights, float* lp_out, RowState* state,
                                   double (&sum)[3]) {
  for (int64_t i = i0 + threadIdx.x; i < i1; i += THREADS) {
    const int64_t t = target_of(r, i);
    double lp = 0.0;
    RowState st = {0.0f, 0.0f, 0.0f};
    if (t >= 0) {
      const Stat rs = row_stat(stats, i, parts, r.c);
      const float below = DONE ? state[i].g : z_below_m<T>(r, i, t, rs.m);
      lp = logprob_of(r, below, rs.s);
      const double w = weight_of(p, i, weights);
      st = {0.0f, rs.m, 1.0f / rs.s};
      if (w != 0.0) {
        add_policy_terms(p, i, lp, w, sum);
        // with the bits of the kernels that find g by themselves
        if (!DONE && state != nullptr) st.g = policy_g(p, i, quick_logprob_of(r, below, rs.s), (float)w);
      }
    }
    lp_out[i] = (float)lp;
    if (!DONE && state != nullptr) state[i] = st;
  }
}

// One workgroup over all rows: weights, lp, state (where kept); sums[3] = loss, KL, clipped share.
template <typename T, int THREADS>
__device__ inline void policy_all(const Rows& r, const Policy& p, int parts, const Stat* stats, double* weights,
                                  float* lp_out, RowState* state, float* sums) {
  __shared__ double red[THREADS / 64];
  policy_weights<THREADS>(r, p, weights);
  __syncthreads();
  double sum[3] = {0.0, 0.0, 0.0};
  policy_rows<T, THREADS, false>(r, p, 0, r.n, parts, stats, weights, lp_out, state, sum);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const double x = block_sum64<THREADS>(sum[k], red);
    if (threadIdx.x == 0) sums[k] = (float)x;
  }
}

template <typename T>
__global__ __launch_bounds__(kFinish) void policy_finish(const Rows r, const Policy p, int parts, const Stat* stats,
                                                         double* weights, float* lp_out, RowState* state, float* sums) {
  policy_all<T, kFinish>(r, p, parts, stats, weights, lp_out, state, sums);
}

// Few rows in parts: every workgroup of the gradient finds its row's weight and g for itself, while
// its logits are on their way, and one more does what policy_finish does: two launches for three
// (bf16 rows of 151936 logits: 4 rows 11.2 us for 13.7, 90 rows 22.1 for 25.3, 250 rows 40.6 for 45.7).  Grid (parts, rows + 1); the gradient is not in the logits' place.  Held to 64
// registers of the 113 that the 64-bit terms ask for: 37 rows of f32 18 to 20 us, as with fp32 terms.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, 8) void policy_few_kernel(const Rows r, const Policy p, int parts, int part_len,
                                                             const Stat* stats, float* lp_out, float* sums, float scale,
                                                             T* d, int64_t d_stride) {
  __shared__ double weights[kFewSegments];
  const int64_t i = (int64_t)blockIdx.y - 1;
  if (i < 0) {
    if (blockIdx.x == 0) policy_all<T, THREADS>(r, p, parts, stats, weights, lp_out, nullptr, sums);
    return;
  }
  int e0, e1;
  part_range(r.v, parts, part_len, (int)blockIdx.x, e0, e1);
  const int64_t t = target_of(r, i);
  T* out = d + i * d_stride;
  if (t < 0) {
    write_zeros<T, THREADS>(out, e0, e1);
    return;
  }
  const T* row = (const T*)r.z + i * r.stride;
  const float f_t = t < r.v ? (float)row[t] : __builtin_nanf("");
  write_gradient<T, THREADS>(row, out, e0, e1, t, f_t, r.c, [&] {
    const Stat st = row_stat(stats, i, parts, r.c);
    const double lp = quick_logprob_of(r, f_t - st.m, st.s);
    const float g1 = policy_g(p, i, lp, 1.0f);
    policy_weights<THREADS>(r, p, weights);
    __syncthreads();
    const float w = (float)weight_of(p, i, weights);
    return RowState{(w != 0.0f ? w * g1 : 0.0f) * scale, st.m, 1.0f / st.s};
  });
}

// Many rows: the weights first,
__global__ __launch_bounds__(kFinish) void policy_weights_kernel(const Rows r, const Policy p, double* weights,
                                                                 int* finished) {
  if (threadIdx.x == 0) *finished = 0;
  policy_weights<kFinish>(r, p, weights);
}

// then a workgroup a row, its statistics and its gradient: the second reading of the row (300 KB
// of a 150,000-word vocabulary in bf16) comes from the caches,
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void policy_row_kernel(const Rows r, const Policy p, const double* weights,
                                                             Stat* stats, RowState* state, float scale, T* d,
                                                             int64_t d_stride) {
  __shared__ Stat red[THREADS / 64];
  const int64_t i = blockIdx.y + (int64_t)gridDim.y * blockIdx.z;
  if (i >= r.n) return;
  const int64_t t = target_of(r, i);
  T* out = d + i * d_stride;
  if (t < 0) {
    write_zeros<T, THREADS>(out, 0, r.v);
    return;
  }
  const T* row = (const T*)r.z + i * r.stride;
  const float f_t = t < r.v ? (float)row[t] : __builtin_nanf("");
  Stat st = thread_stats<T, THREADS>(row, 0, r.v, r.c);
  st = block_stats<THREADS>(st, r.c, red);
  if (threadIdx.x == 0) {
    stats[i] = st;
    state[i].g = f_t - st.m;
  }
  const float w = (float)weight_of(p, i, weights);
  const float g = w != 0.0f ? policy_g(p, i, quick_logprob_of(r, f_t - st.m, st.s), w) : 0.0f;
  write_gradient<T, THREADS>(row, out, 0, r.v, t, f_t, r.c, [&] { return RowState{g * scale, st.m, 1.0f / st.s}; });
}

// or, of longer rows, with the first NV chunks a thread held in registers from the one to the other
// (16 KB a chunk of 1,024 threads: NV 20 is a whole CU's and holds all of 151,936 bf16),
template <typename T, int NV>
__global__ __launch_bounds__(1024) void policy_held_kernel(const Rows r, const Policy p, const double* weights,
                                                                 Stat* stats, RowState* state, float scale, T* d,
                                                                 int64_t d_stride) {
  constexpr int THREADS = 1024, VEC = Logit<T>::kVec, STRIDE = THREADS * VEC, K = 4;
  static_assert(NV % K == 0, "whole groups");
  __shared__ Stat red[THREADS / 64];
  const int64_t i = blockIdx.y + (int64_t)gridDim.y * blockIdx.z;
  if (i >= r.n) return;
  const int64_t t = target_of(r, i);
  T* out = d + i * d_stride;
  if (t < 0) {
    write_zeros<T, THREADS>(out, 0, r.v);
    return;
  }
  const T* row = (const T*)r.z + i * r.stride;
  const float f_t = t < r.v ? (float)row[t] : __builtin_nanf("");
  // held chunks past the row's end re-read its last whole one and are left out below
  const int e0 = (int)threadIdx.x * VEC, whole = r.v / VEC * VEC;
  Chunk q[NV / K][K];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const uint32_t at = (uint32_t)min(e0 + k * STRIDE, whole - VEC) * (uint32_t)sizeof(T);
    q[k / K][k % K] = stream_in((const char*)row + at);
  }
  // in thread_stats' order, so with its bits
  Stat st = {kLowest, 0.0f};
#pragma unroll
  for (int k = 0; k < NV; k += K) {
    if (e0 + (k + K - 1) * STRIDE + VEC <= r.v) {
      add_chunks<T, K>(q[k / K], r.c, st);
    } else {
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (e0 + (k + j) * STRIDE + VEC <= r.v) {
          const Chunk one[1] = {q[k / K][j]};
          add_chunks<T, 1>(one, r.c, st);
        }
    }
  }
  st = thread_stats<T, THREADS>(row, NV * STRIDE, r.v, r.c, st);
  // the incomplete last chunk of a row that ends among the held ones
  const bool has_tail = whole < NV * STRIDE && (whole - e0) % STRIDE == 0 && whole >= e0;
  if (has_tail)
    for (int e = whole; e < r.v; ++e) {
      const float f = (float)row[e], m = fmaxf(st.m, f);
      st = {m, st.s * pow2((st.m - m) * r.c) + pow2((f - m) * r.c)};
    }
  st = block_stats<THREADS>(st, r.c, red);
  if (threadIdx.x == 0) {
    stats[i] = st;
    state[i].g = f_t - st.m;
  }
  const float w = (float)weight_of(p, i, weights);
  const float g = (w != 0.0f ? policy_g(p, i, quick_logprob_of(r, f_t - st.m, st.s), w) : 0.0f) * scale;
  const float inv_s = 1.0f / st.s, k1 = -g * inv_s, c = r.c, m = st.m;
  auto value = [&](float f) { return k1 * pow2((f - m) * c); };
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (e0 + k * STRIDE + VEC > r.v) continue;
    // opaque: the values unpacked for the statistics are not kept (they would spill)
    Chunk held = q[k / K][k % K];
#pragma unroll
    for (int x = 0; x < 4; ++x) asm volatile("" : "+v"(held.w[x]));
    float f[VEC];
    Logit<T>::unpack(held, f);
#pragma unroll
    for (int x = 0; x < VEC; ++x) f[x] = value(f[x]);
    stream_out((char*)out + (uint32_t)(e0 + k * STRIDE) * (uint32_t)sizeof(T), Logit<T>::pack(f));
  }
  if (has_tail)
    for (int e = whole; e < r.v; ++e) out[e] = (T)value((float)row[e]);
  if (t < NV * STRIDE && t < r.v && (int)(t / VEC) % THREADS == (int)threadIdx.x) out[t] = (T)(g + value(f_t));
  if (NV * STRIDE < r.v) write_gradient<T, THREADS>(row, out, NV * STRIDE, r.v, t, f_t, c, [&] { return RowState{g, m, inv_s}; });
}

// and the rows' terms, 256 rows a workgroup; the last workgroup to finish adds the workgroups' sums,
// in order.
template <typename T, bool DONE>
__global__ __launch_bounds__(256) void policy_terms_kernel(const Rows r, const Policy p, const Stat* stats,
                                                           const double* weights, float* lp_out, RowState* state,
                                                           double* partial, int* finished, float* sums) {
  __shared__ double red[4];
  __shared__ int last;
  double sum[3] = {0.0, 0.0, 0.0};
  const int64_t i0 = (int64_t)blockIdx.x * 256;
  policy_rows<T, 256, DONE>(r, p, i0, min(i0 + 256, r.n), 1, stats, weights, lp_out, state, sum);
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const double x = block_sum64<256>(sum[k], red);
    if (threadIdx.x == 0)
      __hip_atomic_store(partial + blockIdx.x * 3 + k, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(finished, 1) == (int)gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!last) return;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    double x = 0.0;
    for (unsigned q = threadIdx.x; q < gridDim.x; q += 256)
      x += __hip_atomic_load(partial + q * 3 + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    x = block_sum64<256>(x, red);
    if (threadIdx.x == 0) sums[k] = (float)x;
  }
}

struct Preference {
  Segments seg;          // 2 pairs segments, non-decreasing over the rows: chosen 2 p, rejected 2 p + 1
  const float* ref_lp;   // [2 pairs]
  float beta, smoothing;
};

__device__ inline int64_t held_segment(const Preference& p, int64_t i) {
  const int64_t s = segment_of(p.seg, i);
  return s < 0 ? (int64_t)-1 : s > p.seg.n ? p.seg.n : s;
}

// A wavefront: the sum of rows [start, end) of lp.
__device__ inline double sequence_sum(const double* lp, int64_t start, int64_t end) {
  double sum = 0.0;
  for (int64_t i = start + (threadIdx.x & 63); i < end; i += 64) sum += lp[i];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
  return sum;
}

struct Pair {
  double h, loss;
  float g;  // dL / d the chosen answer's sum; the rejected one's is -g
};

__device__ inline Pair pair_of(const Preference& p, int64_t q, double chosen, double rejected, bool unordered) {
  const double h = unordered ? __builtin_nan("") : (double)p.beta * ((chosen - (double)p.ref_lp[2 * q]) -
                                                                    (rejected - (double)p.ref_lp[2 * q + 1]));
  const double e = exp(-fabs(h)), tail = log1p(e);  // -log sigma(h) = tail + max(-h, 0)
  const double small = e / (1.0 + e), large = 1.0 / (1.0 + e);
  const double up = h >= 0.0 ? large : small, down = h >= 0.0 ? small : large;  // sigma(h), sigma(-h)
  const double eps = (double)p.smoothing;
  // an answer the policy cannot give (lp -inf) makes h infinite: a term of no weight stays out
  const double lost = eps < 1.0 ? (1.0 - eps) * fmax(-h, 0.0) : 0.0, won = eps > 0.0 ? eps * fmax(h, 0.0) : 0.0;
  return {h, (tail + lost + won) + (h != h ? h : 0.0),
          (float)((double)p.beta * (eps * up - (1.0 - eps) * down) / (double)(p.seg.n / 2))};
}

// One workgroup: lp, the sequences' sums, margins, loss and state (where kept).  starts [2 pairs + 1],
// d_seq and seq_sum [2 pairs] and lp64 [n] (given with has_lp) are scratch.
template <typename T, int THREADS>
__device__ inline void preference_all(const Rows& r, const Preference& p, int parts, const Stat* stats, int64_t* starts,
                                      float* d_seq, double* seq_sum, double* lp64, float* lp_out, float* seq_out,
                                      float* margins, RowState* state, float* loss_out, bool has_lp, bool has_grad) {
  __shared__ double red[THREADS / 64];
  __shared__ int unordered;
  const int tid = threadIdx.x;
  const int64_t count = p.seg.n, pairs = count / 2;
  if (tid == 0) unordered = 0;
  __syncthreads();
  for (int64_t i = tid; i < r.n; i += THREADS) {
    const int64_t t = target_of(r, i);
    // starts[s]: the first row of segment s or a later one
    const int64_t s = held_segment(p, i), before = i > 0 ? held_segment(p, i - 1) : -1;
    for (int64_t q = before + 1; q <= s; ++q) starts[q] = i;
    if (before > s) unordered = 1;
    if (i == r.n - 1)
      for (int64_t q = s + 1; q <= count; ++q) starts[q] = r.n;
    double lp = 0.0;
    RowState st = {0.0f, 0.0f, 0.0f};
    if (t >= 0) {
      const Stat rs = row_stat(stats, i, parts, r.c);
      lp = has_lp ? lp64[i] : logprob_of(r, z_below_m<T>(r, i, t, rs.m), rs.s);
      st = {0.0f, rs.m, 1.0f / rs.s};
    }
    lp64[i] = lp;
    lp_out[i] = (float)lp;
    if (state != nullptr) state[i] = st;
  }
  if (r.n == 0)
    for (int64_t q = tid; q <= count; q += THREADS) starts[q] = 0;
  __syncthreads();
  for (int64_t s = tid >> 6; s < count; s += THREADS / 64) {
    // segments out of order have no sums (several rows may have written a start): NaN
    const double sum = unordered ? __builtin_nan("") : sequence_sum(lp64, starts[s], starts[s + 1]);
    if ((tid & 63) == 0) {
      seq_sum[s] = sum;
      seq_out[s] = (float)sum;
    }
  }
  __syncthreads();
  double loss = 0.0;
  for (int64_t q = tid; q < pairs; q += THREADS) {
    const Pair x = pair_of(p, q, seq_sum[2 * q], seq_sum[2 * q + 1], unordered);
    loss += x.loss;
    d_seq[2 * q] = x.g;
    d_seq[2 * q + 1] = -x.g;
    margins[q] = (float)x.h;
  }
  loss = block_sum64<THREADS>(loss, red);
  if (tid == 0) loss_out[0] = (float)(loss / (double)max(pairs, (int64_t)1));
  if (has_grad) return;  // the gradient kernel finds g itself
  __syncthreads();
  for (int64_t i = tid; i < r.n; i += THREADS) {
    const int64_t s = segment_of(p.seg, i);
    if (s >= 0 && s < count && target_of(r, i) >= 0) state[i].g = d_seq[s];
  }
}

template <typename T>
__global__ __launch_bounds__(kFinish) void preference_finish(const Rows r, const Preference p, int parts,
                                                             const Stat* stats, int64_t* starts, float* d_seq,
                                                             double* seq_sum, double* lp64, float* lp_out, float* seq_out,
                                                             float* margins, RowState* state, float* loss_out,
                                                             bool has_lp, bool has_grad) {
  preference_all<T, kFinish>(r, p, parts, stats, starts, d_seq, seq_sum, lp64, lp_out, seq_out, margins, state, loss_out,
                             has_lp, has_grad);
}

// Few rows in parts (at most kFewRows): as policy_few_kernel; a workgroup sums its row's pair itself
// (4 rows 11.8 us for 14.6, 90 rows 21.2 for 24.6, 250 rows 40.9 for 45.5).  Held to 64 registers, two
// workgroups of 1024 to a CU, it spills 16 in the pair's arithmetic; with the 83 it asks for, one to a
// CU, 37 rows of f32 take 23.4 us for 19.1 and the three launches 21.3.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, 8) void preference_few_kernel(const Rows r, const Preference p, int parts,
                                                                 int part_len, const Stat* stats, int64_t* starts,
                                                                 float* d_seq, double* seq_sum, double* lp64,
                                                                 float* lp_out, float* seq_out, float* margins,
                                                                 float* loss_out, float scale, T* d, int64_t d_stride) {
  static_assert(THREADS >= kFewRows, "a row a thread");
  __shared__ double lps[kFewRows], sums[2];
  __shared__ int64_t bounds[3];
  __shared__ int unordered;
  const int64_t i = (int64_t)blockIdx.y - 1;
  if (i < 0) {
    if (blockIdx.x == 0)
      preference_all<T, THREADS>(r, p, parts, stats, starts, d_seq, seq_sum, lp64, lp_out, seq_out, margins, nullptr,
                                 loss_out, false, true);
    return;
  }
  int e0, e1;
  part_range(r.v, parts, part_len, (int)blockIdx.x, e0, e1);
  const int64_t t = target_of(r, i);
  T* out = d + i * d_stride;
  if (t < 0) {
    write_zeros<T, THREADS>(out, e0, e1);
    return;
  }
  const T* row = (const T*)r.z + i * r.stride;
  const float f_t = t < r.v ? (float)row[t] : __builtin_nanf("");
  write_gradient<T, THREADS>(row, out, e0, e1, t, f_t, r.c, [&] {
    const Stat st = row_stat(stats, i, parts, r.c);
    const int64_t mine = segment_of(p.seg, i), first = mine & ~(int64_t)1;
    if (threadIdx.x == 0) unordered = 0;
    __syncthreads();
    const int64_t j = threadIdx.x;
    if (j < r.n) {
      const int64_t s = held_segment(p, j), before = j > 0 ? held_segment(p, j - 1) : -1;
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        if (before < first + q && first + q <= s) bounds[q] = j;
        if (j == r.n - 1 && s < first + q) bounds[q] = r.n;
      }
      if (before > s) unordered = 1;
      const int64_t tj = target_of(r, j);
      double lp = 0.0;
      if (tj >= 0 && s >= first && s <= first + 1) {
        const Stat sj = row_stat(stats, j, parts, r.c);
        lp = logprob_of(r, z_below_m<T>(r, j, tj, sj.m), sj.s);
      }
      lps[j] = lp;
    }
    __syncthreads();
    const bool in = mine >= 0 && mine < p.seg.n;
    if (in && threadIdx.x < 128) {
      const int w = threadIdx.x >> 6;
      const double sum = sequence_sum(lps, bounds[w], bounds[w + 1]);
      if ((threadIdx.x & 63) == 0) sums[w] = sum;
    }
    __syncthreads();
    const float g = in ? pair_of(p, first / 2, sums[0], sums[1], unordered).g : 0.0f;
    return RowState{(mine & 1 ? -g : g) * scale, st.m, 1.0f / st.s};
  });
}

// ---- host side --------------------------------------------------------------------------------

int value_bytes(int dtype) { return dtype == EG_DTYPE_F32 ? 4 : 2; }

// How a pass over the logits is cut: threads a workgroup, and parts of a row.
struct Cut {
  int threads, parts, part_len;
};

constexpr int64_t kGroupsWanted = 512;  // two workgroups a CU
constexpr int kPartBytes = 16384;       // the shortest part worth a workgroup

Cut make_cut(int64_t n, int64_t v, int dtype) {
  const int64_t size = value_bytes(dtype), vec = 16 / size;
  int64_t parts = n > 0 ? std::min(kGroupsWanted / n, v * size / kPartBytes) : 1;
  parts = std::max<int64_t>(parts, 1);
  const int64_t len = ((v + parts - 1) / parts + vec - 1) / vec * vec;
  parts = (v + len - 1) / len;
  return {len * size > 32768 ? 1024 : 256, (int)parts, (int)len};
}

// Log-probabilities take a launch less with a workgroup a whole row: 5.5 us against 8.2 for 64 KB a
// row, 9.8 against 8.1 for one row of 300 KB, 12.7 against 16.2 for 200 such rows, 8.0 against 8.5 for 64 of
// 200 KB.  Of longer rows 64 are few: 12.3 us for 63 in parts at 9.8 (300 KB), 15.9 at 12.4 (608 KB); by the
// slopes the sides meet at about 120 and 100 rows.
constexpr int64_t kWholeRowBytes = 128 << 10, kWholeRows = 64;

// policy_held_kernel holds 8 chunks a thread of rows above kHeldShort bytes, 20 above kHeldLong.  1,024 rows
// against policy_row_kernel: 66 KB 41.6 us for 38.6, 100 KB 59.9 for 66.4; 8 against 20 chunks: 140 KB 69.7 and
// 69.1 (75.6 not held), 260 KB 131 and 120 (136), 608 KB (fp32) 284 and 257 (312).
constexpr int64_t kHeldShort = 80 << 10, kHeldLong = 128 << 10;

Cut whole_rows(int64_t v, int dtype) { return {v * value_bytes(dtype) > 32768 ? 1024 : 256, 1, (int)v}; }

int check_logits(const eg_logits* l, Rows* r) {
  EG_CHECK_ARG(l != nullptr, "logits is NULL");
  EG_CHECK_ARG(l->dtype == EG_DTYPE_F32 || l->dtype == EG_DTYPE_BF16 || l->dtype == EG_DTYPE_F16,
               "logits dtype=%d must be f32, bf16 or f16", l->dtype);
  EG_CHECK_ARG(l->n >= 0, "n=%lld rows must not be negative", (long long)l->n);
  EG_CHECK_ARG(l->v >= 1 && l->v <= 0x7fffffff - 65536, "vocabulary v=%lld must be in [1, 2^31 - 65536)",
               (long long)l->v);
  EG_CHECK_ARG(l->n <= 1 || l->row_stride >= l->v, "row_stride=%lld must be at least v=%lld",
               (long long)l->row_stride, (long long)l->v);
  EG_CHECK_ARG(l->temperature > 0.0f && l->temperature < 3.0e38f, "temperature=%g must be positive and finite",
               (double)l->temperature);
  EG_CHECK_ARG(l->n == 0 || (l->data != nullptr && l->targets != nullptr), "logits data or targets is NULL");
  EG_CHECK_ARG((uintptr_t)l->data % value_bytes(l->dtype) == 0, "logits data is not aligned to its type");
  *r = {l->data, l->n, l->row_stride, l->targets, (int32_t)l->v, l->targets_i32 != 0, kLog2e / l->temperature,
        1.0 / (double)l->temperature};
  return EG_OK;
}

int check_segments(const void* ids, int32_t i32, int64_t n, Segments* s) {
  EG_CHECK_ARG(n >= 0, "n_segments=%lld must not be negative", (long long)n);
  *s = {ids, n, i32 != 0};
  return EG_OK;
}

// Workspace of a loss: the parts' statistics, then scratch of the rows (8 bytes each) and of the
// segments (24 bytes each).
int64_t stats_bytes(int64_t n, const Cut& cut) { return (n * cut.parts * (int64_t)sizeof(Stat) + 15) / 16 * 16; }

dim3 row_grid(const Cut& cut, int64_t n) {
  const int64_t y = std::min<int64_t>(n, 32768);
  return dim3((unsigned)cut.parts, (unsigned)y, (unsigned)((n + y - 1) / y));
}

// Whether the gradient's workgroups find what they need of the loss themselves: rows in parts, and the
// gradient not in the logits' place (other rows' logits are read meanwhile).
bool few_rows(const Rows& r, const Cut& cut, const void* d) {
  return d != nullptr && d != r.z && r.n >= 1 && r.n <= kFewRows && cut.parts > 1;
}

template <typename F>
int by_dtype(int dtype, F&& f) {
  switch (dtype) {
    case EG_DTYPE_F32: return f(float{});
    case EG_DTYPE_BF16: return f(__bf16{});
    default: return f(_Float16{});
  }
}

int launch_stats(const Rows& r, int dtype, const Cut& cut, Stat* stats, hipStream_t stream, const WholeRow& whole = {}) {
  if (r.n == 0) return EG_OK;
  return by_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    const dim3 grid = row_grid(cut, r.n);
    if (cut.threads == 1024)
      row_stats_kernel<T, 1024><<<grid, 1024, 0, stream>>>(r, cut.parts, cut.part_len, stats, whole);
    else
      row_stats_kernel<T, 256><<<grid, 256, 0, stream>>>(r, cut.parts, cut.part_len, stats, whole);
    return launch_status("row_stats_kernel");
  });
}

int launch_grad(const Rows& r, int dtype, const Cut& cut, const RowState* state, const float* upstream, float scale,
                void* d, int64_t d_stride, hipStream_t stream, const Segments& seg = {}, const float* d_seq = nullptr) {
  if (r.n == 0) return EG_OK;
  return by_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    const dim3 grid = row_grid(cut, r.n);
    if (cut.threads == 1024)
      logits_grad_kernel<T, 1024><<<grid, 1024, 0, stream>>>(r, cut.parts, cut.part_len, state, seg, d_seq, upstream,
                                                             scale, (T*)d, d_stride);
    else
      logits_grad_kernel<T, 256><<<grid, 256, 0, stream>>>(r, cut.parts, cut.part_len, state, seg, d_seq, upstream,
                                                           scale, (T*)d, d_stride);
    return launch_status("logits_grad_kernel");
  });
}

int check_grad(const eg_logits* l, const void* d, int64_t d_stride) {
  EG_CHECK_ARG(l->n == 0 || d != nullptr, "d_logits is NULL");
  EG_CHECK_ARG(l->n <= 1 || d_stride >= l->v, "d_stride=%lld must be at least v=%lld", (long long)d_stride,
               (long long)l->v);
  EG_CHECK_ARG((uintptr_t)d % value_bytes(l->dtype) == 0, "d_logits is not aligned to its type");
  EG_CHECK_ARG(d != l->data || d_stride == l->row_stride || l->n <= 1,
               "d_logits in place of the logits must have their row stride");
  const int64_t size = value_bytes(l->dtype);
  EG_CHECK_ARG(d == l->data || !overlap({d, l->n, l->v, d_stride, 1, size}, {l->data, l->n, l->v, l->row_stride, 1, size}),
               "d_logits overlap the logits: they may be in their place or apart from them");
  return EG_OK;
}

// An argument that is read while the gradient is written.
int check_apart(const eg_logits* l, const void* d, int64_t d_stride, const void* x, int64_t count, int64_t size,
                const char* name) {
  EG_CHECK_ARG(d == nullptr || x == nullptr ||
                   !overlap({d, l->n, l->v, d_stride, 1, value_bytes(l->dtype)}, {x, 1, count, count, 1, size}),
               "d_logits overlap %s", name);
  return EG_OK;
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" {

int64_t eg_loss_workspace_size(int64_t n, int64_t v, int32_t dtype, int64_t n_segments) {
  if (n < 0 || v < 1 || n_segments < 0) return -1;
  return stats_bytes(n, make_cut(n, v, dtype)) + (n_segments + 1) * 24 + n * 8 + 64;
}

#define EG_CHECK_WORKSPACE(need)                                                                              \
  do {                                                                                                        \
    if ((need) > 0 && (workspace == nullptr || workspace_bytes < (need)))                                     \
      return ::eg::set_error(EG_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, \
                             (long long)(need));                                                              \
    EG_CHECK_ARG((uintptr_t)workspace % 16 == 0, "workspace must be 16-byte aligned");                        \
  } while (0)

int eg_token_logprobs(const eg_logits* logits, float* logprobs, void* workspace, int64_t workspace_bytes,
                      void* stream) {
  Rows r;
  if (int rc = check_logits(logits, &r); rc != EG_OK) return rc;
  EG_CHECK_ARG(r.n == 0 || logprobs != nullptr, "logprobs is NULL");
  if (r.n == 0) return EG_OK;
  // one launch where a workgroup has a row alone
  if (r.n >= kWholeRows || r.v * (int64_t)value_bytes(logits->dtype) <= kWholeRowBytes)
    return launch_stats(r, logits->dtype, whole_rows(r.v, logits->dtype), nullptr, (hipStream_t)stream, {logprobs, nullptr});
  const Cut cut = make_cut(r.n, r.v, logits->dtype);
  EG_CHECK_WORKSPACE(stats_bytes(r.n, cut));
  Stat* stats = (Stat*)workspace;
  if (int rc = launch_stats(r, logits->dtype, cut, stats, (hipStream_t)stream); rc != EG_OK) return rc;
  return by_dtype(logits->dtype, [&](auto zero) {
    using T = decltype(zero);
    logprobs_finish<T><<<dim3((unsigned)((r.n + 255) / 256)), 256, 0, (hipStream_t)stream>>>(r, cut.parts, stats,
                                                                                            logprobs);
    return launch_status("logprobs_finish");
  });
}

int eg_policy_loss(const eg_logits* logits, const eg_policy* policy, float* logprobs, float* sums, float* state,
                   void* d_logits, int64_t d_stride, float grad_scale, void* workspace, int64_t workspace_bytes,
                   void* stream) {
  Rows r;
  if (int rc = check_logits(logits, &r); rc != EG_OK) return rc;
  EG_CHECK_ARG(policy != nullptr && sums != nullptr, "policy or sums is NULL");
  EG_CHECK_ARG(r.n == 0 || (logprobs != nullptr && state != nullptr && policy->advantages != nullptr),
               "logprobs, state or advantages is NULL");
  EG_CHECK_ARG(policy->reduction >= EG_REDUCE_SUM && policy->reduction <= EG_REDUCE_SEQUENCE, "reduction=%d",
               policy->reduction);
  EG_CHECK_ARG(policy->clip_low >= 0.0f && policy->clip_low <= 1.0f && policy->clip_high >= 0.0f,
               "clip (%g, %g): 0 <= low <= 1 and high >= 0 are needed", (double)policy->clip_low,
               (double)policy->clip_high);
  Policy p = {policy->advantages, policy->old_logprobs, policy->ref_logprobs, {nullptr, 0, 0}, policy->reduction,
              policy->clip_low, policy->clip_high, policy->kl_coef};
  if (p.reduction == EG_REDUCE_SEQUENCE) {
    if (int rc = check_segments(policy->segment_ids, policy->segment_ids_i32, policy->n_segments, &p.seg); rc != EG_OK)
      return rc;
    EG_CHECK_ARG(r.n == 0 || policy->segment_ids != nullptr, "segment_ids is NULL");
  }
  if (d_logits != nullptr) {
    if (int rc = check_grad(logits, d_logits, d_stride); rc != EG_OK) return rc;
    const int64_t target = logits->targets_i32 != 0 ? 4 : 8, id = policy->segment_ids_i32 != 0 ? 4 : 8;
    const struct { const void* x; int64_t size; const char* name; } read[] = {
        {logits->targets, target, "targets"}, {p.advantages, 4, "advantages"}, {p.old_lp, 4, "old_logprobs"},
        {p.ref_lp, 4, "ref_logprobs"}, {p.seg.ids, id, "segment_ids"}};
    for (const auto& a : read)
      if (int rc = check_apart(logits, d_logits, d_stride, a.x, r.n, a.size, a.name); rc != EG_OK) return rc;
  }
  const Cut cut = make_cut(r.n, r.v, logits->dtype);
  const int64_t first = stats_bytes(r.n, cut);
  EG_CHECK_WORKSPACE(first + (p.seg.n + 1) * 24 + r.n * 8 + 64);
  Stat* stats = (Stat*)workspace;
  double* partial = (double*)((char*)workspace + first);  // 3 of every 256 rows
  double* weights = partial + r.n;
  int* finished = (int*)(weights + p.seg.n + 1);
  const hipStream_t st = (hipStream_t)stream;
  RowState* kept = (RowState*)state;
  const bool many = cut.parts == 1 && r.n >= kGroupsWanted;
  if (many) {
    policy_weights_kernel<<<1, kFinish, 0, st>>>(r, p, weights, finished);
    if (int rc = launch_status("policy_weights_kernel"); rc != EG_OK) return rc;
  }
  if (many && d_logits != nullptr) {
    const int rc = by_dtype(logits->dtype, [&](auto zero) {
      using T = decltype(zero);
      const dim3 grid = row_grid(cut, r.n);
      const float scale = grad_scale / logits->temperature;
      const int64_t bytes = r.v * (int64_t)sizeof(T);
      auto held = [&](auto kernel) { kernel<<<grid, 1024, 0, st>>>(r, p, weights, stats, kept, scale, (T*)d_logits, d_stride); };
      if (bytes > kHeldLong)
        held(policy_held_kernel<T, 20>);
      else if (bytes > kHeldShort)
        held(policy_held_kernel<T, 8>);
      else if (cut.threads == 1024)
        policy_row_kernel<T, 1024><<<grid, 1024, 0, st>>>(r, p, weights, stats, kept, scale, (T*)d_logits, d_stride);
      else
        policy_row_kernel<T, 256><<<grid, 256, 0, st>>>(r, p, weights, stats, kept, scale, (T*)d_logits, d_stride);
      return launch_status("policy_row_kernel");
    });
    if (rc != EG_OK) return rc;
  } else if (int rc = launch_stats(r, logits->dtype, cut, stats, st); rc != EG_OK) {
    return rc;
  }
  if (few_rows(r, cut, d_logits) && p.seg.n <= kFewSegments)
    return by_dtype(logits->dtype, [&](auto zero) {
      using T = decltype(zero);
      const dim3 grid((unsigned)cut.parts, (unsigned)r.n + 1);
      const float scale = grad_scale / logits->temperature;
      if (cut.threads == 1024)
        policy_few_kernel<T, 1024><<<grid, 1024, 0, st>>>(r, p, cut.parts, cut.part_len, stats, logprobs, sums, scale,
                                                          (T*)d_logits, d_stride);
      else
        policy_few_kernel<T, 256><<<grid, 256, 0, st>>>(r, p, cut.parts, cut.part_len, stats, logprobs, sums, scale,
                                                        (T*)d_logits, d_stride);
      return launch_status("policy_few_kernel");
    });
  const int rc = by_dtype(logits->dtype, [&](auto zero) {
    using T = decltype(zero);
    const dim3 grid((unsigned)((r.n + 255) / 256));
    if (many && d_logits != nullptr)
      policy_terms_kernel<T, true><<<grid, 256, 0, st>>>(r, p, stats, weights, logprobs, kept, partial, finished, sums);
    else if (many)
      policy_terms_kernel<T, false><<<grid, 256, 0, st>>>(r, p, stats, weights, logprobs, kept, partial, finished, sums);
    else
      policy_finish<T><<<1, kFinish, 0, st>>>(r, p, cut.parts, stats, weights, logprobs, kept, sums);
    return launch_status("policy_finish");
  });
  if (rc != EG_OK || d_logits == nullptr || many) return rc;
  return launch_grad(r, logits->dtype, cut, (const RowState*)state, nullptr, grad_scale / logits->temperature, d_logits,
                     d_stride, st);
}

int eg_preference_loss(const eg_logits* logits, const eg_preference* preference, float* logprobs,
                       float* sequence_logprobs, float* margins, float* loss, float* state, void* d_logits,
                       int64_t d_stride, float grad_scale, void* workspace, int64_t workspace_bytes, void* stream) {
  Rows r;
  if (int rc = check_logits(logits, &r); rc != EG_OK) return rc;
  EG_CHECK_ARG(preference != nullptr && loss != nullptr, "preference or loss is NULL");
  EG_CHECK_ARG(preference->n_pairs >= 1, "n_pairs=%lld must be at least 1", (long long)preference->n_pairs);
  EG_CHECK_ARG(preference->ref_logprobs != nullptr && sequence_logprobs != nullptr && margins != nullptr,
               "ref_logprobs, sequence_logprobs or margins is NULL");
  EG_CHECK_ARG(r.n == 0 || (logprobs != nullptr && state != nullptr && preference->segment_ids != nullptr),
               "logprobs, state or segment_ids is NULL");
  EG_CHECK_ARG(preference->label_smoothing >= 0.0f && preference->label_smoothing <= 1.0f,
               "label_smoothing=%g must be in [0, 1]", (double)preference->label_smoothing);
  if (d_logits != nullptr) {
    if (int rc = check_grad(logits, d_logits, d_stride); rc != EG_OK) return rc;
    const int64_t target = logits->targets_i32 != 0 ? 4 : 8, id = preference->segment_ids_i32 != 0 ? 4 : 8;
    const struct { const void* x; int64_t count, size; const char* name; } read[] = {
        {logits->targets, r.n, target, "targets"}, {preference->segment_ids, r.n, id, "segment_ids"},
        {preference->ref_logprobs, 2 * preference->n_pairs, 4, "ref_logprobs"}};
    for (const auto& a : read)
      if (int rc = check_apart(logits, d_logits, d_stride, a.x, a.count, a.size, a.name); rc != EG_OK) return rc;
  }
  Preference p;
  if (int rc = check_segments(preference->segment_ids, preference->segment_ids_i32, 2 * preference->n_pairs, &p.seg);
      rc != EG_OK)
    return rc;
  p.ref_lp = preference->ref_logprobs;
  p.beta = preference->beta;
  p.smoothing = preference->label_smoothing;
  const Cut cut = make_cut(r.n, r.v, logits->dtype);
  const int64_t first = stats_bytes(r.n, cut);
  EG_CHECK_WORKSPACE(first + (p.seg.n + 1) * 24 + r.n * 8);
  Stat* stats = (Stat*)workspace;
  int64_t* starts = (int64_t*)((char*)workspace + first);
  double* seq_sum = (double*)(starts + p.seg.n + 1);
  double* lp64 = seq_sum + p.seg.n;
  float* d_seq = (float*)(lp64 + r.n);
  const bool whole = cut.parts == 1;  // a row's workgroup gives its lp
  if (int rc = launch_stats(r, logits->dtype, cut, stats, (hipStream_t)stream, {nullptr, whole ? lp64 : nullptr});
      rc != EG_OK)
    return rc;
  if (few_rows(r, cut, d_logits))
    return by_dtype(logits->dtype, [&](auto zero) {
      using T = decltype(zero);
      const dim3 grid((unsigned)cut.parts, (unsigned)r.n + 1);
      const float scale = grad_scale / logits->temperature;
      if (cut.threads == 1024)
        preference_few_kernel<T, 1024><<<grid, 1024, 0, (hipStream_t)stream>>>(
            r, p, cut.parts, cut.part_len, stats, starts, d_seq, seq_sum, lp64, logprobs, sequence_logprobs, margins, loss,
            scale, (T*)d_logits, d_stride);
      else
        preference_few_kernel<T, 256><<<grid, 256, 0, (hipStream_t)stream>>>(
            r, p, cut.parts, cut.part_len, stats, starts, d_seq, seq_sum, lp64, logprobs, sequence_logprobs, margins, loss,
            scale, (T*)d_logits, d_stride);
      return launch_status("preference_few_kernel");
    });
  int rc = by_dtype(logits->dtype, [&](auto zero) {
    using T = decltype(zero);
    preference_finish<T><<<1, kFinish, 0, (hipStream_t)stream>>>(r, p, cut.parts, stats, starts, d_seq, seq_sum,
                                                                 lp64, logprobs, sequence_logprobs, margins,
                                                                 (RowState*)state, loss, whole, d_logits != nullptr);
    return launch_status("preference_finish");
  });
  if (rc != EG_OK || d_logits == nullptr) return rc;
  return launch_grad(r, logits->dtype, cut, (const RowState*)state, nullptr, grad_scale / logits->temperature,
                     d_logits, d_stride, (hipStream_t)stream, p.seg, d_seq);
}

int eg_logits_grad(const eg_logits* logits, const float* state, const float* upstream, float grad_scale,
                   void* d_logits, int64_t d_stride, void* stream) {
  Rows r;
  if (int rc = check_logits(logits, &r); rc != EG_OK) return rc;
  EG_CHECK_ARG(r.n == 0 || state != nullptr, "state is NULL");
  if (int rc = check_grad(logits, d_logits, d_stride); rc != EG_OK) return rc;
  if (int rc = check_apart(logits, d_logits, d_stride, logits->targets, r.n, logits->targets_i32 != 0 ? 4 : 8, "targets");
      rc != EG_OK)
    return rc;
  if (int rc = check_apart(logits, d_logits, d_stride, state, 3 * r.n, 4, "state"); rc != EG_OK) return rc;
  return launch_grad(r, logits->dtype, make_cut(r.n, r.v, logits->dtype), (const RowState*)state, upstream,
                     grad_scale / logits->temperature, d_logits, d_stride, (hipStream_t)stream);
}

}  // extern "C"
