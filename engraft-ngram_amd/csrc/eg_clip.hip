// The norm of all gradients of a step, and their clipping:
//
//   N = sqrt(sum over all tensors of g^2),   out = g max_norm / N where N > max_norm, g otherwise
//
// Bound by its bytes.  Two kinds of launch: every workgroup adds the squares of its tiles (4,096 values
// of one tensor each, 2,048 where there are less than 2^20 in all) in 64 bits, which neither overflow nor lose small tensors beside large
// ones, and writes its sum; then every workgroup adds all of these sums (a few KB from L2, in one order) and
// writes its tiles' values, from the last one on: what was read last is in the caches.  The
// tensors are kernel arguments, 48 a launch, so that nothing is copied to the device.
#include <algorithm>
#include <string>
#include <vector>

#include "eg_fp8.h"

namespace eg {
namespace {

constexpr int kTensors = 48;      // a launch
constexpr int kThreads = 256;
constexpr int kMostGroups = 512;  // workgroups a launch: 1,024 take 1 to 2 us more for 131 MB, 4,096 7 to 13

struct ClipTensor {
  const void* g;
  void* out;
  int64_t cols, g_stride, out_stride;
  int64_t values;
  int32_t g_dtype, out_dtype;
  int64_t first_tile;             // of the launch's
};

struct ClipArgs {
  ClipTensor t[kTensors];
  int count;
  int64_t tiles;
  double* sums;                   // this launch's, one a workgroup
};

// The tensor of a tile.
__device__ inline int tensor_of(const ClipArgs& a, int64_t tile) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.t[mid].first_tile <= tile) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ inline double wave_sum64(double x) {
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) x += __shfl_xor(x, i);
  return x;
}

// f(a zero of the type)
template <typename F>
__device__ inline void device_type(int32_t dtype, const F& f) {
  if (dtype == EG_DTYPE_F32) f((float)0);
  else if (dtype == EG_DTYPE_BF16) f((__bf16)0);
  else f((_Float16)0);
}

// Whole rows are one row; otherwise a value's place is found by its row.
__device__ inline int64_t place(int64_t i, int64_t cols, int64_t stride) { return cols == stride ? i : i / cols * stride + i % cols; }

// Values i .. i + 7 of a tensor (zeros past its end).
template <typename T>
__device__ inline void read8(const ClipTensor& t, int64_t i, float (&v)[8]) {
  const T* const g = (const T*)t.g;
  const int64_t left = t.values - i;
  if (t.cols == t.g_stride) {
    load8(g + i, left > 8 ? 8 : (int)left, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < left ? (float)g[place(i + k, t.cols, t.g_stride)] : 0.0f;
  }
}

// Outputs apart from the gradients are written past the caches, which hold the gradients' first reading: 131 MB take
// 69.5 us so, 78.7 through them.
template <typename T>
__device__ inline void write8(const ClipTensor& t, int64_t i, const float (&v)[8]) {
  T* const o = (T*)t.out;
  const int64_t left = t.values - i;
  if (t.cols == t.out_stride && left >= 8 && t.out != t.g) {
    typedef i32x4 unaligned __attribute__((aligned(2)));
    T x[8];
    Raw8<T> r;
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = (T)v[k];
    __builtin_memcpy(&r, x, sizeof(r));
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k) __builtin_nontemporal_store(r.w[k], (unaligned*)(o + i) + k);
  } else if (t.cols == t.out_stride) {
    store8(o + i, left > 8 ? 8 : (int)left, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) o[place(i + k, t.cols, t.out_stride)] = (T)v[k];
  }
}

// A tile is READS times eight values a thread; all of its loads are on their way before the first is waited for.
template <typename T, int READS>
__device__ inline void read_tile(const ClipTensor& t, int64_t tile, float (&v)[READS][8]) {
  constexpr int kTile = READS * kThreads * 8, kReads = READS;
  const int64_t i0 = (tile - t.first_tile) * kTile + threadIdx.x * 8;
  if (t.cols == t.g_stride && (tile - t.first_tile + 1) * kTile <= t.values) {
    Raw8<T> r[kReads];
#pragma unroll
    for (int j = 0; j < kReads; ++j) r[j] = load_raw<false>((const T*)t.g + i0 + j * kThreads * 8, 0, 8);
#pragma unroll
    for (int j = 0; j < kReads; ++j) values_of<false, T>(r[j], 0, 8, v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kReads; ++j) read8<T>(t, i0 + j * kThreads * 8, v[j]);
  }
}

template <int READS>
__global__ __launch_bounds__(kThreads) void squares_kernel(const ClipArgs a) {
  __shared__ double part[kThreads / 64];
  double s = 0.0;
  for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const ClipTensor& t = a.t[tensor_of(a, tile)];
    device_type(t.g_dtype, [&](auto z) {
      float v[READS][8];
      read_tile<decltype(z)>(t, tile, v);
#pragma unroll
      for (int j = 0; j < READS; ++j)
#pragma unroll
        for (int k = 0; k < 8; ++k) s += (double)v[j][k] * (double)v[j][k];
    });
  }
  s = wave_sum64(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int i = 0; i < kThreads / 64; ++i) s += part[i];
    a.sums[blockIdx.x] = s;
  }
}

// The root of the sum of `count` sums, in every thread.
__device__ inline double root_of_sums(const double* sums, int64_t count, double* part) {
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += kThreads) s += sums[i];
  s = wave_sum64(s);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0.0;
  for (int i = 0; i < kThreads / 64; ++i) s += part[i];
  return sqrt(s);
}

template <int READS>
__global__ __launch_bounds__(kThreads) void scale_kernel(const ClipArgs a, const double* sums, int64_t count, float max_norm, float* norm) {
  __shared__ double part[kThreads / 64];
  double root = 0.0, factor = 1.0;  // (as a float the factor could leave the normal numbers)
  bool clips = false;
  for (int64_t k = blockIdx.x; k < a.tiles; k += gridDim.x) {
    const int64_t tile = a.tiles - 1 - k;
    const ClipTensor& t = a.t[tensor_of(a, tile)];
    if (k != blockIdx.x && !clips && t.out == t.g) continue;  // as they are
    float v[READS][8];
    device_type(t.g_dtype, [&](auto z) { read_tile<decltype(z)>(t, tile, v); });
    if (k == blockIdx.x) {  // (the first tile's loads are on their way meanwhile)
      root = root_of_sums(sums, count, part);
      clips = root > (double)max_norm && root <= 1.7976931348623157e308;
      if (clips) factor = (double)max_norm / root;
      if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)root;
      if (!clips && t.out == t.g) continue;
    }
    if (clips) {
#pragma unroll
      for (int j = 0; j < READS; ++j)
#pragma unroll
        for (int q = 0; q < 8; ++q) v[j][q] = (float)((double)v[j][q] * factor);
    }
    const int64_t i0 = (tile - t.first_tile) * (READS * kThreads * 8) + threadIdx.x * 8;
    device_type(t.out_dtype, [&](auto y) {
#pragma unroll
      for (int j = 0; j < READS; ++j) write8<decltype(y)>(t, i0 + j * kThreads * 8, v[j]);
    });
  }
}

__global__ __launch_bounds__(kThreads) void norm_of_sums_kernel(const double* sums, int64_t count, float* norm) {
  __shared__ double part[kThreads / 64];
  const double root = root_of_sums(sums, count, part);
  if (threadIdx.x == 0) *norm = (float)root;
}

// Launches of at most kTensors tensors: [first, last) of those that hold values.
struct Launch {
  ClipArgs args;
  int groups;
};

// Values of a tile: few, so that more workgroups share them, where there are less than 2^20 in all.
int tile_of(const eg_clip_tensor* tensors, int64_t count) {
  int64_t values = 0;
  for (int64_t i = 0; i < count && values < (1 << 20); ++i) values += std::max<int64_t>(tensors[i].rows * tensors[i].cols, 0);
  return values < (1 << 20) ? kThreads * 8 : 2 * kThreads * 8;
}

int64_t tiles_of(const eg_clip_tensor& t, int tile) { return (t.rows * t.cols + tile - 1) / tile; }

int groups_of(int64_t tiles) { return (int)std::min<int64_t>(tiles, kMostGroups); }

int check_tensors(const eg_clip_tensor* tensors, int64_t count) {
  EG_CHECK_ARG(count >= 0 && (tensors != nullptr || count == 0), "clip: count=%lld", (long long)count);
  bool outs = false, none = false;
  for (int64_t i = 0; i < count; ++i) {
    const eg_clip_tensor& t = tensors[i];
    EG_CHECK_ARG(t.rows >= 0 && t.cols >= 0 && t.rows < (1ll << 40) && t.cols < (1ll << 40) &&
                     (t.cols == 0 || t.rows <= (1ll << 44) / t.cols),
                 "clip: tensor %lld is %lld x %lld", (long long)i, (long long)t.rows, (long long)t.cols);
    if (t.rows == 0 || t.cols == 0) continue;
    if (const int rc = check_values(t.g, t.g_dtype, t.rows, t.cols, t.g_stride, "clip: a gradient"); rc != EG_OK) return rc;
    (t.out != nullptr ? outs : none) = true;
    if (t.out != nullptr)
      if (const int rc = check_values(t.out, t.out_dtype, t.rows, t.cols, t.out_stride, "clip: an output"); rc != EG_OK) return rc;
  }
  EG_CHECK_ARG(!(outs && none), "clip: some tensors have an output and some none");
  return EG_OK;
}

// The first two gradients (of operands by address) that share a value, which would count twice.
bool find_twice(const std::vector<Operand>& all, const Operand*& x, const Operand*& y) {
  for (size_t i = 0; i < all.size(); ++i) {
    if (all[i].kind != Operand::kGrad) continue;
    for (size_t j = i + 1; j < all.size() && all[j].extent.at < all[i].extent.end(); ++j) {
      if (all[j].kind != Operand::kGrad || !overlap(all[i].extent, all[j].extent)) continue;
      x = &all[i];
      y = &all[j];
      return true;
    }
  }
  return false;
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" {

int64_t eg_clip_workspace_size(const eg_clip_tensor* tensors, int64_t count) {
  if (check_tensors(tensors, count) != EG_OK) return -1;
  const int tile = tile_of(tensors, count);
  int64_t sums = 0, tiles = 0;
  int held = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (tensors[i].rows <= 0 || tensors[i].cols <= 0) continue;
    tiles += tiles_of(tensors[i], tile);
    if (++held == kTensors) {
      sums += groups_of(tiles);
      tiles = held = 0;
    }
  }
  return (sums + groups_of(tiles)) * 8;
}

int eg_clip_grads(const eg_clip_tensor* tensors, int64_t count, float max_norm, float* norm, void* workspace,
                  int64_t workspace_bytes, void* stream) try {
  if (const int rc = check_tensors(tensors, count); rc != EG_OK) return rc;
  EG_CHECK_ARG(norm != nullptr, "clip: NULL norm");
  EG_CHECK_ARG((uintptr_t)norm % 4 == 0, "clip: misaligned norm");
  EG_CHECK_ARG(max_norm >= 0.0f, "clip: max_norm=%g", (double)max_norm);
  const int64_t need = eg_clip_workspace_size(tensors, count);
  if (workspace_bytes < need)
    return set_error(EG_ERR_WORKSPACE, "clip needs %lld bytes of workspace, got %lld", (long long)need, (long long)workspace_bytes);
  EG_CHECK_ARG(need == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0), "clip: the workspace must be 16-byte aligned");
  // a tensor's output is a param here and its gradient a grad: it may be in its own gradient's place, of the
  // same type and stride, and must not overlap anything else; the norm and the workspace (as momenta) must not at all
  std::vector<Operand> operands = {{Operand::kMomentum, (size_t)count, {norm, 1, 1, 1, 1, 4}},
                                   {Operand::kMomentum, (size_t)count + 1, {workspace, 1, need, need, 1, 1}}};
  bool scales = false;
  for (int64_t i = 0; i < count; ++i) {
    const eg_clip_tensor& t = tensors[i];
    if (t.rows == 0 || t.cols == 0) continue;
    operands.push_back({Operand::kGrad, (size_t)i, {t.g, t.rows, t.cols, t.g_stride, 1, item_size(t.g_dtype)}});
    if (t.out == nullptr) continue;
    scales = true;
    const Extent out(t.out, t.rows, t.cols, t.out_stride, 1, item_size(t.out_dtype));
    const bool in_place = t.out == t.g && t.out_dtype == t.g_dtype && (t.out_stride == t.g_stride || t.rows == 1);
    EG_CHECK_ARG(in_place || !overlap(out, operands.back().extent), "clip: output %lld overlaps its gradient and is not in its place", (long long)i);
    operands.push_back({Operand::kParam, (size_t)i, out});
  }
  const Operand *x, *y;
  if (find_overlap(operands, x, y) || (scales && find_twice(operands, x, y))) {
    auto name = [&](const Operand* o) -> std::string {
      if (o->kind == Operand::kMomentum) return o->matrix == (size_t)count ? "the norm" : "the workspace";
      return (o->kind == Operand::kParam ? "output " : "gradient ") + std::to_string(o->matrix);
    };
    return set_error(EG_ERR_ARG, "clip: %s overlaps %s", name(x).c_str(), name(y).c_str());
  }
  const int tile = tile_of(tensors, count);
  const bool small = tile == kThreads * 8;
  std::vector<Launch> launches;
  double* at = (double*)workspace;
  for (int64_t i = 0; i < count; ++i) {
    const eg_clip_tensor& t = tensors[i];
    if (t.rows == 0 || t.cols == 0) continue;
    if (launches.empty() || launches.back().args.count == kTensors) launches.push_back({});
    ClipArgs& a = launches.back().args;
    const bool g_whole = t.rows == 1 || t.g_stride == t.cols, out_whole = t.rows == 1 || t.out_stride == t.cols;
    a.t[a.count++] = {t.g, t.out, t.cols, g_whole ? t.cols : t.g_stride, out_whole ? t.cols : t.out_stride, t.rows * t.cols,
                      t.g_dtype, t.out_dtype, a.tiles};
    a.tiles += tiles_of(t, tile);
  }
  int64_t sums = 0;
  for (Launch& l : launches) {
    l.groups = groups_of(l.args.tiles);
    l.args.sums = at + sums;
    sums += l.groups;
    (small ? squares_kernel<1> : squares_kernel<2>)<<<l.groups, kThreads, 0, (hipStream_t)stream>>>(l.args);
    if (const int rc = launch_status("squares_kernel"); rc != EG_OK) return rc;
  }
  if (!scales) {
    norm_of_sums_kernel<<<1, kThreads, 0, (hipStream_t)stream>>>(at, sums, norm);
    return launch_status("norm_of_sums_kernel");
  }
  for (size_t i = launches.size(); i-- > 0;) {
    (small ? scale_kernel<1> : scale_kernel<2>)<<<launches[i].groups, kThreads, 0, (hipStream_t)stream>>>(launches[i].args, at, sums, max_norm, i == 0 ? norm : nullptr);
    if (const int rc = launch_status("scale_kernel"); rc != EG_OK) return rc;
  }
  return EG_OK;
} catch (...) {
  return set_error(EG_ERR_HIP, "clip: no host memory for %lld tensors", (long long)count);
}

}  // extern "C"
