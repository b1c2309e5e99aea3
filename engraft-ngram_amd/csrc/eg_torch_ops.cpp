// The losses', the weight updates', the 8-bit products' and the norms' calls from torch tensors: argument
// checks, output and workspace allocation and the library call in one C++ function
// each.  From Python through ctypes the same calls take 10 us (a loss) to 100 us (a
// step of 16 matrices) of interpreter time, more than the kernels of a small one.
// Host code only, in the autograd module; the entry points are the library's own,
// handed over as addresses.
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <cstdint>
#include <map>
#include <optional>
#include <sstream>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "eg_overlap.h"
#include "engraft_ngram.h"

namespace {

using torch::Tensor;
using MaybeTensor = std::optional<Tensor>;

struct Entry {
  decltype(&eg_loss_workspace_size) loss_workspace = nullptr;
  decltype(&eg_token_logprobs) token_logprobs = nullptr;
  decltype(&eg_policy_loss) policy = nullptr;
  decltype(&eg_preference_loss) preference = nullptr;
  decltype(&eg_logits_grad) logits_grad = nullptr;
  decltype(&eg_muon_workspace_size) muon_workspace = nullptr;
  decltype(&eg_muon_check) muon_check = nullptr;
  decltype(&eg_muon_step) muon = nullptr;
  decltype(&eg_fp8_quantize) fp8_quantize = nullptr;
  decltype(&eg_fp8_quantize_weight) fp8_quantize_weight = nullptr;
  decltype(&eg_fp8_dequantize) fp8_dequantize = nullptr;
  decltype(&eg_fp8_product) fp8_product = nullptr;
  decltype(&eg_fp8_product_workspace_size) fp8_product_workspace = nullptr;
  decltype(&eg_fp8_linear) fp8_linear = nullptr;
  decltype(&eg_fp8_linear_workspace_size) fp8_linear_workspace = nullptr;
  decltype(&eg_add_rms_norm) norm = nullptr;
  decltype(&eg_add_rms_norm_grad) norm_grad = nullptr;
  decltype(&eg_add_rms_norm_grad_workspace_size) norm_grad_workspace = nullptr;
  decltype(&eg_clip_grads) clip = nullptr;
  decltype(&eg_clip_workspace_size) clip_workspace = nullptr;
  decltype(&eg_last_error) last_error = nullptr;
};
Entry g;
pybind11::handle g_error;  // _lib.EgError, held for good (it may not be released after the interpreter)

// The ctypes path's exceptions: EG_ERR_ARG a ValueError, any other status an EgError.
void check(int rc) {
  if (rc == EG_OK) return;
  const std::string msg = g.last_error();
  if (rc == EG_ERR_ARG) throw std::invalid_argument(msg);
  PyErr_SetObject(g_error.ptr(), g_error(rc, msg).ptr());
  throw pybind11::error_already_set();
}

template <typename... Parts>
[[noreturn]] void refuse(const Parts&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw std::invalid_argument(s.str());
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return EG_DTYPE_F32;
    case torch::kBFloat16: return EG_DTYPE_BF16;
    case torch::kFloat16: return EG_DTYPE_F16;
    default: return -1;
  }
}

// The library wrote t: torch's in-place operations count as its version, which saved tensors
// and the PLE block's kept weight planes go by.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ---- losses -------------------------------------------------------------------------------------

Tensor integers(const Tensor& x, int64_t n, const char* name, const torch::Device& dev) {
  if (x.device() != dev || x.dim() != 1 || x.size(0) != n)
    refuse(name, " must be [", n, "] on ", dev, ", got ", x.sizes(), " on ", x.device());
  if (x.scalar_type() != torch::kInt64 && x.scalar_type() != torch::kInt32)
    refuse(name, " must be int64 or int32, got ", x.scalar_type());
  return x.contiguous();
}

Tensor floats(const Tensor& x, int64_t n, const char* name, const torch::Device& dev) {
  if (x.device() != dev || x.dim() != 1 || x.size(0) != n || !x.is_floating_point())
    refuse(name, " must be floating [", n, "] on ", dev, ", got ", x.scalar_type(), " ", x.sizes(), " on ", x.device());
  return x.to(torch::kFloat32).contiguous();
}

int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1)); }

struct Logits {
  eg_logits c;
  Tensor targets;
};

Logits make_logits(const Tensor& z, const Tensor& targets, double temperature) {
  if (z.dim() != 2 || dtype_code(z) < 0 || !z.is_cuda())
    refuse("logits must be f32, bf16 or f16 [n, vocab] on the GPU, got ", z.scalar_type(), " ", z.sizes(), " on ",
           z.device());
  if (z.size(1) > 1 && z.stride(1) != 1)
    refuse("logits must have unit stride within a row, got strides ", z.strides());
  Logits l;
  l.targets = integers(targets, z.size(0), "targets", z.device());
  l.c = {z.size(0) > 0 ? z.data_ptr() : nullptr,
         dtype_code(z),
         l.targets.scalar_type() == torch::kInt32,
         z.size(0),
         z.size(1),
         row_stride(z),
         z.size(0) > 0 ? l.targets.data_ptr() : nullptr,
         (float)temperature};
  return l;
}

// One buffer of a call: its rows' state (12 bytes each), then the workspace.
struct Scratch {
  Tensor buffer;
  char* at;
  int64_t first, size;
};

Scratch make_scratch(const Logits& l, int64_t segments, bool state, const Tensor& like) {
  Scratch s;
  s.size = g.loss_workspace(l.c.n, l.c.v, l.c.dtype, segments);
  if (s.size < 0) refuse("a loss of ", l.c.n, " rows, a vocabulary of ", l.c.v, " and ", segments, " segments");
  s.first = state ? (12 * l.c.n + 15) / 16 * 16 : 0;
  s.buffer = torch::empty({s.first + s.size}, like.options().dtype(torch::kUInt8));
  s.at = (char*)s.buffer.data_ptr();
  return s;
}

Tensor empty_floats(int64_t n, const Tensor& like) { return torch::empty({n}, like.options().dtype(torch::kFloat32)); }

// Where a gradient is written: `out`, or a new tensor; undefined without one.
Tensor gradient(const Tensor& z, bool wanted, const MaybeTensor& out) {
  if (!wanted) return Tensor();
  if (!out) return torch::empty(z.sizes(), z.options());
  if (out->sizes() != z.sizes() || out->scalar_type() != z.scalar_type() || out->device() != z.device() ||
      (out->size(1) > 1 && out->stride(1) != 1))
    refuse("out must be ", z.scalar_type(), " ", z.sizes(), " on ", z.device(), " with unit stride within a row");
  return *out;
}

void* rows_of(const Tensor& d, int64_t n) { return d.defined() && n > 0 ? d.data_ptr() : nullptr; }

Tensor part(const Tensor& t, int64_t first, int64_t count) { return t.as_strided({count}, {1}, first); }
Tensor scalar(const Tensor& t, int64_t at) { return t.as_strided({}, {}, at); }

const float* values(const Tensor& t) { return (const float*)t.data_ptr(); }

Tensor token_logprobs(const Tensor& logits, const Tensor& targets, double temperature, int64_t stream) {
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const c10::OptionalDeviceGuard on(logits.is_cuda() ? std::optional<c10::Device>(logits.device()) : std::nullopt);
  const Logits l = make_logits(logits, targets, temperature);
  Tensor lp = empty_floats(l.c.n, logits);
  const Scratch s = make_scratch(l, 0, false, logits);
  check(g.token_logprobs(&l.c, (float*)lp.data_ptr(), s.at, s.size, (void*)stream));
  return lp;
}

// (state and workspace, loss, KL, clipped share, log-probabilities, d_logits)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, MaybeTensor> policy(const Tensor& logits, const Tensor& targets, const Tensor& advantages,
                                          const MaybeTensor& old_lp, const MaybeTensor& ref_lp, const MaybeTensor& ids,
                                          int64_t segments, double low, double high, double kl_coef,
                                          double temperature, int64_t reduction, bool grad,
                                          const MaybeTensor& out, double grad_scale, int64_t stream) {
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const c10::OptionalDeviceGuard on(logits.is_cuda() ? std::optional<c10::Device>(logits.device()) : std::nullopt);
  const Logits l = make_logits(logits, targets, temperature);
  const int64_t n = l.c.n;
  const auto dev = logits.device();
  const Tensor a = floats(advantages, n, "advantages", dev);
  eg_policy p = {};
  p.advantages = values(a);
  Tensor o, r, i;
  if (old_lp) p.old_logprobs = values(o = floats(*old_lp, n, "old_logprobs", dev));
  if (ref_lp) p.ref_logprobs = values(r = floats(*ref_lp, n, "ref_logprobs", dev));
  p.reduction = (int32_t)reduction;
  if (reduction == EG_REDUCE_SEQUENCE) {
    i = integers(*ids, n, "segment_ids", dev);
    p.segment_ids = i.data_ptr();
    p.segment_ids_i32 = i.scalar_type() == torch::kInt32;
    p.n_segments = segments;
  }
  p.clip_low = (float)low;
  p.clip_high = (float)high;
  p.kl_coef = (float)kl_coef;
  const Scratch s = make_scratch(l, std::max<int64_t>(p.n_segments, 0), true, logits);
  const Tensor d = gradient(logits, grad, out);
  Tensor sums = empty_floats(3, logits), lp = empty_floats(n, logits);
  check(g.policy(&l.c, &p, (float*)lp.data_ptr(), (float*)sums.data_ptr(), (float*)s.at, rows_of(d, n),
                 d.defined() ? row_stride(d) : 0, (float)grad_scale, s.at + s.first, s.size, (void*)stream));
  if (out) written(d);
  return {s.buffer, scalar(sums, 0), scalar(sums, 1), scalar(sums, 2), lp, d.defined() ? MaybeTensor(d) : std::nullopt};
}

// (state and workspace, loss, margins, the sequences' sums, log-probabilities, d_logits)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, MaybeTensor> preference(const Tensor& logits, const Tensor& targets, const Tensor& ids,
                                              const Tensor& ref_lp, double beta, double smoothing, double temperature,
                                              bool grad, const MaybeTensor& out, double grad_scale, int64_t stream) {
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const c10::OptionalDeviceGuard on(logits.is_cuda() ? std::optional<c10::Device>(logits.device()) : std::nullopt);
  const Logits l = make_logits(logits, targets, temperature);
  const int64_t n = l.c.n;
  const auto dev = logits.device();
  if (ref_lp.dim() != 1 || ref_lp.size(0) < 2 || ref_lp.size(0) % 2 != 0)
    refuse("ref_logprobs must be [2 * pairs] (chosen, rejected, ...), got ", ref_lp.sizes());
  const int64_t count = ref_lp.size(0), pairs = count / 2;
  const Tensor r = floats(ref_lp, count, "ref_logprobs", dev), i = integers(ids, n, "segment_ids", dev);
  const eg_preference p = {i.data_ptr(), values(r), pairs, i.scalar_type() == torch::kInt32, (float)beta,
                           (float)smoothing};
  const Scratch s = make_scratch(l, count, true, logits);
  const Tensor d = gradient(logits, grad, out);
  Tensor sums = empty_floats(1 + pairs + count, logits), lp = empty_floats(n, logits);
  float* to = (float*)sums.data_ptr();
  check(g.preference(&l.c, &p, (float*)lp.data_ptr(), to + 1 + pairs, to + 1, to, (float*)s.at, rows_of(d, n),
                     d.defined() ? row_stride(d) : 0, (float)grad_scale, s.at + s.first, s.size, (void*)stream));
  if (out) written(d);
  return {s.buffer, scalar(sums, 0), part(sums, 1, pairs), part(sums, 1 + pairs, count), lp,
          d.defined() ? MaybeTensor(d) : std::nullopt};
}

Tensor logits_grad(const Tensor& logits, const Tensor& targets, double temperature, const Tensor& state,
                   const Tensor& upstream, int64_t stream) {
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const c10::OptionalDeviceGuard on(logits.is_cuda() ? std::optional<c10::Device>(logits.device()) : std::nullopt);
  const Tensor d = gradient(logits, true, std::nullopt);
  const Logits l = make_logits(logits, targets, temperature);
  const Tensor up = upstream.to(torch::kFloat32);
  check(g.logits_grad(&l.c, values(state), values(up), 1.0f, rows_of(d, l.c.n), row_stride(d), (void*)stream));
  return d;
}

// ---- the orthogonalised step --------------------------------------------------------------------

void check_matrix(const Tensor& t, const char* name, const Tensor* like) {
  if ((t.dim() != 2 && t.dim() != 3) || dtype_code(t) < 0 || !t.is_cuda())
    refuse(name, " must be f32, bf16 or f16 [rows, cols] or [count, rows, cols] on the GPU, got ", t.scalar_type(), " ",
           t.sizes(), " on ", t.device());
  if (like != nullptr && (t.sizes() != like->sizes() || t.device() != like->device()))
    refuse(name, " must be ", like->sizes(), " on ", like->device(), ", got ", t.sizes(), " on ", t.device());
}

void check_writable(const Tensor& t, const char* name) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.stride(i) == 0 && t.size(i) > 1)
      refuse(name, " is written and must not be expanded, got strides ", t.strides());
}

// A momentum step of params (update), or the orthogonalised grads written to params (no momenta): of
// all of them, or of none where one is refused or the workspace is not to be had.
// planes 0: two, but for a bf16 X alone, which is rounded to 8 bits when it is written: one.
void muon(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& momenta,
          const std::vector<float>& coefficients, int64_t steps, int64_t planes, bool nesterov, double momentum,
          double eps, double keep, double lr, bool update, int64_t stream) {
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const c10::OptionalDeviceGuard on(!params.empty() && params[0].is_cuda() ? std::optional<c10::Device>(params[0].device()) : std::nullopt);
  if (params.size() != grads.size() || (update && params.size() != momenta.size()))
    refuse(params.size(), " params, ", grads.size(), " grads and ", momenta.size(), " momenta");
  // matrices of one shape, types and strides share their launches
  using Key = std::tuple<int64_t, int64_t, int, int, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t>;
  struct Group {
    std::vector<size_t> members;
    eg_muon call;
    std::vector<void*> params;
    std::vector<const void*> grads;
    std::vector<float*> momenta;
  };
  std::map<Key, Group> groups;
  std::vector<eg::Operand> operands;  // of all groups: one may not write what another's launches still read
  size_t matrices = 0;
  for (size_t i = 0; i < params.size(); ++i) {
    const Tensor &w = params[i], &d = grads[i];
    if (update) check_matrix(w, "params", nullptr);
    if (w.device() != params[0].device())
      refuse("params must be on one device, got ", params[0].device(), " and ", w.device());
    check_matrix(d, update ? "grads" : "x", update ? &w : nullptr);
    if (!update) check_matrix(w, "out", &d);
    check_writable(w, update ? "params" : "out");
    if (update) {
      check_matrix(momenta[i], "momenta", &w);
      if (momenta[i].scalar_type() != torch::kFloat32) refuse("momenta must be f32, got ", momenta[i].scalar_type());
      check_writable(momenta[i], "momenta");
    }
    if (w.numel() == 0) continue;
    const int64_t r = w.dim() - 2, c = w.dim() - 1;
    const Tensor* m = update ? &momenta[i] : nullptr;
    Group& to = groups[Key{w.size(r), w.size(c), dtype_code(w), dtype_code(d), w.stride(r), w.stride(c), d.stride(r),
                           d.stride(c), m ? m->stride(r) : 0, m ? m->stride(c) : 0}];
    to.members.push_back(i);
    const int64_t count = w.dim() == 3 ? w.size(0) : 1;
    for (int64_t k = 0; k < count; ++k) {
      auto matrix = [&](const Tensor& t, eg::Operand::Kind kind) {
        char* at = (char*)t.data_ptr() + (count > 1 ? k * t.stride(0) * (int64_t)t.element_size() : 0);
        operands.push_back({kind, matrices, {at, t.size(r), t.size(c), t.stride(r), t.stride(c), (int64_t)t.element_size()}});
        return at;
      };
      to.params.push_back(matrix(w, eg::Operand::kParam));
      to.grads.push_back(matrix(d, eg::Operand::kGrad));
      if (m) to.momenta.push_back((float*)matrix(*m, eg::Operand::kMomentum));
      ++matrices;
    }
  }
  // everything that can be refused comes before the first launch; the groups are checked by themselves first
  int64_t need = 0;
  for (auto& [key, group] : groups) {
    eg_muon& o = group.call = {};
    int64_t* const strides[3] = {o.param_stride, o.grad_stride, o.momentum_stride};
    std::tie(o.rows, o.cols, o.param_dtype, o.grad_dtype, strides[0][0], strides[0][1], strides[1][0], strides[1][1],
             strides[2][0], strides[2][1]) = key;
    o.count = (int32_t)group.params.size();
    // one plane's X is 1.1e-3 of itself off: less than bf16's rounding of X, but a step's weights are the
    // fp32 update's only with two (with one, 1.3 to 4.6 % of bf16 weights round the other way)
    o.planes = planes != 0 ? (int32_t)planes : !update && o.param_dtype == EG_DTYPE_BF16 ? 1 : 2;
    o.params = group.params.data();
    o.grads = group.grads.data();
    o.momenta = update ? group.momenta.data() : nullptr;
    o.coefficients = coefficients.data();
    o.steps = (int32_t)steps;
    o.nesterov = nesterov;
    o.momentum = (float)momentum;
    o.eps = (float)eps;
    o.keep = update ? (float)keep : 0.0f;
    o.rate = update ? (float)(lr * std::sqrt(std::max(1.0, (double)o.rows / (double)o.cols))) : -1.0f;
    check(g.muon_check(&o));
    need = std::max(need, g.muon_workspace(o.rows, o.cols, o.count, o.planes));
  }
  if (groups.empty()) return;
  if (groups.size() > 1) {
    const eg::Operand *x, *y;
    if (eg::find_overlap(operands, x, y))
      refuse(eg::name_of(x->kind), " of matrix ", x->matrix, " overlap ", eg::name_of(y->kind), " of matrix ", y->matrix);
  }
  // from torch's allocator on the current stream, which owns it until the work is done; the groups
  // take turns with it
  const Tensor ws = torch::empty({need}, params[0].options().dtype(torch::kUInt8));
  for (auto& [key, group] : groups) {
    const int rc = g.muon(&group.call, ws.data_ptr(), need, (void*)stream);
    for (const size_t i : group.members) {  // some launches may be on their way whatever came of the rest
      written(params[i]);
      if (update) written(momenta[i]);
    }
    check(rc);
  }
}

// ---- products of 8-bit blocks --------------------------------------------------------------------

// torch::empty on like's GPU, without the dispatcher's way there (0.3 us of 1.1)
Tensor fresh(at::IntArrayRef sizes, torch::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

// A forward-mode derivative of an input, which requires_grad does not show, would be lost.
void no_tangent(const Tensor& t) {
  if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    throw std::runtime_error("forward-mode derivatives are not implemented for this operator");
}

std::optional<c10::Device> gpu_of(const Tensor& t) {
  return t.is_cuda() ? std::optional<c10::Device>(t.device()) : std::nullopt;
}

torch::ScalarType type_of(int64_t code, const char* name) {
  switch (code) {
    case EG_DTYPE_F32: return torch::kFloat32;
    case EG_DTYPE_BF16: return torch::kBFloat16;
    case EG_DTYPE_F16: return torch::kFloat16;
    default: refuse(name, " must be f32, bf16 or f16");
  }
}

// Rows of unit stride that lie apart: the tensor itself, or a copy (of a transpose, of expanded rows).
Tensor rows_2d(const Tensor& t, const char* name) {
  if (t.dim() != 2 || dtype_code(t) < 0 || !t.is_cuda())
    refuse(name, " must be f32, bf16 or f16 [rows, cols] on the GPU, got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
  const bool fits = (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
  return fits ? t : t.contiguous();
}

eg_fp8_matrix blocks_of(const Tensor& q, const Tensor& scales, int64_t k, int32_t block_rows, const char* name, const torch::Device& dev) {
  if (q.dim() != 2 || q.scalar_type() != torch::kFloat8_e4m3fn || q.device() != dev || !q.is_cuda())
    refuse(name, ": q must be float8_e4m3fn [rows, k in whole blocks] on ", dev, ", got ", q.scalar_type(), " ", q.sizes(), " on ", q.device());
  const int64_t rows = q.size(0), blocks = (k + 127) / 128;
  if (k < 1 || q.size(1) < blocks * 128 || (q.size(1) > 1 && q.stride(1) != 1))
    refuse(name, ": rows of q must hold the ", blocks, " blocks of k=", k, " at unit stride, got ", q.sizes(), " with strides ", q.strides());
  if (scales.dim() != 2 || scales.scalar_type() != torch::kFloat8_e8m0fnu || scales.device() != dev ||
      scales.size(0) != (rows + block_rows - 1) / block_rows || scales.size(1) < (blocks + 3) / 4 * 4 ||
      (scales.size(1) > 1 && scales.stride(1) != 1))
    refuse(name, ": scales must be float8_e8m0fnu [", (rows + block_rows - 1) / block_rows, ", ", (blocks + 3) / 4 * 4, "] on ", dev,
           " at unit stride, got ", scales.scalar_type(), " ", scales.sizes(), " on ", scales.device());
  return {rows > 0 ? q.data_ptr() : nullptr, rows > 0 ? (uint8_t*)scales.data_ptr() : nullptr, rows, k, row_stride(q),
          row_stride(scales), block_rows};
}

std::pair<Tensor, Tensor> empty_blocks(int64_t rows, int64_t k, int64_t block_rows, const Tensor& like) {
  const int64_t blocks = (k + 127) / 128;
  return {fresh({rows, blocks * 128}, torch::kFloat8_e4m3fn, like),
          fresh({(rows + block_rows - 1) / block_rows, (blocks + 3) / 4 * 4}, torch::kFloat8_e8m0fnu, like)};
}

// (q, scales)
std::tuple<Tensor, Tensor> fp8_quantize(const Tensor& x_, int64_t stream) {
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const c10::OptionalDeviceGuard on(gpu_of(x_));
  const Tensor x = rows_2d(x_, "x");
  if (x.size(1) < 1) refuse("x must have at least one column");
  const auto [q, scales] = empty_blocks(x.size(0), x.size(1), 1, x);
  const eg_fp8_matrix out = blocks_of(q, scales, x.size(1), 1, "x", x.device());
  check(g.fp8_quantize(rows_of(x, x.size(0)), dtype_code(x), row_stride(x), &out, (void*)stream));
  return {q, scales};
}

// (q, scales, the transpose's q and scales)
std::tuple<Tensor, Tensor, MaybeTensor, MaybeTensor> fp8_quantize_weight(const Tensor& w, bool transpose, int64_t stream) {
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const c10::OptionalDeviceGuard on(gpu_of(w));
  if (w.dim() != 2 || dtype_code(w) < 0 || !w.is_cuda() || w.size(0) < 1 || w.size(1) < 1)
    refuse("a weight must be f32, bf16 or f16 [n, k] on the GPU, got ", w.scalar_type(), " ", w.sizes(), " on ", w.device());
  const auto [q, scales] = empty_blocks(w.size(0), w.size(1), 128, w);
  const eg_fp8_matrix out = blocks_of(q, scales, w.size(1), 128, "weight", w.device());
  if (!transpose) {
    check(g.fp8_quantize_weight(w.data_ptr(), dtype_code(w), w.stride(0), w.stride(1), &out, nullptr, (void*)stream));
    return {q, scales, std::nullopt, std::nullopt};
  }
  const auto [qt, scales_t] = empty_blocks(w.size(1), w.size(0), 128, w);
  const eg_fp8_matrix out_t = blocks_of(qt, scales_t, w.size(0), 128, "weight", w.device());
  check(g.fp8_quantize_weight(w.data_ptr(), dtype_code(w), w.stride(0), w.stride(1), &out, &out_t, (void*)stream));
  return {q, scales, qt, scales_t};
}

Tensor fp8_dequantize(const Tensor& q, const Tensor& scales, int64_t k, int64_t block_rows, int64_t dtype, int64_t stream) {
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const c10::OptionalDeviceGuard on(gpu_of(q));
  const eg_fp8_matrix m = blocks_of(q, scales, k, (int32_t)block_rows, "blocks", q.device());
  const Tensor out = fresh({m.rows, k}, type_of(dtype, "dtype"), q);
  check(g.fp8_dequantize(&m, rows_of(out, m.rows), (int32_t)dtype, k, (void*)stream));
  return out;
}

struct Outputs {
  std::vector<Tensor> y;
  eg_fp8_matrix b[2];
  void* at[2] = {nullptr, nullptr};
  int64_t ld[2] = {0, 0};
  bool two;
};

// The weight's rows in one group, or in two from row `split` on, and an output for each.
Outputs outputs(int64_t m, const eg_fp8_matrix& w, int64_t split, int64_t dtype, const Tensor& like) {
  Outputs o;
  o.two = split > 0;
  if (o.two && (split % 128 != 0 || split >= w.rows)) refuse("split must be a multiple of 128 below the weight's ", w.rows, " rows, got ", split);
  o.b[0] = o.b[1] = w;
  if (o.two) {
    o.b[0].rows = split;
    o.b[1].rows = w.rows - split;
    o.b[1].q = (char*)w.q + split * w.stride;
    o.b[1].scales = w.scales + split / 128 * w.scale_stride;
  }
  for (int i = 0; i < (o.two ? 2 : 1); ++i) {
    o.y.push_back(fresh({m, o.b[i].rows}, type_of(dtype, "out_dtype"), like));
    o.at[i] = o.y[i].numel() > 0 ? o.y[i].data_ptr() : nullptr;
    o.ld[i] = o.b[i].rows;
  }
  return o;
}

// `differentiable`: for a caller whose x may have a derivative
std::vector<Tensor> fp8_linear(const Tensor& x_, const Tensor& q, const Tensor& scales, int64_t k, int64_t split, int64_t dtype, int64_t stream,
                               bool differentiable) {
  if (differentiable) no_tangent(x_);
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const c10::OptionalDeviceGuard on(gpu_of(x_));
  const Tensor x = rows_2d(x_, "x");
  const eg_fp8_matrix w = blocks_of(q, scales, k, 128, "weight", x.device());
  if (x.size(1) != k) refuse("x must be [m, ", k, "], got ", x.sizes());
  Outputs o = outputs(x.size(0), w, split, dtype, x);
  const int64_t need = g.fp8_linear_workspace(x.size(0), o.b[0].rows, o.two ? o.b[1].rows : 0, k);
  if (need < 0) refuse("a product of ", x.sizes(), " values");
  const Tensor ws = need > 0 ? fresh({need}, torch::kUInt8, x) : Tensor();
  check(g.fp8_linear(rows_of(x, x.size(0)), dtype_code(x), x.size(0), row_stride(x), &o.b[0], o.two ? &o.b[1] : nullptr, o.at[0], o.ld[0],
                     o.at[1], o.ld[1], (int32_t)dtype, need > 0 ? ws.data_ptr() : nullptr, need, (void*)stream));
  return o.y;
}

std::vector<Tensor> fp8_product(const Tensor& xq, const Tensor& x_scales, const Tensor& q, const Tensor& scales, int64_t k, int64_t split,
                                int64_t dtype, int64_t stream) {
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const c10::OptionalDeviceGuard on(gpu_of(xq));
  const eg_fp8_matrix a = blocks_of(xq, x_scales, k, 1, "x", xq.device()), w = blocks_of(q, scales, k, 128, "weight", xq.device());
  Outputs o = outputs(a.rows, w, split, dtype, xq);
  const int64_t need = g.fp8_product_workspace(a.rows, o.b[0].rows, o.two ? o.b[1].rows : 0, k);
  if (need < 0) refuse("a product of ", a.rows, " rows of ", k, " values");
  const Tensor ws = need > 0 ? fresh({need}, torch::kUInt8, xq) : Tensor();
  check(g.fp8_product(&a, &o.b[0], o.two ? &o.b[1] : nullptr, o.at[0], o.ld[0], o.at[1], o.ld[1], (int32_t)dtype,
                      need > 0 ? ws.data_ptr() : nullptr, need, (void*)stream));
  return o.y;
}

// ---- norms ---------------------------------------------------------------------------------------

void check_vector(const MaybeTensor& w, int64_t d, const char* name, const torch::Device& dev) {
  if (w && (w->dim() != 1 || w->size(0) != d || dtype_code(*w) < 0 || w->device() != dev))
    refuse(name, " must be f32, bf16 or f16 [", d, "] on ", dev, ", got ", w->scalar_type(), " ", w->sizes(), " on ", w->device());
}

// (y or its q, y's scales, h, rstd); dtype -1: blocks; `differentiable`: for a caller whose inputs may have a derivative
std::tuple<Tensor, MaybeTensor, Tensor, MaybeTensor> norm(const Tensor& x_, const MaybeTensor& residual, const MaybeTensor& weight, double eps,
                                                          int64_t dtype, bool stats, int64_t stream, bool differentiable) {
  if (differentiable) {
    no_tangent(x_);
    if (residual) no_tangent(*residual);
    if (weight) no_tangent(*weight);
  }
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const c10::OptionalDeviceGuard on(gpu_of(x_));
  const Tensor x = rows_2d(x_, "x");
  const int64_t rows = x.size(0), d = x.size(1);
  if (d < 1) refuse("x must have at least one column");
  Tensor r;
  if (residual) {
    r = rows_2d(*residual, "residual");
    if (r.sizes() != x.sizes() || r.device() != x.device()) refuse("residual must be ", x.sizes(), " on ", x.device(), ", got ", r.sizes(), " on ", r.device());
    if (r.scalar_type() != x.scalar_type() && r.scalar_type() != torch::kFloat32)
      refuse("residual must be of x's type or f32, got ", r.scalar_type(), " beside ", x.scalar_type());
  }
  check_vector(weight, d, "weight", x.device());
  const Tensor w = weight ? weight->to(torch::kFloat32).contiguous() : Tensor();
  const Tensor h = residual ? fresh({rows, d}, r.scalar_type(), r) : x;
  const Tensor rstd = stats ? fresh({rows}, torch::kFloat32, x) : Tensor();
  eg_norm o = {};
  o.x = rows_of(x, rows);
  o.x_dtype = dtype_code(x);
  o.x_stride = row_stride(x);
  if (residual) {
    o.residual = rows_of(r, rows);
    o.r_dtype = dtype_code(r);
    o.r_stride = row_stride(r);
  }
  if (weight) o.weight = values(w);
  o.eps = (float)eps;
  o.rows = rows;
  o.d = d;
  float* const stat = stats && rows > 0 ? (float*)rstd.data_ptr() : nullptr;
  void* const sum = residual ? rows_of(h, rows) : nullptr;
  if (dtype < 0) {
    const auto [q, scales] = empty_blocks(rows, d, 1, x);
    const eg_fp8_matrix y = blocks_of(q, scales, d, 1, "y", x.device());
    check(g.norm(&o, sum, d, nullptr, 0, 0, &y, stat, (void*)stream));
    return {q, scales, h, stats ? MaybeTensor(rstd) : std::nullopt};
  }
  const Tensor y = fresh({rows, d}, type_of(dtype, "out_dtype"), x);
  check(g.norm(&o, sum, d, rows_of(y, rows), (int32_t)dtype, d, nullptr, stat, (void*)stream));
  return {y, std::nullopt, h, stats ? MaybeTensor(rstd) : std::nullopt};
}

// (d_x of `dtype`, the same of `dtype2` (-1: none), the weight's of its type)
std::tuple<Tensor, MaybeTensor, MaybeTensor> norm_grad(const Tensor& d_y_, const Tensor& h_, const Tensor& rstd_, const MaybeTensor& weight,
                                                       const MaybeTensor& d_res, int64_t dtype, int64_t dtype2, bool weight_grad, int64_t stream) {
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const c10::OptionalDeviceGuard on(gpu_of(h_));
  const Tensor h = rows_2d(h_, "h"), d_y = rows_2d(d_y_, "d_y");
  const int64_t rows = h.size(0), d = h.size(1);
  if (d < 1) refuse("h must have at least one column");
  if (d_y.sizes() != h.sizes() || d_y.device() != h.device()) refuse("d_y must be ", h.sizes(), " on ", h.device(), ", got ", d_y.sizes(), " on ", d_y.device());
  if (rstd_.dim() != 1 || rstd_.size(0) != rows || rstd_.scalar_type() != torch::kFloat32 || rstd_.device() != h.device())
    refuse("rstd must be f32 [", rows, "] on ", h.device(), ", got ", rstd_.scalar_type(), " ", rstd_.sizes(), " on ", rstd_.device());
  const Tensor rstd = rstd_.contiguous();
  check_vector(weight, d, "weight", h.device());
  if (weight_grad && !weight) refuse("the weight's gradient without a weight");
  const Tensor w = weight ? weight->to(torch::kFloat32).contiguous() : Tensor();
  Tensor dr;
  if (d_res) {
    dr = rows_2d(*d_res, "d_residual");
    if (dr.sizes() != h.sizes() || dr.device() != h.device() || dr.scalar_type() != h.scalar_type())
      refuse("d_residual must be ", h.scalar_type(), " ", h.sizes(), " on ", h.device(), ", got ", dr.scalar_type(), " ", dr.sizes(), " on ", dr.device());
  }
  eg_norm_grad o = {};
  o.d_y = rows_of(d_y, rows);
  o.dy_dtype = dtype_code(d_y);
  o.dy_stride = row_stride(d_y);
  o.h = rows_of(h, rows);
  o.h_dtype = dtype_code(h);
  o.h_stride = row_stride(h);
  if (d_res) {
    o.d_residual = rows_of(dr, rows);
    o.dr_stride = row_stride(dr);
  }
  if (weight) o.weight = values(w);
  o.rstd = rows > 0 ? (const float*)rstd.data_ptr() : nullptr;
  o.rows = rows;
  o.d = d;
  const Tensor d_x = fresh({rows, d}, type_of(dtype, "the gradient's type"), h);
  const Tensor d_x2 = dtype2 >= 0 ? fresh({rows, d}, type_of(dtype2, "the gradient's type"), h) : Tensor();
  const Tensor d_w = weight_grad ? fresh({d}, torch::kFloat32, w) : Tensor();
  const int64_t need = weight_grad ? g.norm_grad_workspace(rows, d) : 0;
  const Tensor ws = need > 0 ? fresh({need}, torch::kUInt8, h) : Tensor();
  check(g.norm_grad(&o, rows_of(d_x, rows), (int32_t)dtype, d, rows_of(d_x2, rows), (int32_t)dtype2, d, weight_grad ? (float*)d_w.data_ptr() : nullptr,
                    need > 0 ? ws.data_ptr() : nullptr, std::max<int64_t>(need, 0), (void*)stream));
  return {d_x, dtype2 >= 0 ? MaybeTensor(d_x2) : std::nullopt, weight_grad ? MaybeTensor(d_w.to(weight->scalar_type())) : std::nullopt};
}

// ---- the norm of all gradients --------------------------------------------------------------------

struct Rows {
  int64_t rows, cols, stride;
};

// A tensor's values as rows of unit stride, in the order of its dimensions; in any order that leaves no
// gaps where `any_order`.
Rows rows_of_any(const Tensor& t, bool any_order, const char* name) {
  if (t.is_contiguous() || (any_order && t.is_non_overlapping_and_dense())) return {1, t.numel(), t.numel()};
  std::vector<std::pair<int64_t, int64_t>> dims;  // size and stride, those that continue one another as one
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.size(i) == 1) continue;
    if (!dims.empty() && dims.back().second == t.size(i) * t.stride(i))
      dims.back() = {dims.back().first * t.size(i), t.stride(i)};
    else
      dims.push_back({t.size(i), t.stride(i)});
  }
  if (dims.size() == 2 && dims[1].second == 1 && dims[0].second >= dims[1].first) return {dims[0].first, dims[1].first, dims[0].second};
  refuse(name, " must be without gaps, or rows of unit stride, got ", t.sizes(), " with strides ", t.strides());
}

// The norm; with `outs` (or in place) the clipped gradients too.
Tensor clip(const std::vector<Tensor>& grads, const std::optional<std::vector<Tensor>>& outs, double max_norm, int64_t stream) {
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  if (grads.empty()) refuse("no gradients");
  if (outs && outs->size() != grads.size()) refuse(grads.size(), " gradients and ", outs->size(), " outputs");
  const c10::OptionalDeviceGuard on(gpu_of(grads[0]));
  std::vector<eg_clip_tensor> tensors;
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor& t = grads[i];
    if (dtype_code(t) < 0 || !t.is_cuda() || t.device() != grads[0].device())
      refuse("gradients must be f32, bf16 or f16 on one GPU, got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
    eg_clip_tensor c = {};
    c.g_dtype = dtype_code(t);
    const Tensor* o = outs ? &(*outs)[i] : nullptr;
    if (o != nullptr && (dtype_code(*o) < 0 || o->device() != t.device() || o->sizes() != t.sizes()))
      refuse("an output must be f32, bf16 or f16 ", t.sizes(), " on ", t.device(), ", got ", o->scalar_type(), " ", o->sizes(), " on ", o->device());
    const bool alike = o == nullptr || o->strides() == t.strides();
    Rows a = rows_of_any(t, alike, "a gradient"), b = o ? rows_of_any(*o, alike, "an output") : a;
    if (a.rows == 1 && b.rows > 1) a = {b.rows, b.cols, b.cols};
    if (b.rows == 1 && a.rows > 1) b = {a.rows, a.cols, a.cols};
    if (a.cols != b.cols) refuse("an output's rows of ", b.cols, " values for a gradient's of ", a.cols);
    c.rows = a.rows;
    c.cols = a.cols;
    c.g_stride = a.stride;
    c.out_stride = b.stride;
    if (t.numel() > 0) {
      c.g = t.data_ptr();
      c.out = o ? o->data_ptr() : nullptr;
    }
    if (o) c.out_dtype = dtype_code(*o);
    tensors.push_back(c);
  }
  const Tensor result = fresh({}, torch::kFloat32, grads[0]);
  const int64_t need = g.clip_workspace(tensors.data(), (int64_t)tensors.size());
  const Tensor ws = fresh({std::max<int64_t>(need, 16)}, torch::kUInt8, grads[0]);
  check(g.clip(tensors.data(), (int64_t)tensors.size(), (float)max_norm, (float*)result.data_ptr(), ws.data_ptr(), std::max<int64_t>(need, 0),
               (void*)stream));
  if (outs)
    for (const Tensor& o : *outs) written(o);
  return result;
}

void init_ops(const std::map<std::string, int64_t>& at, pybind11::object error) {
  auto set = [&](auto& fn, const char* name) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at.at(name)); };
  set(g.loss_workspace, "eg_loss_workspace_size");
  set(g.token_logprobs, "eg_token_logprobs");
  set(g.policy, "eg_policy_loss");
  set(g.preference, "eg_preference_loss");
  set(g.logits_grad, "eg_logits_grad");
  set(g.muon_workspace, "eg_muon_workspace_size");
  set(g.muon_check, "eg_muon_check");
  set(g.muon, "eg_muon_step");
  set(g.fp8_quantize, "eg_fp8_quantize");
  set(g.fp8_quantize_weight, "eg_fp8_quantize_weight");
  set(g.fp8_dequantize, "eg_fp8_dequantize");
  set(g.fp8_product, "eg_fp8_product");
  set(g.fp8_product_workspace, "eg_fp8_product_workspace_size");
  set(g.fp8_linear, "eg_fp8_linear");
  set(g.fp8_linear_workspace, "eg_fp8_linear_workspace_size");
  set(g.norm, "eg_add_rms_norm");
  set(g.norm_grad, "eg_add_rms_norm_grad");
  set(g.norm_grad_workspace, "eg_add_rms_norm_grad_workspace_size");
  set(g.clip, "eg_clip_grads");
  set(g.clip_workspace, "eg_clip_workspace_size");
  set(g.last_error, "eg_last_error");
  g_error = error.release();
}

}  // namespace

void bind_ops(pybind11::module_& m) {
  m.def("init_ops", &init_ops, "addresses of the library's entry points by name, and the error class");
  m.def("token_logprobs", &token_logprobs);
  m.def("policy", &policy);
  m.def("preference", &preference);
  m.def("logits_grad", &logits_grad);
  m.def("muon", &muon);
  m.def("fp8_quantize", &fp8_quantize);
  m.def("fp8_quantize_weight", &fp8_quantize_weight);
  m.def("fp8_dequantize", &fp8_dequantize);
  m.def("fp8_linear", &fp8_linear);
  m.def("fp8_product", &fp8_product);
  m.def("norm", &norm);
  m.def("norm_grad", &norm_grad);
  m.def("clip", &clip);
}
