// The losses' and the orthogonalised step's calls from torch tensors: argument
// checks, output and workspace allocation and the library call in one C++ function
// each.  From Python through ctypes the same calls take 10 us (a loss) to 100 us (a
// step of 16 matrices) of interpreter time, more than the kernels of a small one.
// Host code only, in the autograd module; the entry points are the library's own,
// handed over as addresses.
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
}
