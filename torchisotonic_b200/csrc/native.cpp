// The losses and the optimizer step as Python calls them: torch tensors and autograd over the C ABI
// of include/tiso.h (libtiso.so), as a CPython extension module. Their kernels are short for the
// usual sizes of a token batch, and what a pass costs is the host: with the same calls made from
// Python (ctypes, a Python autograd function) a pass forward and backward took 98 to 110 us of host
// time, 54 of them for an autograd function that does nothing; most of the rest was the interpreter,
// in the forward and, after a hand-over of its lock, in the autograd engine's thread.
//
// The losses take their arguments as they are given and answer None where one of them is to be
// converted or refused, which losses.py does (checked there first, a call took 2 to 6 us more);
// adamw's, lists of tensors, are checked here.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <cstdint>
#include <limits>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/tiso.h"

namespace {

using at::ScalarType;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int rc) {
  if (rc != TISO_OK)
    throw std::runtime_error(std::string("torchisotonic_b200: ") + tiso_last_error() + " (status " +
                             std::to_string(rc) + ")");
}

int dtype_of(ScalarType t) {
  switch (t) {
    case at::kHalf: return TISO_F16;
    case at::kBFloat16: return TISO_BF16;
    case at::kFloat: return TISO_F32;
    case at::kDouble: return TISO_F64;
    default: throw py::type_error("unsupported dtype");
  }
}

ScalarType acc_of(const Tensor& x) {
  return x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat;
}

void* data(const Tensor& t) { return t.data_ptr(); }
void* data(const std::optional<Tensor>& t) { return t ? t->data_ptr() : nullptr; }

Tensor empty(const Tensor& like, at::IntArrayRef sizes, ScalarType type) {
  return at::empty(sizes, like.options().dtype(type));
}

void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

// A Python object's tensor, or NULL for another object.
const Tensor* tensor_in(py::handle h) {
  return THPVariable_Check(h.ptr()) ? &THPVariable_Unpack(h.ptr()) : nullptr;
}

// The capture that the current stream is in, 0 for none.
int64_t capture_of(const Tensor& t) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  const auto stream = c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
  if (cudaStreamGetCaptureInfo(stream, &status, &id) != cudaSuccess) {
    (void)cudaGetLastError();  // the launch says what is wrong
    return 0;
  }
  return status == cudaStreamCaptureStatusActive ? static_cast<int64_t>(id) : 0;
}

// Whether a tensor needs no conversion: of this type, contiguous, and where and of the sizes that go
// with the others.
bool ready(const Tensor* t, ScalarType type, at::IntArrayRef sizes, at::Device device) {
  return t && t->scalar_type() == type && t->device() == device && t->sizes() == sizes &&
         t->is_contiguous();
}

// Refuses tensors with a tangent: the result would be without one, and nothing would tell.
void need_no_tangent(const Tensor& t) {
  if (!t._fw_grad(0).defined()) return;
  PyErr_SetString(PyExc_NotImplementedError,
                  "torchisotonic_b200's losses have no forward-mode derivative");
  throw py::error_already_set();
}
void need_no_tangent(const std::optional<Tensor>& t) {
  if (t) need_no_tangent(*t);
}

bool ready_rows(const Tensor* x, double temperature) {
  if (!x || !x->is_cuda() || x->dim() < 1 || x->size(-1) < 1 || !(temperature > 0)) return false;
  const ScalarType type = x->scalar_type();
  return type == at::kHalf || type == at::kBFloat16 || type == at::kFloat || type == at::kDouble;
}

bool ready_logits(const Tensor* x, const Tensor* targets, double temperature) {
  return ready_rows(x, temperature) &&
         ready(targets, at::kLong, x->sizes().slice(0, x->dim() - 1), x->device());
}

// x ([..., vocab]) as rows of logits, and the tensor whose memory they are: x itself when its last
// dimension is contiguous and the leading ones reduce to two strides, else a contiguous copy.
struct Logits {
  Tensor held;
  tiso_rows rows;

  explicit Logits(const Tensor& x) : held(x) {
    const int64_t dims = x.dim(), vocab = x.size(-1);
    const bool contiguous = x.is_contiguous();
    if (!contiguous && (dims > 3 || (x.stride(-1) != 1 && vocab != 1))) held = x.contiguous();
    const int64_t n = held.numel() / vocab;
    if (contiguous || held.is_contiguous()) {
      rows = {held.data_ptr(), n, n > 0 ? n : 1, 0, vocab, vocab};
    } else if (dims == 3) {
      rows = {held.data_ptr(), n, held.size(1) > 0 ? held.size(1) : 1, held.stride(0),
              held.stride(1), vocab};
    } else {  // one row whose elements are apart only where there is one of them, or two dimensions
      rows = {held.data_ptr(), n, n > 0 ? n : 1, 0, dims == 2 ? held.stride(0) : vocab, vocab};
    }
  }
};

// The steps that the torch.library operators call take tensors as a caller of those operators gives
// them: refused here, by what each has to be.
[[noreturn]] void refuse(const std::string& what) { throw py::value_error(what); }

void need_cuda(const Tensor& t, const char* name) {
  if (!t.is_cuda())
    throw std::runtime_error(
        std::string("torchisotonic_b200 runs on CUDA tensors only (no CPU fallback); move ") + name +
        " to a CUDA device");
}

void need(const Tensor& t, const char* name, ScalarType type, at::IntArrayRef sizes,
          const Tensor& beside) {
  need_no_tangent(t);
  if (t.scalar_type() != type)
    throw py::type_error(std::string(name) + " must be of dtype " + c10::toString(type));
  if (!ready(&t, type, sizes, beside.device())) {
    std::string text;
    for (const int64_t n : sizes) text += (text.empty() ? "" : ", ") + std::to_string(n);
    refuse(std::string(name) + " must be contiguous, of sizes [" + text +
           "] and on the first argument's device");
  }
}

void need(const std::optional<Tensor>& t, const char* name, ScalarType type,
          at::IntArrayRef sizes, const Tensor& beside) {
  if (t) need(*t, name, type, sizes, beside);
}

// An upstream gradient: one number, where the loss is.
void need_scalar(const Tensor& t, ScalarType type, const Tensor& beside) {
  need(t, "upstream", type, t.numel() == 1 ? t.sizes() : at::IntArrayRef(), beside);
}

void need_rows(const Tensor& x) {
  need_cuda(x, "logits");
  need_no_tangent(x);
  if (!x.is_floating_point() || x.element_size() == 1)
    throw py::type_error("logits must be float16, bfloat16, float32 or float64");
  if (x.dim() < 1 || x.size(-1) < 1)
    refuse("logits must have a last dimension of at least one element");
}

void need_logits(const Tensor& x, const Tensor& targets) {
  need_rows(x);
  need(targets, "targets", at::kLong, x.sizes().slice(0, x.dim() - 1), x);
}

void need_list(const Tensor& x, const Tensor& ids) {
  if (ids.dim() != x.dim() || ids.sizes().slice(0, x.dim() - 1) != x.sizes().slice(0, x.dim() - 1))
    refuse("ids must have logits' leading dimensions and one of entries");
  need(ids, "ids", at::kLong, ids.sizes(), x);
}

void need_answers(const Tensor& logps, const std::optional<Tensor>& mask, const Tensor& offsets) {
  need_cuda(logps, "logps");
  need_no_tangent(logps);
  if (logps.scalar_type() != at::kFloat && logps.scalar_type() != at::kDouble)
    throw py::type_error("logps must be float32 or float64");
  if (logps.dim() != 1 || !logps.is_contiguous()) refuse("logps must be contiguous and 1-D");
  need(mask, "mask", at::kBool, logps.sizes(), logps);
  if (offsets.dim() != 1 || offsets.numel() < 3 || offsets.numel() % 2 == 0)
    refuse("offsets must be 1-D with 2 * pairs + 1 entries, pairs >= 1");
  need(offsets, "offsets", at::kLong, offsets.sizes(), logps);
}

// A gradient under create_graph: what depends on it raises when it is differentiated.
Tensor once(const Tensor& grad) {
  if (!grad.defined() || !at::GradMode::is_enabled()) return grad;
  auto raises = std::make_shared<torch::autograd::DelayedError>(
      "torchisotonic_b200's losses are differentiable once", 1);
  return (*raises)({grad.detach().requires_grad_()})[0];
}

// ---------------------------------------------------------------------------------------------
// Token log-probabilities

std::tuple<Tensor, Tensor> logprobs(const Tensor& x, const Tensor& targets, double temperature,
                                    int64_t ignore_index, bool with_stats) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Logits logits(x);
  const ScalarType acc = acc_of(x);
  Tensor out = empty(x, targets.sizes(), acc);
  Tensor stats = with_stats ? empty(x, {2 * logits.rows.rows}, acc) : Tensor();
  check(tiso_logprobs(dtype_of(x.scalar_type()), &logits.rows, targets.data_ptr<int64_t>(),
                      ignore_index, temperature, data(out),
                      with_stats ? data(stats) : nullptr, stream_of(x)));
  return {out, stats};
}

Tensor logprobs_grad(const Tensor& x, const Tensor& targets, double temperature,
                     const Tensor& stats, const Tensor& coef) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Logits logits(x);
  Tensor grad = empty(x, x.sizes(), x.scalar_type());
  check(tiso_logprobs_grad(dtype_of(x.scalar_type()), &logits.rows, targets.data_ptr<int64_t>(),
                           temperature, data(stats), dtype_of(coef.scalar_type()), data(coef),
                           nullptr, data(grad), stream_of(x)));
  return grad;
}

struct Logprobs : torch::autograd::Function<Logprobs> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& targets,
                        double temperature, int64_t ignore_index) {
    auto [out, stats] = logprobs(x, targets, temperature, ignore_index, true);
    ctx->save_for_backward({x, targets, stats});
    ctx->saved_data["temperature"] = temperature;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor grad = logprobs_grad(saved[0], saved[1], ctx->saved_data["temperature"].toDouble(),
                                      saved[2], grads[0].contiguous());
    return {once(grad), Tensor(), Tensor(), Tensor()};
  }
};

std::optional<Tensor> token_logprobs(py::handle logits, py::handle y, double temperature,
                                     int64_t ignore_index) {
  const Tensor *x = tensor_in(logits), *targets = tensor_in(y);
  if (!ready_logits(x, targets, temperature)) return std::nullopt;
  need_no_tangent(*x);
  if (x->requires_grad() && at::GradMode::is_enabled())
    return Logprobs::apply(*x, *targets, temperature, ignore_index);
  return std::get<0>(logprobs(*x, *targets, temperature, ignore_index, false));
}

// ---------------------------------------------------------------------------------------------
// Preference loss

struct Preference : torch::autograd::Function<Preference> {
  static tiso_preference_args args_of(const Tensor& logps, const std::optional<Tensor>& refs,
                                      const std::optional<Tensor>& mask, const Tensor& offsets) {
    tiso_preference_args args{};
    args.logps = data(logps);
    args.ref_logps = data(refs);
    args.mask = static_cast<const uint8_t*>(data(mask));
    args.offsets = offsets.data_ptr<int64_t>();
    args.tokens = logps.numel();
    args.pairs = (offsets.numel() - 1) / 2;
    args.beta = 1.0;
    return args;
  }

  // loss, rewards and, kept for the backward, the sequences' coefficients (the workspace is behind
  // them: one allocation)
  static std::tuple<Tensor, Tensor, Tensor> run(const Tensor& logps,
                                                const std::optional<Tensor>& refs,
                                                const std::optional<Tensor>& mask,
                                                const Tensor& offsets, int64_t kind, bool average,
                                                double beta, double label_smoothing,
                                                double margin) {
    const c10::cuda::CUDAGuard guard(logps.device());
    const ScalarType type = logps.scalar_type();
    tiso_preference_args args = args_of(logps, refs, mask, offsets);
    args.kind = static_cast<int>(kind);
    args.average = average;
    args.beta = beta;
    args.label_smoothing = label_smoothing;
    args.margin = margin;
    size_t bytes = 0;
    check(tiso_preference_workspace_size(args.pairs, &bytes));
    const int64_t each = logps.element_size(), behind = (2 * args.pairs * each + 7) / 8 * 8;
    Tensor loss = empty(logps, {}, type), rewards = empty(logps, {2, args.pairs}, type);
    Tensor coef = empty(logps, {(behind + static_cast<int64_t>(bytes)) / each}, type);
    check(tiso_preference(dtype_of(type), &args, data(loss), data(rewards), data(coef),
                          static_cast<char*>(data(coef)) + behind, bytes, stream_of(logps)));
    return {loss, rewards, coef};
  }

  static std::tuple<Tensor, Tensor> run_grad(const Tensor& logps, const std::optional<Tensor>& mask,
                                             const Tensor& offsets, const Tensor& coef,
                                             const Tensor& upstream, bool want, bool want_ref) {
    const c10::cuda::CUDAGuard guard(logps.device());
    const tiso_preference_args args = args_of(logps, std::nullopt, mask, offsets);
    Tensor grad, grad_ref;
    if (want) grad = empty(logps, logps.sizes(), logps.scalar_type());
    if (want_ref) grad_ref = empty(logps, logps.sizes(), logps.scalar_type());
    check(tiso_preference_grad(dtype_of(logps.scalar_type()), &args, data(coef), data(upstream),
                               want ? data(grad) : nullptr, want_ref ? data(grad_ref) : nullptr,
                               stream_of(logps)));
    return {grad, grad_ref};
  }

  static variable_list forward(AutogradContext* ctx, const Tensor& logps,
                               const std::optional<Tensor>& refs, const std::optional<Tensor>& mask,
                               const Tensor& offsets, int64_t kind, bool average, double beta,
                               double label_smoothing, double margin) {
    auto [loss, rewards, coef] =
        run(logps, refs, mask, offsets, kind, average, beta, label_smoothing, margin);
    ctx->save_for_backward({logps, mask.value_or(Tensor()), offsets, coef});
    ctx->saved_data["ref"] = refs.has_value() && refs->requires_grad();
    ctx->saved_data["logps"] = logps.requires_grad();
    ctx->mark_non_differentiable({rewards});
    ctx->set_materialize_grads(false);
    return {loss, rewards};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(9);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto mask = saved[1].defined() ? std::optional<Tensor>(saved[1]) : std::nullopt;
    auto [grad, grad_ref] =
        run_grad(saved[0], mask, saved[2], saved[3], grads[0], ctx->saved_data["logps"].toBool(),
                 ctx->saved_data["ref"].toBool());
    out[0] = once(grad);
    out[1] = once(grad_ref);
    return out;
  }
};

std::optional<std::tuple<Tensor, Tensor>> preference_loss(py::handle of_logps, py::handle of_refs,
                                                          py::handle of_mask, py::handle of_offsets,
                                                          int64_t kind, bool average, double beta,
                                                          double label_smoothing, double margin) {
  const Tensor *logps = tensor_in(of_logps), *offsets = tensor_in(of_offsets);
  if (!logps || !logps->is_cuda() || logps->dim() != 1 || !offsets || offsets->dim() != 1 ||
      offsets->numel() < 3 || offsets->numel() % 2 == 0)
    return std::nullopt;
  const ScalarType type = logps->scalar_type();
  const at::Device device = logps->device();
  if (kind < 0 || !(beta > 0) || !(label_smoothing >= 0 && label_smoothing < 0.5) ||
      (type != at::kFloat && type != at::kDouble) || !ready(logps, type, logps->sizes(), device) ||
      !ready(offsets, at::kLong, offsets->sizes(), device))
    return std::nullopt;
  std::optional<Tensor> refs, mask;
  if (!of_refs.is_none()) {
    const Tensor* t = tensor_in(of_refs);
    if (!ready(t, type, logps->sizes(), device)) return std::nullopt;
    refs = *t;
  }
  if (!of_mask.is_none()) {
    const Tensor* t = tensor_in(of_mask);
    if (!ready(t, at::kBool, logps->sizes(), device)) return std::nullopt;
    mask = *t;
  }
  need_no_tangent(*logps);
  need_no_tangent(refs);
  if (at::GradMode::is_enabled() &&
      (logps->requires_grad() || (refs.has_value() && refs->requires_grad()))) {
    const variable_list out = Preference::apply(*logps, refs, mask, *offsets, kind, average, beta,
                                                label_smoothing, margin);
    return std::make_tuple(out[0], out[1]);
  }
  auto [loss, rewards, coef] =
      Preference::run(*logps, refs, mask, *offsets, kind, average, beta, label_smoothing, margin);
  return std::make_tuple(loss, rewards);
}

// ---------------------------------------------------------------------------------------------
// Policy loss

struct PolicySettings {
  Tensor targets, old_logps, advantages;
  std::optional<Tensor> ref_logps, weight;
  int64_t ignore_index;
  double temperature, clip_low, clip_high, kl_coef;
};

struct PolicyResult {
  Tensor out, logps, kept, grad;  // out: loss, kl, clip fraction
};

// kept: n numbers coef, up to 2 n stats, the workspace (one allocation, in double).
PolicyResult policy(const Tensor& x, const PolicySettings& s, bool with_grad) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Logits logits(x);
  const ScalarType acc = acc_of(x);
  const int dtype = dtype_of(x.scalar_type());
  const int64_t n = logits.rows.rows;
  tiso_policy_args args{};
  args.old_logps = data(s.old_logps);
  args.ref_logps = data(s.ref_logps);
  args.advantages = data(s.advantages);
  args.weight = data(s.weight);
  args.weight_is_byte = s.weight && s.weight->scalar_type() == at::kBool;
  args.clip_low = s.clip_low;
  args.clip_high = s.clip_high;
  args.kl_coef = s.kl_coef;
  size_t bytes = 0;
  check(tiso_policy_workspace_size(dtype, n, &bytes));
  PolicyResult r{empty(x, {3}, acc), empty(x, s.targets.sizes(), acc),
                 empty(x, {3 * n + static_cast<int64_t>((bytes + 7) / 8)}, at::kDouble), Tensor()};
  if (with_grad) r.grad = empty(x, x.sizes(), x.scalar_type());
  double* at = r.kept.data_ptr<double>();
  check(tiso_policy(dtype, &logits.rows, s.targets.data_ptr<int64_t>(), s.ignore_index,
                    s.temperature, &args, data(r.logps), at, at + n, data(r.out),
                    with_grad ? data(r.grad) : nullptr, at + 3 * n, bytes, stream_of(x)));
  return r;
}

// Loss, kl and clip fraction as tensors of their own: parts of `out` that autograd does not take for
// views, whose change in place (loss /= n) it would refuse.
variable_list parts(const Tensor& out) {
  const at::AutoDispatchBelowADInplaceOrView guard;
  return {out.select(0, 0), out.select(0, 1), out.select(0, 2)};
}

// The gradient in x times upstream. grad: what policy wrote, the gradient for upstream 1, overwritten
// unless it is; or undefined, for a new tensor.
Tensor policy_grad(const Tensor& x, const Tensor& targets, double temperature, const Tensor& kept,
                   const Tensor& upstream, Tensor grad) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Logits logits(x);
  const int64_t n = logits.rows.rows;
  Tensor coef = kept;
  const void* scalar = data(upstream);
  if (!grad.defined()) {
    grad = empty(x, x.sizes(), x.scalar_type());
    coef = kept.narrow(0, 0, n) * upstream;
    scalar = nullptr;
  }
  check(tiso_logprobs_grad(dtype_of(x.scalar_type()), &logits.rows, targets.data_ptr<int64_t>(),
                           temperature, kept.data_ptr<double>() + n, TISO_F64, data(coef), scalar,
                           data(grad), stream_of(x)));
  return grad;
}

// A gradient that was written with its loss is kept for the backward, which gives it away the first time
// (and rewrites it unless the upstream gradient is the expected one). Only a backward of the same capture, or
// both outside of any, may have it: a captured backward is replayed, and would leave it as its reader
// left it; a captured forward is replayed over it.
void keep_ready(AutogradContext* ctx, const Tensor& grad) {
  ctx->saved_data["grad"] = grad;
  ctx->saved_data["capture"] = capture_of(grad);
}
// It, or undefined.
Tensor take_ready(AutogradContext* ctx) {
  const auto at = ctx->saved_data.find("grad");
  if (at == ctx->saved_data.end()) return Tensor();
  Tensor grad = at->second.toTensor();
  if (capture_of(grad) != ctx->saved_data["capture"].toInt()) return Tensor();
  ctx->saved_data.erase(at);
  return grad;
}

struct Policy : torch::autograd::Function<Policy> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const PolicySettings& s) {
    PolicyResult r = policy(x, s, true);
    ctx->save_for_backward({x, s.targets, r.kept});
    ctx->saved_data["temperature"] = s.temperature;
    keep_ready(ctx, r.grad);
    variable_list out = parts(r.out);
    out.push_back(r.logps);
    ctx->mark_non_differentiable({out[1], out[2], out[3]});
    ctx->set_materialize_grads(false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor ready = take_ready(ctx);
    Tensor grad;
    {
      const at::NoGradGuard no_grad;
      grad = policy_grad(saved[0], saved[1], ctx->saved_data["temperature"].toDouble(), saved[2],
                         grads[0], ready);
    }
    return {once(grad), Tensor()};
  }
};

std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor>> policy_loss(
    py::handle logits, py::handle y, int64_t ignore_index, double temperature, py::handle old_logps,
    py::handle advantages, py::handle ref_logps, py::handle weight, double clip_low,
    double clip_high, double kl_coef) {
  const Tensor *x = tensor_in(logits), *targets = tensor_in(y);
  if (!ready_logits(x, targets, temperature) || !(clip_low >= 0 && clip_high >= 0))
    return std::nullopt;
  const bool grad_mode = at::GradMode::is_enabled();
  const auto constant = [&](py::handle h, bool may_be_bool) -> const Tensor* {
    const Tensor* t = tensor_in(h);
    const bool is_bool = may_be_bool && t && t->scalar_type() == at::kBool;
    return ready(t, is_bool ? at::kBool : acc_of(*x), targets->sizes(), x->device()) &&
                   !(grad_mode && t->requires_grad())
               ? t
               : nullptr;
  };
  const Tensor *old = constant(old_logps, false), *adv = constant(advantages, false);
  if (!old || !adv) return std::nullopt;
  PolicySettings s{*targets,     *old,        *adv,     std::nullopt, std::nullopt,
                   ignore_index, temperature, clip_low, clip_high,    kl_coef};
  if (!ref_logps.is_none()) {
    const Tensor* t = constant(ref_logps, false);
    if (!t) return std::nullopt;
    s.ref_logps = *t;
  }
  if (!weight.is_none()) {
    const Tensor* t = constant(weight, true);
    if (!t) return std::nullopt;
    s.weight = *t;
  }
  for (const Tensor* t : {x, old, adv}) need_no_tangent(*t);
  need_no_tangent(s.ref_logps);
  need_no_tangent(s.weight);
  if (x->requires_grad() && grad_mode) {
    const variable_list out = Policy::apply(*x, s);
    return std::make_tuple(out[0], out[3], out[1], out[2]);
  }
  const PolicyResult r = policy(*x, s, false);
  const variable_list out = parts(r.out);
  return std::make_tuple(out[0], r.logps, out[1], out[2]);
}

// ---------------------------------------------------------------------------------------------
// A token's scores

struct ScoresResult {
  Tensor logps, entropy, top_logps, top_ids, stats;  // logps: undefined without targets
};

ScoresResult scores(const Tensor& x, const std::optional<Tensor>& targets, int64_t top,
                    double temperature, int64_t ignore_index, bool with_stats) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Logits logits(x);
  const ScalarType acc = acc_of(x);
  const at::IntArrayRef shape = x.sizes().slice(0, x.dim() - 1);
  c10::SmallVector<int64_t, 8> lists(shape.begin(), shape.end());
  lists.push_back(top);
  ScoresResult r;
  if (targets) r.logps = empty(x, shape, acc);
  r.entropy = empty(x, shape, acc);
  r.top_logps = empty(x, lists, acc);
  r.top_ids = empty(x, lists, at::kLong);
  if (with_stats) r.stats = empty(x, {3 * logits.rows.rows}, acc);
  check(tiso_scores(dtype_of(x.scalar_type()), &logits.rows,
                    targets ? targets->data_ptr<int64_t>() : nullptr, ignore_index, temperature, top,
                    targets ? data(r.logps) : nullptr, data(r.entropy), data(r.top_logps),
                    r.top_ids.data_ptr<int64_t>(), with_stats ? data(r.stats) : nullptr,
                    stream_of(x)));
  return r;
}

// coef_logp, coef_entropy: contiguous, or undefined
Tensor scores_grad(const Tensor& x, const std::optional<Tensor>& targets, double temperature,
                   const Tensor& stats, const Tensor& coef_logp, const Tensor& coef_entropy) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Logits logits(x);
  Tensor grad = empty(x, x.sizes(), x.scalar_type());
  check(tiso_scores_grad(dtype_of(x.scalar_type()), &logits.rows,
                         targets ? targets->data_ptr<int64_t>() : nullptr, temperature, data(stats),
                         coef_logp.defined() ? data(coef_logp) : nullptr,
                         coef_entropy.defined() ? data(coef_entropy) : nullptr, data(grad),
                         stream_of(x)));
  return grad;
}

struct Scores : torch::autograd::Function<Scores> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x,
                               const std::optional<Tensor>& targets, int64_t top, double temperature,
                               int64_t ignore_index) {
    ScoresResult r = scores(x, targets, top, temperature, ignore_index, true);
    ctx->save_for_backward({x, targets.value_or(Tensor()), r.stats});
    ctx->saved_data["temperature"] = temperature;
    ctx->mark_non_differentiable({r.top_logps, r.top_ids});
    ctx->set_materialize_grads(false);
    variable_list out{r.entropy, r.top_logps, r.top_ids};
    if (targets) out.push_back(r.logps);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(5);
    const Tensor coef_entropy = grads[0].defined() ? grads[0].contiguous() : Tensor();
    const Tensor coef_logp =
        grads.size() > 3 && grads[3].defined() ? grads[3].contiguous() : Tensor();
    if (!coef_entropy.defined() && !coef_logp.defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto targets = saved[1].defined() ? std::optional<Tensor>(saved[1]) : std::nullopt;
    out[0] = once(scores_grad(saved[0], targets, ctx->saved_data["temperature"].toDouble(), saved[2],
                              coef_logp, coef_entropy));
    return out;
  }
};

constexpr int64_t kMostListed = 128;

std::optional<std::tuple<std::optional<Tensor>, Tensor, Tensor, Tensor>> token_scores(
    py::handle logits, py::handle y, int64_t top, double temperature, int64_t ignore_index) {
  const Tensor* x = tensor_in(logits);
  if (!ready_rows(x, temperature) || top < 0 || top > kMostListed || top > x->size(-1))
    return std::nullopt;
  std::optional<Tensor> targets;
  if (!y.is_none()) {
    const Tensor* t = tensor_in(y);
    if (!ready(t, at::kLong, x->sizes().slice(0, x->dim() - 1), x->device())) return std::nullopt;
    targets = *t;
  }
  need_no_tangent(*x);
  if (x->requires_grad() && at::GradMode::is_enabled()) {
    const variable_list out = Scores::apply(*x, targets, top, temperature, ignore_index);
    return std::make_tuple(targets ? std::optional<Tensor>(out[3]) : std::nullopt, out[0], out[1],
                           out[2]);
  }
  const ScoresResult r = scores(*x, targets, top, temperature, ignore_index, false);
  return std::make_tuple(targets ? std::optional<Tensor>(r.logps) : std::nullopt, r.entropy,
                         r.top_logps, r.top_ids);
}

// ---------------------------------------------------------------------------------------------
// Distillation

struct DistillSettings {
  Tensor ids, logps;
  std::optional<Tensor> weight;
  int64_t kind;
  bool drop;
  double mix, temperature, upstream;
  int64_t ignore_index;
};

struct DistillResult {
  Tensor loss, divergence, kept, grad;
};

// kept: for a gradient n numbers coef, 2 n stats and n top listed (in doubles' places), then the
// workspace (one allocation, in double).
int64_t kept_of(int64_t n, int64_t top, ScalarType acc) {
  return acc == at::kDouble ? n * (3 + top) : n + (n * (2 + top) + 1) / 2;
}

DistillResult distill(const Tensor& x, const DistillSettings& s, bool with_kept, bool with_grad) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Logits logits(x);
  const ScalarType acc = acc_of(x);
  const int dtype = dtype_of(x.scalar_type());
  const int64_t n = logits.rows.rows, top = s.ids.size(-1);
  tiso_distill_args args{};
  args.ids = s.ids.data_ptr<int64_t>();
  args.logps = data(s.logps);
  args.weight = data(s.weight);
  args.weight_is_byte = s.weight && s.weight->scalar_type() == at::kBool;
  args.top = top;
  args.kind = static_cast<int>(s.kind);
  args.drop = s.drop;
  args.mix = s.mix;
  args.upstream = s.upstream;
  size_t bytes = 0;
  check(tiso_distill_workspace_size(dtype, n, &bytes));
  const int64_t behind = with_kept ? kept_of(n, top, acc) : 0;
  DistillResult r{empty(x, {}, acc), empty(x, x.sizes().slice(0, x.dim() - 1), acc),
                  empty(x, {behind + static_cast<int64_t>((bytes + 7) / 8)}, at::kDouble), Tensor()};
  if (with_grad) r.grad = empty(x, x.sizes(), x.scalar_type());
  double* at = r.kept.data_ptr<double>();
  char* stats = reinterpret_cast<char*>(at + n);
  const int64_t each = acc == at::kDouble ? 8 : 4;
  check(tiso_distill(dtype, &logits.rows, s.ignore_index, s.temperature, &args, data(r.divergence),
                     with_kept ? at : nullptr, with_kept ? stats : nullptr,
                     with_kept ? stats + 2 * n * each : nullptr, data(r.loss),
                     with_grad ? data(r.grad) : nullptr, at + behind, bytes, stream_of(x)));
  return r;
}

// The gradient times upstream. grad: what distill wrote for `expected`, overwritten unless upstream is
// that; or undefined, for a new tensor.
Tensor distill_grad(const Tensor& x, const Tensor& ids, double temperature, int64_t ignore_index,
                    const Tensor& kept, double expected, const Tensor& upstream, Tensor grad) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Logits logits(x);
  const int64_t n = logits.rows.rows, top = ids.size(-1);
  if (!grad.defined()) {
    grad = empty(x, x.sizes(), x.scalar_type());
    expected = std::numeric_limits<double>::quiet_NaN();
  }
  const double* at = kept.data_ptr<double>();
  const char* stats = reinterpret_cast<const char*>(at + n);
  check(tiso_distill_grad(dtype_of(x.scalar_type()), &logits.rows, ignore_index, temperature,
                          ids.data_ptr<int64_t>(), top, at, stats,
                          stats + 2 * n * (acc_of(x) == at::kDouble ? 8 : 4), expected,
                          data(upstream), data(grad), stream_of(x)));
  return grad;
}

struct Distill : torch::autograd::Function<Distill> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const DistillSettings& s) {
    DistillResult r = distill(x, s, true, true);
    ctx->save_for_backward({x, s.ids, r.kept});
    ctx->saved_data["temperature"] = s.temperature;
    ctx->saved_data["ignore_index"] = s.ignore_index;
    ctx->saved_data["upstream"] = s.upstream;
    keep_ready(ctx, r.grad);
    ctx->mark_non_differentiable({r.divergence});
    ctx->set_materialize_grads(false);
    return {r.loss, r.divergence};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    const Tensor ready = take_ready(ctx);
    return {once(distill_grad(saved[0], saved[1], ctx->saved_data["temperature"].toDouble(),
                              ctx->saved_data["ignore_index"].toInt(), saved[2],
                              ctx->saved_data["upstream"].toDouble(), grads[0], ready)),
            Tensor()};
  }
};

std::optional<std::tuple<Tensor, Tensor>> distillation_loss(
    py::handle logits, py::handle of_ids, py::handle of_logps, py::handle of_weight, int64_t kind,
    bool drop, double mix, double temperature, double upstream, int64_t ignore_index) {
  const Tensor *x = tensor_in(logits), *ids = tensor_in(of_ids), *logps = tensor_in(of_logps);
  if (!ready_rows(x, temperature) || !ids || ids->dim() != x->dim() || kind < 0 ||
      !(mix > 0 && mix < 1) || (kind == TISO_DISTILL_REVERSE && drop))
    return std::nullopt;
  const at::IntArrayRef shape = x->sizes().slice(0, x->dim() - 1);
  const at::Device device = x->device();
  if (ids->sizes().slice(0, x->dim() - 1) != shape || ids->size(-1) < 1 ||
      ids->size(-1) > kMostListed || !ready(ids, at::kLong, ids->sizes(), device) ||
      !ready(logps, acc_of(*x), ids->sizes(), device))
    return std::nullopt;
  const bool grad_mode = at::GradMode::is_enabled();
  if (grad_mode && logps->requires_grad()) return std::nullopt;
  DistillSettings s{*ids, *logps, std::nullopt, kind, drop, mix, temperature, upstream, ignore_index};
  if (!of_weight.is_none()) {
    const Tensor* t = tensor_in(of_weight);
    if (!t || !ready(t, t->scalar_type() == at::kBool ? at::kBool : acc_of(*x), shape, device) ||
        (grad_mode && t->requires_grad()))
      return std::nullopt;
    s.weight = *t;
  }
  need_no_tangent(*x);
  need_no_tangent(*logps);
  need_no_tangent(s.weight);
  if (x->requires_grad() && grad_mode) {
    const variable_list out = Distill::apply(*x, s);
    return std::make_tuple(out[0], out[1]);
  }
  const DistillResult r = distill(*x, s, false, false);
  return std::make_tuple(r.loss, r.divergence);
}

// ---------------------------------------------------------------------------------------------
// AdamW

// The tensors of a sequence, and what keeps them alive.
struct Tensors {
  py::object held;
  std::vector<const Tensor*> all;

  explicit Tensors(const py::handle& sequence)
      : held(py::reinterpret_steal<py::object>(
            PySequence_Fast(sequence.ptr(), "params, grads, states and scales must be sequences"))) {
    if (!held) throw py::error_already_set();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(held.ptr());
    PyObject** items = PySequence_Fast_ITEMS(held.ptr());
    all.reserve(static_cast<size_t>(n));
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (!THPVariable_Check(items[i]))
        throw py::type_error("params, grads, states and scales must be torch.Tensors");
      all.push_back(&THPVariable_Unpack(items[i]));
    }
  }
};

// indices: the tensors' places among all of the step's; empty for those in the lists.
void adamw(const py::list& lists, int64_t step, double lr, double beta1, double beta2, double eps,
           double weight_decay, uint32_t seed, const std::vector<int64_t>& indices) {
  std::vector<Tensors> held;
  std::vector<std::vector<const Tensor*>> all;
  for (const py::handle& list : lists) {
    held.emplace_back(list);
    all.push_back(held.back().all);
  }
  const size_t count = all[0].size();
  for (const auto& list : all)
    if (list.size() != count)
      throw py::value_error("params, grads, states and scales must be of one length");
  if (!indices.empty() && indices.size() != count)
    throw py::value_error("indices must be as many as params");
  if (count == 0) return;
  const at::Device device = all[0][0]->device();
  for (const auto& list : all)
    for (const Tensor* t : list)
      if (!t->is_contiguous())
        throw py::value_error("params, grads, states and scales must be contiguous");
  if (!device.is_cuda())
    throw std::runtime_error(
        "torchisotonic_b200 runs on CUDA tensors only (no CPU fallback); "
        "move params to a CUDA device");
  for (const auto& list : all)
    for (const Tensor* t : list)
      if (t->device() != device)
        throw py::value_error("params, grads, states and scales must be on one device");
  const ScalarType state = all[2][0]->scalar_type();
  for (size_t k = 1; k < 4; ++k)
    for (size_t i = 0; i < count; ++i)
      if (all[k][i]->numel() != all[0][i]->numel())
        throw py::value_error("grads and states must be shaped like their parameters");
  if (state != at::kFloat && state != at::kFloat8_e4m3fn)
    throw py::type_error("optimizer states must be float32 or float8_e4m3fn tensors");
  for (size_t k = 2; k < 4; ++k)
    for (const Tensor* t : all[k])
      if (t->scalar_type() != state) throw py::type_error("optimizer states must be of one dtype");
  const bool small = state == at::kFloat8_e4m3fn;
  if (small != (all.size() == 6))
    throw py::value_error("scales go with float8_e4m3fn states, and only with them");
  for (size_t k = 4; k < all.size(); ++k)
    for (size_t i = 0; i < count; ++i) {
      if (all[k][i]->scalar_type() != at::kFloat)
        throw py::type_error("scales must be float32 tensors");
      if (all[k][i]->numel() != (all[0][i]->numel() + 255) / 256)
        throw py::value_error("a scale tensor must hold ceil(n / 256) numbers");
    }
  for (size_t i = 0; i < count; ++i) {
    const ScalarType p = all[0][i]->scalar_type(), g = all[1][i]->scalar_type();
    if ((p != at::kFloat && p != at::kHalf && p != at::kBFloat16) || (g != p && g != at::kFloat))
      throw py::type_error(
          "params must be float32, bfloat16 or float16, grads like their parameter or float32");
  }
  // a call for each pair of types
  std::vector<bool> done(count, false);
  std::vector<tiso_adamw_tensor> table;
  table.reserve(count);
  const tiso_adamw_args args{lr, beta1, beta2, eps, weight_decay, step, seed};
  const c10::cuda::CUDAGuard guard(device);
  for (size_t from = 0; from < count; ++from) {
    if (done[from]) continue;
    const ScalarType p = all[0][from]->scalar_type(), g = all[1][from]->scalar_type();
    table.clear();
    for (size_t i = from; i < count; ++i) {
      if (done[i] || all[0][i]->scalar_type() != p || all[1][i]->scalar_type() != g) continue;
      done[i] = true;
      table.push_back({all[0][i]->data_ptr(), all[1][i]->data_ptr(), all[2][i]->data_ptr(),
                       all[3][i]->data_ptr(), small ? all[4][i]->data_ptr<float>() : nullptr,
                       small ? all[5][i]->data_ptr<float>() : nullptr, all[0][i]->numel(),
                       indices.empty() ? static_cast<int64_t>(i) : indices[i]});
    }
    check(tiso_adamw(dtype_of(p), dtype_of(g), small ? 8 : 32, static_cast<int64_t>(table.size()),
                     table.data(), &args, stream_of(*all[0][0])));
  }
  for (size_t k = 0; k < all.size(); ++k)  // autograd's check of saved tensors sees the change
    if (k != 1)
      for (const Tensor* t : all[k]) t->unsafeGetTensorImpl()->bump_version();
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.doc() = "The losses and the optimizer step over libtiso.so (see losses.py and optim.py)";
  m.def("token_logprobs", &token_logprobs);
  m.def("preference_loss", &preference_loss);
  m.def("policy_loss", &policy_loss);
  m.def("token_scores", &token_scores);
  m.def("distillation_loss", &distillation_loss);
  m.def("adamw", &adamw);
  // the steps alone, for the torch.library operators
  m.def("logprobs", [](const Tensor& x, const Tensor& targets, double temperature,
                       int64_t ignore_index) {
    need_logits(x, targets);
    return logprobs(x, targets, temperature, ignore_index, true);
  });
  m.def("logprobs_grad", [](const Tensor& x, const Tensor& targets, double temperature,
                            const Tensor& stats, const Tensor& coef) {
    need_logits(x, targets);
    need(stats, "stats", acc_of(x), {2 * targets.numel()}, x);
    need(coef, "coef", coef.scalar_type() == at::kDouble ? at::kDouble : acc_of(x), targets.sizes(),
         x);
    return logprobs_grad(x, targets, temperature, stats, coef);
  });
  m.def("preference", [](const Tensor& logps, const std::optional<Tensor>& refs,
                         const std::optional<Tensor>& mask, const Tensor& offsets, int64_t kind,
                         bool average, double beta, double label_smoothing, double margin) {
    need_answers(logps, mask, offsets);
    need(refs, "refs", logps.scalar_type(), logps.sizes(), logps);
    return Preference::run(logps, refs, mask, offsets, kind, average, beta, label_smoothing, margin);
  });
  m.def("preference_grad", [](const Tensor& logps, const std::optional<Tensor>& mask,
                              const Tensor& offsets, const Tensor& coef, const Tensor& upstream) {
    need_answers(logps, mask, offsets);
    need(coef, "coef", logps.scalar_type(), {offsets.numel() - 1}, logps);
    need_scalar(upstream, logps.scalar_type(), logps);
    return std::get<0>(Preference::run_grad(logps, mask, offsets, coef, upstream, true, false));
  });
  m.def("policy", [](const Tensor& x, const Tensor& targets, int64_t ignore_index,
                     double temperature, const Tensor& old_logps, const Tensor& advantages,
                     const std::optional<Tensor>& ref_logps, const std::optional<Tensor>& weight,
                     double clip_low, double clip_high, double kl_coef) {
    need_logits(x, targets);
    const ScalarType acc = acc_of(x);
    need(old_logps, "old_logps", acc, targets.sizes(), x);
    need(advantages, "advantages", acc, targets.sizes(), x);
    need(ref_logps, "ref_logps", acc, targets.sizes(), x);
    need(weight, "weight", weight && weight->scalar_type() == at::kBool ? at::kBool : acc,
         targets.sizes(), x);
    const PolicyResult r = policy(x, {targets, old_logps, advantages, ref_logps, weight,
                                      ignore_index, temperature, clip_low, clip_high, kl_coef},
                                  false);
    return std::make_tuple(r.out, r.logps, r.kept);
  });
  m.def("policy_grad", [](const Tensor& x, const Tensor& targets, double temperature,
                          const Tensor& kept, const Tensor& upstream) {
    need_logits(x, targets);
    need(kept, "kept", at::kDouble, {targets.numel() * (acc_of(x) == at::kDouble ? 3 : 2)}, x);
    need_scalar(upstream, acc_of(x), x);
    return policy_grad(x, targets, temperature, kept, upstream, Tensor());
  });
  m.def("scores", [](const Tensor& x, const std::optional<Tensor>& targets, int64_t top,
                     double temperature, int64_t ignore_index) {
    need_rows(x);
    need(targets, "targets", at::kLong, x.sizes().slice(0, x.dim() - 1), x);
    const ScoresResult r = scores(x, targets, top, temperature, ignore_index, true);
    return std::make_tuple(targets ? r.logps : empty(x, {0}, acc_of(x)), r.entropy, r.top_logps,
                           r.top_ids, r.stats);
  });
  m.def("scores_grad", [](const Tensor& x, const std::optional<Tensor>& targets, double temperature,
                          const Tensor& stats, const std::optional<Tensor>& coef_logp,
                          const Tensor& coef_entropy) {
    need_rows(x);
    const at::IntArrayRef shape = x.sizes().slice(0, x.dim() - 1);
    need(targets, "targets", at::kLong, shape, x);
    need(stats, "stats", acc_of(x), {3 * (x.numel() / x.size(-1))}, x);
    need(coef_logp, "coef_logp", acc_of(x), shape, x);
    need(coef_entropy, "coef_entropy", acc_of(x), shape, x);
    return scores_grad(x, targets, temperature, stats, coef_logp.value_or(Tensor()), coef_entropy);
  });
  m.def("distill", [](const Tensor& x, const Tensor& ids, const Tensor& logps,
                      const std::optional<Tensor>& weight, int64_t kind, bool drop, double mix,
                      double temperature, int64_t ignore_index) {
    need_rows(x);
    need_list(x, ids);
    need(logps, "logps", acc_of(x), ids.sizes(), x);
    need(weight, "weight", weight && weight->scalar_type() == at::kBool ? at::kBool : acc_of(x),
         x.sizes().slice(0, x.dim() - 1), x);
    const DistillResult r = distill(
        x, {ids, logps, weight, kind, drop, mix, temperature, 1.0, ignore_index}, true, false);
    return std::make_tuple(r.loss, r.divergence, r.kept);
  });
  m.def("distill_grad", [](const Tensor& x, const Tensor& ids, double temperature,
                           int64_t ignore_index, const Tensor& kept, const Tensor& upstream) {
    need_rows(x);
    need_list(x, ids);
    need(kept, "kept", at::kDouble, {kept_of(x.numel() / x.size(-1), ids.size(-1), acc_of(x))}, x);
    need_scalar(upstream, acc_of(x), x);
    return distill_grad(x, ids, temperature, ignore_index, kept, 0.0, upstream, Tensor());
  });
}
