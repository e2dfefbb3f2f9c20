// The block operators (norm, experts, AdamW) for torch: tensors in, tensors
// out, autograd nodes, over the C ABI of libmlpk (include/mlpk.h).
//
// One eager call in Python through ctypes costs 12 to 20 us of host time, and a
// backward pass in Python some 60 more (the engine's thread has to take the
// interpreter's lock); many of these calls are of small kernels, so the binding
// is native.  It has no kernels and no checks' messages: where the arguments are
// not what an operator takes, a call returns None and the Python layer says why.
// It does so too where torch's dispatcher would not go straight to a CUDA kernel
// (a mode, a tracer, a transform, a tensor subclass): the Python layer then calls
// the operators torch.ops.mlpk.*, which those see, or says that there is no rule.
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <string>
#include <vector>

#include "../../include/mlpk.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

constexpr int kNormMaxWidth = 32768;
constexpr int kExpertMax = 1024;

// A status that is not MLPK_OK; Python sees it as _lib.MlpkError.
struct MlpkFailure : std::runtime_error {
  MlpkFailure(const char* fn, int status)
      : std::runtime_error(std::string(fn) + " failed: " + mlpk_status_string(status) +
                           (status == MLPK_ERR_CUDA ? std::string(": ") + mlpk_last_cuda_error() : std::string())),
        fn(fn), status(status) {}
  const char* fn;
  int status;
};
void check(const char* fn, int status) {
  if (status != MLPK_OK) throw MlpkFailure(fn, status);
}

int code(at::ScalarType t) {  // below 0: not a type of the block operators
  switch (t) {
    case at::kHalf: return MLPK_DT_F16;
    case at::kFloat: return MLPK_DT_F32;
    case at::kBFloat16: return MLPK_DT_BF16;
    default: return -1;
  }
}
int code(const Tensor& t) { return code(t.scalar_type()); }
bool weight_type(const Tensor& w, const Tensor& x) {
  return w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat;
}

Tensor aligned(const Tensor& t) {
  if (!t.defined()) return t;
  Tensor c = t.is_contiguous() ? t : t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
mlpk_stream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
// Absent inputs of an autograd node: a node counts the defined ones alone.
std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
bool needs_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Whether the dispatcher would take these tensors to a CUDA kernel with nothing
// but backward-mode autograd before it: no dispatch mode, tracer,
// functionalization or function transform is active, none is a subclass or a
// lazy view, and none has a tangent.
bool direct(std::initializer_list<const Tensor*> ts) {
  static const c10::DispatchKeySet ordinary =
      c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::ADInplaceOrView,
                           c10::DispatchKey::BackendSelect}) |
      c10::autocast_dispatch_keyset;
  const auto local = c10::impl::tls_local_dispatch_key_set();
  c10::DispatchKeySet keys = local.included_;
  for (const Tensor* t : ts) {
    if (!t->defined()) continue;
    if (t->_fw_grad(/*level=*/0).defined()) return false;
    keys = keys | t->key_set();
  }
  return ((keys - local.excluded_ - ordinary).raw_repr() >> c10::num_backends) == 0;
}
// What a backward says where an operator's gradient would drop a tangent.
void refuse_tangents(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(),
                "the gradient of this operator has no forward-mode derivative");
}
// The operator torch.ops.mlpk.<name>.
template <class... Args>
c10::IValue operate(const char* name, Args&&... args) {
  torch::jit::Stack stack;
  torch::jit::push(stack, std::forward<Args>(args)...);
  c10::Dispatcher::singleton().findSchemaOrThrow(name, "").callBoxed(&stack);
  return std::move(stack.at(0));
}

// A gradient in a backward that is itself recorded (create_graph).  The
// operators have no second derivatives: if the gradient depends on a tensor that
// needs one, asking for its derivative raises.
Tensor once(const Tensor& grad, std::initializer_list<const Tensor*> depends_on) {
  if (!grad.defined() || !needs_grad(depends_on)) return grad;
  auto node =
      std::make_shared<torch::autograd::DelayedError>("the gradient of this operator cannot be differentiated again", 1);
  return (*node)({grad.detach().requires_grad_(true)})[0];
}

// ------------------------------------------------------------------ norm
struct Normed {
  Tensor y, h, rstd;
};
Normed norm_forward(const Tensor& x_in, const Tensor& w_in, const Tensor& r_in, double eps, bool want_rstd) {
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = aligned(x_in), w = aligned(w_in), r = aligned(r_in);
  const int64_t width = x.size(-1), rows = x.numel() / width;
  Normed n;
  n.y = at::empty_like(x);
  if (r.defined()) n.h = at::empty_like(x);
  if (want_rstd) n.rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  check("mlpk_rms_norm",
        mlpk_rms_norm(rows, static_cast<int>(width), code(x), ptr(x), ptr(r), ptr(w), code(w.defined() ? w : x),
                      static_cast<float>(eps), ptr(n.y), ptr(n.h), static_cast<float*>(ptr(n.rstd)), stream_of(x)));
  return n;
}

// (dx, dw): dx is the residual's gradient too; dw only if wanted.
std::tuple<Tensor, Tensor> norm_backward(const Tensor& x_in, const Tensor& w_in, const Tensor& r_in,
                                         const Tensor& rstd, const Tensor& gy_in, const Tensor& gh_in, bool want_dw) {
  if (!gy_in.defined())  // y was not used: the norm adds nothing
    return {gh_in, want_dw && gh_in.defined() ? at::zeros_like(w_in) : Tensor()};
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = aligned(x_in), w = aligned(w_in), r = aligned(r_in), gy = aligned(gy_in), gh = aligned(gh_in);
  const int64_t width = x.size(-1), rows = x.numel() / width;
  Tensor dx = at::empty_like(x), dw, work;
  if (want_dw) {
    dw = at::empty_like(w);
    const int64_t bytes = mlpk_rms_norm_bwd_workspace_size(rows, static_cast<int>(width), code(x));
    work = at::empty({std::max<int64_t>(bytes, 16)}, x.options().dtype(at::kByte));
  }
  check("mlpk_rms_norm_bwd",
        mlpk_rms_norm_bwd(rows, static_cast<int>(width), code(x), ptr(x), ptr(r), static_cast<float*>(ptr(rstd)),
                          ptr(w), code(w.defined() ? w : x), ptr(gy), ptr(gh), ptr(dx), ptr(dw), ptr(work),
                          work.defined() ? work.numel() : 0, stream_of(x)));
  return {dx, dw};
}

struct NormNode : torch::autograd::Function<NormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                               const std::optional<Tensor>& residual, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor w = weight.value_or(Tensor()), r = residual.value_or(Tensor());
    Normed n = norm_forward(x, w, r, eps, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, w, r, n.rstd});
    return r.defined() ? variable_list{n.y, n.h} : variable_list{n.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dx, dw;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &r = saved[2], &gy = grads[0];
    const Tensor gh = grads.size() > 1 ? grads[1] : Tensor();
    const size_t r_at = w.defined() ? 2 : 1;  // the residual's place among the inputs there are
    {
      const at::NoGradGuard no_grad;
      const bool want_dw = w.defined() && ctx->needs_input_grad(1);
      if (!gy.defined() || direct({&gy, &gh, &x, &w, &r})) {
        std::tie(dx, dw) = norm_backward(x, w, r, saved[3], gy, gh, want_dw);
      } else {
        refuse_tangents({&gy, &gh, &x, &w, &r});
        const std::vector<Tensor> got =
            operate("mlpk::rms_norm_bwd", x, maybe(r), maybe(w), saved[3], gy, maybe(gh), want_dw).toTensorVector();
        dx = got[0];
        if (want_dw) dw = got[1];
      }
    }
    if (gy.defined()) {  // else dx is gh itself
      dx = once(dx, {&gy, &gh, &x, &w, &r});
      dw = once(dw, {&gy, &x, &r});
    }
    return {ctx->needs_input_grad(0) ? dx : Tensor(), dw, r.defined() && ctx->needs_input_grad(r_at) ? dx : Tensor(),
            Tensor()};
  }
};

bool norm_takes(const Tensor& x, const Tensor& w, const Tensor& r, double eps) {
  if (!x.is_cuda() || code(x) < 0 || x.dim() < 1 || !(eps >= 0.0)) return false;
  const int64_t width = x.size(-1);
  if (width < 1 || width > kNormMaxWidth) return false;
  if (w.defined() && (w.dim() != 1 || w.size(0) != width || w.device() != x.device() || !weight_type(w, x)))
    return false;
  return !r.defined() || (r.sizes() == x.sizes() && r.scalar_type() == x.scalar_type() && r.device() == x.device());
}

py::object rms_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& residual,
                    double eps) {
  const Tensor w = weight.value_or(Tensor()), r = residual.value_or(Tensor());
  if (!norm_takes(x, w, r, eps) || !direct({&x, &w, &r})) return py::none();
  variable_list out;
  {
    py::gil_scoped_release no_gil;
    if (needs_grad({&x, &w, &r})) {
      out = NormNode::apply(x, maybe(w), maybe(r), eps);
    } else {
      Normed n = norm_forward(x, w, r, eps, false);
      out.push_back(std::move(n.y));
      if (r.defined()) out.push_back(std::move(n.h));
    }
  }
  return r.defined() ? py::object(py::make_tuple(out[0], out[1])) : py::cast(out[0]);
}

py::object norm_fp8(const Tensor& x_in, const std::optional<Tensor>& weight, const std::optional<Tensor>& residual,
                    double eps, int64_t group) {
  Tensor q, scale, h;
  {
    py::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(x_in.device());
    const Tensor x = aligned(x_in), w = aligned(weight.value_or(Tensor())), r = aligned(residual.value_or(Tensor()));
    const int64_t width = x.size(-1), rows = x.numel() / width;
    q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = group ? (width + group - 1) / group : 1;
    scale = at::empty(shape, x.options().dtype(at::kFloat));
    if (r.defined()) h = at::empty_like(x);
    check("mlpk_rms_norm_fp8",
          mlpk_rms_norm_fp8(rows, static_cast<int>(width), code(x), ptr(x), ptr(r), ptr(w),
                            code(w.defined() ? w : x), static_cast<float>(eps), static_cast<int>(group), ptr(q),
                            static_cast<float*>(ptr(scale)), ptr(h), stream_of(x)));
  }
  return h.defined() ? py::make_tuple(q, scale, h) : py::make_tuple(q, scale);
}
// None also where a gradient would be needed.
py::object rms_norm_fp8(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& residual,
                        double eps, int64_t group) {
  const Tensor w = weight.value_or(Tensor()), r = residual.value_or(Tensor());
  if (!norm_takes(x, w, r, eps) || (group != 0 && group != 128) || needs_grad({&x, &w, &r}) || !direct({&x, &w, &r}))
    return py::none();
  return norm_fp8(x, weight, residual, eps, group);
}

// ------------------------------------------------------------------ experts
py::object sort_ids(const Tensor& ids_in, int64_t experts) {
  const bool wide = ids_in.scalar_type() == at::kLong;
  Tensor row_of, offsets;
  {
    py::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(ids_in.device());
    const Tensor ids = aligned(ids_in);
    row_of = at::empty(ids.sizes(), ids.options().dtype(at::kInt));
    offsets = at::empty({experts + 1}, ids.options().dtype(at::kInt));
    const int64_t bytes = mlpk_expert_sort_workspace_size(ids.numel(), static_cast<int>(experts));
    const Tensor work = bytes > 0 ? at::empty({bytes}, ids.options().dtype(at::kByte)) : Tensor();
    check("mlpk_expert_sort",
          mlpk_expert_sort(ids.numel(), static_cast<int>(experts), ptr(ids), wide ? 8 : 4,
                           static_cast<int32_t*>(ptr(row_of)), static_cast<int32_t*>(ptr(offsets)), ptr(work), bytes,
                           stream_of(ids)));
  }
  return py::make_tuple(row_of, offsets);
}

py::object expert_sort(const Tensor& ids, int64_t experts) {
  if (!ids.is_cuda() || ids.dim() != 2 || !(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt) ||
      experts < 1 || experts > kExpertMax || ids.size(1) < 1 || ids.numel() > 0x7fffffff || !direct({&ids}))
    return py::none();
  return sort_ids(ids, experts);
}

const int32_t* kept(const Tensor& offsets) { return offsets.data_ptr<int32_t>() + offsets.size(0) - 1; }

Tensor dispatch_rows(const Tensor& x_in, const Tensor& row_in, const Tensor& offsets) {
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = aligned(x_in), row_of = aligned(row_in);
  Tensor xs = at::empty({row_of.numel(), x.size(1)}, x.options());
  check("mlpk_expert_dispatch",
        mlpk_expert_dispatch(row_of.size(0), static_cast<int>(row_of.size(1)), static_cast<int>(x.size(1)), code(x),
                             ptr(x), row_of.data_ptr<int32_t>(), kept(offsets), ptr(xs), stream_of(x)));
  return xs;
}

Tensor combine_rows(const Tensor& y_in, const Tensor& w_in, const Tensor& row_in, const Tensor& offsets) {
  const c10::cuda::CUDAGuard guard(y_in.device());
  const Tensor y = aligned(y_in), row_of = aligned(row_in), w = w_in.defined() ? w_in.contiguous() : w_in;
  Tensor out = at::empty({row_of.size(0), y.size(1)}, y.options());
  check("mlpk_expert_combine",
        mlpk_expert_combine(row_of.size(0), static_cast<int>(row_of.size(1)), static_cast<int>(y.size(1)), code(y),
                            ptr(y), ptr(w), code(w.defined() ? w : y), row_of.data_ptr<int32_t>(), kept(offsets),
                            ptr(out), stream_of(y)));
  return out;
}

// (dy, dw), those that are wanted.
std::tuple<Tensor, Tensor> combine_backward(const Tensor& g_in, const Tensor& y_in, const Tensor& w_in,
                                            const Tensor& row_in, const Tensor& offsets, bool want_dy, bool want_dw) {
  const c10::cuda::CUDAGuard guard(y_in.device());
  const Tensor g = aligned(g_in), y = aligned(y_in), row_of = aligned(row_in);
  const Tensor w = w_in.defined() ? w_in.contiguous() : w_in;
  Tensor dy = want_dy ? at::empty_like(y) : Tensor(), dw = want_dw ? at::empty_like(w) : Tensor();
  check("mlpk_expert_combine_bwd",
        mlpk_expert_combine_bwd(row_of.size(0), static_cast<int>(row_of.size(1)), static_cast<int>(y.size(1)), code(y),
                                ptr(g), ptr(y), ptr(w), code(w.defined() ? w : y), row_of.data_ptr<int32_t>(),
                                kept(offsets), ptr(dy), ptr(dw), stream_of(y)));
  return {dy, dw};
}

struct DispatchNode : torch::autograd::Function<DispatchNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& row_of, const Tensor& offsets) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({row_of, offsets});
    return {dispatch_rows(x, row_of, offsets)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dx;
    {
      const at::NoGradGuard no_grad;
      const variable_list saved = ctx->get_saved_variables();
      if (direct({&grads[0], &saved[0], &saved[1]})) {
        dx = combine_rows(grads[0], Tensor(), saved[0], saved[1]);
      } else {
        refuse_tangents({&grads[0]});
        dx = operate("mlpk::expert_combine", grads[0], std::optional<Tensor>(), saved[0], saved[1]).toTensor();
      }
    }
    return {once(dx, {&grads[0]}), Tensor(), Tensor()};
  }
};

struct CombineNode : torch::autograd::Function<CombineNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& y, const std::optional<Tensor>& weights,
                               const Tensor& row_of, const Tensor& offsets) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor w = weights.value_or(Tensor());
    ctx->save_for_backward({y, w, row_of, offsets});
    return {combine_rows(y, w, row_of, offsets)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    Tensor dy, dw;
    const variable_list saved = ctx->get_saved_variables();
    {
      const at::NoGradGuard no_grad;
      const bool want_dy = ctx->needs_input_grad(0), want_dw = saved[1].defined() && ctx->needs_input_grad(1);
      if (direct({&grads[0], &saved[0], &saved[1], &saved[2], &saved[3]})) {
        std::tie(dy, dw) = combine_backward(grads[0], saved[0], saved[1], saved[2], saved[3], want_dy, want_dw);
      } else {
        refuse_tangents({&grads[0], &saved[0], &saved[1]});
        const std::vector<Tensor> got = operate("mlpk::expert_combine_bwd", grads[0], saved[0], maybe(saved[1]), saved[2],
                                                saved[3], want_dy, want_dw)
                                            .toTensorVector();
        if (want_dy) dy = got.front();
        if (want_dw) dw = got.back();
      }
    }
    return {once(dy, {&grads[0], &saved[1]}), once(dw, {&grads[0], &saved[0]}), Tensor(), Tensor()};
  }
};

bool rows_take(const Tensor& t, int64_t rows, const Tensor& row_of, const Tensor& offsets) {
  return t.is_cuda() && code(t) >= 0 && t.dim() == 2 && t.size(0) == rows && t.size(1) >= 1 && row_of.dim() == 2 &&
         row_of.scalar_type() == at::kInt && offsets.scalar_type() == at::kInt && offsets.dim() == 1 &&
         offsets.size(0) > 1 && offsets.is_contiguous() && t.device() == row_of.device() &&
         t.device() == offsets.device() && direct({&t, &row_of, &offsets});
}

py::object expert_dispatch(const Tensor& x, const Tensor& row_of, const Tensor& offsets) {
  if (row_of.dim() != 2 || !rows_take(x, row_of.size(0), row_of, offsets)) return py::none();
  Tensor xs;
  {
    py::gil_scoped_release no_gil;
    xs = needs_grad({&x}) ? DispatchNode::apply(x, row_of, offsets)[0] : dispatch_rows(x, row_of, offsets);
  }
  return py::cast(xs);
}

py::object expert_combine(const Tensor& y, const std::optional<Tensor>& weights, const Tensor& row_of,
                          const Tensor& offsets) {
  const Tensor w = weights.value_or(Tensor());
  if (!rows_take(y, row_of.numel(), row_of, offsets)) return py::none();
  if (w.defined() && (w.sizes() != row_of.sizes() || w.device() != y.device() || !weight_type(w, y) || !direct({&w})))
    return py::none();
  Tensor out;
  {
    py::gil_scoped_release no_gil;
    out = needs_grad({&y, &w}) ? CombineNode::apply(y, maybe(w), row_of, offsets)[0] : combine_rows(y, w, row_of, offsets);
  }
  return py::cast(out);
}

// ------------------------------------------------------------------ AdamW
// Some tensors of one type and device with their places in the flat state and
// in its step counts.
class AdamwBucket {
 public:
  AdamwBucket(std::vector<Tensor> params, std::vector<int64_t> off, std::vector<int32_t> tick, int bits,
              const Tensor& exp_avg, const Tensor& exp_avg_sq, const std::optional<Tensor>& avg_scale,
              const std::optional<Tensor>& sq_scale, const std::optional<Tensor>& master, const Tensor& ticks)
      : params_(std::move(params)), off_(std::move(off)), tick_(std::move(tick)), device_(params_[0].device()),
        type_(params_[0].scalar_type()),
        keep_{exp_avg, exp_avg_sq, avg_scale.value_or(Tensor()), sq_scale.value_or(Tensor()),
              master.value_or(Tensor()), ticks} {
    state_.bits = bits;
    state_.exp_avg = ptr(keep_[0]);
    state_.exp_avg_sq = ptr(keep_[1]);
    state_.exp_avg_scale = static_cast<float*>(ptr(keep_[2]));
    state_.exp_avg_sq_scale = static_cast<float*>(ptr(keep_[3]));
    state_.master = static_cast<float*>(ptr(keep_[4]));
    state_.ticks = static_cast<int64_t*>(ptr(keep_[5]));
    for (const Tensor& p : params_) {
      numel_.push_back(p.numel());
      strides_.push_back(p.strides().vec());
    }
  }

  void step(double lr, const std::optional<Tensor>& lr_tensor, double beta1, double beta2, double eps,
            double weight_decay, bool maximize, const std::optional<Tensor>& grad_scale,
            const std::optional<Tensor>& found_inf) {
    const at::NoGradGuard no_grad;
    mlpk_adamw_args args = {};
    args.lr = lr;
    args.beta1 = beta1;
    args.beta2 = beta2;
    args.eps = eps;
    args.weight_decay = weight_decay;
    args.maximize = maximize;
    args.lr_ptr = scalar(lr_tensor);
    args.grad_scale = scalar(grad_scale);
    args.found_inf = scalar(found_inf);
    // Gradients in the parameters' type, then those in fp32 beside 16-bit
    // parameters: a launch for each.
    Part same, wide;
    for (size_t i = 0; i < params_.size(); ++i) {
      const Tensor& p = params_[i];
      const Tensor& g = p.grad();
      if (!g.defined()) continue;
      TORCH_CHECK(p.scalar_type() == type_ && p.device() == device_ && p.numel() == numel_[i] &&
                      p.strides() == at::IntArrayRef(strides_[i]),
                  "a parameter changed its type, device, size or strides after its first step");
      TORCH_CHECK_VALUE(g.device() == device_ && !g.is_sparse(), "a gradient must be a dense tensor on ", device_);
      TORCH_CHECK_TYPE(g.scalar_type() == type_ || g.scalar_type() == at::kFloat, "gradients must be ", type_,
                       " or float32, got ", g.scalar_type());
      Part& part = g.scalar_type() == type_ ? same : wide;
      const void* gp = g.data_ptr();
      if (g.strides() != p.strides()) {  // the elements are taken in the parameter's order of memory
        part.copies.push_back(at::empty_like(p, p.options().dtype(g.scalar_type())).copy_(g));
        gp = part.copies.back().data_ptr();
      }
      part.numel.push_back(numel_[i]);
      part.off.push_back(off_[i]);
      part.tick.push_back(tick_[i]);
      part.p.push_back(p.data_ptr());
      part.g.push_back(gp);
      p.unsafeGetTensorImpl()->bump_version();
    }
    const c10::cuda::CUDAGuard guard(device_);
    for (const Part* part : {&same, &wide})
      if (!part->p.empty())
        check("mlpk_adamw_step",
              mlpk_adamw_step(static_cast<int>(part->p.size()), part->numel.data(), part->p.data(), part->g.data(),
                              part->off.data(), part->tick.data(), code(type_),
                              part == &same ? code(type_) : MLPK_DT_F32, &state_, &args,
                              c10::cuda::getCurrentCUDAStream(device_.index()).stream()));
  }

 private:
  struct Part {
    std::vector<int64_t> numel, off;
    std::vector<int32_t> tick;
    std::vector<void*> p;
    std::vector<const void*> g;
    std::vector<Tensor> copies;
  };
  const float* scalar(const std::optional<Tensor>& t) const {
    if (!t || !t->defined()) return nullptr;
    TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->device() == device_ && t->numel() == 1,
                      "lr, grad_scale and found_inf must be float32 values on ", device_);
    return t->data_ptr<float>();
  }

  std::vector<Tensor> params_;
  std::vector<int64_t> off_, numel_;
  std::vector<int32_t> tick_;
  std::vector<std::vector<int64_t>> strides_;
  at::Device device_;
  at::ScalarType type_;
  std::vector<Tensor> keep_;
  mlpk_adamw_state state_ = {};
};

}  // namespace

#ifndef MLPK_BUILT_FOR  // the versions of torch and Python, from build.py
#define MLPK_BUILT_FOR "unknown"
#endif

PYBIND11_MODULE(mlpk_torch, m) {
  m.attr("built_for") = MLPK_BUILT_FOR;
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const MlpkFailure& e) {
      const py::object cls = py::module_::import("mlp_megakernel_b200._lib").attr("MlpkError");
      PyErr_SetObject(cls.ptr(), cls(e.fn, e.status).ptr());
    }
  });
  // The public calls.
  m.def("rms_norm", &rms_norm);
  m.def("rms_norm_fp8", &rms_norm_fp8);
  m.def("expert_sort", &expert_sort);
  m.def("expert_dispatch", &expert_dispatch);
  m.def("expert_combine", &expert_combine);
  // What the torch.ops.mlpk operators run, below autograd and with arguments
  // that have been checked.
  m.def("norm_forward", [](const Tensor& x, const std::optional<Tensor>& w, const std::optional<Tensor>& r,
                           double eps) {
    const Normed n = norm_forward(x, w.value_or(Tensor()), r.value_or(Tensor()), eps, true);
    return std::make_tuple(n.y, n.h, n.rstd);
  });
  m.def("norm_backward", [](const Tensor& x, const std::optional<Tensor>& r, const std::optional<Tensor>& w,
                            const Tensor& rstd, const Tensor& gy, const std::optional<Tensor>& gh, bool want_dw) {
    return norm_backward(x, w.value_or(Tensor()), r.value_or(Tensor()), rstd, gy, gh.value_or(Tensor()), want_dw);
  });
  m.def("norm_fp8", &norm_fp8);
  m.def("sort_ids", &sort_ids);
  m.def("dispatch_rows", &dispatch_rows);
  m.def("combine_rows", [](const Tensor& y, const std::optional<Tensor>& w, const Tensor& row_of,
                           const Tensor& offsets) { return combine_rows(y, w.value_or(Tensor()), row_of, offsets); });
  m.def("combine_backward", [](const Tensor& g, const Tensor& y, const std::optional<Tensor>& w, const Tensor& row_of,
                               const Tensor& offsets, bool want_dy, bool want_dw) {
    return combine_backward(g, y, w.value_or(Tensor()), row_of, offsets, want_dy, want_dw);
  });
  // Whether two lists hold the same objects in the same order.
  m.def("same_items", [](const py::list& a, const py::list& b) {
    const Py_ssize_t n = PyList_GET_SIZE(a.ptr());
    if (n != PyList_GET_SIZE(b.ptr())) return false;
    for (Py_ssize_t i = 0; i < n; ++i)
      if (PyList_GET_ITEM(a.ptr(), i) != PyList_GET_ITEM(b.ptr(), i)) return false;
    return true;
  });
  py::class_<AdamwBucket>(m, "AdamwBucket")
      .def(py::init<std::vector<Tensor>, std::vector<int64_t>, std::vector<int32_t>, int, const Tensor&, const Tensor&,
                    const std::optional<Tensor>&, const std::optional<Tensor>&, const std::optional<Tensor>&,
                    const Tensor&>())
      .def("step", &AdamwBucket::step, py::call_guard<py::gil_scoped_release>());
}
