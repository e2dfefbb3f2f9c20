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

// The same, where the node knows whether the gradient depends on such a tensor.
Tensor once_if(const Tensor& grad, const Tensor& upstream, bool depends) {
  if (!depends || !grad.defined() || !at::GradMode::is_enabled()) return once(grad, {&upstream});
  const Tensor needing = upstream.detach().requires_grad_(true);
  return once(grad, {&needing});
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

// ------------------------------------------------------------------ feed-forward
constexpr int64_t kFfMaxRows = 0x7fffffff - 256, kFfMaxWidth = 1 << 20;
constexpr int kActs = 6;

bool operand_type(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
bool ff_width(int64_t w) { return w >= 8 && w % 8 == 0 && w <= kFfMaxWidth; }
int64_t rows_of(const Tensor& x) { return x.numel() / x.size(-1); }
std::vector<int64_t> with_width(const Tensor& x, int64_t width) {
  std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
  s.back() = width;
  return s;
}

// A weight [in][out] where it lies: contiguous, or the transpose of a contiguous
// tensor; anything else is copied.
struct Weight {
  Tensor t;
  int layout;
};
Weight weight_in(const Tensor& w, int layout) {
  if (layout == MLPK_W_OUT_IN) return {aligned(w.t()), layout};
  return {aligned(w), layout};
}
int layout_of(const Tensor& w) {
  return !w.is_contiguous() && w.t().is_contiguous() ? MLPK_W_OUT_IN : MLPK_W_IN_OUT;
}
Weight weight_of(const Tensor& w) { return weight_in(w, layout_of(w)); }
// A weight's gradient in its layout: [the memory, the tensor [in][out]].
std::pair<Tensor, Tensor> grad_of(const Tensor& w, int layout) {
  if (layout == MLPK_W_OUT_IN) {
    const Tensor m = at::empty({w.size(1), w.size(0)}, w.options());
    return {m, m.t()};
  }
  const Tensor m = at::empty({w.size(0), w.size(1)}, w.options());
  return {m, m};
}

// Values that a forward keeps: of its type, or 8 bits and their scales.
struct Kept {
  Tensor v, scale;
  int kind() const { return !v.defined() ? MLPK_KEEP_NONE : scale.defined() ? MLPK_KEEP_FP8 : MLPK_KEEP_16; }
  float* scales() const { return static_cast<float*>(ptr(scale)); }
};
// As the kernels take it: a hook on saved tensors may give back other strides.
Kept aligned(const Kept& k) { return {aligned(k.v), aligned(k.scale)}; }
// Whether values [..., width] of that many rows are what a forward keeps for `go`'s
// backward, in all but the layout: of its type, or in 8 bits with scales (the
// values in rows of `pitch`).
bool kept_for(const Kept& k, const Tensor& go, int64_t rows, int64_t width, int64_t pitch) {
  const Tensor &v = k.v, &s = k.scale;
  if (!v.defined() || v.device() != go.device() || v.dim() < 1) return false;
  if (!s.defined()) return v.scalar_type() == go.scalar_type() && v.size(-1) == width && v.numel() == rows * width;
  return v.scalar_type() == at::kFloat8_e4m3fn && v.size(-1) == pitch && v.numel() == rows * pitch &&
         s.scalar_type() == at::kFloat && s.device() == go.device() && s.dim() >= 1 && s.size(-1) == (width + 127) / 128 &&
         s.numel() == rows * s.size(-1);
}
bool weight_for(const Tensor& w, const Tensor& go) {
  return w.dim() == 2 && w.scalar_type() == go.scalar_type() && w.device() == go.device();
}
void check_saved(bool ok) { TORCH_CHECK(ok, "a saved tensor is not what the forward saved (a hook changed its shape, type or device)"); }
Kept keep_for(const Tensor& x, int64_t rows, int64_t width, int64_t keep) {
  Kept k;
  if (keep == MLPK_KEEP_16) k.v = at::empty({rows, width}, x.options());
  if (keep == MLPK_KEEP_FP8) {
    k.v = at::empty({rows, mlpk_fp8_pitch(static_cast<int>(width))}, x.options().dtype(at::kFloat8_e4m3fn));
    k.scale = at::empty({rows, (width + 127) / 128}, x.options().dtype(at::kFloat));
  }
  return k;
}

Kept checkpoint(const Tensor& x_in) {
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = aligned(x_in);
  const int64_t width = x.size(-1), rows = rows_of(x);
  Kept k;
  k.v = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  k.scale = at::empty(with_width(x, (width + 127) / 128), x.options().dtype(at::kFloat));
  check("mlpk_fp8_checkpoint", mlpk_fp8_checkpoint(rows, static_cast<int>(width), code(x), ptr(x), ptr(k.v), k.scales(),
                                                   stream_of(x)));
  return k;
}
Tensor restore(const Tensor& q_in, const Tensor& scale_in, at::ScalarType type) {
  const c10::cuda::CUDAGuard guard(q_in.device());
  const Tensor q = aligned(q_in), scale = aligned(scale_in);
  const int64_t width = q.size(-1);
  Tensor x = at::empty(q.sizes(), q.options().dtype(type));
  check("mlpk_fp8_restore", mlpk_fp8_restore(rows_of(q), static_cast<int>(width), code(type), ptr(q),
                                             static_cast<float*>(ptr(scale)), ptr(x), stream_of(q)));
  return x;
}

Tensor workspace(int64_t bytes, const Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
// out = act(x w + b) + r, and what is kept of x w + b.
Tensor linear_forward(const Tensor& x_in, const Weight& w, int64_t n, const Tensor& b_in, const Tensor& r_in, int64_t act,
                      Kept* z) {
  const Tensor x = aligned(x_in), b = aligned(b_in), r = aligned(r_in);
  Tensor out = at::empty(with_width(x, n), x.options());
  const int k = static_cast<int>(x.size(-1)), m = static_cast<int>(n), keep = z ? z->kind() : MLPK_KEEP_NONE;
  const int64_t rows = rows_of(x), bytes = mlpk_linear_workspace_size(rows, k, m, code(x), w.layout, keep);
  const Tensor work = workspace(bytes, x);
  check("mlpk_linear", mlpk_linear(rows, k, m, code(x), ptr(x), ptr(w.t), w.layout, ptr(b), code(b.defined() ? b : x),
                                   static_cast<int>(act), ptr(r), ptr(out), keep, z ? ptr(z->v) : nullptr,
                                   z ? z->scales() : nullptr, ptr(work), std::max<int64_t>(bytes, 0), stream_of(x)));
  return out;
}
std::pair<Tensor, Kept> linear_kept(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r, int64_t act,
                                    int64_t keep) {
  const c10::cuda::CUDAGuard guard(x.device());
  Kept z = keep_for(x, rows_of(x), w.size(1), keep);
  Tensor out = linear_forward(x, weight_of(w), w.size(1), b, r, act, &z);
  return {std::move(out), std::move(z)};
}

// The gradients of x (of one product, or the sum of two) and of the weights.
Tensor dx_of(const Tensor& shaped, std::initializer_list<Tensor> dz, std::initializer_list<Weight> w, int64_t d_in) {
  const Tensor& first = *dz.begin();
  Tensor dx = at::empty(with_width(shaped, d_in), first.options());
  const void *zp[2], *wp[2];
  int n = 0;
  for (const Tensor& t : dz) zp[n++] = ptr(t);
  n = 0;
  for (const Weight& t : w) wp[n++] = ptr(t.t);
  const int k = static_cast<int>(d_in), m = static_cast<int>(first.size(-1)), layout = w.begin()->layout;
  const int64_t rows = rows_of(first), bytes = mlpk_linear_dx_workspace_size(rows, k, m, code(first), n, layout);
  const Tensor work = workspace(bytes, first);
  check("mlpk_linear_dx", mlpk_linear_dx(rows, k, m, code(first), n, zp, wp, layout, ptr(dx), ptr(work),
                                         std::max<int64_t>(bytes, 0), stream_of(first)));
  return dx;
}
void dw_of(const Tensor& x_in, std::initializer_list<Tensor> dz, std::initializer_list<Tensor> dw, int layout) {
  const Tensor x = aligned(x_in);
  const void* zp[2];
  void* wp[2];
  int n = 0;
  for (const Tensor& t : dz) zp[n++] = ptr(t);
  n = 0;
  for (const Tensor& t : dw) wp[n++] = ptr(t);
  const int k = static_cast<int>(x.size(-1)), m = static_cast<int>(dz.begin()->size(-1));
  const int64_t rows = rows_of(x), bytes = mlpk_linear_dw_workspace_size(rows, k, m, code(x), n, layout);
  const Tensor work = workspace(bytes, x);
  check("mlpk_linear_dw",
        mlpk_linear_dw(rows, k, m, code(x), n, ptr(x), zp, wp, layout, ptr(work), std::max<int64_t>(bytes, 0), stream_of(x)));
}

struct LinearGrads {
  Tensor dx, dw, db;
};
LinearGrads linear_backward(const Tensor& go_in, const Kept& x, const Tensor& w_in, const Kept& z_in, int64_t act,
                            at::ScalarType db_type, bool want_dx, bool want_dw, bool want_db) {
  const c10::cuda::CUDAGuard guard(go_in.device());
  const Tensor go = aligned(go_in);
  const int64_t rows = rows_of(go), n = go.size(-1);
  check_saved(weight_for(w_in, go) && w_in.size(1) == n &&
              (act == MLPK_ACT_NONE || kept_for(z_in, go, rows, n, mlpk_fp8_pitch(static_cast<int>(n)))) &&
              (!want_dw || kept_for(x, go, rows, w_in.size(0), w_in.size(0))));
  const Kept z = aligned(z_in);
  LinearGrads got;
  Tensor dz = go;
  if (act != MLPK_ACT_NONE || want_db) {
    if (act != MLPK_ACT_NONE) dz = want_dx || want_dw ? at::empty_like(go) : Tensor();
    Tensor work;
    int64_t bytes = 0;
    if (want_db) {
      got.db = at::empty({n}, go.options().dtype(db_type));
      bytes = mlpk_linear_dz_workspace_size(rows, static_cast<int>(n), code(go));
      work = workspace(bytes, go);
    }
    check("mlpk_linear_dz",
          mlpk_linear_dz(rows, static_cast<int>(n), code(go), static_cast<int>(act), ptr(go),
                         act != MLPK_ACT_NONE ? z.kind() : MLPK_KEEP_NONE, ptr(z.v), z.scales(),
                         act != MLPK_ACT_NONE ? ptr(dz) : nullptr, ptr(got.db), code(db_type), ptr(work),
                         std::max<int64_t>(bytes, 0), stream_of(go)));
  }
  const Weight w = weight_of(w_in);
  if (want_dx) got.dx = dx_of(go, {dz}, {w}, w_in.size(0));
  if (want_dw) {
    Tensor memory;
    std::tie(memory, got.dw) = grad_of(w_in, w.layout);
    dw_of(x.scale.defined() ? restore(x.v, x.scale, go.scalar_type()) : x.v, {dz}, {memory}, w.layout);
  }
  return got;
}

std::tuple<Tensor, Kept, Kept> gated_forward(const Tensor& x_in, const Tensor& wg_in, const Tensor& wu_in,
                                             const Tensor& wd_in, const Tensor& r, int64_t act, int64_t keep) {
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = aligned(x_in);
  const int64_t rows = rows_of(x), width = wg_in.size(1);
  const int layout = layout_of(wg_in) == layout_of(wu_in) ? layout_of(wg_in) : MLPK_W_IN_OUT;
  const Weight wg = weight_in(wg_in, layout), wu = weight_in(wu_in, layout);
  Kept g = keep_for(x, rows, width, keep), u = keep_for(x, rows, width, keep);
  const Tensor h = at::empty({rows, width}, x.options());
  check("mlpk_gated", mlpk_gated(rows, static_cast<int>(x.size(-1)), static_cast<int>(width), code(x),
                                 static_cast<int>(act), ptr(x), ptr(wg.t), ptr(wu.t), layout, ptr(h), g.kind(), ptr(g.v),
                                 g.scales(), ptr(u.v), u.scales(), stream_of(x)));
  Tensor out = linear_forward(h, weight_of(wd_in), wd_in.size(1), Tensor(), r, MLPK_ACT_NONE, nullptr);
  return {out.view(with_width(x, wd_in.size(1))), std::move(g), std::move(u)};
}

struct GatedGrads {
  Tensor dx, dwg, dwu, dwd;
};
GatedGrads gated_backward(const Tensor& go_in, const Kept& x, const Tensor& wg_in, const Tensor& wu_in, const Tensor& wd_in,
                          const Kept& g_in, const Kept& u_in, int64_t act, bool want_dx, bool want_dgu, bool want_dd) {
  const c10::cuda::CUDAGuard guard(go_in.device());
  const Tensor go = aligned(go_in);
  check_saved(weight_for(wd_in, go) && wd_in.size(1) == go.size(-1) && weight_for(wg_in, go) && weight_for(wu_in, go));
  const int64_t rows = rows_of(go), width = wd_in.size(0), pitch = mlpk_fp8_pitch(static_cast<int>(width));
  check_saved(wg_in.size(1) == width && wu_in.sizes() == wg_in.sizes() && kept_for(g_in, go, rows, width, pitch) &&
              kept_for(u_in, go, rows, width, pitch) && g_in.kind() == u_in.kind() &&
              (!want_dgu || kept_for(x, go, rows, wg_in.size(0), wg_in.size(0))));
  const Kept g = aligned(g_in), u = aligned(u_in);
  const Weight wd = weight_of(wd_in);
  Tensor dg = at::empty({rows, width}, go.options()), du = at::empty_like(dg), h = at::empty_like(dg);
  check("mlpk_gated_bwd",
        mlpk_gated_bwd(rows, static_cast<int>(width), static_cast<int>(go.size(-1)), code(go), static_cast<int>(act),
                       ptr(go), ptr(wd.t), wd.layout, g.kind(), ptr(g.v), g.scales(), ptr(u.v), u.scales(), ptr(dg),
                       ptr(du), ptr(h), stream_of(go)));
  GatedGrads got;
  Tensor memory, other;
  if (want_dd) {
    std::tie(memory, got.dwd) = grad_of(wd_in, wd.layout);
    dw_of(h, {go}, {memory}, wd.layout);
  }
  h.reset();
  const int layout = layout_of(wg_in) == layout_of(wu_in) ? layout_of(wg_in) : MLPK_W_IN_OUT;
  if (want_dx) got.dx = dx_of(go, {dg, du}, {weight_in(wg_in, layout), weight_in(wu_in, layout)}, wg_in.size(0));
  if (want_dgu) {
    std::tie(memory, got.dwg) = grad_of(wg_in, layout);
    std::tie(other, got.dwu) = grad_of(wu_in, layout);
    dw_of(x.scale.defined() ? restore(x.v, x.scale, go.scalar_type()) : x.v, {dg, du}, {memory, other}, layout);
  }
  return got;
}

// What a node keeps of its input, if a weight's gradient needs it.
Kept input_kept(const Tensor& x, bool wanted, bool fp8) {
  if (!wanted) return {};
  if (!fp8) return {x, Tensor()};
  return checkpoint(x);
}

struct LinearNode : torch::autograd::Function<LinearNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias,
                               const std::optional<Tensor>& residual, int64_t act, bool fp8) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
    const bool any = x.requires_grad() || w.requires_grad() || (b.defined() && b.requires_grad());
    auto [out, z] = linear_kept(x, w, b, r, act, act != MLPK_ACT_NONE && any ? (fp8 ? MLPK_KEEP_FP8 : MLPK_KEEP_16) : 0);
    const Kept k = input_kept(x, w.requires_grad(), fp8);
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = static_cast<int64_t>(b.defined() ? b.scalar_type() : at::ScalarType::Undefined);
    ctx->saved_data["residual"] = r.defined();
    ctx->saved_data["x_needs"] = x.requires_grad();
    ctx->save_for_backward({k.v, k.scale, w, z.v, z.scale});
    return {out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &go = grads[0], &w = saved[2];
    const int64_t act = ctx->saved_data["act"].toInt();
    const auto db_type = static_cast<at::ScalarType>(ctx->saved_data["bias"].toInt());
    const bool has_b = db_type != at::ScalarType::Undefined, has_r = ctx->saved_data["residual"].toBool();
    const bool want_dx = ctx->needs_input_grad(0), want_dw = ctx->needs_input_grad(1);
    const bool want_db = has_b && ctx->needs_input_grad(2), want_dr = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
    LinearGrads got;
    if (!go.defined()) return variable_list(6);
    if (want_dx || want_dw || want_db) {
      const at::NoGradGuard no_grad;
      const at::ScalarType type = has_b ? db_type : go.scalar_type();
      if (direct({&go, &saved[0], &saved[1], &w, &saved[3], &saved[4]})) {
        got = linear_backward(go, {saved[0], saved[1]}, w, {saved[3], saved[4]}, act, type, want_dx, want_dw, want_db);
      } else {
        refuse_tangents({&go, &saved[0], &w});
        const std::vector<Tensor> t =
            operate("mlpk::linear_bwd", go, maybe(saved[0]), maybe(saved[1]), w, maybe(saved[3]), maybe(saved[4]), act,
                    type, want_dx, want_dw, want_db)
                .toTensorVector();
        size_t i = 0;
        if (want_dx) got.dx = t[i++];
        if (want_dw) got.dw = t[i++];
        if (want_db) got.db = t[i++];
      }
    }
    // Whether a gradient depends on an input that needs one itself (wanted in this
    // pass or not): through z on x, w and b, which are not all without one.
    const bool by_z = act != MLPK_ACT_NONE;
    return {once_if(got.dx, go, by_z || w.requires_grad()),
            once_if(got.dw, go, by_z || ctx->saved_data["x_needs"].toBool()), once_if(got.db, go, by_z),
            want_dr ? go : Tensor(), Tensor(), Tensor()};
  }
};

struct GatedNode : torch::autograd::Function<GatedNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                               const std::optional<Tensor>& residual, int64_t act, bool fp8) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor r = residual.value_or(Tensor());
    const bool any = x.requires_grad() || wg.requires_grad() || wu.requires_grad() || wd.requires_grad();
    auto [out, g, u] = gated_forward(x, wg, wu, wd, r, act, any ? (fp8 ? MLPK_KEEP_FP8 : MLPK_KEEP_16) : 0);
    const Kept k = input_kept(x, wg.requires_grad() || wu.requires_grad(), fp8);
    ctx->saved_data["act"] = act;
    ctx->saved_data["residual"] = r.defined();
    ctx->saved_data["x_needs"] = x.requires_grad();
    ctx->save_for_backward({k.v, k.scale, wg, wu, wd, g.v, g.scale, u.v, u.scale});
    return {out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &go = grads[0], &x = saved[0], &wg = saved[2], &wu = saved[3], &wd = saved[4];
    const int64_t act = ctx->saved_data["act"].toInt();
    const bool want_dx = ctx->needs_input_grad(0), want_g = ctx->needs_input_grad(1), want_u = ctx->needs_input_grad(2);
    const bool want_d = ctx->needs_input_grad(3), any = want_dx || want_g || want_u || want_d;
    const bool want_dr = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(4);
    GatedGrads got;
    if (!go.defined()) return variable_list(7);
    if (any) {
      const at::NoGradGuard no_grad;
      if (direct({&go, &x, &saved[1], &wg, &wu, &wd, &saved[5], &saved[6], &saved[7], &saved[8]})) {
        got = gated_backward(go, {x, saved[1]}, wg, wu, wd, {saved[5], saved[6]}, {saved[7], saved[8]}, act, want_dx,
                             want_g || want_u, want_d);
      } else {
        refuse_tangents({&go, &x, &wg, &wu, &wd});
        const std::vector<Tensor> t =
            operate("mlpk::gated_mlp_bwd", go, maybe(x), maybe(saved[1]), wg, wu, wd, saved[5], maybe(saved[6]), saved[7],
                    maybe(saved[8]), act, want_dx, want_g || want_u, want_d)
                .toTensorVector();
        size_t i = 0;
        if (want_dx) got.dx = t[i++];
        if (want_g || want_u) {
          got.dwg = t[i++];
          got.dwu = t[i++];
        }
        if (want_d) got.dwd = t[i++];
      }
    }
    // Whether a gradient depends on an input that needs one itself: w_up's does not
    // on w_up, w_down's not on w_down.
    const bool x_or_g = ctx->saved_data["x_needs"].toBool() || wg.requires_grad();
    return {once_if(got.dx, go, true),
            once_if(want_g ? got.dwg : Tensor(), go, true),
            once_if(want_u ? got.dwu : Tensor(), go, x_or_g || wd.requires_grad()),
            once_if(got.dwd, go, x_or_g || wu.requires_grad()),
            want_dr ? go : Tensor(),
            Tensor(),
            Tensor()};
  }
};

bool ff_x(const Tensor& x) {
  return x.is_cuda() && operand_type(x) && x.dim() >= 1 && ff_width(x.size(-1)) && rows_of(x) <= kFfMaxRows;
}
bool ff_weight(const Tensor& w, const Tensor& x, int64_t d_in) {
  return w.dim() == 2 && w.size(0) == d_in && ff_width(w.size(1)) && w.scalar_type() == x.scalar_type() &&
         w.device() == x.device();
}
bool ff_residual(const Tensor& r, const Tensor& x, int64_t d_out) {
  return !r.defined() || (r.sizes() == at::IntArrayRef(with_width(x, d_out)) && r.scalar_type() == x.scalar_type() &&
                          r.device() == x.device());
}

py::object linear(const Tensor& x, const Tensor& w, const std::optional<Tensor>& bias,
                  const std::optional<Tensor>& residual, int64_t act, bool fp8) {
  const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
  if (act < 0 || act >= kActs || !ff_x(x) || !ff_weight(w, x, x.size(-1)) || !ff_residual(r, x, w.size(1)) ||
      (b.defined() && (b.dim() != 1 || b.size(0) != w.size(1) || b.device() != x.device() || !weight_type(b, x))) ||
      !direct({&x, &w, &b, &r}))
    return py::none();
  Tensor out;
  {
    py::gil_scoped_release no_gil;
    out = needs_grad({&x, &w, &b, &r}) ? LinearNode::apply(x, w, maybe(b), maybe(r), act, fp8)[0]
                                       : linear_kept(x, w, b, r, act, MLPK_KEEP_NONE).first;
  }
  return py::cast(out);
}

py::object gated_mlp(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd,
                     const std::optional<Tensor>& residual, int64_t act, bool fp8) {
  const Tensor r = residual.value_or(Tensor());
  if (act < 0 || act >= kActs || !ff_x(x) || !ff_weight(wg, x, x.size(-1)) || !ff_weight(wu, x, x.size(-1)) ||
      wu.size(1) != wg.size(1) || !ff_weight(wd, x, wg.size(1)) || !ff_residual(r, x, wd.size(1)) ||
      !direct({&x, &wg, &wu, &wd, &r}))
    return py::none();
  Tensor out;
  {
    py::gil_scoped_release no_gil;
    out = needs_grad({&x, &wg, &wu, &wd, &r}) ? GatedNode::apply(x, wg, wu, wd, maybe(r), act, fp8)[0]
                                              : std::get<0>(gated_forward(x, wg, wu, wd, r, act, MLPK_KEEP_NONE));
  }
  return py::cast(out);
}

py::object fp8_checkpoint(const Tensor& x) {
  if (!x.is_cuda() || code(x) < 0 || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > 0x7fffffff || needs_grad({&x}) ||
      !direct({&x}))
    return py::none();
  Kept k;
  {
    py::gil_scoped_release no_gil;
    k = checkpoint(x);
  }
  return py::make_tuple(k.v, k.scale);
}
py::object fp8_restore(const Tensor& q, const Tensor& scale, at::ScalarType type) {
  if (!q.is_cuda() || q.scalar_type() != at::kFloat8_e4m3fn || q.dim() < 1 || q.size(-1) < 1 ||
      q.size(-1) > 0x7fffffff || scale.scalar_type() != at::kFloat || scale.device() != q.device() ||
      scale.sizes() != at::IntArrayRef(with_width(q, (q.size(-1) + 127) / 128)) || !direct({&q, &scale}))
    return py::none();
  Tensor x;
  {
    py::gil_scoped_release no_gil;
    x = restore(q, scale, type);
  }
  return py::cast(x);
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
  m.def("linear", &linear);
  m.def("gated_mlp", &gated_mlp);
  m.def("fp8_checkpoint", &fp8_checkpoint);
  m.def("fp8_restore", &fp8_restore);
  using Maybe = std::optional<Tensor>;
  m.def("linear_forward", [](const Tensor& x, const Tensor& w, const Maybe& b, const Maybe& r, int64_t act, int64_t keep) {
    const auto [out, z] = linear_kept(x, w, b.value_or(Tensor()), r.value_or(Tensor()), act, keep);
    return std::make_tuple(out, maybe(z.v), maybe(z.scale));
  });
  m.def("linear_backward", [](const Tensor& go, const Maybe& x, const Maybe& x_scale, const Tensor& w, const Maybe& z,
                              const Maybe& z_scale, int64_t act, bool db32, bool want_dx, bool want_dw, bool want_db) {
    const LinearGrads g = linear_backward(go, {x.value_or(Tensor()), x_scale.value_or(Tensor())}, w,
                                          {z.value_or(Tensor()), z_scale.value_or(Tensor())}, act,
                                          db32 ? at::kFloat : go.scalar_type(), want_dx, want_dw, want_db);
    return std::make_tuple(maybe(g.dx), maybe(g.dw), maybe(g.db));
  });
  m.def("gated_forward", [](const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const Maybe& r,
                            int64_t act, int64_t keep) {
    const auto [out, g, u] = gated_forward(x, wg, wu, wd, r.value_or(Tensor()), act, keep);
    return std::make_tuple(out, maybe(g.v), maybe(g.scale), maybe(u.v), maybe(u.scale));
  });
  m.def("gated_backward", [](const Tensor& go, const Maybe& x, const Maybe& x_scale, const Tensor& wg, const Tensor& wu,
                             const Tensor& wd, const Tensor& g, const Maybe& g_scale, const Tensor& u,
                             const Maybe& u_scale, int64_t act, bool want_dx, bool want_dgu, bool want_dd) {
    const GatedGrads t = gated_backward(go, {x.value_or(Tensor()), x_scale.value_or(Tensor())}, wg, wu, wd,
                                        {g, g_scale.value_or(Tensor())}, {u, u_scale.value_or(Tensor())}, act, want_dx,
                                        want_dgu, want_dd);
    return std::make_tuple(maybe(t.dx), maybe(t.dwg), maybe(t.dwu), maybe(t.dwd));
  });
  m.def("checkpoint", [](const Tensor& x) {
    const Kept k = checkpoint(x);
    return std::make_tuple(k.v, k.scale);
  });
  m.def("restore", &restore);
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
