// Python entry points of the norms, SwiGLU and the vocabulary loss (motif_b200/ops.py), with their gradients:
// argument checks, allocation, the call of the C ABI and the autograd node in one compiled step, and a
// backward pass that needs no Python.  As Python autograd functions over ctypes a forward and backward pass
// of a small norm took 130 us of host time, more than its elementary operations; here it takes 61 to 69, as torch.neg
// does (67): the autograd engine's own.  A loss alone takes 12.
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/engine.h>
#include <torch/csrc/autograd/graph_task.h>

#include <atomic>
#include <string>

#include "host.hpp"

namespace {

using namespace mb_host;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// Kernels that backward passes have launched (on the autograd engine's threads), for launch trackers.
std::atomic<int64_t> backward_kernels{0};
struct Counted {
  const int64_t before = motif_b200_launches();
  ~Counted() { backward_kernels += motif_b200_launches() - before; }
};

bool grad_needed(const Tensor& t) { return t.defined() && t.requires_grad(); }
// A forward-mode tangent is refused, not dropped.
void no_tangent(const Tensor& t) {
  if (t.defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
    throw Refusal{PyExc_NotImplementedError, "motif_b200 ops have no forward-mode derivatives"};
}
// In a backward pass, whose errors travel through the autograd engine: torch's own exceptions.
void check_backward(const char* name, int rc) {
  if (rc == MB_OK) return;
  const std::string what = std::string(name) + ": " + motif_b200_last_error();
  TORCH_CHECK_NOT_IMPLEMENTED(rc != MB_ERR_UNSUPPORTED, what);
  TORCH_CHECK(rc != MB_ERR_CUDA, what);
  TORCH_CHECK_VALUE(false, what);
}
// A backward pass that is itself recorded (create_graph=True): its results would look like constants, and the
// terms of a second derivative that pass through here be dropped.
void first_order() {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::GradMode::is_enabled(),
                              "motif_b200 ops have no second derivatives (create_graph=True)");
}

// The values that t stands for as they lie in memory (a copy of a view that is negated lazily).
Tensor resolved(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
// t as rows of its last dimension whose elements lie next to each other (a copy where they do not).
Tensor rows_of(const Tensor& lazy) {
  const Tensor t = resolved(lazy);
  Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / std::max<int64_t>(t.size(-1), 1), t.size(-1)});
  return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}
const Tensor& cuda(const char* name, PyObject* o) {
  const Tensor& t = tensor(name, o);
  if (!t.is_cuda()) refuse(std::string(name) + " must live on CUDA");
  return t;
}
Tensor weight_of(const char* op, PyObject* o, int64_t n, const Tensor& x) {
  if (o == Py_None) return Tensor();
  const Tensor& w = cuda("weight", o);
  if (w.dim() != 1 || w.size(0) != n)
    refuse(std::string(op) + ": weight must be [" + std::to_string(n) + "], got " + shape_of(w));
  if (w.device() != x.device()) refuse(std::string(op) + ": weight is on " + w.device().str() + ", x on " + x.device().str());
  dtype_code(w.scalar_type());
  return w;
}
// x's shape with another last dimension.
std::vector<int64_t> shape_with(const Tensor& x, int64_t last) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = last;
  return s;
}
// Plain [n] memory of a weight.
Tensor flat(const Tensor& w) { return w.defined() ? resolved(w).contiguous() : w; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// What a backward pass finds saved may be other than what its forward pass saved (a hook's mistake, an exchanged
// .data): the kernels go by the sizes of dy, so x has to be of them, `last` in its last dimension.
void came_back(const char* op, const Tensor& x, const Tensor& dy, int64_t last) {
  TORCH_CHECK(x.device() == dy.device() && x.scalar_type() == dy.scalar_type() && x.sizes().vec() == shape_with(dy, last), op,
              ": the input saved by its forward pass came back as another");
}

// ------------------------------------------------------------------ norms
struct NormFunction : torch::autograd::Function<NormFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, double eps, bool gated) {
    const c10::Device dev = x.device();
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor r = rows_of(x), w = weight ? flat(*weight) : Tensor();
    const int64_t n = r.size(1) / (gated ? 2 : 1);
    Tensor y = fresh(shape_with(x, n), x.scalar_type(), dev);
    check("motif_b200_rms_norm_train",
          motif_b200_rms_norm_train(r.data_ptr(), ptr(w), w.defined() ? dtype_code(w.scalar_type()) : MB_F32,
                                    y.data_ptr(), r.size(0), n, r.stride(0), n, gated, (float)eps,
                                    dtype_code(x.scalar_type()), stream_of(dev)));
    ctx->save_for_backward({x, weight ? *weight : Tensor()});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["gated"] = gated;
    ctx->saved_data["weight"] = (int64_t)(weight ? weight->scalar_type() : at::ScalarType::Undefined);
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order();
    const Counted counted;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1];
    const bool gated = ctx->saved_data["gated"].toBool();
    const float eps = (float)ctx->saved_data["eps"].toDouble();
    const c10::Device dev = grads[0].device();
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t n = grads[0].size(-1);
    came_back("rms_norm", x, grads[0], gated ? 2 * n : n);
    TORCH_CHECK(ctx->saved_data["weight"].toInt() ==
                        (weight.defined() ? (int64_t)weight.scalar_type() : (int64_t)at::ScalarType::Undefined) &&
                    (!weight.defined() || (weight.device() == dev && weight.sizes() == at::IntArrayRef({n}))),
                "rms_norm: the weight saved by its forward pass came back as another");
    const Tensor r = rows_of(x), dy = rows_of(grads[0]), w = flat(weight);
    const int64_t m = r.size(0);
    Tensor dx = fresh(x.sizes(), x.scalar_type(), dev), dw;
    const int wd = w.defined() ? dtype_code(w.scalar_type()) : MB_F32, dc = dtype_code(x.scalar_type());
    int64_t bytes = 0;
    c10::DataPtr ws;
    if (w.defined() && ctx->needs_input_grad(1)) {
      dw = fresh({n}, w.scalar_type(), dev);
      bytes = motif_b200_rms_norm_backward_workspace_bytes(m, n, dc);
      ws = c10::cuda::CUDACachingAllocator::get()->allocate((size_t)bytes);
    }
    check_backward("motif_b200_rms_norm_backward",
                   motif_b200_rms_norm_backward(r.data_ptr(), ptr(w), wd, dy.data_ptr(), dx.data_ptr(), ptr(dw), m, n,
                                                r.stride(0), dy.stride(0), r.size(1), gated, eps, ws.get(), bytes, dc,
                                                stream_of(dev)));
    return {ctx->needs_input_grad(0) ? dx : Tensor(), dw, Tensor(), Tensor()};
  }
};

// x, weight or None, eps, gated
PyObject* norm(PyObject* const* a) {
  const int gated = PyObject_IsTrue(a[3]);
  if (gated < 0) throw Refusal{nullptr, ""};
  const char* op = gated ? "gated_rms_norm" : "rms_norm";
  const Tensor& x = cuda("x", a[0]);
  if (x.dim() < 1) refuse(std::string(op) + ": x must have a last dimension");
  if (gated && x.size(-1) % 2) refuse("gated_rms_norm: x must be [..., 2 * dim], got " + shape_of(x));
  const int64_t n = x.size(-1) / (gated ? 2 : 1);
  const int dc = dtype_code(x.scalar_type());
  const Tensor w = weight_of(op, a[1], n, x);
  const double eps = number(a[2]);
  no_tangent(x);
  no_tangent(w);
  Tensor y;
  {
    const NoGil others;
    if (at::GradMode::is_enabled() && (grad_needed(x) || grad_needed(w))) {
      y = NormFunction::apply(x, w.defined() ? OptTensor(w) : OptTensor(), eps, gated != 0);
    } else {
      const c10::Device dev = x.device();
      const c10::cuda::CUDAGuard guard(dev);
      const at::AutoDispatchBelowADInplaceOrView plain;
      const Tensor r = rows_of(x), wt = w.defined() ? flat(w.to(x.scalar_type())) : w;
      y = fresh(shape_with(x, n), x.scalar_type(), dev);
      auto* call = gated ? motif_b200_gated_rms_norm : motif_b200_rms_norm;
      if (r.size(0) || !n)
        check(gated ? "motif_b200_gated_rms_norm" : "motif_b200_rms_norm",
              call(r.data_ptr(), ptr(wt), y.data_ptr(), r.size(0), n, r.stride(0), n, (float)eps, dc, stream_of(dev)));
    }
  }
  return wrap(y);
}

// ------------------------------------------------------------------ SwiGLU
struct SwiGLUFunction : torch::autograd::Function<SwiGLUFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x) {
    const c10::Device dev = x.device();
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor r = rows_of(x);
    const int64_t n = r.size(1) / 2;
    Tensor y = fresh(shape_with(x, n), x.scalar_type(), dev);
    check("motif_b200_swiglu_train",
          motif_b200_swiglu_train(r.data_ptr(), y.data_ptr(), r.size(0), n, r.stride(0), n,
                                  dtype_code(x.scalar_type()), stream_of(dev)));
    ctx->save_for_backward({x});
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order();
    const Counted counted;
    const Tensor x = ctx->get_saved_variables()[0];
    const c10::Device dev = grads[0].device();
    const c10::cuda::CUDAGuard guard(dev);
    came_back("swiglu", x, grads[0], 2 * grads[0].size(-1));
    const Tensor r = rows_of(x), dy = rows_of(grads[0]);
    Tensor dx = fresh(x.sizes(), x.scalar_type(), dev);
    check_backward("motif_b200_swiglu_backward",
                   motif_b200_swiglu_backward(r.data_ptr(), dy.data_ptr(), dx.data_ptr(), r.size(0), dy.size(1),
                                              r.stride(0), dy.stride(0), r.size(1), dtype_code(x.scalar_type()),
                                              stream_of(dev)));
    return {dx};
  }
};

// x, split along the last dimension
PyObject* swiglu(PyObject* const* a) {
  const Tensor& x = cuda("x", a[0]);
  if (x.dim() < 1 || x.size(-1) % 2) refuse("SwiGLU needs an even split dimension, got " + shape_of(x));
  const int dc = dtype_code(x.scalar_type());
  no_tangent(x);
  Tensor y;
  {
    const NoGil others;
    if (at::GradMode::is_enabled() && x.requires_grad()) {
      y = SwiGLUFunction::apply(x);
    } else {
      const c10::Device dev = x.device();
      const c10::cuda::CUDAGuard guard(dev);
      const at::AutoDispatchBelowADInplaceOrView plain;
      const Tensor r = rows_of(x);
      const int64_t n = r.size(1) / 2;
      y = fresh(shape_with(x, n), x.scalar_type(), dev);
      if (r.size(0) || !n)
        check("motif_b200_swiglu", motif_b200_swiglu(r.data_ptr(), y.data_ptr(), r.size(0), n, r.stride(0), n, dc,
                                                     stream_of(dev)));
    }
  }
  return wrap(y);
}

// ------------------------------------------------------------------ vocabulary loss
struct Loss {
  Tensor loss, state;
  int64_t backward_bytes;
};
Loss loss_forward(const Tensor& x, const Tensor& weight, const Tensor& labels, int64_t ignore, int64_t reduction) {
  const c10::Device dev = x.device();
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor r = rows_of(x), w = rows_of(weight), lab = resolved(labels).to(at::kLong).contiguous();
  const int64_t n = r.size(0), d = r.size(1), v = w.size(0);
  const int dc = dtype_code(x.scalar_type());
  int64_t bytes[3];
  check("motif_b200_linear_cross_entropy_bytes",
        motif_b200_linear_cross_entropy_bytes(w.data_ptr(), w.stride(0), n, v, d, dc, bytes));
  Loss out;
  out.state = fresh({bytes[0]}, at::kByte, dev);
  out.loss = reduction == 0 ? fresh(labels.sizes(), at::kFloat, dev) : fresh({}, at::kFloat, dev);
  out.backward_bytes = bytes[2];
  const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate((size_t)bytes[1]);
  check("motif_b200_linear_cross_entropy",
        motif_b200_linear_cross_entropy(r.data_ptr(), r.stride(0), w.data_ptr(), w.stride(0), lab.data_ptr<int64_t>(),
                                        ignore, (int)reduction, out.loss.data_ptr<float>(), n, v, d,
                                        out.state.data_ptr(), bytes[0], ws.get(), bytes[1], dc, stream_of(dev)));
  return out;
}

// What saved-tensor hooks (offloading, packing) give back may lie elsewhere, with other strides: `t` as plain memory
// at a boundary of `bytes`.
Tensor plain(const Tensor& t, uintptr_t bytes) {
  if (t.is_contiguous() && !t.is_neg() && (uintptr_t)t.data_ptr() % bytes == 0) return t;
  return resolved(t).clone(at::MemoryFormat::Contiguous);
}
// w [V, d] with rows that begin at 16-byte boundaries.
Tensor aligned_rows(const Tensor& w) {
  const int64_t step = 16 / w.element_size();
  if ((uintptr_t)w.data_ptr() % 16 == 0 && w.stride(0) % step == 0 && w.stride(0) >= w.size(1)) return w;
  Tensor out = at::empty({w.size(0), (w.size(1) + step - 1) / step * step}, w.options()).narrow(1, 0, w.size(1));
  return out.copy_(w);
}

// Where one gradient arrives for all tokens, the forward pass computes the gradients as well, in one pass over
// the logits, and the backward pass multiplies them with what arrived.  (fp16, whose range is too small for that,
// and one gradient per token: the logits are computed again in the backward pass.)
struct LossFunction : torch::autograd::Function<LossFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& labels, int64_t ignore,
                        int64_t reduction) {
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["words"] = weight.size(0);
    ctx->saved_data["dtype"] = (int64_t)weight.scalar_type();
    const bool again = reduction == 0 || x.scalar_type() == at::kHalf;
    ctx->saved_data["again"] = again;
    if (again) {
      Loss out = loss_forward(x, weight, labels, ignore, reduction);
      ctx->save_for_backward({weight, out.state});
      ctx->saved_data["bytes"] = out.backward_bytes;
      ctx->saved_data["state"] = out.state.numel();
      return out.loss;
    }
    const c10::Device dev = x.device();
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor r = rows_of(x), w = rows_of(weight), lab = resolved(labels).to(at::kLong).contiguous();
    const int64_t n = r.size(0), d = r.size(1), v = w.size(0);
    const int dc = dtype_code(x.scalar_type());
    Tensor loss = fresh({}, at::kFloat, dev), dx, dw;
    if (x.requires_grad()) dx = fresh(x.sizes(), x.scalar_type(), dev);
    if (weight.requires_grad()) dw = fresh({v, d}, x.scalar_type(), dev);
    const int64_t bytes = motif_b200_linear_cross_entropy_train_workspace_bytes(w.data_ptr(), w.stride(0), n, v, d, dc);
    check("motif_b200_linear_cross_entropy_train", bytes < 0 ? MB_ERR_SHAPE : MB_OK);
    const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate((size_t)bytes);
    check("motif_b200_linear_cross_entropy_train",
          motif_b200_linear_cross_entropy_train(r.data_ptr(), r.stride(0), w.data_ptr(), w.stride(0),
                                                lab.data_ptr<int64_t>(), ignore, (int)reduction,
                                                loss.data_ptr<float>(), ptr(dx), ptr(dw), n, v, d, ws.get(), bytes, dc,
                                                stream_of(dev)));
    // saved-tensor hooks may keep what they are handed: then the backward pass writes elsewhere
    ctx->saved_data["own"] = !at::SavedTensorDefaultHooks::get_hooks().has_value();
    ctx->save_for_backward({dx, dw});
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    first_order();
    const Counted counted;
    const variable_list saved = ctx->get_saved_variables();
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const int64_t reduction = ctx->saved_data["reduction"].toInt();
    const int64_t v = ctx->saved_data["words"].toInt(), d = shape.back();
    const auto dtype = (at::ScalarType)ctx->saved_data["dtype"].toInt();
    const int dc = dtype_code(dtype);
    const c10::Device dev = grads[0].device();
    const c10::cuda::CUDAGuard guard(dev);
    // what hooks hand back is read as what was saved (and memory is indexed with what lies in the state)
    auto came_back = [&](const Tensor& t, at::ScalarType type, at::IntArrayRef sizes) {
      TORCH_CHECK(t.device() == dev && t.scalar_type() == type && t.sizes() == sizes,
                  "linear_cross_entropy: the tensors saved by its forward pass came back as others");
    };
    Tensor dx, dw;
    if (!ctx->saved_data["again"].toBool()) {
      Tensor sx = saved[0], sw = saved[1];
      if (sx.defined()) {
        came_back(sx, dtype, shape);
        sx = plain(sx, 16);
      }
      if (sw.defined()) {
        came_back(sw, dtype, {v, d});
        sw = plain(sw, 16);
      }
      // a graph that is not kept has no other use for them: they are multiplied where they are (not while a CUDA
      // graph captures this pass, which may run again by itself)
      const bool keep = !ctx->saved_data["own"].toBool() || torch::autograd::get_current_graph_task_keep_graph() ||
                        c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
      if (sx.defined() && ctx->needs_input_grad(0)) dx = keep ? fresh(shape, dtype, dev) : sx;
      if (sw.defined() && ctx->needs_input_grad(1)) dw = keep ? fresh({v, d}, dtype, dev) : sw;
      check_backward("motif_b200_scale_gradients",
                     motif_b200_scale_gradients(dx.defined() ? sx.data_ptr() : nullptr, ptr(dx),
                                                dx.defined() ? dx.numel() : 0, dw.defined() ? sw.data_ptr() : nullptr,
                                                ptr(dw), dw.defined() ? dw.numel() : 0,
                                                resolved(grads[0]).data_ptr<float>(), dc, stream_of(dev)));
      return {dx, dw, Tensor(), Tensor(), Tensor()};
    }
    came_back(saved[0], dtype, {v, d});
    came_back(saved[1], at::kByte, {ctx->saved_data["state"].toInt()});
    const int64_t bytes = ctx->saved_data["bytes"].toInt();
    const Tensor state = plain(saved[1], 256), up = reduction == 0 ? resolved(grads[0]).reshape({-1}) : resolved(grads[0]);
    Tensor w = rows_of(saved[0]);
    int64_t n = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) n *= shape[i];
    // a weight that the forward pass read where it was and that came back with other strides
    int64_t now[3];
    check_backward("motif_b200_linear_cross_entropy_bytes",
                   motif_b200_linear_cross_entropy_bytes(w.data_ptr(), w.stride(0), n, v, d, dc, now));
    if (now[0] > state.numel()) w = aligned_rows(w);
    if (ctx->needs_input_grad(0)) dx = fresh(shape, dtype, dev);
    if (ctx->needs_input_grad(1)) dw = fresh({v, d}, dtype, dev);
    const c10::DataPtr ws = c10::cuda::CUDACachingAllocator::get()->allocate((size_t)bytes);
    check_backward("motif_b200_linear_cross_entropy_backward",
                   motif_b200_linear_cross_entropy_backward(
                       w.data_ptr(), w.stride(0), up.data_ptr<float>(), reduction == 0 ? up.stride(0) : 0,
                       (int)reduction, ptr(dx), ptr(dw), n, v, d, state.data_ptr(), state.numel(), ws.get(), bytes,
                       dc, stream_of(dev)));
    return {dx, dw, Tensor(), Tensor(), Tensor()};
  }
};

// x, weight, labels, ignore_index, reduction (0 none, 1 mean, 2 sum)
PyObject* loss(PyObject* const* a) {
  const Tensor &x = cuda("x", a[0]), &w = cuda("weight", a[1]), &labels = cuda("labels", a[2]);
  const int64_t ignore = whole(a[3]), reduction = whole(a[4]);
  if (x.dim() < 1 || w.dim() != 2 || w.size(1) != x.size(-1))
    refuse("x [..., d] and weight [V, d] expected, got " + shape_of(x) + " and " + shape_of(w));
  const at::IntArrayRef lead = x.sizes().slice(0, (size_t)x.dim() - 1);
  if (labels.sizes() != lead) refuse("labels must be x's shape " + shape_of(x) + " without the last, got " + shape_of(labels));
  if (!at::isIntegralType(labels.scalar_type(), false)) refuse("labels must be whole numbers, got " + kind_of(labels));
  dtype_code(x.scalar_type());
  if (w.scalar_type() != x.scalar_type()) refuse("x and weight must share one dtype, got " + kind_of(x) + " and " + kind_of(w));
  if (w.device() != x.device() || labels.device() != x.device())
    refuse("x, weight and labels must share one device, got " + x.device().str() + ", " + w.device().str() + " and " +
           labels.device().str());
  if (!w.numel()) refuse("weight must not be empty, got " + shape_of(w));
  no_tangent(x);
  no_tangent(w);
  Tensor out;
  {
    const NoGil others;
    if (at::GradMode::is_enabled() && (grad_needed(x) || grad_needed(w))) {
      out = LossFunction::apply(x, w, labels, ignore, reduction);
    } else {
      const at::AutoDispatchBelowADInplaceOrView plain;
      out = loss_forward(x, w, labels, ignore, reduction).loss;
    }
  }
  return wrap(out);
}

// Kernels launched by backward passes so far.
PyObject* backward_launches(PyObject* const*) { return PyLong_FromLongLong(backward_kernels.load()); }

PyMethodDef methods[] = {method<norm, 4>("rms_norm"), method<swiglu, 1>("swiglu"),
                         method<loss, 5>("linear_cross_entropy"), method<backward_launches, 0>("backward_launches"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_train_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__train_host(void) { return PyModule_Create(&module); }
