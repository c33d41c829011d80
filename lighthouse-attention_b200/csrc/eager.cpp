// Eager calls of the norm and the losses with their autograd nodes, in C++.
//
// The kernels of these operators take a few to a few hundred microseconds; a call
// through a custom op or a Python autograd function costs 50 to 150 us of host
// time, forward and backward.  The functions here check the plain case (dense
// tensors of one device, aligned, of the supported types and shapes), allocate,
// and call the C entry points of liblighthouse_b200.so, whose addresses Python
// hands over once (bind).  For any other case they return None and do nothing:
// the Python functions then take their own path, which copies what is strided,
// refuses what is wrong and says why.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <map>
#include <string>

#include "../../include/lighthouse_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
  decltype(&lh_last_error) last_error;
  decltype(&lh_rms_norm_fwd) norm_fwd;
  decltype(&lh_rms_norm_bwd_workspace_size) norm_ws;
  decltype(&lh_rms_norm_bwd) norm_bwd;
  decltype(&lh_linear_loss_workspace_size) loss_ws;
  decltype(&lh_linear_loss_kept_size) loss_kept;
  decltype(&lh_linear_xent_fwd) xent_fwd;
  decltype(&lh_linear_xent_bwd) xent_bwd;
  decltype(&lh_linear_distill_fwd) distill_fwd;
  decltype(&lh_linear_distill_bwd) distill_bwd;
} api{};

template <class F>
void set(F& f, const std::map<std::string, uintptr_t>& m, const char* name) {
  f = reinterpret_cast<F>(m.at(name));
}
void bind(const std::map<std::string, uintptr_t>& m) {
  set(api.last_error, m, "lh_last_error");
  set(api.norm_fwd, m, "lh_rms_norm_fwd");
  set(api.norm_ws, m, "lh_rms_norm_bwd_workspace_size");
  set(api.norm_bwd, m, "lh_rms_norm_bwd");
  set(api.loss_ws, m, "lh_linear_loss_workspace_size");
  set(api.loss_kept, m, "lh_linear_loss_kept_size");
  set(api.xent_fwd, m, "lh_linear_xent_fwd");
  set(api.xent_bwd, m, "lh_linear_xent_bwd");
  set(api.distill_fwd, m, "lh_linear_distill_fwd");
  set(api.distill_bwd, m, "lh_linear_distill_bwd");
}

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, ": lighthouse_b200 error ", rc, ": ", api.last_error()); }

int dtype_code(at::ScalarType t) { return t == at::kBFloat16 ? LH_DTYPE_BF16 : t == at::kFloat ? LH_DTYPE_F32 : -1; }
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0; }

// A dense, aligned CUDA tensor that nothing wraps or intercepts.
bool plain(const Tensor& t) {
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() && !t.is_conj() && !t.is_neg() &&
         !t.key_set().has_any(c10::python_ks | c10::functorch_transforms_ks) && aligned(t);
}
bool intercepted() { return c10::impl::TorchDispatchModeTLS::any_modes_set(); }

Tensor empty(at::IntArrayRef size, at::ScalarType dtype, at::Device dev) {
  return at::detail::empty_cuda(size, dtype, dev, std::nullopt);
}
Tensor dense16(const Tensor& t) {
  Tensor c = t.resolve_neg().contiguous();          // the bit that says minus is not in the memory
  return aligned(c) ? c : c.clone();
}
void* stream(at::Device dev) { return at::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// A saved tensor, dense and aligned again: hooks on saved tensors may give back other strides, and must not
// give back anything else.
Tensor unpacked(const Tensor& t, at::IntArrayRef size, at::ScalarType type, at::Device dev) {
  TORCH_CHECK(t.defined() && t.layout() == at::kStrided && t.sizes() == size && t.scalar_type() == type && t.device() == dev,
              "lighthouse_b200: a saved tensor came back with another shape, type or device");
  return dense16(t);
}

// Gradients of these functions have no graph of their own: a second derivative raises.
variable_list once(variable_list out) {
  if (at::GradMode::is_enabled()) {
    for (Tensor& t : out)
      if (t.defined()) {
        auto err = std::make_shared<torch::autograd::DelayedError>(
            "trying to differentiate twice through a lighthouse_b200 function, which is differentiable once", 1);
        t = (*err)({t.detach().requires_grad_(true)})[0];
      }
  }
  return out;
}

// ---------------------------------------------------------------- norm
bool norm_case(const Tensor& x, const Tensor& r, const Tensor& w) {
  if (!api.norm_fwd || intercepted() || !plain(x) || !plain(w) || (r.defined() && !plain(r)) || x.dim() < 1) return false;
  const int64_t D = x.size(-1);
  return D % 8 == 0 && D >= 8 && D <= 16384 && x.numel() > 0 && x.numel() / D < (1ll << 31) && w.dim() == 1 && w.size(0) == D &&
         (!r.defined() || r.sizes() == x.sizes()) && dtype_code(x.scalar_type()) >= 0 && dtype_code(w.scalar_type()) >= 0 &&
         (!r.defined() || dtype_code(r.scalar_type()) >= 0) && w.device() == x.device() &&
         (!r.defined() || r.device() == x.device());
}

struct NormOut { Tensor y, h, rstd, scale; };

NormOut norm_forward(const Tensor& x, const Tensor& r, const Tensor& w, double eps, at::ScalarType out, int64_t group,
                     bool with_rstd) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t D = x.size(-1), N = x.numel() / D;
  const bool fp8 = out == at::kFloat8_e4m3fn;
  NormOut o;
  o.y = empty(x.sizes(), out, x.device());
  if (r.defined()) o.h = empty(x.sizes(), r.scalar_type(), x.device());
  if (with_rstd) o.rstd = empty({N}, at::kFloat, x.device());
  if (fp8) {
    auto sizes = x.sizes().vec();
    sizes.back() = group ? (D + 127) / 128 : 1;
    o.scale = empty(sizes, at::kFloat, x.device());
  }
  check(api.norm_fwd(x.const_data_ptr(), dtype_code(x.scalar_type()), r.defined() ? r.const_data_ptr() : nullptr,
                     r.defined() ? dtype_code(r.scalar_type()) : 0, w.const_data_ptr(), dtype_code(w.scalar_type()), N,
                     (int)D, (float)eps, o.y.mutable_data_ptr(), fp8 ? (int)LH_DTYPE_E4M3 : dtype_code(out),
                     fp8 ? (float*)o.scale.mutable_data_ptr() : nullptr, (int)group,
                     o.h.defined() ? o.h.mutable_data_ptr() : nullptr,
                     with_rstd ? (float*)o.rstd.mutable_data_ptr() : nullptr, stream(x.device())),
        "rms_norm");
  return o;
}

struct NormFn : torch::autograd::Function<NormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& residual,
                               const Tensor& w, double eps, at::ScalarType out) {
    const Tensor r = residual.value_or(Tensor());
    NormOut o = norm_forward(x, r, w, eps, out, 0, true);
    ctx->save_for_backward({r.defined() ? o.h : x, w, o.rstd});
    ctx->saved_data["x"] = (int64_t)x.scalar_type();
    ctx->saved_data["h"] = (int64_t)(r.defined() ? r : x).scalar_type();
    ctx->saved_data["w"] = (int64_t)w.scalar_type();
    ctx->saved_data["res"] = r.defined();
    ctx->set_materialize_grads(false);
    return r.defined() ? variable_list{o.y, o.h} : variable_list{o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto x_type = (at::ScalarType)ctx->saved_data["x"].toInt();
    const bool res = ctx->saved_data["res"].toBool();
    const Tensor dh_in = res ? grads[1] : Tensor();
    if (!grads[0].defined())                      // only the stream's new value was used
      return once({dh_in.defined() ? dh_in.to(x_type) : Tensor(), dh_in, Tensor(), Tensor(), Tensor()});
    const Tensor dy = dense16(grads[0]), dh = dh_in.defined() ? dense16(dh_in) : Tensor();
    const c10::cuda::CUDAGuard guard(dy.device());
    const int64_t D = dy.size(-1), N = dy.numel() / D;
    const Tensor h = unpacked(saved[0], dy.sizes(), (at::ScalarType)ctx->saved_data["h"].toInt(), dy.device());
    const Tensor w = unpacked(saved[1], {D}, (at::ScalarType)ctx->saved_data["w"].toInt(), dy.device());
    const Tensor rstd = unpacked(saved[2], {N}, at::kFloat, dy.device());
    const Tensor dx = empty(h.sizes(), x_type, h.device());
    const Tensor dr = res ? empty(h.sizes(), h.scalar_type(), h.device()) : Tensor();
    const Tensor dw = empty({D}, w.scalar_type(), h.device());
    const size_t n = api.norm_ws(N, (int)D);
    const Tensor ws = empty({(int64_t)n}, at::kByte, h.device());
    check(api.norm_bwd(dy.const_data_ptr(), dtype_code(dy.scalar_type()), dh.defined() ? dh.const_data_ptr() : nullptr,
                       h.const_data_ptr(), dtype_code(h.scalar_type()), w.const_data_ptr(), dtype_code(w.scalar_type()),
                       (const float*)rstd.const_data_ptr(), N, (int)D, dx.mutable_data_ptr(), dtype_code(x_type),
                       res ? dr.mutable_data_ptr() : nullptr, dw.mutable_data_ptr(), ws.mutable_data_ptr(), n,
                       stream(h.device())),
          "rms_norm_bwd");
    return once({dx, dr, dw, Tensor(), Tensor()});
  }
};

py::object rms_norm(const Tensor& x, const Tensor& w, double eps, std::optional<at::ScalarType> out) {
  const at::ScalarType t = out.value_or(x.scalar_type());
  if (dtype_code(t) < 0 || !norm_case(x, Tensor(), w)) return py::none();
  return py::cast(NormFn::apply(x, std::optional<Tensor>(), w, eps, t)[0]);
}
py::object add_rms_norm(const Tensor& x, const Tensor& r, const Tensor& w, double eps, std::optional<at::ScalarType> out) {
  const at::ScalarType t = out.value_or(x.scalar_type());
  if (dtype_code(t) < 0 || !norm_case(x, r, w)) return py::none();
  const variable_list o = NormFn::apply(x, std::optional<Tensor>(r), w, eps, t);
  return py::make_tuple(o[0], o[1]);
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
py::object norm_fp8(const Tensor& x, const Tensor& r, const Tensor& w, double eps, int64_t group) {
  if ((group != 0 && group != 128) || !norm_case(x, r, w)) return py::none();
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(r) || wants_grad(w))) return py::none();
  const NormOut o = norm_forward(x, r, w, eps, at::kFloat8_e4m3fn, group, false);
  return r.defined() ? py::make_tuple(o.y, o.scale, o.h) : py::make_tuple(o.y, o.scale);
}
py::object rms_norm_fp8(const Tensor& x, const Tensor& w, double eps, int64_t group) {
  return norm_fp8(x, Tensor(), w, eps, group);
}

// ---------------------------------------------------------------- losses
bool loss_case(const Tensor& h, const Tensor& w, int64_t reduction) {
  if (!api.xent_fwd || intercepted() || reduction < 0 || reduction > 2 || !plain(h) || !plain(w) || h.dim() != 2 || w.dim() != 2)
    return false;
  const int64_t N = h.size(0), D = h.size(1), V = w.size(0), most = 1 << 22;
  return h.scalar_type() == at::kBFloat16 && w.scalar_type() == at::kBFloat16 && w.size(1) == D && h.device() == w.device() &&
         D % 8 == 0 && D >= 8 && D <= 65536 && N >= 1 && N <= most && V >= 1 && V <= most;
}
bool rows_case(const Tensor& t, const Tensor& h, int64_t dim) {
  return t.defined() && t.is_cuda() && t.is_contiguous() && !t.is_neg() && t.dim() == dim && t.size(0) == h.size(0) && t.device() == h.device() &&
         !t.key_set().has_any(c10::python_ks | c10::functorch_transforms_ks);
}

struct LossFn : torch::autograd::Function<LossFn> {
  // target (N) and K = 0, or teacher logits and indices (N, K)
  static Tensor forward(AutogradContext* ctx, const Tensor& h, const Tensor& w, const Tensor& target,
                        const std::optional<Tensor>& teacher, double temperature, int64_t ignore, int64_t reduction,
                        bool gradients) {
    const Tensor tl = teacher.value_or(Tensor());
    const c10::cuda::CUDAGuard guard(h.device());
    const int64_t N = h.size(0), D = h.size(1), V = w.size(0), K = tl.defined() ? tl.size(1) : 0;
    const Tensor loss = reduction == LH_REDUCE_NONE ? empty({N}, at::kFloat, h.device()) : empty({}, at::kFloat, h.device());
    const Tensor kept = empty({(int64_t)api.loss_kept((int)N, (int)V, (int)K, (int)reduction, gradients)}, at::kByte, h.device());
    const size_t n = api.loss_ws((int)N, (int)V, (int)D, (int)K, 0);
    const Tensor ws = empty({(int64_t)n}, at::kByte, h.device());
    if (K)
      check(api.distill_fwd(h.const_data_ptr(), w.const_data_ptr(), tl.const_data_ptr(), dtype_code(tl.scalar_type()),
                            (const int64_t*)target.const_data_ptr(), (int)N, (int)V, (int)D, (int)K, (float)temperature,
                            (int)reduction, (float*)loss.mutable_data_ptr(), kept.mutable_data_ptr(),
                            (size_t)kept.numel(), ws.mutable_data_ptr(), n, stream(h.device())),
            "linear_distill");
    else
      check(api.xent_fwd(h.const_data_ptr(), w.const_data_ptr(), (const int64_t*)target.const_data_ptr(), ignore, (int)N,
                         (int)V, (int)D, (int)reduction, (float*)loss.mutable_data_ptr(), kept.mutable_data_ptr(),
                         (size_t)kept.numel(), ws.mutable_data_ptr(), n, stream(h.device())),
            "linear_xent");
    ctx->save_for_backward({h, w, K ? Tensor() : target, kept});
    ctx->saved_data["K"] = K;
    ctx->saved_data["T"] = temperature;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["N"] = N;
    ctx->saved_data["V"] = V;
    ctx->saved_data["D"] = D;
    ctx->saved_data["kept"] = kept.numel();
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor g = dense16(grads[0]);
    const c10::cuda::CUDAGuard guard(g.device());
    auto number = [&](const char* name) { return ctx->saved_data[name].toInt(); };
    const int64_t N = number("N"), V = number("V"), D = number("D"), K = number("K");
    const int reduction = (int)number("reduction");
    const Tensor h = unpacked(saved[0], {N, D}, at::kBFloat16, g.device());
    const Tensor w = unpacked(saved[1], {V, D}, at::kBFloat16, g.device());
    const Tensor target = K ? Tensor() : unpacked(saved[2], {N}, at::kLong, g.device());
    const Tensor kept = unpacked(saved[3], {number("kept")}, at::kByte, g.device());
    // a frozen projection, or hidden states that nothing learns from: half of the gradients' products
    Tensor dh, dw;
    if (ctx->needs_input_grad(0)) dh = empty(h.sizes(), at::kBFloat16, h.device());
    if (ctx->needs_input_grad(1)) dw = empty(w.sizes(), at::kBFloat16, h.device());
    if (!dh.defined() && !dw.defined()) return variable_list(8);
    void *dhp = dh.defined() ? dh.mutable_data_ptr() : nullptr, *dwp = dw.defined() ? dw.mutable_data_ptr() : nullptr;
    const size_t n = api.loss_ws((int)N, (int)V, (int)D, (int)K, 1);
    const Tensor ws = empty({(int64_t)n}, at::kByte, h.device());
    if (K)
      check(api.distill_bwd(h.const_data_ptr(), w.const_data_ptr(), (int)N, (int)V, (int)D, (int)K,
                            (float)ctx->saved_data["T"].toDouble(), reduction, kept.const_data_ptr(),
                            (size_t)kept.numel(), (const float*)g.const_data_ptr(), dhp, dwp, ws.mutable_data_ptr(), n, stream(h.device())),
            "linear_distill_bwd");
    else
      check(api.xent_bwd(h.const_data_ptr(), w.const_data_ptr(), (const int64_t*)target.const_data_ptr(), (int)N, (int)V,
                         (int)D, reduction, kept.const_data_ptr(), (size_t)kept.numel(), (const float*)g.const_data_ptr(), dhp, dwp, ws.mutable_data_ptr(),
                         n, stream(h.device())),
            "linear_xent_bwd");
    return once({dh, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

bool wants_grad(const Tensor& h, const Tensor& w) {
  return at::GradMode::is_enabled() && (wants_grad(h) || wants_grad(w));
}
py::object linear_xent(const Tensor& h, const Tensor& w, const Tensor& target, int64_t ignore, int64_t reduction) {
  if (!loss_case(h, w, reduction) || !rows_case(target, h, 1) || target.scalar_type() != at::kLong) return py::none();
  return py::cast(LossFn::apply(h, w, target, std::optional<Tensor>(), 1.0, ignore, reduction, wants_grad(h, w)));
}
py::object linear_distill(const Tensor& h, const Tensor& w, const Tensor& tl, const Tensor& ti, double temperature,
                          int64_t reduction) {
  if (!loss_case(h, w, reduction) || !rows_case(tl, h, 2) || !rows_case(ti, h, 2) || ti.scalar_type() != at::kLong ||
      dtype_code(tl.scalar_type()) < 0 || tl.size(1) != ti.size(1) || tl.size(1) < 1 || tl.size(1) > 256 ||
      !(temperature >= 1e-18 && temperature <= 1e18))
    return py::none();
  return py::cast(LossFn::apply(h, w, ti, std::optional<Tensor>(tl.detach()), temperature, 0, reduction, wants_grad(h, w)));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("rms_norm", &rms_norm);
  m.def("add_rms_norm", &add_rms_norm);
  m.def("rms_norm_fp8", &rms_norm_fp8);
  m.def("add_rms_norm_fp8", &norm_fp8);
  m.def("linear_xent", &linear_xent);
  m.def("linear_distill", &linear_distill);
}
