// Autograd and argument checks of gsr.layers and gsr.optim around libgsr's C ABI (module gsr._torch).
//
// Small calls are bound by the host: a backward pass runs on the autograd engine's own thread, where
// interpreted bookkeeping around a 4 us kernel costs ten times the kernel.  This module does that
// bookkeeping natively.  It computes nothing: every result comes from a gsr_* call on the
// caller's current stream, and all memory from torch's allocator.  Layer norm of 16000 x 8 forward and
// backward 70 us a pass, 145 with the same nodes in Python; an AdamW step of 8 tensors 7.6.
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <utility>
#include <vector>

#include "gsr.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// libgsr's calls, taken by bind() from the library that the ctypes binding has loaded (so that both sides
// of the package use one library, wherever it lies).
struct Calls {
  decltype(&::gsr_last_error) last_error;
  decltype(&::gsr_layer_norm_fwd) layer_norm_fwd;
  decltype(&::gsr_layer_norm_workspace) layer_norm_workspace;
  decltype(&::gsr_layer_norm_bwd) layer_norm_bwd;
  decltype(&::gsr_gated_fwd) gated_fwd;
  decltype(&::gsr_gated_kept) gated_kept;
  decltype(&::gsr_gated_workspace) gated_workspace;
  decltype(&::gsr_gated_bwd) gated_bwd;
  decltype(&::gsr_adamw_step) adamw_step;
  decltype(&::gsr_adamw_decode_root) adamw_decode_root;
} gsr;

void bind(const std::string& path) {
  void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(lib, "cannot load ", path, ": ", dlerror());
  Calls c;
  const auto take = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(dlsym(lib, name));
    TORCH_CHECK(f, path, " has no ", name);
  };
  take(c.last_error, "gsr_last_error");
  take(c.layer_norm_fwd, "gsr_layer_norm_fwd");
  take(c.layer_norm_workspace, "gsr_layer_norm_workspace");
  take(c.layer_norm_bwd, "gsr_layer_norm_bwd");
  take(c.gated_fwd, "gsr_gated_fwd");
  take(c.gated_kept, "gsr_gated_kept");
  take(c.gated_workspace, "gsr_gated_workspace");
  take(c.gated_bwd, "gsr_gated_bwd");
  take(c.adamw_step, "gsr_adamw_step");
  take(c.adamw_decode_root, "gsr_adamw_decode_root");
  gsr = c;   // only a library that has them all
}

int type_of(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return GSR_F32;
    case at::kBFloat16: return GSR_BF16;
    case at::kHalf: return GSR_F16;
    default: TORCH_CHECK_VALUE(false, what, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

at::ScalarType scalar_of(int type) { return type == GSR_F32 ? at::kFloat : type == GSR_BF16 ? at::kBFloat16 : at::kHalf; }

void check(int rc, const char* name) {
  if (rc == 0) return;
  TORCH_CHECK_VALUE(rc != GSR_EINVAL, name, ": ", gsr.last_error());
  TORCH_CHECK(false, name, " failed (code ", rc, "): ", gsr.last_error());
}

void on_device(const Tensor& t, const char* who) {
  TORCH_CHECK(t.is_cuda(), who, ": libgsr runs on a CUDA (ROCm/HIP) device; got a tensor on '", t.device(),
              "'. Move the module and its inputs to 'cuda' (there is no CPU path).");
}

void* stream_of(const c10::Device& d) {
  return c10::hip::getCurrentHIPStream(d.index()).stream();
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// The optional tensors of a call as tensors that may be undefined.
Tensor or_none(const std::optional<Tensor>& t) { return t ? *t : Tensor(); }
std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
// t as it lies in memory: a view that negates what it reads (is_neg) is written out.
Tensor as_held(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
Tensor packed(const Tensor& t) { return as_held(t.defined() && !t.is_contiguous() ? t.contiguous() : t); }
// A tensor with a tangent is refused: calls that need no autograd node would drop it without a word.
void no_tangent(const Tensor& t, const char* who) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), who, ": no forward-mode derivative");
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// x as rows of unit stride: a view where it is one matrix of evenly spaced rows, else a copy.
struct Rows {
  Tensor t;
  int64_t rows, stride;
};

Rows rows_of(const Tensor& x, int64_t dim) {
  Tensor t = x.dim() == 2 ? x : x.reshape({-1, dim});
  if ((dim > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < dim)) t = t.contiguous();
  t = as_held(t);
  const int64_t rows = t.size(0);
  return {t, rows, rows > 1 ? t.stride(0) : dim};
}

// Under create_graph the gradients carry a node whose own backward raises (differentiable once).
variable_list once(variable_list grads, const char* who) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)   // (a node is only made for inputs that require a gradient)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      std::string(who) + ": trying to differentiate twice a function that can be differentiated once", grads.size());
  return (*node)(std::move(grads));
}

// ------------------------------------------------------------------ layer norm
Tensor norm_forward(const Rows& r, const Tensor& x, const Tensor& w, const Tensor& b, double eps, const Tensor& stats) {
  const c10::OptionalDeviceGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options());
  const Tensor& p = w.defined() ? w : b.defined() ? b : x;
  check(gsr.layer_norm_fwd(r.t.data_ptr(), r.rows, x.size(-1), r.stride, type_of(x, "x"), ptr(w), ptr(b), type_of(p, "weight"),
                           (float)eps, y.data_ptr(), stats.defined() ? stats.data_ptr<float>() : nullptr,
                           stream_of(x.device())),
        "gsr_layer_norm_fwd");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                        const std::optional<Tensor>& bias, double eps) {
    const Tensor w = or_none(weight), b = or_none(bias);
    const Rows r = rows_of(x, x.size(-1));
    Tensor stats = at::empty({r.rows, 2}, x.options().dtype(at::kFloat));
    Tensor y = norm_forward(r, x, w, b, eps, stats);
    ctx->save_for_backward({r.t, w, stats});
    ctx->saved_data["shape"] = x.sizes();
    ctx->saved_data["bias"] = b.defined();
    ctx->saved_data["wtype"] = (int64_t)type_of(w.defined() ? w : b.defined() ? b : x, "weight");
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    no_tangent(grads[0], "layer_norm");
    const int64_t rows = x.size(0), dim = x.size(1), stride = rows > 1 ? x.stride(0) : dim;
    const int wtype = (int)ctx->saved_data["wtype"].toInt(), xtype = type_of(x, "x");
    Tensor dx, dw, db, ws;
    {
      const at::AutoGradMode off(false);
      const c10::OptionalDeviceGuard guard(x.device());
      const Rows g = rows_of(grads[0].scalar_type() == x.scalar_type() ? grads[0] : grads[0].to(x.scalar_type()), dim);
      const auto params = x.options().dtype(scalar_of(wtype));
      if (ctx->needs_input_grad(0)) dx = at::empty(ctx->saved_data["shape"].toIntVector(), x.options());
      const size_t bias_at = w.defined() ? 2 : 1;   // (tensors that were not given have no place among the inputs)
      if (w.defined() && ctx->needs_input_grad(1)) dw = at::empty({dim}, params);
      if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(bias_at)) db = at::empty({dim}, params);
      size_t bytes = 0;
      if (dw.defined() || db.defined()) {
        bytes = gsr.layer_norm_workspace(rows, dim, xtype);
        ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
      }
      check(gsr.layer_norm_bwd(x.data_ptr(), g.t.data_ptr(), rows, dim, stride, g.stride, xtype, ptr(w), wtype,
                               stats.data_ptr<float>(), ptr(dx), ptr(dw), ptr(db), ptr(ws), bytes, stream_of(x.device())),
            "gsr_layer_norm_bwd");
    }
    return once({dx, dw, db, Tensor()}, "layer_norm");
  }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
  type_of(x, "layer_norm: x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "layer_norm: x must be [..., dim] with dim >= 1, got ", x.sizes());
  const Tensor w = packed(or_none(weight)), b = packed(or_none(bias));
  for (const auto& [t, name] : {std::pair<const Tensor&, const char*>{w, "weight"}, {b, "bias"}}) {
    if (!t.defined()) continue;
    type_of(t, name);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == x.size(-1), "layer_norm: ", name, " must be [", x.size(-1), "], got ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == x.device(), "layer_norm: ", name, " is on ", t.device(), ", x on ", x.device());
  }
  TORCH_CHECK_VALUE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
                    "layer_norm: weight and bias must have one type");
  TORCH_CHECK_VALUE(eps >= 0, "layer_norm: eps must not be negative, got ", eps);
  for (const Tensor* t : {&x, &w, &b}) no_tangent(*t, "layer_norm");
  on_device(x, "layer_norm");
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b))) return LayerNorm::apply(x, given(w), given(b), eps);
  return norm_forward(rows_of(x, x.size(-1)), x, w, b, eps, Tensor());
}

// ----------------------------------------------------------------- gated block
Tensor gated_forward(const Rows& r, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& bg, const Tensor& bu,
                     int64_t act, const Tensor& kept) {
  const c10::OptionalDeviceGuard guard(x.device());
  const int type = type_of(x, "x");
  const int64_t dim = x.size(-1), hidden = wg.size(0);
  auto shape = x.sizes().vec();
  shape.back() = hidden;
  Tensor h = at::empty(shape, x.options()), ws;
  const size_t bytes = gsr.gated_workspace(r.rows, dim, hidden, type, 0);
  if (bytes) ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
  check(gsr.gated_fwd(r.t.data_ptr(), r.rows, dim, r.stride, type, wg.data_ptr(), wu.data_ptr(), hidden, ptr(bg), ptr(bu), (int)act,
                      h.data_ptr(), ptr(kept), ptr(ws), bytes, stream_of(x.device())),
        "gsr_gated_fwd");
  return h;
}

struct Gated : torch::autograd::Function<Gated> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu,
                        const std::optional<Tensor>& b_gate, const std::optional<Tensor>& b_up, int64_t act) {
    const Tensor bg = or_none(b_gate), bu = or_none(b_up);
    const Rows r = rows_of(x, x.size(-1));
    Tensor kept;
    if (const size_t bytes = gsr.gated_kept(r.rows, x.size(-1), wg.size(0), type_of(x, "x")))
      kept = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    ctx->save_for_backward({r.t, wg, wu, bg, bu, kept});
    ctx->saved_data["shape"] = x.sizes();
    ctx->saved_data["act"] = act;
    return gated_forward(r, x, wg, wu, bg, bu, act, kept);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &bg = saved[3], &bu = saved[4], &kept = saved[5];
    no_tangent(grads[0], "gated_linear");
    const int64_t rows = x.size(0), dim = x.size(1), stride = rows > 1 ? x.stride(0) : dim, hidden = wg.size(0);
    const int type = type_of(x, "x");
    Tensor d[5];
    {
      const at::AutoGradMode off(false);
      const c10::OptionalDeviceGuard guard(x.device());
      const Rows g = rows_of(grads[0].scalar_type() == x.scalar_type() ? grads[0] : grads[0].to(x.scalar_type()), hidden);
      if (ctx->needs_input_grad(0)) d[0] = at::empty(ctx->saved_data["shape"].toIntVector(), x.options());
      for (int i = 1; i < (bg.defined() ? 5 : 3); ++i)
        if (ctx->needs_input_grad(i)) d[i] = at::empty(i < 3 ? wg.sizes() : wg.sizes().slice(0, 1), x.options());
      const size_t bytes = gsr.gated_workspace(rows, dim, hidden, type, 1);
      const Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
      check(gsr.gated_bwd(x.data_ptr(), rows, dim, stride, type, wg.data_ptr(), wu.data_ptr(), hidden, ptr(bg), ptr(bu),
                          (int)ctx->saved_data["act"].toInt(), g.t.data_ptr(), g.stride, ptr(kept), ptr(d[0]), ptr(d[1]), ptr(d[2]), ptr(d[3]),
                          ptr(d[4]), ws.data_ptr(), bytes, stream_of(x.device())),
            "gsr_gated_bwd");
    }
    return once({d[0], d[1], d[2], d[3], d[4], Tensor()}, "gated_linear");
  }
};

Tensor gated_linear(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const std::optional<Tensor>& b_gate,
                    const std::optional<Tensor>& b_up, int64_t act) {
  type_of(x, "gated_linear: x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "gated_linear: x must be [..., dim] with dim >= 1, got ", x.sizes());
  const int64_t dim = x.size(-1);
  TORCH_CHECK_VALUE(w_gate.dim() == 2 && w_gate.size(1) == dim && w_gate.size(0) >= 1 && w_up.sizes() == w_gate.sizes(),
                    "gated_linear: w_gate and w_up must be [hidden, ", dim, "], got ", w_gate.sizes(), " and ", w_up.sizes());
  TORCH_CHECK_VALUE(b_gate.has_value() == b_up.has_value(), "gated_linear: b_gate and b_up go together");
  const int64_t hidden = w_gate.size(0);
  const Tensor wg = packed(w_gate), wu = packed(w_up), bg = packed(or_none(b_gate)), bu = packed(or_none(b_up));
  for (const Tensor* t : {&wg, &wu, &bg, &bu}) {
    if (!t->defined()) continue;
    TORCH_CHECK_VALUE(t->dim() == 2 || (t->dim() == 1 && t->size(0) == hidden), "gated_linear: the biases must be [", hidden,
                      "], got ", t->sizes());
    TORCH_CHECK_VALUE(t->scalar_type() == x.scalar_type(), "gated_linear: weights and biases must have x's type ", x.scalar_type(),
                      ", got ", t->scalar_type());
    TORCH_CHECK_VALUE(t->device() == x.device(), "gated_linear: a weight or bias is on ", t->device(), ", x on ", x.device());
  }
  TORCH_CHECK_VALUE(dim <= 1 << 20 && hidden <= 1 << 20 && x.numel() / dim <= 1 << 26,
                    "gated_linear: at most 2^26 rows and 2^20 columns, got ", x.sizes(), ", ", w_gate.sizes());
  for (const Tensor* t : {&x, &wg, &wu, &bg, &bu}) no_tangent(*t, "gated_linear");
  on_device(x, "gated_linear");
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(wg) || wants_grad(wu) || wants_grad(bg) || wants_grad(bu)))
    return Gated::apply(x, wg, wu, given(bg), given(bu), act);
  return gated_forward(rows_of(x, dim), x, wg, wu, bg, bu, act, Tensor());
}

// ----------------------------------------------------------------- AdamW step
int64_t units_of(int64_t numel) { return (numel + GSR_ADAMW_BLOCK - 1) / GSR_ADAMW_BLOCK; }

// Whether a and b order their elements in memory alike (dimensions of one element do not count).
bool same_layout(const Tensor& a, const Tensor& b) {
  if (a.sizes() != b.sizes()) return false;
  if (a.numel() == 0) return true;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) != 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}

// The tensors of a list, read in place: converting hundreds of them one by one costs more than the step.
class Tensors {
  py::object seq_;   // keeps them alive
  std::vector<const Tensor*> t_;

 public:
  Tensors(py::handle list, const char* what) : seq_(py::reinterpret_steal<py::object>(PySequence_Fast(list.ptr(), what))) {
    if (!seq_) throw py::error_already_set();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq_.ptr());
    PyObject** items = PySequence_Fast_ITEMS(seq_.ptr());
    t_.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      TORCH_CHECK_TYPE(THPVariable_Check(items[i]), what, ", got a ", Py_TYPE(items[i])->tp_name);
      t_.push_back(&THPVariable_Unpack(items[i]));
    }
  }
  size_t size() const { return t_.size(); }
  const Tensor& operator[](size_t i) const { return *t_[i]; }
};

void adamw_step(py::handle param_list, py::handle grad_list, py::handle m_list, py::handle v_list, double lr,
                const std::optional<Tensor>& lr_dev, double beta1, double beta2, double eps, double weight_decay, int64_t step,
                py::handle step_list, py::handle m_unit_list, py::handle v_unit_list, bool unbiased) {
  const Tensors params(param_list, "adamw_step: params must be a list of tensors"),
      grads(grad_list, "adamw_step: grads must be a list of tensors"), ms(m_list, "adamw_step: exp_avgs must be a list of tensors"),
      vs(v_list, "adamw_step: exp_avg_sqs must be a list of tensors");
  const auto maybe = [](py::handle list, const char* what) { return list.is_none() ? std::nullopt : std::optional<Tensors>(Tensors(list, what)); };
  const auto steps = maybe(step_list, "adamw_step: step must be a number, a tensor or a list of tensors"),
             m_units = maybe(m_unit_list, "adamw_step: exp_avg_units must be a list of tensors"),
             v_units = maybe(v_unit_list, "adamw_step: exp_avg_root_units must be a list of tensors");
  const size_t count = params.size();
  TORCH_CHECK_VALUE(m_units.has_value() == v_units.has_value(), "adamw_step: exp_avg_units and exp_avg_root_units go together");
  const bool byte = m_units.has_value();
  TORCH_CHECK_VALUE(grads.size() == count && ms.size() == count && vs.size() == count &&
                        (!byte || (m_units->size() == count && v_units->size() == count)),
                    "adamw_step: ", count, " params, but lists of other lengths");
  TORCH_CHECK_VALUE(!steps || steps->size() == count, "adamw_step: ", count, " params, but ", steps ? steps->size() : 0, " steps");
  TORCH_CHECK_VALUE(lr_dev || lr >= 0, "adamw_step: lr must not be negative, got ", lr);
  TORCH_CHECK_VALUE(!lr_dev || (lr_dev->numel() == 1 && lr_dev->scalar_type() == at::kFloat),
                    "adamw_step: a tensor lr must be one float32 value");
  const auto held = [](const Tensor& t) {
    TORCH_CHECK_VALUE(!t.is_neg(), "adamw_step: views that negate what they read are taken as gradients only");
  };
  if (lr_dev) held(*lr_dev);
  TORCH_CHECK_VALUE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "adamw_step: betas must be in [0, 1), got ", beta1, ", ", beta2);
  TORCH_CHECK_VALUE(eps >= 0 && weight_decay >= 0, "adamw_step: eps and weight_decay must not be negative, got ", eps, ", ", weight_decay);
  TORCH_CHECK_VALUE(steps || step >= 1, "adamw_step: step must be at least 1, got ", step);
  if (count == 0) return;
  const auto device = params[0].device();
  TORCH_CHECK_VALUE(!lr_dev || lr_dev->device() == device, "adamw_step: lr must be on ", device);
  struct Group {
    int p, g;
    std::vector<gsr_adamw_tensor> list;
  };
  std::vector<Group> groups;
  std::vector<std::pair<uintptr_t, uintptr_t>> written[5];   // what is written, a list each
  std::vector<Tensor> kept;   // gradients copied into their parameter's layout
  const auto writes = [&](int list, const Tensor& t) {
    const auto at = (uintptr_t)t.data_ptr();
    written[list].emplace_back(at, at + t.numel() * t.element_size());
    return (void*)at;
  };
  for (auto& w : written) w.reserve(count);
  const auto mtype = byte ? at::kFloat8_e4m3fn : at::kFloat, vtype = byte ? at::kByte : at::kFloat;
  for (size_t i = 0; i < count; ++i) {
    const Tensor &p = params[i], &m = ms[i], &v = vs[i];
    const int pt = type_of(p, "adamw_step: a parameter"), gt = type_of(grads[i], "adamw_step: a gradient");
    for (const Tensor* t : {&p, &grads[i], &m, &v})
      TORCH_CHECK_VALUE(t->device() == device, "adamw_step: tensor ", i, ", its gradient or a moment is on ", t->device(),
                        ", the first tensor on ", device);
    TORCH_CHECK_VALUE(m.scalar_type() == mtype && v.scalar_type() == vtype, "adamw_step: exp_avg must be torch.",
                      byte ? "float8_e4m3fn" : "float32", " and exp_avg_sq torch.", byte ? "uint8" : "float32", ", got ",
                      m.scalar_type(), " and ", v.scalar_type());
    TORCH_CHECK_VALUE(grads[i].layout() == at::kStrided && grads[i].sizes() == p.sizes(), "adamw_step: gradient ", i,
                      " must be dense and ", p.sizes(), ", got ", grads[i].sizes());
    TORCH_CHECK_VALUE(p.is_non_overlapping_and_dense(), "adamw_step: parameter ", i, " does not fill its memory (strides ",
                      p.strides(), ")");
    TORCH_CHECK_VALUE(same_layout(m, p) && same_layout(v, p), "adamw_step: moments must have their parameter's shape and strides ",
                      p.sizes(), ", ", p.strides());
    for (const Tensor* t : {&p, &m, &v}) held(*t);
    const int64_t n = p.numel();
    if (byte)
      for (const Tensor* u : {&(*m_units)[i], &(*v_units)[i]})
        TORCH_CHECK_VALUE(u->scalar_type() == at::kFloat && u->dim() == 1 && u->size(0) == units_of(n) && u->is_contiguous() &&
                              u->device() == device,
                          "adamw_step: units ", i, " must be contiguous float32 [", units_of(n), "] on ", device, ", got ",
                          u->scalar_type(), " ", u->sizes());
    if (byte) held((*m_units)[i]), held((*v_units)[i]);
    if (steps)
      TORCH_CHECK_VALUE((*steps)[i].numel() == 1 && (*steps)[i].scalar_type() == at::kLong && (*steps)[i].device() == device,
                        "adamw_step: step ", i, " must be one int64 value on ", device);
    if (n == 0) continue;
    Tensor g = grads[i];
    if (!same_layout(g, p) || g.is_neg()) {
      g = at::empty_strided(p.sizes(), p.strides(), g.options()).copy_(g);
      kept.push_back(g);
    }
    gsr_adamw_tensor t{};
    t.p = writes(0, p), t.g = g.data_ptr(), t.m = writes(1, m), t.v = writes(2, v), t.n = n;
    if (byte) t.m_unit = (float*)writes(3, (*m_units)[i]), t.v_unit = (float*)writes(4, (*v_units)[i]);
    if (steps) t.step = (*steps)[i].data_ptr<int64_t>();
    auto at = std::find_if(groups.begin(), groups.end(), [&](const Group& x) { return x.p == pt && x.g == gt; });
    if (at == groups.end()) {
      at = groups.insert(at, Group{pt, gt, {}});
      at->list.reserve(count);
    }
    at->list.push_back(t);
  }
  // Nothing is written twice: all of it in order of its addresses (each list mostly is in order).
  for (auto& w : written)
    if (!std::is_sorted(w.begin(), w.end())) std::sort(w.begin(), w.end());
  size_t at[5] = {};
  for (uintptr_t end = 0;;) {
    int first = -1;
    for (int k = 0; k < 5; ++k)
      if (at[k] < written[k].size() && (first < 0 || written[k][at[k]] < written[first][at[first]])) first = k;
    if (first < 0) break;
    const auto& w = written[first][at[first]++];
    TORCH_CHECK_VALUE(w.first >= end, "adamw_step: a tensor is listed twice, or tensors to be written overlap");
    end = w.second;
  }
  on_device(params[0], "adamw_step");
  gsr_adamw_args args{};
  args.lr = lr, args.beta1 = beta1, args.beta2 = beta2, args.eps = eps, args.weight_decay = weight_decay;
  args.step = steps ? 0 : step;
  args.lr_dev = lr_dev ? lr_dev->data_ptr<float>() : nullptr;
  args.bits = byte ? 8 : 32;
  args.rounding = unbiased ? GSR_ROUND_UNBIASED : GSR_ROUND_NEAREST;
  const c10::OptionalDeviceGuard guard(device);
  void* stream = stream_of(device);
  for (const Group& g : groups)
    check(gsr.adamw_step(g.list.data(), (int32_t)g.list.size(), g.p, g.g, &args, stream), "gsr_adamw_step");
  for (size_t i = 0; i < count; ++i)
    if (!params[i].is_inference()) params[i].unsafeGetTensorImpl()->bump_version();
}

Tensor decode_root(const Tensor& codes, const Tensor& units) {
  TORCH_CHECK_VALUE(codes.scalar_type() == at::kByte && codes.is_contiguous(), "decode_root: codes must be contiguous uint8, got ",
                    codes.scalar_type());
  TORCH_CHECK_VALUE(units.scalar_type() == at::kFloat && units.dim() == 1 && units.size(0) == units_of(codes.numel()) &&
                        units.is_contiguous() && units.device() == codes.device(),
                    "decode_root: units must be contiguous float32 [", units_of(codes.numel()), "] on ", codes.device(), ", got ",
                    units.scalar_type(), " ", units.sizes(), " on ", units.device());
  TORCH_CHECK_VALUE(!units.is_neg(), "decode_root: units must not be a view that negates what it reads");
  on_device(codes, "decode_root");
  const c10::OptionalDeviceGuard guard(codes.device());
  Tensor out = at::empty(codes.sizes(), codes.options().dtype(at::kFloat));
  check(gsr.adamw_decode_root(codes.data_ptr<uint8_t>(), units.data_ptr<float>(), codes.numel(), out.data_ptr<float>(),
                              stream_of(codes.device())),
        "gsr_adamw_decode_root");
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("layer_norm", &layer_norm);
  m.def("gated_linear", &gated_linear);
  m.def("adamw_step", &adamw_step);
  m.def("decode_root", &decode_root);
  m.attr("ABI_VERSION") = GSR_ABI_VERSION;
}
