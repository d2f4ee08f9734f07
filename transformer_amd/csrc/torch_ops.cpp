// The training-layer operators as torch calls with autograd: allocation of outputs and workspaces from torch's allocator,
// the launches (include/mslayers.h) on the current stream, and the backward nodes.
//
// In C++ because a step's small calls are bound by the host: the backward of a call runs in a thread of the autograd engine, on
// another core than the caller's, where a node in Python took 25 to 50 us.  The checks of arguments are the Python modules'
// (attention.py, rotary.py, norm.py, swiglu.py): they make a plan per layout, which holds all that the C calls need, and hand
// over operands that the kernels take as they lie.
#include <torch/extension.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <memory>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/mslayers.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

struct CallError : std::runtime_error {
  int code;
  std::string what_;
  CallError(int code, const char* what) : std::runtime_error(std::string(what) + ": error " + std::to_string(code)), code(code), what_(what) {}
};

void check(int32_t code, const char* what) {
  if (code != MSD_OK) throw CallError(code, what);
}

void* at_(const Tensor& x) { return x.defined() ? x.data_ptr() : nullptr; }
Tensor contiguous_like(const Tensor& x) { return at::empty_like(x, x.options(), at::MemoryFormat::Contiguous); }
Tensor bytes(const Tensor& x, int64_t n) { return at::empty({n}, x.options().dtype(at::kByte)); }
bool wanted(const Tensor& x) { return x.defined() && x.requires_grad(); }

// A call is launches of the library, which neither a trace records (it would keep the outputs' allocation and nothing else) nor
// forward-mode differentiation sees (an output without a tangent stands for a tangent of zero): refused, in the backward too.
bool has_tangent(const Tensor& x) { return x.defined() && x._fw_grad(0).defined(); }
bool has_tangent(const MaybeTensor& x) { return x && has_tangent(*x); }
template <class... X>
void only_run(const char* what, const X&... x) {
  using c10::impl::TorchDispatchModeKey;
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY))
    throw std::runtime_error(std::string(what) + " cannot be traced: a trace does not record its kernels");
  if ((has_tangent(x) || ...)) throw std::runtime_error(std::string(what) + " has no forward-mode derivative");
}

// The calls go to x's device, with its current stream
struct Place {
  c10::DeviceGuard guard;
  hipStream_t stream;
  explicit Place(const Tensor& x) : guard(x.device()), stream(c10::hip::getCurrentHIPStream(x.get_device()).stream()) {}
};

// Hooks on saved tensors hand them back as they like: strides are taken as they come, all else has to be what was saved (the
// kernels would read other values, or past the end).
void restored(const Tensor& x, at::ScalarType type, at::IntArrayRef sizes, at::Device device) {
  if (!x.defined() || x.scalar_type() != type || x.sizes() != sizes || x.device() != device)
    throw std::runtime_error("a saved tensor has come back with another type, shape or device");
}
at::ScalarType scalar_type(int32_t type) { return type == MSD_F32 ? at::kFloat : at::kBFloat16; }

// What a backward node returns.  Second derivatives are refused where one is asked for, not where gradients are only recorded.
variable_list first_order(variable_list g, bool recorded) {
  if (!recorded) return g;
  for (auto& x : g)
    if (x.defined()) x = x.detach().requires_grad_(true);
  const auto n = int64_t(g.size());
  auto refuse = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that is differentiable once", n);
  return (*refuse)(std::move(g));
}

// The stride between x's rows (its last axis) where one describes them all and a row is contiguous
std::optional<int64_t> row_stride(const Tensor& x) {
  const int64_t n = x.dim();
  if (x.is_contiguous()) return x.size(n - 1);
  if (x.stride(n - 1) != 1 && x.size(n - 1) > 1) return std::nullopt;
  std::optional<int64_t> row;
  int64_t inner = 1;   // rows of the axes behind
  for (int64_t i = n - 2; i >= 0; inner *= x.size(i--)) {
    if (x.size(i) == 1) continue;
    if (!row) {
      if (inner != 1) return std::nullopt;
      row = x.stride(i);
    } else if (x.stride(i) != *row * inner) {
      return std::nullopt;
    }
  }
  return row.value_or(x.size(n - 1));
}
// x, or a contiguous copy, and the stride between its rows
std::pair<Tensor, int64_t> rows_of(const Tensor& x) {
  if (const auto s = row_stride(x)) return {x, *s};
  return {x.contiguous(), x.size(x.dim() - 1)};
}

// Strides of x (sequences, rows, heads, d) or (rows, heads, d); 0 along an axis of one (or none)
void head_strides(const Tensor& x, int64_t (&s)[3]) {
  const int64_t n = x.dim();
  for (int i = 0; i < 3; ++i) {
    const int64_t axis = n - 4 + i;
    s[i] = axis < 0 || x.size(axis) <= 1 ? 0 : x.stride(axis);
  }
}
bool heads_contiguous(const Tensor& x) { return x.size(-1) == 1 || x.stride(-1) == 1; }

// ---- attention ----
struct AttnPlan : torch::CustomClassHolder {
  msd_attn a;
  int64_t forward_bytes, backward_bytes;
  bool q_zero, k_zero;    // the sequences leave rows out
  Tensor table, host;     // of the sequences
  uint64_t table_stream;  // that the table was made on
  // keeps the table's memory until what is launched on this stream is done with it
  void use_table(hipStream_t s) const {
    if (table.defined() && reinterpret_cast<uint64_t>(s) != table_stream)
      table.record_stream(c10::impl::VirtualGuardImpl(table.device().type()).getStream(table.device()));
  }
};
using Attn = c10::intrusive_ptr<AttnPlan>;

// Whether x can be read where it lies: heads contiguous, on 16-byte boundaries, within reach (128 rows and `group` heads)
bool attn_reads(const Tensor& x, int64_t group) {
  if (x.is_contiguous()) return reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  const int64_t n = x.dim();
  if (!heads_contiguous(x) || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16) return false;
  for (int64_t i = 0; i + 1 < n; ++i)
    if (x.size(i) > 1 && x.stride(i) % 8) return false;
  const int64_t row = x.size(n - 3) > 1 ? x.stride(n - 3) : 0, head = x.size(n - 2) > 1 ? x.stride(n - 2) : 0;
  return 128 * row + group * head < int64_t(1) << 30;
}

// x, or a copy that can be read, and its strides
Tensor attn_operand(const Tensor& x, int64_t group, int64_t (&s)[3]) {
  const Tensor y = attn_reads(x, group) ? x : x.clone(at::MemoryFormat::Contiguous);
  head_strides(y, s);
  return y;
}

Tensor attn_output(const Tensor& like, bool zero) {
  Tensor x = contiguous_like(like);
  return zero ? x.zero_() : x;
}

Tensor attn_run(const Tensor& q, const Tensor& k, const Tensor& v, const AttnPlan& p, Tensor* lse, Tensor* low) {
  Place on(q);
  Tensor out = attn_output(q, p.q_zero), ws;
  if (lse) {
    *lse = at::empty(q.sizes().slice(0, q.dim() - 1), q.options().dtype(at::kFloat));
    *low = at::empty(q.sizes(), q.options().dtype(at::kByte));
  }
  if (p.forward_bytes) ws = bytes(q, p.forward_bytes);
  p.use_table(on.stream);
  check(msd_attn_forward(&p.a, at_(q), at_(k), at_(v), at_(out), lse ? at_(*low) : nullptr,
                         lse ? static_cast<float*>(at_(*lse)) : nullptr, at_(ws), on.stream),
        "msd_attn_forward");
  return out;
}

struct Attention : torch::autograd::Function<Attention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Attn& p) {
    Tensor lse, low, out = attn_run(q, k, v, *p, &lse, &low);
    ctx->save_for_backward({q, k, v, out, low, lse});
    ctx->saved_data["plan"] = c10::IValue::make_capsule(p);
    return {out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    only_run("the gradient of attention", g[0]);
    const bool recorded = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    const auto x = ctx->get_saved_variables();   // (with the strides that hooks on saved tensors have given them, if any)
    const auto capsule = ctx->saved_data["plan"].toCapsule();
    const AttnPlan& p = static_cast<const AttnPlan&>(*capsule);
    msd_attn a = p.a;
    const auto q_sizes = g[0].sizes();
    const int64_t dense[4] = {a.n_seqs, a.k_len, a.n_kv_heads, a.d_head}, flat[3] = {a.k_rows, a.n_kv_heads, a.d_head};
    const auto k_sizes = g[0].dim() == 4 ? at::IntArrayRef(dense) : at::IntArrayRef(flat);
    for (int i : {0, 3}) restored(x[i], at::kBFloat16, q_sizes, g[0].device());
    for (int i : {1, 2}) restored(x[i], at::kBFloat16, k_sizes, g[0].device());
    restored(x[4], at::kByte, q_sizes, g[0].device());
    restored(x[5], at::kFloat, q_sizes.slice(0, q_sizes.size() - 1), g[0].device());
    Place on(g[0]);
    const int64_t group = a.n_heads / a.n_kv_heads;
    const Tensor q = attn_operand(x[0], group, a.q_stride), k = attn_operand(x[1], 1, a.k_stride), v = attn_operand(x[2], 1, a.v_stride);
    const Tensor dout = attn_operand(g[0], group, a.dout_stride), out = x[3].contiguous(), low = x[4].contiguous(), lse = x[5].contiguous();
    Tensor dq = attn_output(q, p.q_zero), dk = attn_output(k, p.k_zero), dv = attn_output(v, p.k_zero), ws;
    if (p.backward_bytes) ws = bytes(q, p.backward_bytes);
    p.use_table(on.stream);
    check(msd_attn_backward(&a, at_(q), at_(k), at_(v), at_(out), at_(low), static_cast<const float*>(at_(lse)), at_(dout),
                            at_(dq), at_(dk), at_(dv), at_(ws), on.stream),
          "msd_attn_backward");
    return first_order({dq, dk, dv, Tensor()}, recorded);
  }
};

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const Attn& p) {
  only_run("attention", q, k, v);
  if (at::GradMode::is_enabled() && (wanted(q) || wanted(k) || wanted(v))) return Attention::apply(q, k, v, p)[0];
  return attn_run(q, k, v, *p, nullptr, nullptr);
}

// ---- rotary positions ----
struct RopePlan : torch::CustomClassHolder {
  msd_rope forward, backward;   // (the strides of gradients and of the saved positions are set in the call)
};
using Rope = c10::intrusive_ptr<RopePlan>;

std::pair<Tensor, Tensor> rope_run(const msd_rope& r, const Tensor& q, const Tensor& k, const Tensor& turns, const Tensor& positions) {
  Place on(q);
  Tensor q_out = contiguous_like(q), k_out;
  if (k.defined()) k_out = contiguous_like(k);
  check(msd_rope_apply(&r, at_(q), at_(k), at_(positions), static_cast<const double*>(at_(turns)), at_(q_out), at_(k_out), on.stream),
        "msd_rope_apply");
  return {q_out, k_out};
}

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const MaybeTensor& k, const Tensor& turns,
                               const MaybeTensor& positions, const Rope& p) {
    const Tensor pos = positions.value_or(Tensor());
    auto [a, b] = rope_run(p->forward, q, k.value_or(Tensor()), turns, pos);
    ctx->save_for_backward({turns, pos});
    ctx->saved_data["plan"] = c10::IValue::make_capsule(p);
    if (!b.defined()) return {a};
    return {a, b};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    only_run("the gradient of rotary", g[0], g.size() > 1 ? g[1] : Tensor());
    const bool recorded = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    const auto x = ctx->get_saved_variables();
    const auto capsule = ctx->saved_data["plan"].toCapsule();
    msd_rope r = static_cast<const RopePlan&>(*capsule).backward;
    restored(x[0], at::kDouble, r.d_rot / 2, g[0].device());
    const Tensor positions = x[1];
    if (r.position_bytes) {
      const int64_t sizes[2] = {r.batch, r.tokens};
      restored(positions, r.position_bytes == 8 ? at::kLong : at::kInt,
               at::IntArrayRef(sizes).slice(positions.defined() && positions.dim() == 2 ? 0 : 1), g[0].device());
      r.position_stride[0] = positions.dim() == 2 ? positions.stride(0) : 0;
      r.position_stride[1] = positions.stride(-1);
    }
    Tensor dq = g[0], dk = g.size() > 1 ? g[1] : Tensor();
    if (!heads_contiguous(dq)) dq = dq.contiguous();
    if (dk.defined() && !heads_contiguous(dk)) dk = dk.contiguous();
    head_strides(dq, r.q_stride);
    if (dk.defined()) head_strides(dk, r.k_stride);
    auto [a, b] = rope_run(r, dq, dk, x[0].contiguous(), positions);
    return first_order({a, b, Tensor(), Tensor(), Tensor()}, recorded);
  }
};

variable_list rotary(const Tensor& q, const MaybeTensor& k, const Tensor& turns, const MaybeTensor& positions, const Rope& p) {
  only_run("rotary", q, k, turns);
  // (a RotaryFrequencies can be given another vector after its own checks, and the plan knows its length only)
  if (turns.scalar_type() != at::kDouble || turns.dim() != 1 || turns.numel() != p->forward.d_rot / 2 || !turns.is_contiguous() ||
      turns.device() != q.device())
    throw std::invalid_argument("turns must be a contiguous float64 vector of d_rot / 2 values on q's GPU");
  if (at::GradMode::is_enabled() && turns.requires_grad())
    throw std::invalid_argument("the frequencies take no gradient: hand over turns.detach()");
  if (at::GradMode::is_enabled() && (wanted(q) || (k && wanted(*k)))) return Rotary::apply(q, k, turns, positions, p);
  auto [a, b] = rope_run(p->forward, q, k.value_or(Tensor()), turns, positions.value_or(Tensor()));
  if (!b.defined()) return {a};
  return {a, b};
}

// ---- RMSNorm ----
struct RmsPlan : torch::CustomClassHolder {
  int64_t rows, x_stride, residual_stride, held, parts;   // held: bytes of a checkpoint; parts: floats of the backward's workspace
  int32_t d, type, scale_type;
  float eps;
};
using Rms = c10::intrusive_ptr<RmsPlan>;

struct RmsOut {
  Tensor y, sum, rstd, held;
};
RmsOut rms_run(const Tensor& x, const Tensor& scale, const Tensor& residual, const RmsPlan& p, bool keep) {
  Place on(x);
  RmsOut o;
  o.y = contiguous_like(x);
  if (residual.defined()) o.sum = contiguous_like(x);
  if (keep) o.rstd = at::empty({p.rows}, x.options().dtype(at::kFloat));
  if (keep && p.held) o.held = bytes(x, p.held);
  check(msd_rms_forward(at_(x), p.x_stride, at_(residual), p.residual_stride, at_(scale), p.scale_type, p.rows, p.d, p.type, p.eps,
                        at_(o.y), at_(o.sum), static_cast<float*>(at_(o.rstd)), at_(o.held), on.stream),
        "msd_rms_forward");
  return o;
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& scale, const MaybeTensor& residual, const Rms& p) {
    const Tensor w = scale.contiguous();
    RmsOut o = rms_run(x, w, residual.value_or(Tensor()), *p, true);
    ctx->save_for_backward({o.held.defined() ? o.held : o.sum.defined() ? o.sum : x, w, o.rstd});
    ctx->saved_data["plan"] = c10::IValue::make_capsule(p);
    ctx->saved_data["scale"] = scale.requires_grad();
    ctx->set_materialize_grads(false);
    if (!o.sum.defined()) return {o.y};
    return {o.y, o.sum};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    only_run("the gradient of rms_norm", g[0], g.size() > 1 ? g[1] : Tensor());
    const bool recorded = at::GradMode::is_enabled(), sums = g.size() > 1;
    at::NoGradGuard no_grad;
    const Tensor dsum = sums ? g[1] : Tensor();
    if (!g[0].defined())   // only the sum was used: the norm adds nothing
      return first_order({dsum, Tensor(), dsum, Tensor()}, recorded);
    const auto s = ctx->get_saved_variables();
    const auto capsule = ctx->saved_data["plan"].toCapsule();
    const RmsPlan& p = static_cast<const RmsPlan&>(*capsule);
    if (p.held) restored(s[0], at::kByte, p.held, g[0].device());
    else restored(s[0], scalar_type(p.type), g[0].sizes(), g[0].device());
    restored(s[1], scalar_type(p.scale_type), int64_t(p.d), g[0].device());
    restored(s[2], at::kFloat, p.rows, g[0].device());
    Place on(g[0]);
    const auto [kept, kept_stride] = p.held ? std::pair<Tensor, int64_t>{s[0].contiguous(), 0} : rows_of(s[0]);
    const Tensor scale = s[1].contiguous(), rstd = s[2].contiguous();
    const auto [dy, dy_stride] = rows_of(g[0]);
    const auto [ds, ds_stride] = dsum.defined() ? rows_of(dsum) : std::pair<Tensor, int64_t>{Tensor(), 0};
    Tensor dx = contiguous_like(dy), dscale, ws;
    if (ctx->saved_data["scale"].toBool()) {
      dscale = at::empty_like(scale);
      ws = at::empty({p.parts}, rstd.options());
    }
    check(msd_rms_backward(p.held ? nullptr : at_(kept), kept_stride, static_cast<const float*>(at_(rstd)),
                           p.held ? at_(kept) : nullptr, at_(scale), p.scale_type, at_(dy), dy_stride, at_(ds), ds_stride, p.rows, p.d,
                           p.type, at_(dx), at_(dscale), at_(ws), on.stream),
          "msd_rms_backward");
    return first_order({dx, dscale, sums ? dx : Tensor(), Tensor()}, recorded);
  }
};

variable_list rms_norm(const Tensor& x, const Tensor& scale, const MaybeTensor& residual, const Rms& p) {
  only_run("rms_norm", x, scale, residual);
  if (at::GradMode::is_enabled() && (wanted(x) || wanted(scale) || (residual && wanted(*residual))))
    return RmsNorm::apply(x, scale, residual, p);
  RmsOut o = rms_run(x, scale.contiguous(), residual.value_or(Tensor()), *p, false);
  if (!o.sum.defined()) return {o.y};
  return {o.y, o.sum};
}

// ---- SwiGLU ----
struct GluPlan : torch::CustomClassHolder {
  int64_t rows, gate_stride, up_stride, held;
  int32_t d, type;
};
using Glu = c10::intrusive_ptr<GluPlan>;

Tensor glu_run(const Tensor& gate, const Tensor& up, const GluPlan& p, Tensor* held) {
  Place on(gate);
  Tensor y = contiguous_like(gate);
  if (held && p.held) *held = bytes(gate, p.held);
  check(msd_swiglu_forward(at_(gate), p.gate_stride, at_(up), p.up_stride, p.rows, p.d, p.type, at_(y), held ? at_(*held) : nullptr,
                           on.stream),
        "msd_swiglu_forward");
  return y;
}

struct Swiglu : torch::autograd::Function<Swiglu> {
  static variable_list forward(AutogradContext* ctx, const Tensor& gate, const Tensor& up, const Glu& p) {
    Tensor held, y = glu_run(gate, up, *p, &held);
    ctx->save_for_backward(held.defined() ? variable_list{held} : variable_list{gate, up});
    ctx->saved_data["plan"] = c10::IValue::make_capsule(p);
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    only_run("the gradient of swiglu", g[0]);
    const bool recorded = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    const auto s = ctx->get_saved_variables();
    const auto capsule = ctx->saved_data["plan"].toCapsule();
    const GluPlan& p = static_cast<const GluPlan&>(*capsule);
    if (p.held) restored(s[0], at::kByte, p.held, g[0].device());
    for (size_t i = 0; !p.held && i < 2; ++i) restored(s[i], scalar_type(p.type), g[0].sizes(), g[0].device());
    Place on(g[0]);
    const std::pair<Tensor, int64_t> none;
    const auto [gate, gate_stride] = p.held ? none : rows_of(s[0]);
    const auto [up, up_stride] = p.held ? none : rows_of(s[1]);
    const auto [dy, stride] = rows_of(g[0]);
    const Tensor held = p.held ? s[0].contiguous() : Tensor();
    Tensor dgate = contiguous_like(dy), dup = contiguous_like(dy);
    check(msd_swiglu_backward(at_(gate), gate_stride, at_(up), up_stride, p.held ? at_(held) : nullptr, at_(dy), stride, p.rows, p.d,
                              p.type, at_(dgate), at_(dup), on.stream),
          "msd_swiglu_backward");
    return first_order({dgate, dup, Tensor()}, recorded);
  }
};

Tensor swiglu(const Tensor& gate, const Tensor& up, const Glu& p) {
  only_run("swiglu", gate, up);
  if (at::GradMode::is_enabled() && (wanted(gate) || wanted(up))) return Swiglu::apply(gate, up, p)[0];
  return glu_run(gate, up, *p, nullptr);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  py::register_exception_translator([](std::exception_ptr e) {   // as the ctypes calls' errors
    try {
      if (e) std::rethrow_exception(e);
    } catch (const CallError& x) {
      const py::object type = py::module_::import("transformer_amd._lib").attr("MsdError");
      PyErr_SetObject(type.ptr(), type(x.code, x.what_).ptr());
    }
  });
  const auto free_threads = py::call_guard<py::gil_scoped_release>();
  py::class_<AttnPlan, Attn>(m, "AttnPlan")
      .def(py::init([](uintptr_t a, int64_t forward_bytes, int64_t backward_bytes, bool q_zero, bool k_zero, const MaybeTensor& table,
                       const MaybeTensor& host, uint64_t table_stream) {
        auto p = c10::make_intrusive<AttnPlan>();
        p->a = *reinterpret_cast<const msd_attn*>(a);
        p->forward_bytes = forward_bytes;
        p->backward_bytes = backward_bytes;
        p->q_zero = q_zero;
        p->k_zero = k_zero;
        p->table = table.value_or(Tensor());
        p->host = host.value_or(Tensor());
        p->table_stream = table_stream;
        return p;
      }));
  py::class_<RopePlan, Rope>(m, "RopePlan").def(py::init([](uintptr_t forward, uintptr_t backward) {
    auto p = c10::make_intrusive<RopePlan>();
    p->forward = *reinterpret_cast<const msd_rope*>(forward);
    p->backward = *reinterpret_cast<const msd_rope*>(backward);
    return p;
  }));
  py::class_<RmsPlan, Rms>(m, "RmsPlan")
      .def(py::init([](int64_t rows, int32_t d, int32_t type, int32_t scale_type, float eps, int64_t x_stride, int64_t residual_stride,
                       int64_t held, int64_t parts) {
        auto p = c10::make_intrusive<RmsPlan>();
        p->rows = rows;
        p->d = d;
        p->type = type;
        p->scale_type = scale_type;
        p->eps = eps;
        p->x_stride = x_stride;
        p->residual_stride = residual_stride;
        p->held = held;
        p->parts = parts;
        return p;
      }));
  py::class_<GluPlan, Glu>(m, "GluPlan")
      .def(py::init([](int64_t rows, int32_t d, int32_t type, int64_t gate_stride, int64_t up_stride, int64_t held) {
        auto p = c10::make_intrusive<GluPlan>();
        p->rows = rows;
        p->d = d;
        p->type = type;
        p->gate_stride = gate_stride;
        p->up_stride = up_stride;
        p->held = held;
        return p;
      }));
  m.def("attention", &attention, free_threads);
  m.def("rotary", &rotary, free_threads);
  m.def("rms_norm", &rms_norm, free_threads);
  m.def("swiglu", &swiglu, free_threads);
  m.def("row_stride", &row_stride);
  m.def("restored", [](const Tensor& x, const Tensor& saved) { restored(x, saved.scalar_type(), saved.sizes(), saved.device()); });
}
