// The training-layer operators as torch calls with autograd: allocation of outputs and workspaces from torch's allocator,
// the launches (include/mslayers.h) on the current stream, and the backward nodes.
//
// In C++ because a step's small calls are bound by the host: the backward of a call runs in a thread of the autograd engine, on
// another core than the caller's, where a node in Python took 25 to 50 us.  The checks of arguments are the Python modules'
// (attention.py, rotary.py, norm.py, swiglu.py): they make a plan per layout, which holds all that the C calls need, and hand
// over operands that the kernels take as they lie.  The paged cache's calls check theirs here.
#include <torch/extension.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/mslayers.h"
#include "../../include/mspaged.h"
#include "overlap.h"

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

// ---- the paged cache ----
// A step's sequences: the plan's words, on the device and on the host
struct PagedSteps : torch::CustomClassHolder {
  Tensor table, host;
  uint64_t table_stream;   // that the table was made on
  int32_t word(int i) const { return host.data_ptr<int32_t>()[i]; }
};
using Paged = c10::intrusive_ptr<PagedSteps>;

// keeps a table's memory until what is launched on stream s is done with it
void use_table(const Tensor& table, uint64_t made_on, hipStream_t s) {
  if (reinterpret_cast<uint64_t>(s) != made_on)
    table.record_stream(c10::impl::VirtualGuardImpl(table.device().type()).getStream(table.device()));
}

// (The checks of arguments are here and not in paged_attention.py: a decode step makes these calls in every layer, on sequences that are new
// in every step, and in Python they took longer than the launches.)
template <class... X>
void need(bool ok, const X&... x) {
  if (!ok) throw std::invalid_argument(c10::str(x...));
}

// stride of an axis; 0 along one of one (or none)
int64_t stride_of(const Tensor& x, int64_t axis) { return x.size(axis) > 1 ? x.stride(axis) : 0; }

// Pages (.., n_kv_heads, positions, d_head) of keys and of values, as a call on them
msd_paged paged_call(const Tensor& k, const Tensor& v, const PagedSteps& s, bool layers, bool written) {
  for (const Tensor* x : {&k, &v}) need(x->scalar_type() == at::kBFloat16, "pages must be bfloat16");
  const int64_t n = k.dim();
  need((n == 3 || (layers && n == 4)) && k.sizes() == v.sizes() && k.size(n - 2) % MSD_PAGE == 0,
       "pages of one shape (n_kv_heads, positions, d_head), positions a multiple of ", MSD_PAGE, ", expected, got ", k.sizes(), " and ", v.sizes());
  const int64_t D = k.size(n - 1), positions = k.size(n - 2);
  need(D % 8 == 0 && D > 0 && D <= 128, "d_head must be a multiple of 8 up to 128 (got ", D, ")");
  need(k.size(n - 3) == s.word(MSD_PLAN_KV_HEADS), "pages of ", k.size(n - 3), " heads, sequences of ", s.word(MSD_PLAN_KV_HEADS));
  need(k.is_cuda() && k.device() == v.device() && k.device() == s.table.device(), "pages and sequences must be on one GPU (got ", k.device(), ", ",
       v.device(), " and ", s.table.device(), ")");
  for (const Tensor* x : {&k, &v}) {
    bool aligned = x->stride(n - 1) == 1 && reinterpret_cast<uintptr_t>(x->data_ptr()) % 16 == 0;
    for (int64_t i = 0; i + 1 < n; ++i) aligned &= x->size(i) <= 1 || x->stride(i) % 8 == 0;
    need(aligned, "pages must have contiguous heads on 16-byte boundaries");
    bool near = x->stride(n - 2) < (int64_t(1) << 25);
    for (int64_t i = 0; i + 2 < n; ++i) near &= x->size(i) <= 1 || x->stride(i) < (int64_t(1) << 40);
    need(near, "pages: strides out of reach");
    if (!written) continue;
    std::vector<std::pair<int64_t, int64_t>> axes;   // no two places of the pages are one
    for (int64_t i = 0; i + 1 < n; ++i)
      if (x->size(i) > 1) axes.emplace_back(x->stride(i), x->size(i));
    std::sort(axes.begin(), axes.end());
    int64_t end = D;
    for (const auto& [stride, size] : axes) {
      need(stride >= end, "pages that are written must not overlap");
      end += (size - 1) * stride;
    }
  }
  need(positions < (int64_t(1) << 31) && s.word(MSD_PLAN_PAGES) <= positions / MSD_PAGE, "tables reach page ", s.word(MSD_PLAN_PAGES) - 1,
       ", the pages are ", positions / MSD_PAGE);
  msd_paged a{};
  a.d_head = int32_t(D);
  a.scale = 1;
  a.positions = positions;
  a.k_stride[0] = stride_of(k, n - 3), a.k_stride[1] = stride_of(k, n - 2);
  a.v_stride[0] = stride_of(v, n - 3), a.v_stride[1] = stride_of(v, n - 2);
  a.plan = s.table.data_ptr<int32_t>();
  a.plan_host = s.host.data_ptr<int32_t>();
  return a;
}

// New rows (rows, heads, d_head) that can be read where they lie: x, or a copy of it
Tensor paged_rows(const char* name, const Tensor& x, int64_t heads, const msd_paged& a, const PagedSteps& s, at::Device device) {
  need(x.dim() == 3 && x.size(1) == heads && x.size(2) == a.d_head, name, " (rows, ", heads, ", ", a.d_head, ") expected, got ", x.sizes());
  need(x.scalar_type() == at::kBFloat16, name, " must be bfloat16");
  need(x.device() == device, name, " and the pages must be on one GPU");
  need(s.word(MSD_PLAN_Q_END) <= x.size(0), "sequences reach row ", s.word(MSD_PLAN_Q_END), " of ", x.size(0), " rows of ", name);
  need(x.size(0) < (int64_t(1) << 31) / s.word(MSD_PLAN_HEADS), name, ": rows times heads out of reach");
  return attn_reads(x, heads) ? x : x.clone(at::MemoryFormat::Contiguous);
}

void weights_fit(const Tensor& w, at::IntArrayRef sizes, at::Device device, const char* where) {
  const int64_t n = int64_t(sizes.size());
  need(w.dim() == n + 1 && w.sizes().slice(0, n) == sizes && w.scalar_type() == at::kFloat && w.device() == device && w.size(n) < (int64_t(1) << 31),
       "weights must be float32 (", c10::Join(", ", sizes), ", width) on ", where, " GPU, got ", w.scalar_type(), " ", w.sizes(), " on ", w.device());
}

template <class... X>
void no_gradient(const char* what, const X&... x) {
  if (at::GradMode::is_enabled() && (x.requires_grad() || ...))
    throw std::invalid_argument(std::string(what) + " has no gradient: call it under torch.no_grad(), or hand over detached tensors");
}

// x's memory, from its first place to behind its last
struct Ends {
  uintptr_t first, last;
  explicit Ends(const Tensor& x) : first(reinterpret_cast<uintptr_t>(x.data_ptr())) {
    const auto sizes = x.sizes(), strides = x.strides();
    int64_t n = x.numel() ? 1 : 0;
    for (size_t i = 0; n && i < sizes.size(); ++i) n += (sizes[i] - 1) * strides[i];
    last = first + n * x.element_size();
  }
  bool meet(const Ends& other) const { return first < other.last && other.first < last; }
};

// Of pages of one shape, none of which overlaps with itself
bool share_memory(const Tensor& k, const Tensor& v) {
  std::vector<msd_overlap::Axis> axes;
  const int64_t n = k.dim();
  for (int64_t i = 0; i + 1 < n; ++i) axes.push_back({k.size(i), k.stride(i), v.stride(i)});
  return msd_overlap::share(std::move(axes), k.size(n - 1), static_cast<const uint16_t*>(v.data_ptr()) - static_cast<const uint16_t*>(k.data_ptr()));
}

// Pages that a call is about to write
struct Written {
  const Tensor &k, &v;
  Ends k_ends, v_ends;
  Written(const Tensor& k_pages, const Tensor& v_pages) : k(k_pages), v(v_pages), k_ends(k), v_ends(v) {}
  // (before anything is launched: an inference tensor outside inference mode raises here)
  void mark() const {
    need(!k_ends.meet(v_ends) || !share_memory(k, v), "k_pages and v_pages are the same memory, or share some of it");
    for (const Tensor* x : {&k, &v}) x->unsafeGetTensorImpl()->bump_version();
  }
  // x, or a copy of it where it lies among the pages: new rows are those from before the call
  Tensor apart(const Tensor& x) const {
    const Ends e(x);
    return e.meet(k_ends) || e.meet(v_ends) ? x.clone(at::MemoryFormat::Contiguous) : x;
  }
};

void paged_append(const Tensor& k_new, const Tensor& v_new, const Tensor& k_pages, const Tensor& v_pages, const Paged& steps) {
  only_run("paged_append", k_new, v_new, k_pages, v_pages);
  no_gradient("paged_append", k_new, v_new, k_pages, v_pages);
  const PagedSteps& p = *steps;
  msd_paged a = paged_call(k_pages, v_pages, p, false, true);
  const int64_t heads = p.word(MSD_PLAN_KV_HEADS);
  Place on(k_pages);
  const Written pages(k_pages, v_pages);
  const Tensor k = pages.apart(paged_rows("k", k_new, heads, a, p, k_pages.device()));
  const Tensor v = pages.apart(paged_rows("v", v_new, heads, a, p, k_pages.device()));
  need(k.size(0) == v.size(0), "k of ", k.size(0), " rows, v of ", v.size(0));
  need(!p.word(MSD_PLAN_SHARED), "a page that takes new rows is in use elsewhere too");
  a.q_rows = k.size(0);
  const int64_t k_stride[2] = {stride_of(k, 0), stride_of(k, 1)}, v_stride[2] = {stride_of(v, 0), stride_of(v, 1)};
  use_table(p.table, p.table_stream, on.stream);
  pages.mark();
  check(msd_paged_append(&a, at_(k), k_stride, at_(v), v_stride, at_(k_pages), at_(v_pages), on.stream), "msd_paged_append");
}

variable_list paged_attention(const Tensor& q_new, const Tensor& k_pages, const Tensor& v_pages, const Paged& steps, std::optional<double> scale,
                              const MaybeTensor& weights) {
  only_run("paged_attention", q_new, k_pages, v_pages, weights);
  no_gradient("paged_attention", q_new, k_pages, v_pages);
  if (weights) no_gradient("paged_attention", *weights);
  const PagedSteps& p = *steps;
  msd_paged a = paged_call(k_pages, v_pages, p, false, false);
  const double c = scale.value_or(1 / std::sqrt(double(a.d_head)));
  need(c >= 0x1p-60 && c <= 0x1p60, "scale must lie in [2 ** -60, 2 ** 60] (got ", c, ")");
  a.scale = float(c);
  const int64_t sizes[2] = {p.word(MSD_PLAN_SEQS), p.word(MSD_PLAN_KV_HEADS)};
  if (weights) weights_fit(*weights, sizes, k_pages.device(), "the pages'");
  Place on(k_pages);
  const Tensor q = paged_rows("q", q_new, p.word(MSD_PLAN_HEADS), a, p, k_pages.device());
  a.q_rows = q.size(0);
  a.q_stride[0] = stride_of(q, 0), a.q_stride[1] = stride_of(q, 1);
  Tensor out = attn_output(q, p.word(MSD_PLAN_Q_COUNT) != a.q_rows), held, counted, ws;
  if (weights) {
    held = weights->contiguous();
    counted = at::empty({sizes[0], sizes[1], p.word(MSD_PLAN_LONGEST)}, held.options());
  }
  const int64_t n = msd_paged_attn_workspace_bytes(&a, counted.defined());
  if (n < 0) check(int32_t(n), "msd_paged_attn_workspace_bytes");
  if (n) ws = bytes(q, n);
  use_table(p.table, p.table_stream, on.stream);
  check(msd_paged_attn(&a, at_(q), at_(k_pages), at_(v_pages), at_(out), static_cast<const float*>(at_(held)),
                       held.defined() ? int32_t(held.size(2)) : 0, static_cast<float*>(at_(counted)), at_(ws), on.stream),
        "msd_paged_attn");
  if (!weights) return {out};
  return {out, counted};
}

variable_list paged_evict(const Tensor& k_pages, const Tensor& v_pages, const Tensor& weights, const Paged& steps, const Tensor& to, uint64_t to_stream,
                          int32_t pages, int32_t keep, int32_t recent) {
  only_run("paged_evict", k_pages, v_pages, weights);
  no_gradient("paged_evict", k_pages, v_pages, weights);
  const PagedSteps& p = *steps;
  msd_paged a = paged_call(k_pages, v_pages, p, true, true);
  need(pages <= a.positions / MSD_PAGE, "tables reach page ", pages - 1, ", the pages are ", a.positions / MSD_PAGE);
  a.q_rows = p.word(MSD_PLAN_Q_END);
  const bool layers = k_pages.dim() == 4;
  std::vector<int64_t> sizes;
  if (layers) sizes.push_back(k_pages.size(0));
  sizes.push_back(p.word(MSD_PLAN_SEQS));
  sizes.push_back(p.word(MSD_PLAN_KV_HEADS));
  need(!layers || k_pages.size(0) * k_pages.size(1) < 65536, "layers times heads must stay below 65536 (got ", k_pages.size(0), " and ", k_pages.size(1), ")");
  weights_fit(weights, sizes, k_pages.device(), "the pages'");
  const Written memory(k_pages, v_pages);
  Place on(k_pages);
  const Tensor w = weights.contiguous();
  sizes.push_back(keep);
  Tensor out = at::empty(sizes, w.options()), kept = at::empty(sizes, w.options().dtype(at::kInt));
  const int32_t n_layers = layers ? int32_t(k_pages.size(0)) : 1;
  use_table(p.table, p.table_stream, on.stream);
  use_table(to, to_stream, on.stream);
  memory.mark();
  check(msd_paged_evict(&a, n_layers, layers ? stride_of(k_pages, 0) : 0, layers ? stride_of(v_pages, 0) : 0, at_(k_pages), at_(v_pages),
                        static_cast<const float*>(at_(w)), int32_t(w.size(-1)), keep, recent, static_cast<const int32_t*>(at_(to)),
                        int32_t(to.size(1)), static_cast<float*>(at_(out)), static_cast<int32_t*>(at_(kept)), on.stream),
        "msd_paged_evict");
  return {out, kept};
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
  py::class_<PagedSteps, Paged>(m, "PagedSteps").def(py::init([](const Tensor& table, const Tensor& host, uint64_t table_stream) {
    auto p = c10::make_intrusive<PagedSteps>();
    p->table = table;
    p->host = host;
    p->table_stream = table_stream;
    return p;
  }));
  m.def("attention", &attention, free_threads);
  m.def("rotary", &rotary, free_threads);
  m.def("rms_norm", &rms_norm, free_threads);
  m.def("swiglu", &swiglu, free_threads);
  m.def("paged_append", &paged_append, free_threads);
  m.def("paged_attention", &paged_attention, free_threads);
  m.def("paged_evict", &paged_evict, free_threads);
  m.def("row_stride", &row_stride);
  m.def("restored", [](const Tensor& x, const Tensor& saved) { restored(x, saved.scalar_type(), saved.sizes(), saved.device()); });
}
