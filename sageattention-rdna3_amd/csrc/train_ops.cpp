// Compiled host layer of the training operators: attention with its gradient
// (sageattn_train, sageattn_backward) and rotary positions over several axes
// (rotary_axes), as autograd functions over the C ABI.  The Python functions
// check arguments and their messages; a training step of a small block is bound
// by the host, and the same nodes written in Python cost it ~40 us more.
//
// The backward functions run on the autograd engine's threads, on the device
// and the current stream of their forward call; they raise only std::exception
// types (anything else would end the process there).
#include "host_common.h"

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <vector>

namespace sage_host {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void* current_stream(const at::Tensor& t) {
  return reinterpret_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

void check_std(const char* fn, int64_t rc) {
  if (rc < 0) {
    const char* m = sage_last_error();
    throw std::runtime_error(std::string(fn) + ": " + (m != nullptr ? m : ""));
  }
}

// t with rows that meet the 16-byte access contract and do not overlap
at::Tensor rows_ready(const at::Tensor& t, int64_t layout) {
  const Dims d = bhnd(t, layout);
  const int64_t align = t.element_size() == 4 ? 4 : 8;
  if (t.stride(3) == 1 && (d.n <= 1 || d.sn >= d.d) && d.sb % align == 0 && d.sh % align == 0 && d.sn % align == 0 &&
      reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0)
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return SAGE_DTYPE_F16;
    case at::kBFloat16: return SAGE_DTYPE_BF16;
    default: return SAGE_DTYPE_F32;
  }
}

// The kernels' byte offsets within a head are 32-bit, up to 128 rows past its end (sage_attn_bwd).
bool head_fits(int64_t n, int64_t sn) { return (n + 128) * sn * 2 <= static_cast<int64_t>(UINT32_MAX); }

// rows_ready, with every head's rows within those offsets: [B,N,H,D] of many heads and tokens is copied head by head.
at::Tensor heads_ready(const at::Tensor& t, int64_t layout) {
  const at::Tensor r = rows_ready(t, layout);
  const Dims d = bhnd(r, layout);
  if (d.n <= 1 || head_fits(d.n, d.sn)) return r;
  return layout == 1 ? r.clone(at::MemoryFormat::Contiguous) : r.transpose(1, 2).clone(at::MemoryFormat::Contiguous).transpose(1, 2);
}

// A gradient in the layout of `like` (whose own strides may be those of a view or an expanded tensor): contiguous, or head
// by head where heads_ready would copy it.
at::Tensor grad_like(const at::Tensor& like, int64_t layout) {
  const Dims d = bhnd(like, layout);
  if (layout == 1 || head_fits(d.n, d.h * d.d)) return at::empty(like.sizes(), like.options());
  return at::empty({d.b, d.h, d.n, d.d}, like.options()).transpose(1, 2);
}

// The backward pass's limits, told by the forward call (they start near 2^24 tokens, or 2^24 blocks of 64).
void check_bwd_sizes(const at::Tensor& q, const at::Tensor& k, int64_t layout, bool is_causal) {
  const Dims a = bhnd(q, layout), b = bhnd(k, layout);
  constexpr int64_t kMany = 1 << 24;
  if (a.n < kMany - 128 && b.n < kMany - 128 && a.b * a.h < kMany && a.b * a.h * ((a.n + 63) / 64 + (b.n + 63) / 64) < kMany) return;
  const int64_t rc = sage_attn_bwd_workspace_bytes(dtype_code(q), a.b, a.h, b.h, a.n, b.n, a.d, is_causal ? 1 : 0, 1, 1);
  if (rc < 0) check("sage_attn_bwd_workspace_bytes", static_cast<int>(rc));
  if (!head_fits(std::max(a.n, b.n), a.d))
    throw py::value_error("sageattn_train: the backward pass takes heads of up to " +
                          std::to_string(UINT32_MAX / (2 * a.d) - 128) + " tokens");
}

bool dual(const at::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }

struct AttnGrads {
  at::Tensor dq, dk, dv;
};

AttnGrads attn_bwd(at::Tensor dout, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor out, at::Tensor lse,
                   at::Tensor dlse, int64_t layout, bool is_causal, double sm_scale, bool need_q, bool need_kv,
                   bool own_lse) {
  const c10::DeviceGuard guard(q.device());
  dout = heads_ready(dout, layout);
  q = heads_ready(q, layout);
  k = heads_ready(k, layout);
  v = heads_ready(v, layout);
  out = heads_ready(out, layout);
  lse = lse.contiguous();
  if (dlse.defined()) dlse = dlse.contiguous();
  AttnGrads g;
  if (need_q) g.dq = grad_like(q, layout);
  if (need_kv) {
    g.dk = grad_like(k, layout);
    g.dv = grad_like(v, layout);
  }
  const Dims qd = bhnd(q, layout), kd = bhnd(k, layout);
  const int64_t bytes = sage_attn_bwd_workspace_bytes(dtype_code(q), qd.b, qd.h, kd.h, qd.n, kd.n, qd.d, is_causal ? 1 : 0,
                                                     need_q ? 1 : 0, need_kv ? 1 : 0);
  check_std("sage_attn_bwd_workspace_bytes", bytes);
  at::Tensor ws = at::empty({bytes}, q.options().dtype(at::kByte));
  const at::Tensor* const order[8] = {&dout, &q, &k, &v, &out, &g.dq, &g.dk, &g.dv};
  int64_t strides[24] = {};
  for (int i = 0; i < 8; ++i) {
    if (!order[i]->defined()) continue;
    const Dims d = bhnd(*order[i], layout);
    strides[3 * i] = d.sb;
    strides[3 * i + 1] = d.sh;
    strides[3 * i + 2] = d.sn;
  }
  check_std(own_lse ? "sage_attn_direct_bwd" : "sage_attn_bwd",
            (own_lse ? sage_attn_direct_bwd : sage_attn_bwd)(
                dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                static_cast<const float*>(lse.data_ptr()), static_cast<const float*>(ptr(dlse)), ptr(g.dq), ptr(g.dk),
                ptr(g.dv), dtype_code(q), qd.b, qd.h, kd.h, qd.n, kd.n, qd.d, strides, is_causal ? 1 : 0, sm_scale,
                ws.data_ptr(), bytes, current_stream(q)));
  return g;
}

// Gradients that are not differentiable themselves: under create_graph they get a node that raises when a second
// derivative is asked for (an output without a graph would be taken for a constant).
variable_list once_differentiable(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in;
  for (auto& g : grads)
    if (g.defined()) in.push_back(g.detach().requires_grad_(true));
  torch::autograd::DelayedError fail("sageattn_train: the gradient is not differentiable a second time",
                                     static_cast<int64_t>(in.size()));
  variable_list made = fail.apply(std::move(in));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = made[i++];
  return grads;
}

struct AttnTrain : public torch::autograd::Function<AttnTrain> {
  static variable_list forward(AutogradContext* ctx, at::Tensor q, at::Tensor k, at::Tensor v, int64_t layout,
                               bool is_causal, double sm_scale) {
    auto r = attn_fwd(q, k, v, layout, is_causal, sm_scale, true, false, true, 0, current_stream(q));
    ctx->save_for_backward({q, k, v, r.first, r.second});
    ctx->saved_data["args"] = std::vector<double>{static_cast<double>(layout), is_causal ? 1.0 : 0.0, sm_scale};
    ctx->set_materialize_grads(false);
    return {r.first, r.second};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const bool need_q = ctx->needs_input_grad(0), need_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    variable_list r(6);
    if (!grads[0].defined() && !grads[1].defined()) return r;
    if (dual(grads[0]) || dual(grads[1])) throw std::runtime_error("sageattn_train has no forward-mode derivative");
    at::Tensor dout = grads[0].defined() ? grads[0] : at::zeros_like(s[3]);
    {
      at::NoGradGuard no_grad;
      const auto args = ctx->saved_data["args"].toDoubleVector();
      AttnGrads g = attn_bwd(dout, s[0], s[1], s[2], s[3], s[4], grads[1], static_cast<int64_t>(args[0]),
                             args[1] != 0.0, args[2], need_q, need_kv, true);
      r[0] = g.dq;
      if (ctx->needs_input_grad(1)) r[1] = g.dk;
      if (ctx->needs_input_grad(2)) r[2] = g.dv;
    }
    return once_differentiable(std::move(r));
  }
};

struct RotaryCfg {
  std::vector<int64_t> axes;
  std::vector<double> theta;
  int64_t layout;
  bool interleaved, inverse;
};

// One launch for one or two tensors (an undefined one is left out).
variable_list rotate(at::Tensor x0, at::Tensor x1, const at::Tensor& pos, const RotaryCfg& c) {
  variable_list in = {x0, x1}, out(2);
  int64_t strides[12] = {}, heads[2] = {0, 0}, pos_strides[3], batch = 0, n = 0, d = 0;
  int dtype = 0;
  at::Tensor any;
  for (int i = 0; i < 2; ++i) {
    if (!in[i].defined()) continue;
    in[i] = rows_ready(in[i], c.layout);
    out[i] = at::empty(in[i].sizes(), in[i].options());
    const Dims a = bhnd(in[i], c.layout), o = bhnd(out[i], c.layout);
    const int64_t s[6] = {a.sb, a.sh, a.sn, o.sb, o.sh, o.sn};
    std::copy(s, s + 6, strides + 6 * i);
    heads[i] = a.h;
    batch = a.b, n = a.n, d = a.d;
    dtype = dtype_code(in[i]);
    any = in[i];
  }
  if (!any.defined()) return out;
  const c10::DeviceGuard guard(any.device());
  const bool batched = pos.dim() == 3;
  pos_strides[0] = batched ? pos.stride(0) : 0;
  pos_strides[1] = pos.stride(batched ? 1 : 0);
  pos_strides[2] = pos.stride(batched ? 2 : 1);
  const int type = pos.scalar_type() == at::kInt ? SAGE_POSITION_I32 : pos.scalar_type() == at::kLong ? SAGE_POSITION_I64 : SAGE_POSITION_F32;
  check_std("sage_rotary_axes",
            sage_rotary_axes(ptr(in[0]), ptr(out[0]), heads[0], ptr(in[1]), ptr(out[1]), heads[1], dtype, batch, n, d,
                             strides, pos.data_ptr(), type, pos_strides, static_cast<int>(c.axes.size()), c.axes.data(),
                             c.theta.data(), c.interleaved ? 1 : 0, c.inverse ? 1 : 0, current_stream(any)));
  return out;
}

// Linear in its tensors: the gradient is the turn the other way, through the same node, so it can be differentiated
// again.
struct RotaryAxes : public torch::autograd::Function<RotaryAxes> {
  static variable_list forward(AutogradContext* ctx, const c10::optional<at::Tensor>& q, const c10::optional<at::Tensor>& k,
                               at::Tensor pos, RotaryCfg c) {
    variable_list out = rotate(q ? *q : at::Tensor(), k ? *k : at::Tensor(), pos, c);
    ctx->save_for_backward({pos});
    // one entry: layout, interleaved, inverse, whether q is there, then the axes' thetas and widths
    std::vector<double> args = {static_cast<double>(c.layout), c.interleaved ? 1.0 : 0.0, c.inverse ? 1.0 : 0.0,
                                q.has_value() ? 1.0 : 0.0};
    args.insert(args.end(), c.theta.begin(), c.theta.end());
    args.insert(args.end(), c.axes.begin(), c.axes.end());
    ctx->saved_data["args"] = std::move(args);
    ctx->set_materialize_grads(false);
    variable_list made, fixed;
    for (int i = 0; i < 2; ++i) {
      if (!out[i].defined()) continue;
      made.push_back(out[i]);
      if (!(i == 0 ? q : k)->requires_grad()) fixed.push_back(out[i]);
    }
    ctx->mark_non_differentiable(fixed);  // of an input without a gradient: attention then computes none for it either
    return made;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto args = ctx->saved_data["args"].toDoubleVector();
    const auto theta = args.begin() + 4, axes = theta + (args.end() - theta) / 2;
    const RotaryCfg c{{axes, args.end()}, {theta, axes}, static_cast<int64_t>(args[0]), args[1] != 0.0, args[2] == 0.0};
    const bool has_q = args[3] != 0.0;
    c10::optional<at::Tensor> g[2];
    size_t at = 0;
    if (has_q && at < grads.size()) {
      if (grads[at].defined() && ctx->needs_input_grad(0)) g[0] = grads[at];
      ++at;
    }
    const size_t k_input = has_q ? 1 : 0;  // undefined optionals are not inputs of the node
    if (at < grads.size() && grads[at].defined() && ctx->needs_input_grad(k_input)) g[1] = grads[at];
    variable_list r(4);
    if (!g[0] && !g[1]) return r;
    variable_list made = apply(g[0], g[1], ctx->get_saved_variables()[0], c);
    size_t i = 0;
    if (g[0]) r[0] = made[i++];
    if (g[1]) r[1] = made[i++];
    return r;
  }
};

// ---- the public calls: checks and messages, then the nodes above

void require(bool ok, const std::string& message) {
  if (ok) return;
  PyErr_SetString(PyExc_AssertionError, message.c_str());
  throw py::error_already_set();
}

void require_value(bool ok, const std::string& message) {
  if (!ok) throw py::value_error(message);
}

// A dual tensor need not require grad, and its tangent would be lost without a word.
void refuse_dual(const char* fn, std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors) {
    if (t == nullptr || !dual(*t)) continue;
    PyErr_SetString(PyExc_NotImplementedError, (std::string(fn) + " has no forward-mode derivative").c_str());
    throw py::error_already_set();
  }
}

int64_t layout_code(const py::handle& name) {
  if (py::isinstance<py::str>(name)) {
    const std::string s = py::cast<std::string>(name);
    if (s == "HND") return 1;
    if (s == "NHD") return 0;
  }
  throw py::value_error("tensor_layout must be 'HND' or 'NHD', got " + py::cast<std::string>(py::repr(name)));
}

// The checks of sageattn that hold here too, and its shapes.
void check_qkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t layout) {
  const auto dt = q.scalar_type();
  require(q.is_cuda(), "Input tensors must be on CUDA/HIP device.");
  require(dt == at::kHalf || dt == at::kBFloat16, "Input tensors must be fp16 or bf16.");
  require(k.device() == q.device() && v.device() == q.device(), "All tensors must be on the same device.");
  require(k.scalar_type() == dt && v.scalar_type() == dt, "All tensors must have the same dtype.");
  require_value(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k and v must be 4-D tensors");
  require(q.size(3) == 64 || q.size(3) == 128, "head_dim must be 64 or 128, got " + std::to_string(q.size(3)) + ".");
  require(q.stride(3) == 1 && k.stride(3) == 1 && v.stride(3) == 1, "Last dim of qkv must be contiguous.");
  const int h = layout == 1 ? 1 : 2;
  require_value(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3),
                "incompatible shapes q=" + shape_str(q) + " k=" + shape_str(k) + " v=" + shape_str(v));
  require_value(q.size(h) > 0 && k.size(h) > 0 && q.size(h) % k.size(h) == 0,
                "number of query heads (" + std::to_string(q.size(h)) + ") must be a multiple of kv heads (" +
                    std::to_string(k.size(h)) + ")");
}

double scale_or_default(const std::optional<double>& scale, const at::Tensor& q) {
  return scale ? *scale : std::pow(static_cast<double>(q.size(3)), -0.5);
}

py::object sageattn_train(at::Tensor q, at::Tensor k, at::Tensor v, const py::object& tensor_layout, bool is_causal,
                          std::optional<double> sm_scale, bool return_lse) {
  const int64_t layout = layout_code(tensor_layout);
  check_qkv(q, k, v, layout);
  refuse_dual("sageattn_train", {&q, &k, &v});
  const c10::DeviceGuard guard(q.device());
  if (!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad() || v.requires_grad())) {
    auto r = attn_fwd(q, k, v, layout, is_causal, scale_or_default(sm_scale, q), return_lse, false, true, 0, current_stream(q));
    if (return_lse) return py::make_tuple(r.first, r.second);
    return py::cast(r.first);
  }
  check_bwd_sizes(q, k, layout, is_causal);
  variable_list r = AttnTrain::apply(q, k, v, layout, is_causal, scale_or_default(sm_scale, q));
  if (return_lse) return py::make_tuple(r[0], r[1]);
  return py::cast(r[0]);
}

// k minus its mean over the tokens, as the INT8 path's smooth_k takes it (and rounds it, more coarsely than here).
at::Tensor smoothed(const at::Tensor& key, int64_t layout) {
  const at::Tensor k = rows_ready(key, layout);
  const Dims d = bhnd(k, layout);
  if (d.b == 0 || d.n == 0) return k;
  const int64_t bytes = sage_k_mean_workspace_bytes(d.b, d.h, d.n, d.d);
  check_std("sage_k_mean_workspace_bytes", bytes);
  at::Tensor mean = at::empty({d.b, d.h, d.d}, k.options());
  at::Tensor ws = at::empty({(std::max<int64_t>(bytes, 4) + 3) / 4}, k.options().dtype(at::kFloat));
  check_std("sage_k_mean", sage_k_mean(k.data_ptr(), mean.data_ptr(), ws.data_ptr(), dtype_code(k), d.b, d.h, d.n, d.d,
                                       d.sb, d.sh, d.sn, current_stream(k)));
  return k - mean.unsqueeze(layout == 1 ? 2 : 1);
}

py::object sageattn_backward(at::Tensor dout, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor out, at::Tensor lse,
                             const py::object& tensor_layout, bool is_causal, std::optional<double> sm_scale,
                             const std::optional<at::Tensor>& dlse, bool smooth) {
  const int64_t layout = layout_code(tensor_layout);
  check_qkv(q, k, v, layout);
  for (const auto& [name, t] : {std::pair<const char*, const at::Tensor*>("dout", &dout), {"out", &out}})
    require_value(t->sizes() == q.sizes() && t->scalar_type() == q.scalar_type() && t->device() == q.device(),
                  std::string(name) + " must have the shape, dtype and device of q");
  const Dims d = bhnd(q, layout);
  const std::vector<int64_t> rows = {d.b, d.h, d.n};
  const at::Tensor* const optional_dlse = dlse ? &*dlse : nullptr;
  for (const auto& [name, t] : {std::pair<const char*, const at::Tensor*>("lse", &lse), {"dlse", optional_dlse}})
    require_value(t == nullptr || (t->sizes() == at::IntArrayRef(rows) && t->scalar_type() == at::kFloat && t->device() == q.device()),
                  std::string(name) + " must be [" + std::to_string(d.b) + ", " + std::to_string(d.h) + ", " +
                      std::to_string(d.n) + "] fp32 on the device of q");
  refuse_dual("sageattn_backward", {&dout, &q, &k, &v, &out, &lse, optional_dlse});
  require_value(!smooth || dlse == std::nullopt, "dlse is not taken with smooth_k=True");
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(q.device());
  if (smooth) k = smoothed(k, layout);
  AttnGrads g = attn_bwd(dout, q, k, v, out, lse, dlse ? *dlse : at::Tensor(), layout, is_causal, scale_or_default(sm_scale, q), true, true,
                         false);
  return py::make_tuple(g.dq, g.dk, g.dv);
}

py::object rotary_axes(at::Tensor q, const std::optional<at::Tensor>& k, at::Tensor positions,
                       const std::vector<int64_t>& axes, const py::object& theta, const py::object& tensor_layout,
                       bool interleaved, bool inverse) {
  const int64_t layout = layout_code(tensor_layout);
  const auto dt = q.scalar_type();
  require(q.is_cuda(), "Input tensors must be on CUDA/HIP device.");
  require(dt == at::kHalf || dt == at::kBFloat16 || dt == at::kFloat, "Input tensors must be fp16, bf16, or fp32.");
  require_value(q.dim() == 4, "q and k must be 4-D tensors");
  const int64_t d = q.size(3), b = q.size(0), n = q.size(layout == 1 ? 2 : 1);
  require(d == 64 || d == 128, "head_dim must be 64 or 128, got " + std::to_string(d) + ".");
  if (k) {
    require(k->device() == q.device(), "All tensors must be on the same device.");
    require(k->scalar_type() == dt, "All tensors must have the same dtype.");
    require_value(k->dim() == 4 && k->size(0) == b && k->size(layout == 1 ? 2 : 1) == n && k->size(3) == d,
                  "incompatible shapes q=" + shape_str(q) + " k=" + shape_str(*k));
  }
  int64_t width = 0;
  bool fits = !axes.empty();
  for (int64_t a : axes) {
    fits = fits && a > 0 && a % 2 == 0 && a <= d - width;
    width += fits ? a : 0;
  }
  require_value(fits, "axes_dim must be positive even widths that sum to at most " + std::to_string(d));
  RotaryCfg c{axes, {}, layout, interleaved, inverse};
  if (py::isinstance<py::sequence>(theta) && !py::isinstance<at::Tensor>(theta)) c.theta = py::cast<std::vector<double>>(theta);
  else c.theta.assign(axes.size(), py::cast<double>(theta));
  bool positive = c.theta.size() == axes.size();
  for (double t : c.theta) positive = positive && t > 0.0 && std::isfinite(t);
  require_value(positive, "theta must be positive: one number, or one per axis");
  const auto pt = positions.scalar_type();
  require_value(positions.device() == q.device(), "positions must be on the device of q");
  require_value(pt == at::kInt || pt == at::kLong || pt == at::kFloat, "positions must be int32, int64 or float32");
  const int64_t na = static_cast<int64_t>(axes.size());
  require_value(positions.sizes() == at::IntArrayRef({n, na}) || positions.sizes() == at::IntArrayRef({b, n, na}),
                "positions must be [" + std::to_string(n) + ", " + std::to_string(na) + "] or [" + std::to_string(b) +
                    ", " + std::to_string(n) + ", " + std::to_string(na) + "], got " + shape_str(positions));
  refuse_dual("rotary_axes", {&q, k ? &*k : nullptr, &positions});
  if (!at::GradMode::is_enabled() || !(q.requires_grad() || (k && k->requires_grad()))) {  // no node: ~2 us
    variable_list r = rotate(q, k ? *k : at::Tensor(), positions, c);
    if (!k) return py::cast(r[0]);
    return py::make_tuple(r[0], r[1]);
  }
  variable_list r = RotaryAxes::apply(q, k, positions.detach(), std::move(c));
  if (r.size() == 1) return py::cast(r[0]);
  return py::make_tuple(r[0], r[1]);
}

}  // namespace

void bind_train(py::module_& m) {
  m.def("sageattn_train", &sageattn_train);
  m.def("sageattn_backward", &sageattn_backward);
  m.def("rotary_axes", &rotary_axes);
}

}  // namespace sage_host
