// blocks_aten.cpp -- ATen / autograd front end of include/butd_gated_ffn.h and include/butd_residual_norm.h: checks,
// allocation and the autograd nodes of butd_detr_amd.gated_ffn and butd_detr_amd.residual_norm in C++.  A small layer's pass
// is bound by the host: as Python autograd functions over ctypes a forward + backward took about 145 us of it, the kernels
// of 2048 rows x 288 take 25.
#include <ATen/autocast_mode.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <climits>
#include <optional>
#include <string>
#include <tuple>
#include <unordered_set>
#include <vector>

#include "butd_gated_ffn.h"
#include "butd_pointnet2.h"
#include "butd_residual_norm.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;
typedef std::optional<Tensor> Maybe;

butd_stream_t stream_of(const Tensor &t) { return (butd_stream_t)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void ok(long err, const char *what) { TORCH_CHECK(err == 0, what, ": HIP error ", err, " (", butd_error_string((int)err), ")"); }

int dtype_of(at::ScalarType t) {       // BUTD_FFN_* and BUTD_NORM_* number alike; -1: not served
  return t == at::kFloat ? 0 : t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : -1;
}
static_assert(BUTD_FFN_F32 == BUTD_NORM_F32 && BUTD_FFN_BF16 == BUTD_NORM_BF16 && BUTD_FFN_F16 == BUTD_NORM_F16, "");

const char *python_name(at::ScalarType t) {
  return t == at::kFloat ? "torch.float32" : t == at::kBFloat16 ? "torch.bfloat16" : t == at::kHalf ? "torch.float16" : c10::toString(t);
}
std::string python_shape(at::IntArrayRef s) {
  std::string out = "(";
  for (size_t i = 0; i < s.size(); ++i) out += (i ? ", " : "") + std::to_string(s[i]);
  return out + (s.size() == 1 ? ",)" : ")");
}

void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor value(const Maybe &t) { return t.has_value() ? *t : Tensor(); }
Tensor contiguous(const Tensor &t) { return t.defined() ? t.contiguous() : t; }

// The kernels are no registered operators: a tracer would record the allocation of the outputs and nothing that fills them.
void no_tracing(const char *what) {
  TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                  !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
              what, ": cannot be traced (torch.jit.trace, torch.fx make_fx)");
}

bool wants_grad(std::initializer_list<Tensor> ts, const char *what) {
  for (const Tensor &t : ts)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), what, ": forward-mode derivatives are not implemented");
  if (!at::GradMode::is_enabled()) return false;
  bool wanted = false;
  for (const Tensor &t : ts) wanted |= t.defined() && t.requires_grad();
  if (!wanted) return false;
  // A leaf whose gradient accumulator an eager graph keeps alive belongs to that graph's stream, as an eager graph's output
  // does.  A backward pass captured elsewhere makes that stream wait for the capture; the default stream cannot, which ends the
  // process: refused here, for the operands and for what stands behind views and casts of them that this capture has made.
  const hipStream_t stream = (hipStream_t)stream_of(*ts.begin());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (!stream || hipStreamIsCapturing(stream, &status) != hipSuccess || status == hipStreamCaptureStatusNone) return true;
  std::vector<std::shared_ptr<torch::autograd::Node>> open;
  std::unordered_set<const torch::autograd::Node *> seen;
  const auto visit = [&](const std::shared_ptr<torch::autograd::Node> &node) {
    if (node && seen.insert(node.get()).second) open.push_back(node);
  };
  for (const Tensor &t : ts)
    if (t.defined() && t.requires_grad()) visit(t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn());
  while (!open.empty()) {
    const auto node = open.back();
    open.pop_back();
    const auto s = node->stream();
    if (!s || !s->device().is_cuda()) continue;
    const hipStream_t owner = c10::hip::HIPStreamMasqueradingAsCUDA(*s).stream();
    TORCH_CHECK(owner != nullptr, what, ": captured into a graph while an eager graph of the same leaves is alive on the default "
                "stream; release its outputs first, or detach what is taken from it");
    if (owner == stream)
      for (const auto &edge : node->next_edges()) visit(edge.function);
  }
  return true;
}

// What a backward pass hands back is not differentiable: under create_graph a second derivative raises instead of being zero.
void seal(variable_list &grads, const char *what) {
  if (!at::GradMode::is_enabled()) return;
  variable_list some;
  for (const Tensor &g : grads)
    if (g.defined()) some.push_back(g.requires_grad() ? g : g.detach().requires_grad_(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + ": only first derivatives are implemented", (int64_t)some.size());
  variable_list sealed = (*error)(std::move(some));
  size_t k = 0;
  for (Tensor &g : grads)
    if (g.defined()) g = sealed[k++];
}

// ---- the gated feed-forward block -----------------------------------------------------------------------------------------
// (..., C) as rows: the tensor itself where it has two dimensions and a contiguous last one, else a (contiguous) 2-d form
Tensor rows_of(const Tensor &t) {
  const int64_t cols = t.size(-1);
  if (t.dim() == 2 && t.size(0) > 1 && t.stride(1) == 1 && t.stride(0) >= cols) return t;
  return t.contiguous().view({-1, cols});
}
long ld_of(const Tensor &rows) { return rows.size(0) > 1 ? rows.stride(0) : rows.size(1); }

butd_gated_ffn_args ffn_args(const Tensor &x, const Tensor &gate, const Tensor &up, const Tensor &down, int64_t activation) {
  butd_gated_ffn_args a{};
  a.dtype = dtype_of(x.scalar_type());
  a.activation = (int)activation;
  a.rows = x.size(0);
  a.width = (int)gate.size(1);
  a.hidden = (int)gate.size(0);
  a.x = ptr(x);         a.ld_x = ld_of(x);
  a.w_gate = ptr(gate); a.ld_gate = ld_of(gate);
  a.w_up = ptr(up);     a.ld_up = ld_of(up);
  a.w_down = ptr(down); a.ld_down = ld_of(down);
  a.ld_h = butd_gated_ffn_ld_hidden(a.dtype, a.hidden);
  return a;
}

void ffn_run(const butd_gated_ffn_args &a, const Tensor &ref, bool backward) {
  const char *what = backward ? "butd_gated_ffn_bwd" : "butd_gated_ffn_fwd";
  const long need = backward ? butd_gated_ffn_bwd_workspace(&a) : butd_gated_ffn_fwd_workspace(&a);
  ok(need < 0 ? -need : 0, what);
  Tensor ws;
  if (need) ws = at::empty({need}, ref.options().dtype(at::kByte));
  ok((backward ? butd_gated_ffn_bwd : butd_gated_ffn_fwd)(&a, ptr(ws), need, stream_of(ref)), what);
}

struct FfnOut {
  Tensor y, h, ab;
};
FfnOut ffn_forward(const Tensor &x, const Tensor &gate, const Tensor &up, const Tensor &down, const Tensor &bg, const Tensor &bu,
                   const Tensor &bd, int64_t activation, bool keep) {
  DeviceGuard on_device(x.device());
  butd_gated_ffn_args a = ffn_args(x, gate, up, down, activation);
  a.b_gate = ptr(bg);
  a.b_up = ptr(bu);
  a.b_down = ptr(bd);
  FfnOut o;
  o.h = at::empty({a.rows, a.ld_h}, x.options());
  o.y = at::empty({a.rows, (long)a.width}, x.options());
  if (keep) {
    o.ab = at::empty({2, a.rows, a.ld_h}, x.options().dtype(at::kFloat));
    a.a = o.ab.data_ptr<float>();
    a.b = a.a ? a.a + a.rows * a.ld_h : nullptr;
  }
  a.h = ptr(o.h);
  a.y = ptr(o.y);
  a.ld_y = a.width;
  ffn_run(a, x, false);
  return o;
}

struct GatedFfnNode : torch::autograd::Function<GatedFfnNode> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const Tensor &w_down,
                        const Maybe &b_gate, const Maybe &b_up, const Maybe &b_down, int64_t activation) {
    const Tensor xr = rows_of(x), gate = rows_of(w_gate), up = rows_of(w_up), down = rows_of(w_down);
    FfnOut o = ffn_forward(xr, gate, up, down, contiguous(value(b_gate)), contiguous(value(b_up)), contiguous(value(b_down)),
                           activation, true);
    ctx->save_for_backward({xr, gate, up, down, o.h, o.ab});
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["shape"] = x.sizes();
    ctx->saved_data["biases"] = (int64_t)((b_gate.has_value() ? 1 : 0) | (b_up.has_value() ? 2 : 0) | (b_down.has_value() ? 4 : 0));
    return o.y.view(x.sizes());
  }
  static variable_list backward(AutogradContext *ctx, variable_list dys) {
    variable_list grads(8);                              // one an argument of forward
    if (!dys[0].defined()) return grads;
    {
      const variable_list saved = ctx->get_saved_variables();
      const Tensor &x = saved[0], &gate = saved[1], &up = saved[2], &down = saved[3], &h = saved[4], &ab = saved[5];
      DeviceGuard on_device(x.device());
      at::AutoGradMode off(false);
      const Tensor dy = rows_of(dys[0]);
      butd_gated_ffn_args a = ffn_args(x, gate, up, down, ctx->saved_data["activation"].toInt());
      a.h = ptr(h);
      a.a = ab.data_ptr<float>();
      a.b = a.a ? a.a + a.rows * a.ld_h : nullptr;
      a.dy = ptr(dy);
      a.ld_dy = ld_of(dy);
      a.ld_dx = a.width;
      const int64_t biases = ctx->saved_data["biases"].toInt();
      size_t edge = 0;
      const long E = a.width, F = a.hidden;
      const std::vector<std::vector<int64_t>> shapes = {{a.rows, E}, {F, E}, {F, E}, {E, F}, {F}, {F}, {E}};
      void **const out[7] = {&a.dx, &a.dw_gate, &a.dw_up, &a.dw_down, &a.db_gate, &a.db_up, &a.db_down};
      for (int i = 0; i < 7; ++i) {
        if (i >= 4 && !(biases >> (i - 4) & 1)) continue;  // (an absent bias has no edge)
        if (!ctx->needs_input_grad(edge++)) continue;
        grads[i] = at::empty(shapes[i], x.options());
        *out[i] = ptr(grads[i]);
      }
      ffn_run(a, x, true);
      if (grads[0].defined()) grads[0] = grads[0].view(ctx->saved_data["shape"].toIntVector());
    }
    seal(grads, "gated_ffn");
    return grads;
  }
};

// (grad: of the call's own tensors, where gated_ffn has looked at them already)
Tensor gated_ffn_of(const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const Tensor &w_down, const Maybe &b_gate,
                    const Maybe &b_up, const Maybe &b_down, int64_t activation, std::optional<bool> grad) {
  no_tracing("gated_ffn");
  TORCH_CHECK(x.dim() >= 1 && w_gate.dim() == 2, "gated_ffn: x must be (..., width) and w_gate (hidden, width)");
  const int64_t hidden = w_gate.size(0), width = w_gate.size(1);
  TORCH_CHECK(width >= 1 && hidden >= 1, "gated_ffn: width and hidden must be at least 1");
  TORCH_CHECK(dtype_of(x.scalar_type()) >= 0, "gated_ffn: ", x.scalar_type(), " is not served (float32, bfloat16, float16)");
  TORCH_CHECK(x.size(-1) == width, "gated_ffn: x must be (..., ", width, "), is ", python_shape(x.sizes()));
  const auto need = [&](const char *name, const Tensor &t, at::IntArrayRef shape) {
    TORCH_CHECK(t.sizes() == shape, "gated_ffn: ", name, " must be ", python_shape(shape), ", is ", python_shape(t.sizes()));
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), "gated_ffn: ", name, " must be ", python_name(x.scalar_type()), " as x is, is ",
                python_name(t.scalar_type()));
    TORCH_CHECK(t.device() == x.device(), "gated_ffn: ", name, " must be on ", x.device());
  };
  need("w_gate", w_gate, {hidden, width});
  need("w_up", w_up, {hidden, width});
  need("w_down", w_down, {width, hidden});
  if (b_gate.has_value()) need("b_gate", *b_gate, {hidden});
  if (b_up.has_value()) need("b_up", *b_up, {hidden});
  if (b_down.has_value()) need("b_down", *b_down, {width});
  TORCH_CHECK(x.is_cuda(), "CPU not supported");
  TORCH_CHECK(x.numel() / width <= 1L << 27, "gated_ffn: at most 2^27 rows");
  const Tensor bg = value(b_gate), bu = value(b_up), bd = value(b_down);
  if (grad.has_value() ? *grad : wants_grad({x, w_gate, w_up, w_down, bg, bu, bd}, "gated_ffn"))
    return GatedFfnNode::apply(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation);
  return ffn_forward(rows_of(x), rows_of(w_gate), rows_of(w_up), rows_of(w_down), contiguous(bg), contiguous(bu), contiguous(bd),
                     activation, false)
      .y.view(x.sizes());
}

Tensor gated_ffn(const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const Tensor &w_down, const Maybe &b_gate,
                 const Maybe &b_up, const Maybe &b_down, int64_t activation) {
  if (!x.is_cuda() || !at::autocast::is_autocast_enabled(at::kCUDA))
    return gated_ffn_of(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, std::nullopt);
  // under autocast every operand goes to the type that linear layers take there
  const at::ScalarType type = at::autocast::get_autocast_dtype(at::kCUDA);
  const auto cast = [&](const Tensor &t) { return t.is_cuda() && dtype_of(t.scalar_type()) >= 0 ? t.to(type) : t; };
  const auto cast_maybe = [&](const Maybe &t) { return t.has_value() ? Maybe(cast(*t)) : t; };
  const bool grad = wants_grad({x, w_gate, w_up, w_down, value(b_gate), value(b_up), value(b_down)}, "gated_ffn");
  return gated_ffn_of(cast(x), cast(w_gate), cast(w_up), cast(w_down), cast_maybe(b_gate), cast_maybe(b_up), cast_maybe(b_down),
                      activation, grad);
}

// ---- norms around a block ---------------------------------------------------------------------------------------------------
struct NormConfig {
  int64_t post_kind, pre_kind, gate_kind, per_sample;
  double post_eps, pre_eps, scale;
};

butd_residual_norm_args norm_args(const Tensor &x, const Tensor &residual, const Tensor &gate, const Tensor &w1, const Tensor &b1,
                                  const Tensor &w2, const Tensor &b2, const NormConfig &c) {
  butd_residual_norm_args a{};
  const auto dtype = [&](const Tensor &t, const Tensor &u) {
    return dtype_of(t.defined() ? t.scalar_type() : u.defined() ? u.scalar_type() : x.scalar_type());
  };
  a.x_dtype = dtype_of(x.scalar_type());
  a.stream_dtype = residual.defined() ? dtype_of(residual.scalar_type()) : a.x_dtype;
  a.post_kind = (int)c.post_kind;
  a.pre_kind = (int)c.pre_kind;
  a.gate_kind = (int)c.gate_kind;
  a.post_dtype = dtype(w1, b1);
  a.pre_dtype = dtype(w2, b2);
  a.gate_dtype = dtype(gate, gate);
  a.cols = (int)x.size(-1);
  a.rows = x.numel() / a.cols;
  a.rows_per_sample = c.per_sample;
  a.residual_scale = (float)c.scale;
  a.post_eps = (float)c.post_eps;
  a.pre_eps = (float)c.pre_eps;
  a.x = ptr(x);
  a.residual = ptr(residual);
  a.gate = ptr(gate);
  a.post_weight = ptr(w1);
  a.post_bias = ptr(b1);
  a.pre_weight = ptr(w2);
  a.pre_bias = ptr(b2);
  return a;
}

struct NormOut {
  Tensor stream, normed, stats;
};
// without residual, gate and post norm the stream is x itself: not written again
NormOut norm_forward(const Tensor &x, const Tensor &residual, const Tensor &gate, const Tensor &w1, const Tensor &b1, const Tensor &w2,
                     const Tensor &b2, const NormConfig &c, bool keep) {
  DeviceGuard on_device(x.device());
  butd_residual_norm_args a = norm_args(x, residual, gate, w1, b1, w2, b2, c);
  NormOut o;
  if (residual.defined() || gate.defined() || c.post_kind)
    o.stream = at::empty(x.sizes(), residual.defined() ? residual.options() : x.options());
  if (c.pre_kind) o.normed = at::empty(x.sizes(), x.options());
  if (keep) o.stats = at::empty({4, a.rows}, x.options().dtype(at::kFloat));
  a.stream = ptr(o.stream);
  a.normed = ptr(o.normed);
  a.stats = (float *)ptr(o.stats);
  ok(butd_residual_norm_fwd(&a, stream_of(x)), "butd_residual_norm_fwd");
  return o;
}

struct ResidualNormNode : torch::autograd::Function<ResidualNormNode> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Maybe &residual, const Maybe &gate, const Maybe &w1,
                               const Maybe &b1, const Maybe &w2, const Maybe &b2, int64_t post_kind, int64_t pre_kind,
                               int64_t gate_kind, int64_t per_sample, double post_eps, double pre_eps, double scale) {
    const NormConfig c{post_kind, pre_kind, gate_kind, per_sample, post_eps, pre_eps, scale};
    variable_list t = {x.contiguous()};
    int64_t there = 0;
    int bit = 0;
    for (const Maybe *m : {&residual, &gate, &w1, &b1, &w2, &b2}) {
      t.push_back(contiguous(value(*m)));
      there |= (int64_t)m->has_value() << bit++;
    }
    NormOut o = norm_forward(t[0], t[1], t[2], t[3], t[4], t[5], t[6], c, true);
    t.push_back(o.stats);
    ctx->save_for_backward(t);
    ctx->set_materialize_grads(false);
    ctx->saved_data["there"] = there;
    ctx->saved_data["kinds"] = std::vector<int64_t>{post_kind, pre_kind, gate_kind, per_sample};
    ctx->saved_data["reals"] = std::vector<double>{post_eps, pre_eps, scale};
    variable_list out;
    if (o.stream.defined()) out.push_back(o.stream);
    if (o.normed.defined()) out.push_back(o.normed);
    ctx->saved_data["stream"] = o.stream.defined();
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list ds) {
    variable_list grads(14);                             // one an argument of forward
    const bool stream = ctx->saved_data["stream"].toBool();
    Tensor d_stream = stream ? ds[0] : Tensor(), d_normed = stream ? (ds.size() > 1 ? ds[1] : Tensor()) : ds[0];
    if (!d_stream.defined() && !d_normed.defined()) return grads;
    {
      const variable_list t = ctx->get_saved_variables();
      const Tensor &x = t[0];
      DeviceGuard on_device(x.device());
      at::AutoGradMode off(false);
      const auto k = ctx->saved_data["kinds"].toIntVector();
      const auto r = ctx->saved_data["reals"].toDoubleVector();
      const int64_t there = ctx->saved_data["there"].toInt();
      butd_residual_norm_args a = norm_args(x, t[1], t[2], t[3], t[4], t[5], t[6], NormConfig{k[0], k[1], k[2], k[3], r[0], r[1], r[2]});
      d_stream = contiguous(d_stream);
      d_normed = contiguous(d_normed);
      a.stats = (float *)ptr(t[7]);
      a.d_stream = ptr(d_stream);
      a.d_normed = ptr(d_normed);
      void **const out[7] = {&a.d_x, &a.d_residual, &a.d_gate, &a.d_post_weight, &a.d_post_bias, &a.d_pre_weight, &a.d_pre_bias};
      size_t edge = 0;
      for (int i = 0; i < 7; ++i) {
        if (i && !(there >> (i - 1) & 1)) continue;      // (an absent tensor has no edge)
        if (!ctx->needs_input_grad(edge++)) continue;
        // (no rows: the sums are zeros, a gate per sample's among them)
        grads[i] = a.rows ? at::empty(t[i].sizes(), t[i].options()) : at::zeros(t[i].sizes(), t[i].options());
        *out[i] = ptr(grads[i]);
      }
      const long need = butd_residual_norm_bwd_workspace(&a);
      ok(need < 0 ? -need : 0, "butd_residual_norm_bwd");
      Tensor ws;
      if (need) ws = at::empty({need}, x.options().dtype(at::kByte));
      ok(butd_residual_norm_bwd(&a, ptr(ws), need, stream_of(x)), "butd_residual_norm_bwd");
    }
    seal(grads, "residual_norm");
    return grads;
  }
};

// kinds: BUTD_NORM_* of the two norms.  -> (stream or None, normed or None)
std::tuple<Maybe, Maybe> residual_norm(const Tensor &x, const Maybe &residual, const Maybe &gate, const Maybe &w1, const Maybe &b1,
                                       const Maybe &w2, const Maybe &b2, int64_t post_kind, int64_t pre_kind, double post_eps,
                                       double pre_eps, double scale) {
  no_tracing("residual_norm");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, "residual_norm: x must be (..., cols) with cols >= 1");
  TORCH_CHECK(dtype_of(x.scalar_type()) >= 0, "residual_norm: ", x.scalar_type(), " is not served (float32, bfloat16, float16)");
  const int64_t cols = x.size(-1);
  TORCH_CHECK(cols <= BUTD_NORM_MAX_COLS, "residual_norm: rows of up to ", BUTD_NORM_MAX_COLS, " elements, x has ", cols);
  TORCH_CHECK(x.numel() / cols <= INT_MAX, "residual_norm: at most 2^31 - 1 rows");
  const auto typed = [&](const char *name, const Tensor &t) {
    TORCH_CHECK(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, "residual_norm: ", name, " must be ",
                python_name(x.scalar_type()), " or float32, is ", python_name(t.scalar_type()));
    TORCH_CHECK(t.device() == x.device(), "residual_norm: ", name, " must be on ", x.device());
  };
  if (residual.has_value()) {
    TORCH_CHECK(residual->sizes() == x.sizes(), "residual_norm: residual must be ", python_shape(x.sizes()), ", is ",
                python_shape(residual->sizes()));
    typed("residual", *residual);
  }
  const struct { const char *name; const Maybe &weight, &bias; } norms[2] = {{"post_norm", w1, b1}, {"pre_norm", w2, b2}};
  for (const auto &n : norms) {
    for (const Maybe *p : {&n.weight, &n.bias})
      if (p->has_value()) {
        TORCH_CHECK((*p)->dim() == 1 && (*p)->size(0) == cols, "residual_norm: ", n.name, " must normalise (", cols, ",)");
        typed((std::string(n.name) + (p == &n.weight ? ".weight" : ".bias")).c_str(), **p);
      }
    TORCH_CHECK(!n.weight.has_value() || !n.bias.has_value() || n.weight->scalar_type() == n.bias->scalar_type(), "residual_norm: ",
                n.name, "'s weight and bias must have one dtype");
  }
  int64_t gate_kind = BUTD_GATE_NONE, per_sample = 1;
  if (gate.has_value()) {
    const at::IntArrayRef s = gate->sizes();
    if (s.size() == 1 && s[0] == cols) gate_kind = BUTD_GATE_CHANNEL;
    else if (s == x.sizes()) gate_kind = BUTD_GATE_ELEMENT;
    else if (x.dim() == 3 && s.size() >= 2 && s.size() <= 3 && s[0] == x.size(0) && s.back() == cols && (s.size() == 2 || s[1] == 1))
      gate_kind = BUTD_GATE_SAMPLE;
    TORCH_CHECK(gate_kind != BUTD_GATE_NONE, "residual_norm: gate must be (", cols, ",), of x's shape, or (batch, ", cols,
                ") with x (batch, length, ", cols, "); is ", python_shape(s), " with x ", python_shape(x.sizes()));
    typed("gate", *gate);
    if (gate_kind == BUTD_GATE_SAMPLE) per_sample = x.size(1);
  }
  TORCH_CHECK(x.is_cuda(), "CPU not supported");
  const Tensor r = value(residual), g = value(gate), p1 = value(w1), q1 = value(b1), p2 = value(w2), q2 = value(b2);
  const bool has_stream = r.defined() || g.defined() || post_kind;
  if (!has_stream && !pre_kind) return {Maybe(), Maybe()};
  if (wants_grad({x, r, g, p1, q1, p2, q2}, "residual_norm")) {
    variable_list out = ResidualNormNode::apply(x, residual, gate, w1, b1, w2, b2, post_kind, pre_kind, gate_kind, per_sample,
                                                post_eps, pre_eps, scale);
    return {has_stream ? Maybe(out[0]) : Maybe(), pre_kind ? Maybe(out.back()) : Maybe()};
  }
  NormOut o = norm_forward(x.contiguous(), contiguous(r), contiguous(g), contiguous(p1), contiguous(q1), contiguous(p2), contiguous(q2),
                           NormConfig{post_kind, pre_kind, gate_kind, per_sample, post_eps, pre_eps, scale}, false);
  return {has_stream ? Maybe(o.stream) : Maybe(), pre_kind ? Maybe(o.normed) : Maybe()};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  // (the argument structs go by pointer: their layout has to be the library's)
  TORCH_CHECK(butd_gated_ffn_args_size() == (long)sizeof(butd_gated_ffn_args) &&
                  butd_residual_norm_args_size() == (long)sizeof(butd_residual_norm_args),
              "butd_blocks_aten and libbutd_detr_hip.so were built from different headers: python -m butd_detr_amd.binding.build");
  m.def("gated_ffn", &gated_ffn, py::call_guard<py::gil_scoped_release>());
  m.def("residual_norm", &residual_norm, py::call_guard<py::gil_scoped_release>());
}
