// ops_mlp.cpp -- the host side of the node-wise MLP operators (shadow_gnn_amd/ops_mlp.py): argument checks, autograd nodes and the
// calls of the C entries (include/shadow_hip.h).  Small calls are bound by the host, and a backward pass written in Python also waits
// for the interpreter lock in autograd's thread: forward + backward of a layer norm of 64 x 64 takes 33 to 68 us here, 70 to 134 us so
// (the spread is autograd's thread being woken).
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <string>

#include "shadow_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
typedef std::optional<Tensor> OptTensor;

void check(int rc) {
  TORCH_CHECK(rc == SG_OK, "libshadow_hip status ", rc, ": ", sg_last_error());
}

int dtype_of(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return SL_F32;
    case at::kBFloat16: return SL_BF16;
    case at::kHalf: return SL_F16;
    default: return -1;
  }
}

std::string shape_of(const Tensor &t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); i++) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
std::string say(const Tensor &t) { return std::string(c10::toString(t.scalar_type())) + " " + shape_of(t); }

[[noreturn]] void type_error(const std::string &m) { throw py::type_error(m); }
[[noreturn]] void value_error(const std::string &m) { throw py::value_error(m); }

void float_rows(const char *name, const Tensor &t) {
  if (dtype_of(t) < 0) type_error(std::string(name) + ": " + say(t) + " (float32, bfloat16 or float16)");
  if (t.dim() < 1) value_error(std::string(name) + ": a tensor of rows is needed");
}

void on_device(const Tensor &t) {
  TORCH_CHECK(t.is_cuda(), "shadow_gnn_amd ops need tensors on a ROCm device (no CPU fallback)");
}
void one_device(const Tensor &t) { on_device(t); }
template <typename... More>
void one_device(const Tensor &t, const OptTensor &o, const More &...more) {
  on_device(t);
  if (o) {
    on_device(*o);
    if (o->device() != t.device()) value_error("operands on " + t.device().str() + " and " + o->device().str());
  }
  one_device(t, more...);
}

// Forward-mode derivatives are not provided: a tangent, of an input or of a gradient, is an error, not a silent zero.
void no_tangents(const char *) {}
template <typename... More>
void no_tangents(const char *name, const OptTensor &t, const More &...more) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->defined() || !t->_fw_grad(0).defined(), name, ": forward-mode derivatives are not provided");
  no_tangents(name, more...);
}

bool needs_grad(const Tensor &t) { return t.requires_grad(); }
bool needs_grad(const OptTensor &t) { return t && t->requires_grad(); }
template <typename... Ts>
bool any_grad(const Ts &...ts) { return at::GradMode::is_enabled() && (needs_grad(ts) || ...); }

// the tensor whose memory holds its values (the imaginary part of a conjugate is a view that negates)
Tensor in_memory(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }

// [rows, width] with unit stride along the row and a pitch of at least the width (copied if it has neither)
struct Rows {
  Tensor keep;
  void *p = nullptr;
  int64_t n = 0, F = 0, ld = 0;
};
Rows rows_of(const Tensor &given) {
  const Tensor t = in_memory(given);
  Rows r;
  r.F = t.size(-1);
  r.n = 1;
  for (int64_t i = 0; i + 1 < t.dim(); i++) r.n *= t.size(i);
  r.keep = t.dim() == 2 || t.is_contiguous() ? t : t.reshape({r.n, r.F});
  if (r.keep.is_contiguous()) {
    r.ld = r.F;
  } else {                                     // (two dimensions here)
    r.ld = r.keep.stride(0);
    if ((r.keep.stride(1) != 1 && r.F > 1) || r.ld < r.F) { r.keep = r.keep.contiguous(); r.ld = r.F; }
  }
  r.p = r.keep.data_ptr();
  return r;
}
Rows rows_of(const OptTensor &t) { return t ? rows_of(*t) : Rows(); }
void *ptr(const OptTensor &t) { return t ? t->data_ptr() : nullptr; }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// the device of a launch made current, and torch's current stream on it
struct On {
  c10::DeviceGuard guard;
  void *stream;
  explicit On(const Tensor &t) : guard(t.device()), stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream()) {}
};

uint32_t u32(const char *name, int64_t v) {
  if (v > 0xFFFFFFFFll) value_error(std::string(name) + ": " + std::to_string(v) + " rows");
  return (uint32_t)v;
}

Tensor like(const Tensor &x, at::IntArrayRef shape) { return at::empty(shape, x.options().requires_grad(false)); }
Tensor like(const Tensor &x, at::IntArrayRef shape, at::ScalarType t) { return at::empty(shape, x.options().dtype(t).requires_grad(false)); }

// A gradient of these operators is not differentiable itself: with create_graph its own backward pass is an error, not a silent zero.
// Its inputs are x and dy, and what a gradient depends on where both of them are constants (w, b: they stand in act'(z)).
struct Once : public Function<Once> {
  static Tensor forward(AutogradContext *, const Tensor &g, const Tensor &, const Tensor &, const OptTensor &, const OptTensor &) { return g.view_as(g); }
  static variable_list backward(AutogradContext *, const variable_list &) {
    TORCH_CHECK(false, "the operators of shadow_gnn_amd.ops_mlp are differentiable once");
  }
};
void once(variable_list &grads, const Tensor &x, const Tensor &dy, const OptTensor &w = {}, const OptTensor &b = {}) {
  if (!at::GradMode::is_enabled()) return;
  for (Tensor &g : grads)
    if (g.defined()) g = Once::apply(g, x, dy, w, b);
}

// ------------------------------------------------------------------------------------------------ layer norm
Tensor ln_forward(const Tensor &x, const OptTensor &scale, const OptTensor &offset, double eps, Tensor *stats) {
  const Rows r = rows_of(x);
  const uint32_t n = u32("layer_norm", r.n);
  Tensor y = like(x, x.sizes());
  if (stats) *stats = like(x, {r.n, 2}, at::kFloat);
  if (n) {
    const On on(x);
    const OptTensor &w = scale ? scale : offset;
    check(sl_layer_norm_fwd(dtype_of(x), w ? dtype_of(*w) : SL_F32, r.p, r.ld, ptr(scale), ptr(offset), n, (uint32_t)r.F, (float)eps, y.data_ptr(), r.F,
                            stats ? (float *)stats->data_ptr() : nullptr, on.stream));
  }
  return y;
}

struct LayerNorm : public Function<LayerNorm> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &scale, const OptTensor &offset, double eps) {
    Tensor stats;
    Tensor y = ln_forward(x, scale, offset, eps, &stats);
    ctx->save_for_backward({x, scale.value_or(Tensor()), offset.value_or(Tensor()), stats});
    return y;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &dys) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &scale = saved[1], &offset = saved[2], &stats = saved[3], &dy = dys[0];
    no_tangents("layer_norm", dy);
    size_t edge = 0;
    const bool need_x = ctx->needs_input_grad(edge++), need_s = scale.defined() && ctx->needs_input_grad(edge++), need_o = offset.defined() && ctx->needs_input_grad(edge++);
    variable_list out(4);
    {
      at::NoGradGuard no_grad;
      const Rows r = rows_of(x), d = rows_of(dy);
      const uint32_t n = (uint32_t)r.n, F = (uint32_t)r.F;
      if (need_x) out[0] = like(x, x.sizes());
      if (need_s) out[1] = like(scale, scale.sizes());
      if (need_o) out[2] = like(offset, offset.sizes());
      Tensor part;
      const int64_t floats = need_s || need_o ? (int64_t)sl_layer_norm_partial_floats(n, F) : 0;
      if (floats) part = like(x, {floats}, at::kFloat);
      const Tensor &w = scale.defined() ? scale : offset;
      const On on(x);
      check(sl_layer_norm_bwd(dtype_of(x), w.defined() ? dtype_of(w) : SL_F32, r.p, r.ld, d.p, d.ld, ptr(scale), (const float *)stats.data_ptr(), n, F,
                              ptr(out[0]), r.F, ptr(out[1]), ptr(out[2]), (float *)ptr(part), on.stream));
    }
    once(out, x, dy);
    return out;
  }
};

Tensor layer_norm(const Tensor &x, const OptTensor &scale, const OptTensor &offset, double eps) {
  float_rows("layer_norm", x);
  const int64_t F = x.size(-1);
  if (F < 1 || F > 16384) value_error("layer_norm: rows of " + std::to_string(F) + " elements (1 to 16384)");
  if (!(eps >= 0.0)) value_error("layer_norm: eps " + std::to_string(eps));
  for (const OptTensor *t : {&scale, &offset})
    if (*t) {
      if ((*t)->scalar_type() != x.scalar_type() && (*t)->scalar_type() != at::kFloat) type_error("layer_norm: scale / offset " + say(**t) + " for rows of " + say(x));
      if ((*t)->dim() != 1 || (*t)->size(0) != F) value_error("layer_norm: scale / offset " + say(**t) + " for rows of " + std::to_string(F));
    }
  if (scale && offset && scale->scalar_type() != offset->scalar_type()) type_error("layer_norm: scale " + say(*scale) + " and offset " + say(*offset));
  no_tangents("layer_norm", x, scale, offset);
  one_device(x, scale, offset);
  const OptTensor s = scale ? OptTensor(in_memory(*scale).contiguous()) : scale, o = offset ? OptTensor(in_memory(*offset).contiguous()) : offset;
  if (any_grad(x, s, o)) return LayerNorm::apply(x, s, o, eps);
  return ln_forward(x, s, o, eps, nullptr);
}

// ------------------------------------------------------------------------------------------------ dropout
Tensor drop(const Tensor &x, double p, uint64_t seed, const OptTensor &d_seed, const OptTensor &residual) {
  const Rows r = rows_of(x), q = rows_of(residual);
  Tensor y = like(x, x.sizes());
  if (r.n && r.F) {
    const On on(x);
    check(sl_dropout(dtype_of(x), r.p, r.ld, q.p, q.ld, (uint64_t)r.n, u32("dropout", r.F), (float)p, seed, (const int64_t *)ptr(d_seed), y.data_ptr(), r.F, on.stream));
  }
  return y;
}

struct Dropout : public Function<Dropout> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &residual, const OptTensor &d_seed, double p, int64_t seed) {
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["residual"] = residual.has_value();
    ctx->save_for_backward({d_seed.value_or(Tensor())});
    return drop(x, p, (uint64_t)seed, d_seed, residual);
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &dys) {
    const Tensor d_seed = ctx->get_saved_variables()[0], &dy = dys[0];
    no_tangents("dropout", dy);
    const bool residual = ctx->saved_data["residual"].toBool();
    variable_list out(5);
    if (ctx->needs_input_grad(0)) {
      at::NoGradGuard no_grad;
      out[0] = drop(dy, ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(), d_seed.defined() ? OptTensor(d_seed) : OptTensor(), OptTensor());
    }
    once(out, dy, dy);
    if (residual && ctx->needs_input_grad(1)) out[1] = dy;
    return out;
  }
};

Tensor dropout(const Tensor &x, double p, uint64_t seed, const OptTensor &d_seed, const OptTensor &residual) {
  float_rows("dropout", x);
  if (!(p >= 0.0 && p < 1.0)) value_error("dropout: probability " + std::to_string(p) + " (0 <= p < 1)");
  if (!((float)p < 1.0f)) value_error("dropout: the probability rounds to 1 in fp32");
  if (residual && (residual->sizes() != x.sizes() || residual->scalar_type() != x.scalar_type())) value_error("dropout: residual " + say(*residual) + " for x " + say(x));
  if (d_seed && (d_seed->scalar_type() != at::kLong || d_seed->numel() != 1)) value_error("dropout: a seed tensor is one int64");
  no_tangents("dropout", x, residual);
  one_device(x, residual, d_seed);
  if (any_grad(x, residual)) return Dropout::apply(x, residual, d_seed, p, (int64_t)seed);
  return drop(x, p, seed, d_seed, residual);
}

// ------------------------------------------------------------------------------------------------ the 16-bit Linear
std::vector<int64_t> out_shape(const Tensor &x, int64_t N) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = N;
  return s;
}

Tensor lin_forward(const Tensor &x, const Tensor &W, const OptTensor &b, const OptTensor &residual, int act, Tensor *kept) {
  const Rows r = rows_of(x), w = rows_of(W), q = rows_of(residual);
  const uint32_t M = u32("linear_act", r.n), N = (uint32_t)w.n, K = (uint32_t)w.F;
  Tensor y = like(x, out_shape(x, N));
  if (kept) *kept = like(x, {(int64_t)sl_linear16_kept_bytes(act, M, N) + 16}, at::kByte);
  if (M) {
    const On on(x);
    check(sl_linear16_fwd(dtype_of(x), r.p, r.ld, w.p, w.ld, ptr(b), b && b->scalar_type() == at::kFloat, q.p, q.ld, M, N, K, act, y.data_ptr(), N,
                          kept ? kept->data_ptr() : nullptr, on.stream));
  }
  return y;
}

struct LinearAct : public Function<LinearAct> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &W, const OptTensor &b, const OptTensor &residual, int64_t act) {
    Tensor kept;
    Tensor y = lin_forward(x, W, b, residual, (int)act, act ? &kept : nullptr);
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = b ? (int64_t)b->scalar_type() : (int64_t)-1;
    ctx->saved_data["residual"] = residual.has_value();
    // (for once() alone, which reads no value of it: not a saved tensor, which must not change before the backward pass)
    if (act && needs_grad(b)) ctx->saved_data["b"] = *b;
    ctx->save_for_backward({x, W, kept});
    return y;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &dys) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &W = saved[1], &kept = saved[2], &dy = dys[0];
    no_tangents("linear_act", dy);
    const int act = (int)ctx->saved_data["act"].toInt();
    const int64_t bias = ctx->saved_data["bias"].toInt();
    size_t edge = 2;
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = bias >= 0 && ctx->needs_input_grad(edge++),
               need_r = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(edge);
    variable_list out(5);
    if (need_x || need_w || need_b) {
      at::NoGradGuard no_grad;
      const Rows r = rows_of(x), w = rows_of(W), d = rows_of(dy);
      const uint32_t M = (uint32_t)r.n, N = (uint32_t)w.n, K = (uint32_t)w.F;
      if (need_x) out[0] = like(x, x.sizes());
      Tensor dW;
      if (need_w || need_b) dW = like(x, {(int64_t)N, (int64_t)K});
      if (need_b) out[2] = like(x, {(int64_t)N}, (at::ScalarType)bias);
      const Tensor ws = like(x, {(int64_t)sl_linear16_bwd_scratch_bytes_for(act, r.p, r.ld, w.ld, d.p, d.ld, M, N, K, need_x, need_w || need_b) + 16}, at::kByte);
      const On on(x);
      check(sl_linear16_bwd(dtype_of(x), r.p, r.ld, w.p, w.ld, d.p, d.ld, ptr(kept), M, N, K, act, ptr(out[0]), K, ptr(dW), K, ptr(out[2]),
                            bias == (int64_t)at::kFloat, ws.data_ptr(), on.stream));
      if (need_w) out[1] = dW;
    }
    const auto b = ctx->saved_data.find("b");
    once(out, x, dy, act ? OptTensor(W) : OptTensor(), b != ctx->saved_data.end() ? OptTensor(b->second.toTensor()) : OptTensor());
    if (need_r) out[3] = dy;
    return out;
  }
};

Tensor linear_act(const Tensor &x, const Tensor &W, const OptTensor &b, int64_t act, const OptTensor &residual) {
  if (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kHalf)
    type_error("linear_act: " + say(x) + " (bfloat16 or float16; fp32 products are ops.linear / ops.linear_act_norm)");
  float_rows("linear_act", x);
  if (W.dim() != 2 || W.size(1) != x.size(-1) || W.scalar_type() != x.scalar_type() || W.size(0) < 1 || W.size(1) < 1 || W.size(0) > (1 << 24) || W.size(1) > (1 << 24))
    value_error("linear_act: weight " + say(W) + " for x " + say(x));
  const int64_t N = W.size(0);
  if (b && (b->dim() != 1 || b->size(0) != N || (b->scalar_type() != at::kFloat && b->scalar_type() != x.scalar_type())))
    value_error("linear_act: bias " + say(*b) + " for " + std::to_string(N) + " outputs of " + say(x));
  if (residual && (residual->scalar_type() != x.scalar_type() || residual->sizes() != at::IntArrayRef(out_shape(x, N))))
    value_error("linear_act: residual " + say(*residual) + " for " + std::to_string(N) + " outputs of x " + say(x));
  no_tangents("linear_act", x, W, b, residual);
  one_device(x, OptTensor(W), b, residual);
  const OptTensor bc = b ? OptTensor(in_memory(*b).contiguous()) : b;
  if (any_grad(x, W, bc, residual)) return LinearAct::apply(x, W, bc, residual, act);
  return lin_forward(x, W, bc, residual, (int)act, nullptr);
}

// ------------------------------------------------------------------------------------------------ log probabilities of labels
variable_list lp_forward(const Tensor &x, const Tensor &label, int64_t k) {
  const Rows r = rows_of(x);
  const uint32_t n = u32("label_logprobs", r.n), C = u32("label_logprobs", r.F);
  const at::IntArrayRef lead = x.sizes().slice(0, x.dim() - 1);
  std::vector<int64_t> tops = lead.vec();
  tops.push_back(k);
  variable_list o = {like(x, lead, at::kFloat), like(x, lead, at::kFloat), like(x, tops, at::kFloat), like(x, tops, at::kLong), like(x, {r.n, 2}, at::kFloat)};
  if (n) {
    const size_t need = sl_label_logprobs_scratch_bytes(dtype_of(x), n, C, (uint32_t)k);
    Tensor ws;
    if (need) ws = like(x, {(int64_t)need}, at::kByte);
    const On on(x);
    check(sl_label_logprobs_fwd(dtype_of(x), r.p, r.ld, label.data_ptr(), label.scalar_type() == at::kLong, n, C, (uint32_t)k, (float *)o[0].data_ptr(),
                                (float *)o[1].data_ptr(), (float *)o[4].data_ptr(), (float *)o[2].data_ptr(), (int64_t *)o[3].data_ptr(), ptr(ws), on.stream));
  }
  return o;
}

struct LabelLogprobs : public Function<LabelLogprobs> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &label, int64_t k) {
    variable_list o = lp_forward(x, label, k);
    ctx->saved_data["k"] = k;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({o[3]});
    ctx->save_for_backward({x, label, o[1], o[3], o[4]});
    o.pop_back();
    return o;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &dys) {
    variable_list out(3);
    if (!dys[0].defined() && !dys[1].defined() && !dys[2].defined()) return out;
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &label = saved[1], &ent = saved[2], &idx = saved[3], &stat = saved[4];
    no_tangents("label_logprobs", dys[0], dys[1], dys[2]);
    const uint32_t k = (uint32_t)ctx->saved_data["k"].toInt();
    {
      at::NoGradGuard no_grad;
      Tensor g[3];
      for (int i = 0; i < 3; i++)
        if (dys[i].defined() && dys[i].numel()) g[i] = in_memory(dys[i]).contiguous();
      const Rows r = rows_of(x);
      out[0] = like(x, x.sizes());
      if (r.n) {
        const On on(x);
        check(sl_label_logprobs_bwd(dtype_of(x), r.p, r.ld, label.data_ptr(), label.scalar_type() == at::kLong, (uint32_t)r.n, (uint32_t)r.F, k,
                                    (const float *)stat.data_ptr(), (const float *)ent.data_ptr(), (const int64_t *)idx.data_ptr(), (const float *)ptr(g[0]),
                                    (const float *)ptr(g[1]), (const float *)ptr(g[2]), out[0].data_ptr(), r.F, on.stream));
      }
    }
    once(out, x, dys[0].defined() ? dys[0] : dys[1].defined() ? dys[1] : dys[2]);
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> label_logprobs(const Tensor &x, const Tensor &label, int64_t k) {
  float_rows("label_logprobs", x);
  const int64_t C = x.size(-1);
  if ((label.scalar_type() != at::kInt && label.scalar_type() != at::kLong) || label.sizes() != x.sizes().slice(0, x.dim() - 1))
    value_error("label_logprobs: label " + say(label) + " for logits " + say(x));
  if (C < 1 || k < 0 || k > C || k > 64) value_error("label_logprobs: topk " + std::to_string(k) + " of " + std::to_string(C) + " classes (at most 64)");
  no_tangents("label_logprobs", x);
  one_device(x, OptTensor(label));
  const Tensor lab = label.contiguous();
  const variable_list o = any_grad(x) ? LabelLogprobs::apply(x, lab, k) : lp_forward(x, lab, k);
  return {o[0], o[1], o[2], o[3]};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("layer_norm", &layer_norm);
  m.def("dropout", &dropout);
  m.def("linear_act", &linear_act);
  m.def("label_logprobs", &label_logprobs);
  m.def("abi_version", &sg_abi_version);
}
