// The tensor-level calls and autograd nodes of the state-space operators (state_space.py): the short causal convolution, the selective scan
// and the gated group norm.  No arithmetic happens here.  Errors keep the types that torch_ops.cpp gives them.
#include "torch_call.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int float_code(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return RFA_BF16;
  if (t.scalar_type() == at::kHalf) return RFA_F16;
  if (t.scalar_type() == at::kFloat) return RFA_F32;
  raise(PyExc_TypeError, "rfa_b200: unsupported dtype " + dtype_name(t) + " (fp16, bf16 and fp32 only)");
}
void same_dtype(const char* what, const Tensor& x, std::initializer_list<const Tensor*> others) {
  for (const Tensor* t : others)
    if (t->scalar_type() != x.scalar_type())
      raise(PyExc_TypeError, std::string(what) + ": expected tensors of one dtype, got " + dtype_name(x) + " and " + dtype_name(*t));
}
void need_shape(const char* what, const char* name, const Tensor& t, at::IntArrayRef shape) {
  if (t.sizes() != shape) {
    std::string want = "[";
    for (size_t i = 0; i < shape.size(); ++i) want += (i ? ", " : "") + std::to_string(shape[i]);
    raise(PyExc_AssertionError, std::string(what) + ": " + name + " is " + shape_name(t) + ", expected " + want + "]");
  }
}
void need_f32(const char* what, const char* name, const Tensor& t) {
  if (t.scalar_type() != at::kFloat) raise(PyExc_TypeError, std::string(what) + ": " + name + " must be fp32, got " + dtype_name(t));
}
// A gradient that a caller hands in: of the shape that it is the gradient of, and on its device.
void need_grad(const char* what, const char* name, const OptTensor& g, at::IntArrayRef shape, const Tensor& x) {
  if (!g) return;
  need_shape(what, name, *g, shape);
  require_device(x, {&*g});
}
// Activations are taken with any strides but along the channels.
Tensor unit_last(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// A contiguous copy where a tensor is not contiguous or, being a state that kernels take in 16-byte words, not aligned.
Tensor packed(const Tensor& t) {
  Tensor c = t.contiguous();
  return aligned(c) ? c : c.clone();
}
OptTensor packed(const OptTensor& t) { return t ? OptTensor(packed(*t)) : t; }
const void* maybe(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
void* maybe_out(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
const float* maybe_f(const OptTensor& t) { return t ? t->data_ptr<float>() : nullptr; }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor plain(const OptTensor& t) { return t ? *t : Tensor(); }
Tensor scratch(size_t bytes, const Tensor& like) { return fresh({static_cast<int64_t>(std::max<size_t>(bytes, 16))}, like, at::kByte); }
int as_int(const char* what, int64_t n) {
  if (n > INT_MAX) raise(PyExc_ValueError, std::string(what) + ": a size of " + std::to_string(n));
  return static_cast<int>(n);
}
OptTensor mask_of(const char* what, const OptTensor& mask, int64_t B, int64_t T, const Tensor& like) {
  if (!mask) return mask;
  need_shape(what, "key_padding_mask", *mask, {B, T});
  return mask_bytes(mask, B * T, like);
}
// A kernel wrote to it: autograd is to notice where an earlier graph keeps it.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
bool wants(const OptTensor& t) { return t && t->requires_grad(); }
template <class... Ts> bool records(const Ts&... ts) {      // decided in front of a node, whose own forward records nothing
  return at::GradMode::is_enabled() && (wants(OptTensor(ts)) || ...);
}
void once(const char* what) {
  if (at::GradMode::is_enabled()) raise(PyExc_RuntimeError, std::string(what) + ": the backward pass is not differentiable (create_graph)");
}

// ---- convolution ---------------------------------------------------------------------------------------------------------
struct Conv {
  rfa_causal_conv_t c{};
  Tensor x, weight;
  OptTensor bias, state, mask;
  Conv(const char* what, const Tensor& x_, const Tensor& w_, const OptTensor& bias_, const OptTensor& state_, const OptTensor& mask_, bool silu) {
    require_cuda(x_);
    rank(x_, 3);
    rank(w_, 2);
    const int64_t T = x_.size(0), B = x_.size(1), D = x_.size(2), W = w_.size(1);
    c.dtype = float_code(x_);
    same_dtype(what, x_, {&w_, bias_ ? &*bias_ : &x_, state_ ? &*state_ : &x_});
    require_device(x_, {&w_, bias_ ? &*bias_ : &x_, state_ ? &*state_ : &x_});
    need_shape(what, "weight", w_, {D, W});
    if (bias_) need_shape(what, "bias", *bias_, {D});
    if (W < 1 || W > 8) raise(PyExc_ValueError, std::string(what) + ": a window of " + std::to_string(W) + " tokens (1 to 8)");
    if (state_) need_shape(what, "state", *state_, {B, W - 1, D});
    x = unit_last(x_);
    weight = w_.contiguous();
    if (bias_) bias = bias_->contiguous();
    if (state_) state = state_->contiguous();
    mask = mask_of(what, mask_, B, T, x_);
    c.T = T; c.B = as_int(what, B); c.D = as_int(what, D); c.W = static_cast<int>(W);
    c.silu = silu;
    if (empty()) return;                               // empty tensors have no address
    c.x = x.data_ptr(); c.x_t = x.stride(0); c.x_b = x.stride(1);
    c.weight = weight.data_ptr();
    c.bias = maybe(bias);
    c.state_in = W > 1 ? maybe(state) : nullptr;
    c.mask = static_cast<const uint8_t*>(maybe(mask));
  }
  bool empty() const { return c.T == 0 || c.B == 0 || c.D == 0; }
};

// -> y, and where asked the last inputs: in place of `state` where that is asked too
std::tuple<Tensor, OptTensor> causal_conv_fwd(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& state, const OptTensor& mask,
                                              bool silu, bool return_state, bool in_place) {
  Conv v("causal_conv", x, weight, bias, state, mask, silu);
  if (in_place && state && !state->is_contiguous()) raise(PyExc_ValueError, "causal_conv: the state must be contiguous (it is updated in place)");
  Tensor y = fresh(x.sizes(), x, x.scalar_type());
  OptTensor out;
  const int64_t W = weight.size(1);
  if (return_state) {
    const bool here = in_place && state && (v.c.T <= 1 || v.empty());
    out = here ? *state : fresh({x.size(1), W - 1, x.size(2)}, x, x.scalar_type());
    if (v.empty() && !here) state ? out->copy_(*state) : out->zero_();
  }
  if (v.empty()) return {y, in_place && state ? state : out};
  Call c(x);
  check(rfa_causal_conv_fwd(&v.c, y.data_ptr(), out && W > 1 ? out->data_ptr() : nullptr, c.stream), "rfa_causal_conv_fwd");
  if (out && state && out->is_same(*state)) written(*state);
  if (out && in_place && state && !out->is_same(*state)) {
    state->copy_(*out);
    out = state;
  }
  return {y, out};
}

// -> gx, gweight, gbias, gstate
std::tuple<Tensor, OptTensor, OptTensor, OptTensor> causal_conv_bwd(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& state,
                                                                    const OptTensor& mask, bool silu, Tensor g, OptTensor g_state, bool need_weight,
                                                                    bool need_bias, bool need_state) {
  Conv v("causal_conv", x, weight, bias, state, mask, silu);
  need_grad("causal_conv", "g", g, x.sizes(), x);
  need_grad("causal_conv", "g_state", g_state, {x.size(1), weight.size(1) - 1, x.size(2)}, x);
  Tensor gx = fresh(x.sizes(), x, x.scalar_type());
  OptTensor gw, gb, gs;
  need_state = need_state && state;
  if (need_weight) gw = fresh(weight.sizes(), x, x.scalar_type());
  if (need_bias && bias) gb = fresh(bias->sizes(), x, x.scalar_type());
  if (need_state) gs = fresh(state->sizes(), x, x.scalar_type());
  if (v.empty()) {
    if (gw) gw->zero_();
    if (gb) gb->zero_();
    if (gs) g_state ? gs->copy_(*g_state) : gs->zero_();
    return {gx, gw, gb, gs};
  }
  g = unit_last(g.to(x.scalar_type()));
  if (g_state) g_state = g_state->to(x.scalar_type()).contiguous();
  const size_t bytes = gw || gb ? rfa_causal_conv_workspace_bytes(v.c.T, v.c.B, v.c.D, v.c.W) : 0;
  const Tensor ws = scratch(bytes, x);
  const bool kept = weight.size(1) > 1;
  Call c(x);
  check(rfa_causal_conv_bwd(&v.c, g.data_ptr(), g.stride(0), g.stride(1), kept ? maybe(g_state) : nullptr, gx.data_ptr(), maybe_out(gw), maybe_out(gb),
                            kept ? maybe_out(gs) : nullptr, ws.data_ptr(), ws.numel(), c.stream),
        "rfa_causal_conv_bwd");
  return {gx, gw, gb, gs};
}

struct CausalConvBackward : torch::autograd::Function<CausalConvBackward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& state,
                               const OptTensor& mask, bool silu, bool return_state) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, weight, plain(bias), plain(state), plain(mask)});
    ctx->saved_data["silu"] = silu;
    ctx->saved_data["need"] = static_cast<int64_t>(weight.requires_grad() | wants(bias) << 1 | wants(state) << 2);
    auto [y, out] = causal_conv_fwd(x, weight, bias, state, mask, silu, return_state, false);
    if (!return_state) return {y};
    return {y, *out};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    once("causal_conv");
    const variable_list s = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    const Tensor gy = g[0].defined() ? g[0] : at::zeros_like(s[0]);
    auto [gx, gw, gb, gs] = causal_conv_bwd(s[0], s[1], opt(s[2]), opt(s[3]), opt(s[4]), ctx->saved_data["silu"].toBool(), gy,
                                            g.size() > 1 ? opt(g[1]) : OptTensor(), need & 1, need & 2, need & 4);
    return {gx, plain(gw), plain(gb), plain(gs), Tensor(), Tensor(), Tensor()};
  }
};

Tensor causal_conv_node(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& mask, bool silu) {
  if (!records(x, weight, bias)) return std::get<0>(causal_conv_fwd(x, weight, bias, std::nullopt, mask, silu, false, false));
  return CausalConvBackward::apply(x, weight, bias, OptTensor(), mask, silu, false)[0];
}
std::tuple<Tensor, Tensor> incremental_causal_conv_node(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& state,
                                                        const OptTensor& mask, bool silu) {
  if (!records(x, weight, bias, state)) {
    auto [y, out] = causal_conv_fwd(x, weight, bias, state, mask, silu, true, true);
    return {y, *out};
  }
  const variable_list r = CausalConvBackward::apply(x, weight, bias, state, mask, silu, true);
  return {r[0], r[1]};
}

// ---- selective scan ------------------------------------------------------------------------------------------------------
struct Scan {
  rfa_scan_t c{};
  Tensor x, dt, a, b, cc;
  OptTensor d, bias, s, mask;
  Scan(const Tensor& x_, const Tensor& dt_, const Tensor& a_, const Tensor& b_, const Tensor& c_, const OptTensor& d_, const OptTensor& bias_,
       const OptTensor& s_, const OptTensor& mask_, bool softplus) {
    const char* what = "selective_scan";
    require_cuda(x_);
    rank(x_, 3);
    rank(a_, 2);
    rank(b_, 4);
    const int64_t T = x_.size(0), B = x_.size(1), D = x_.size(2), N = a_.size(1), G = b_.size(2);
    c.dtype = float_code(x_);
    same_dtype(what, x_, {&dt_, &b_, &c_});
    require_device(x_, {&dt_, &a_, &b_, &c_, d_ ? &*d_ : &x_, bias_ ? &*bias_ : &x_, s_ ? &*s_ : &x_});
    need_shape(what, "dt", dt_, {T, B, D});
    need_shape(what, "a", a_, {D, N});
    need_shape(what, "b", b_, {T, B, G, N});
    need_shape(what, "c", c_, {T, B, G, N});
    need_f32(what, "a", a_);
    if (d_) { need_f32(what, "d", *d_); need_shape(what, "d", *d_, {D}); }
    if (bias_) { need_f32(what, "dt_bias", *bias_); need_shape(what, "dt_bias", *bias_, {D}); }
    if (s_) { need_f32(what, "s", *s_); need_shape(what, "s", *s_, {B, D, N}); }
    if (N < 1 || N > 64) raise(PyExc_ValueError, "selective_scan: " + std::to_string(N) + " states per channel (1 to 64)");
    if (G < 1 || D % G) raise(PyExc_ValueError, "selective_scan: " + std::to_string(D) + " channels in " + std::to_string(G) + " groups");
    x = unit_last(x_); dt = unit_last(dt_); b = unit_last(b_); cc = unit_last(c_);
    a = a_.contiguous();
    if (d_) d = d_->contiguous();
    if (bias_) bias = bias_->contiguous();
    s = packed(s_);
    mask = mask_of(what, mask_, B, T, x_);
    c.T = T; c.B = as_int(what, B); c.D = as_int(what, D); c.N = static_cast<int>(N); c.G = as_int(what, G);
    c.softplus = softplus;
    if (empty()) return;
    c.x = x.data_ptr(); c.dt = dt.data_ptr(); c.b = b.data_ptr(); c.c = cc.data_ptr();
    c.x_t = x.stride(0); c.x_b = x.stride(1); c.dt_t = dt.stride(0); c.dt_b = dt.stride(1);
    c.b_t = b.stride(0); c.b_b = b.stride(1); c.b_g = b.stride(2);
    c.c_t = cc.stride(0); c.c_b = cc.stride(1); c.c_g = cc.stride(2);
    c.a = a.data_ptr<float>();
    c.d = maybe_f(d); c.dt_bias = maybe_f(bias); c.s_in = maybe_f(s);
    c.mask = static_cast<const uint8_t*>(maybe(mask));
  }
  bool empty() const { return c.T == 0 || c.B == 0 || c.D == 0; }
};

// -> y; the last state where asked, in place of `s` where that is asked too; the checkpoints of a backward where asked
std::tuple<Tensor, OptTensor, OptTensor> selective_scan_fwd(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c,
                                                            const OptTensor& d, const OptTensor& dt_bias, const OptTensor& s, const OptTensor& mask,
                                                            bool softplus, bool return_state, bool in_place, bool save) {
  Scan v(x, dt, a, b, c, d, dt_bias, s, mask, softplus);
  if (in_place && s && !s->is_contiguous()) raise(PyExc_ValueError, "selective_scan: the state must be contiguous (it is updated in place)");
  Tensor y = fresh(x.sizes(), x, x.scalar_type());
  if (v.empty()) {
    if (!return_state) return {y, std::nullopt, std::nullopt};
    if (in_place && s) return {y, *s, std::nullopt};
    return {y, s ? s->clone() : fresh_zeros({x.size(1), x.size(2), a.size(1)}, x), std::nullopt};
  }
  OptTensor out, kept;
  if (v.c.T == 1 && return_state && !save) {           // one token: the state is read and written once
    const bool here = in_place && s && v.s->is_same(*s);
    out = here ? *s : s ? v.s->is_same(*s) || v.s->is_alias_of(*s) ? v.s->clone() : *v.s : fresh_zeros({x.size(1), x.size(2), a.size(1)}, x);
    {
      Call call(x);
      check(rfa_selective_scan_step(&v.c, y.data_ptr(), out->data_ptr<float>(), call.stream), "rfa_selective_scan_step");
    }
    if (here) written(*s);
  } else {
    if (return_state) out = fresh({x.size(1), x.size(2), a.size(1)}, x, at::kFloat);
    if (save) kept = scratch(rfa_selective_scan_checkpoint_bytes(v.c.T, v.c.B, v.c.D, v.c.N), x);
    const Tensor ws = scratch(rfa_selective_scan_workspace_bytes(v.c.T, v.c.B, v.c.D, v.c.N, v.c.G, 0), x);
    Call call(x);
    check(rfa_selective_scan_fwd(&v.c, y.data_ptr(), out ? out->data_ptr<float>() : nullptr, kept ? static_cast<float*>(kept->data_ptr()) : nullptr,
                                 ws.data_ptr(), ws.numel(), call.stream),
          "rfa_selective_scan_fwd");
  }
  if (out && in_place && s && !out->is_same(*s)) {
    s->copy_(*out);
    out = s;
  }
  return {y, out, kept};
}

// -> gx, gdt, ga, gb, gc, gd, gbias, gs
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, OptTensor, OptTensor, OptTensor> selective_scan_bwd(
    const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const OptTensor& d, const OptTensor& dt_bias, const OptTensor& s,
    const OptTensor& mask, bool softplus, Tensor g, OptTensor g_s, const OptTensor& kept, bool need_state) {
  Scan v(x, dt, a, b, c, d, dt_bias, s, mask, softplus);
  need_grad("selective_scan", "g", g, x.sizes(), x);
  need_grad("selective_scan", "g_s", g_s, {x.size(1), x.size(2), a.size(1)}, x);
  const auto half = x.scalar_type();
  Tensor gx = fresh(x.sizes(), x, half), gdt = fresh(x.sizes(), x, half), ga = fresh(a.sizes(), x, at::kFloat);
  Tensor gb = fresh(b.sizes(), x, half), gc = fresh(b.sizes(), x, half);
  OptTensor gd, gbias, gs;
  if (d) gd = fresh(d->sizes(), x, at::kFloat);
  if (dt_bias) gbias = fresh(dt_bias->sizes(), x, at::kFloat);
  if (need_state && s) gs = fresh(s->sizes(), x, at::kFloat);
  if (v.empty()) {
    ga.zero_(); gb.zero_(); gc.zero_();
    if (gd) gd->zero_();
    if (gbias) gbias->zero_();
    if (gs) g_s ? gs->copy_(*g_s) : gs->zero_();
    return {gx, gdt, ga, gb, gc, gd, gbias, gs};
  }
  const size_t kept_bytes = rfa_selective_scan_checkpoint_bytes(v.c.T, v.c.B, v.c.D, v.c.N);
  if (!kept || !kept->is_contiguous() || kept->nbytes() < kept_bytes) raise(PyExc_ValueError, "selective_scan: a backward pass wants its forward's checkpoints");
  require_device(x, {&*kept});
  g = g.to(half).contiguous();
  if (g_s) g_s = packed(g_s->to(at::kFloat));
  const Tensor ws = scratch(rfa_selective_scan_workspace_bytes(v.c.T, v.c.B, v.c.D, v.c.N, v.c.G, 1), x);
  Call call(x);
  check(rfa_selective_scan_bwd(&v.c, g.data_ptr(), maybe_f(g_s), static_cast<const float*>(kept->data_ptr()), gx.data_ptr(), gdt.data_ptr(),
                               ga.data_ptr<float>(), gb.data_ptr(), gc.data_ptr(), gd ? gd->data_ptr<float>() : nullptr,
                               gbias ? gbias->data_ptr<float>() : nullptr, gs ? gs->data_ptr<float>() : nullptr, ws.data_ptr(), ws.numel(), call.stream),
        "rfa_selective_scan_bwd");
  return {gx, gdt, ga, gb, gc, gd, gbias, gs};
}

struct SelectiveScanBackward : torch::autograd::Function<SelectiveScanBackward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const OptTensor& d,
                               const OptTensor& dt_bias, const OptTensor& s, const OptTensor& mask, bool softplus, bool return_state) {
    ctx->set_materialize_grads(false);
    auto [y, out, kept] = selective_scan_fwd(x, dt, a, b, c, d, dt_bias, s, mask, softplus, return_state, false, true);
    ctx->save_for_backward({x, dt, a, b, c, plain(d), plain(dt_bias), plain(s), plain(mask), plain(kept)});
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["need_s"] = wants(s);
    if (!return_state) return {y};
    return {y, *out};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    once("selective_scan");
    const variable_list t = ctx->get_saved_variables();
    const Tensor gy = g[0].defined() ? g[0] : at::zeros_like(t[0]);
    auto [gx, gdt, ga, gb, gc, gd, gbias, gs] =
        selective_scan_bwd(t[0], t[1], t[2], t[3], t[4], opt(t[5]), opt(t[6]), opt(t[7]), opt(t[8]), ctx->saved_data["softplus"].toBool(), gy,
                           g.size() > 1 ? opt(g[1]) : OptTensor(), opt(t[9]), ctx->saved_data["need_s"].toBool());
    return {gx, gdt, ga, gb, gc, plain(gd), plain(gbias), plain(gs), Tensor(), Tensor(), Tensor()};
  }
};

Tensor selective_scan_node(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const OptTensor& d,
                           const OptTensor& dt_bias, const OptTensor& mask, bool softplus) {
  if (!records(x, dt, a, b, c, d, dt_bias))
    return std::get<0>(selective_scan_fwd(x, dt, a, b, c, d, dt_bias, std::nullopt, mask, softplus, false, false, false));
  return SelectiveScanBackward::apply(x, dt, a, b, c, d, dt_bias, OptTensor(), mask, softplus, false)[0];
}
std::tuple<Tensor, Tensor> incremental_selective_scan_node(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c,
                                                           const OptTensor& d, const OptTensor& dt_bias, const OptTensor& s, const OptTensor& mask,
                                                           bool softplus) {
  if (!records(x, dt, a, b, c, d, dt_bias, s)) {
    auto [y, out, kept] = selective_scan_fwd(x, dt, a, b, c, d, dt_bias, s, mask, softplus, true, true, false);
    return {y, *out};
  }
  const variable_list r = SelectiveScanBackward::apply(x, dt, a, b, c, d, dt_bias, s, mask, softplus, true);
  return {r[0], r[1]};
}

// ---- group norm ----------------------------------------------------------------------------------------------------------
// [..., C] as rows one stride apart, a copy where it is not.
Tensor as_rows(const Tensor& t, int64_t& stride) {
  const int64_t n = t.dim();
  Tensor v = unit_last(t);
  stride = v.size(-1);
  int64_t expect = -1;
  for (int64_t i = n - 2; i >= 0; --i) {
    if (v.size(i) == 1) continue;
    if (expect < 0) stride = v.stride(i);
    else if (v.stride(i) != expect) {
      v = v.contiguous();
      stride = v.size(-1);
      return v;
    }
    expect = v.stride(i) * v.size(i);
  }
  return v;
}

struct Norm {
  rfa_group_norm_t c{};
  Tensor x;
  OptTensor gate, weight, bias;
  Norm(const Tensor& x_, int64_t groups, const OptTensor& w_, const OptTensor& bias_, const OptTensor& gate_, bool silu, double eps) {
    const char* what = "group_norm";
    require_cuda(x_);
    if (x_.dim() < 1) raise(PyExc_ValueError, "group_norm: expected a tensor of channels, got " + shape_name(x_));
    const int64_t C = x_.size(-1);
    c.dtype = float_code(x_);
    same_dtype(what, x_, {w_ ? &*w_ : &x_, bias_ ? &*bias_ : &x_, gate_ ? &*gate_ : &x_});
    require_device(x_, {w_ ? &*w_ : &x_, bias_ ? &*bias_ : &x_, gate_ ? &*gate_ : &x_});
    if (groups < 1 || C % groups || C / groups > 16384)
      raise(PyExc_ValueError, "group_norm: " + std::to_string(C) + " channels in " + std::to_string(groups) + " groups (of at most 16384)");
    if (w_) need_shape(what, "weight", *w_, {C});
    if (bias_) need_shape(what, "bias", *bias_, {C});
    if (gate_) need_shape(what, "gate", *gate_, x_.sizes());
    c.C = as_int(what, C); c.groups = static_cast<int>(groups);
    c.rows = C ? x_.numel() / C : 0;
    c.silu = silu; c.eps = static_cast<float>(eps);
    if (empty()) return;
    x = as_rows(x_, c.x_r);
    if (gate_) gate = as_rows(*gate_, c.gate_r);
    if (w_) weight = w_->contiguous();
    if (bias_) bias = bias_->contiguous();
    c.x = x.data_ptr(); c.gate = maybe(gate); c.weight = maybe(weight); c.bias = maybe(bias);
  }
  bool empty() const { return c.rows == 0 || c.C == 0; }
};

Tensor group_norm_fwd(const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias, const OptTensor& gate, bool silu, double eps) {
  Norm v(x, groups, weight, bias, gate, silu, eps);
  Tensor y = fresh(x.sizes(), x, x.scalar_type());
  if (v.empty()) return y;
  Call c(x);
  check(rfa_group_norm_fwd(&v.c, y.data_ptr(), c.stream), "rfa_group_norm_fwd");
  return y;
}

// -> gx, gweight, gbias, ggate
std::tuple<Tensor, OptTensor, OptTensor, OptTensor> group_norm_bwd(const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias,
                                                                   const OptTensor& gate, bool silu, double eps, Tensor g, bool need_weight, bool need_bias,
                                                                   bool need_gate) {
  Norm v(x, groups, weight, bias, gate, silu, eps);
  need_grad("group_norm", "g", g, x.sizes(), x);
  Tensor gx = fresh(x.sizes(), x, x.scalar_type());
  OptTensor gw, gb, gg;
  if (need_weight && weight) gw = fresh(weight->sizes(), x, x.scalar_type());
  if (need_bias && bias) gb = fresh(bias->sizes(), x, x.scalar_type());
  if (need_gate && gate) gg = fresh(x.sizes(), x, x.scalar_type());
  if (v.empty()) {
    if (gw) gw->zero_();
    if (gb) gb->zero_();
    return {gx, gw, gb, gg};
  }
  int64_t g_r = 0;
  g = as_rows(g.to(x.scalar_type()), g_r);
  const Tensor ws = scratch(gw || gb ? rfa_group_norm_workspace_bytes(v.c.rows, v.c.C, v.c.groups) : 0, x);
  Call c(x);
  check(rfa_group_norm_bwd(&v.c, g.data_ptr(), g_r, gx.data_ptr(), maybe_out(gg), maybe_out(gw), maybe_out(gb), ws.data_ptr(), ws.numel(), c.stream),
        "rfa_group_norm_bwd");
  return {gx, gw, gb, gg};
}

struct GroupNormBackward : torch::autograd::Function<GroupNormBackward> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias, const OptTensor& gate,
                        bool silu, double eps) {
    ctx->save_for_backward({x, plain(weight), plain(bias), plain(gate)});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["silu"] = silu;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["need"] = static_cast<int64_t>(wants(weight) | wants(bias) << 1 | wants(gate) << 2);
    return group_norm_fwd(x, groups, weight, bias, gate, silu, eps);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    once("group_norm");
    const variable_list s = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    auto [gx, gw, gb, gg] = group_norm_bwd(s[0], ctx->saved_data["groups"].toInt(), opt(s[1]), opt(s[2]), opt(s[3]), ctx->saved_data["silu"].toBool(),
                                           ctx->saved_data["eps"].toDouble(), g[0], need & 1, need & 2, need & 4);
    return {gx, Tensor(), plain(gw), plain(gb), plain(gg), Tensor(), Tensor()};
  }
};

Tensor group_norm_node(const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias, const OptTensor& gate, bool silu, double eps) {
  if (!records(x, weight, bias, gate)) return group_norm_fwd(x, groups, weight, bias, gate, silu, eps);
  return GroupNormBackward::apply(x, groups, weight, bias, gate, silu, eps);
}

}  // namespace

void def_state_space(py::module_& m) {
  const auto def = [&](const char* name, auto* f) { m.def(name, f, py::call_guard<py::gil_scoped_release>()); };
  def("causal_conv_fwd", &causal_conv_fwd);
  def("causal_conv_bwd", &causal_conv_bwd);
  def("causal_conv_node", &causal_conv_node);
  def("incremental_causal_conv_node", &incremental_causal_conv_node);
  def("selective_scan_fwd", &selective_scan_fwd);
  def("selective_scan_bwd", &selective_scan_bwd);
  def("selective_scan_node", &selective_scan_node);
  def("incremental_selective_scan_node", &incremental_selective_scan_node);
  def("group_norm_fwd", &group_norm_fwd);
  def("group_norm_bwd", &group_norm_bwd);
  def("group_norm_node", &group_norm_node);
}
