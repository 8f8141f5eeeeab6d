// The tensor-level calls and autograd nodes of decay_attention.py and window_attention.py.  No arithmetic happens here.  Errors keep the types that
// torch_ops.cpp gives them.
#include "torch_checks.h"

namespace {

double scale_of(const std::optional<double>& scale, int64_t width) { return scale ? *scale : width > 0 ? 1.0 / std::sqrt(static_cast<double>(width)) : 1.0; }

// The tensor-core kernels take 16-bit heads of up to 128 whose rows start on 16 bytes.  Other rows of those types are copied for them, widths that are no multiple
// of 8 filled with zeros, which add nothing to a product: a copy reads and writes a row once where the kernels for any rows take several times as long for it.  Below 64
// tokens the copies' launches cost more (8 x 16 heads of 64, forward, tensor cores / any rows, us: 2 tokens 6 / 11, 64 6 / 35, 256 9 / 113; a copy 2 to 3).
bool copies_pay(const Tensor& q, int64_t width) { return (q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16) && width >= 1 && width <= 128 && q.size(0) >= 64; }
bool rows_fit(const Tensor& t) {
  if (!aligned(t) || (t.size(-1) > 1 && t.stride(-1) != 1)) return false;
  for (int64_t d = 0; d + 1 < t.dim(); ++d)
    if (t.size(d) > 1 && (t.stride(d) <= 0 || t.stride(d) % 8)) return false;
  return true;
}
Tensor filled(const Tensor& t) {
  const int64_t rest = (8 - t.size(-1) % 8) % 8;
  if (rest) return at::constant_pad_nd(t, {0, rest});
  return rows_fit(t) ? t : packed(t);
}
Tensor cut(const Tensor& t, int64_t width) { return t.size(-1) == width ? t : t.narrow(-1, 0, width).contiguous(); }
Tensor filled_state(const Tensor& s) {
  const int64_t rows = (8 - s.size(-2) % 8) % 8, cols = (8 - s.size(-1) % 8) % 8;
  return rows || cols ? at::constant_pad_nd(s, {0, cols, 0, rows}) : s;
}
Tensor cut_state(const Tensor& s, int64_t rows, int64_t cols) {
  return s.size(-2) == rows && s.size(-1) == cols ? s : s.narrow(-2, 0, rows).narrow(-1, 0, cols).contiguous();
}

// ---- linear attention with a decay ------------------------------------------------------------------------------------------
struct Decay {
  rfa_decay_t c{};
  Tensor q, k, v, log_decay;
  OptTensor s, mask;
  Decay(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_, const OptTensor& s_, const OptTensor& mask_, const std::optional<double>& scale) {
    const char* what = "decay_attention";
    require_cuda(q_);
    rank(q_, 4);
    rank(v_, 4);
    const int64_t T = q_.size(0), B = q_.size(1), H = q_.size(2), K = q_.size(3), D = v_.size(3);
    c.dtype = float_code(q_);
    same_dtype(what, q_, {&k_, &v_});
    require_device(q_, {&k_, &v_, &g_, s_ ? &*s_ : &q_});
    need_shape(what, "k", k_, {T, B, H, K});
    need_shape(what, "v", v_, {T, B, H, D});
    c.per_head = g_.dim() == 1;
    if (c.per_head) need_shape(what, "log_decay", g_, {H});
    else need_shape(what, "log_decay", g_, {T, B, H});
    c.decay_dtype = float_code(g_);
    if (c.decay_dtype != RFA_F32) same_dtype(what, q_, {&g_});
    if (s_) { need_f32(what, "s", *s_); need_shape(what, "s", *s_, {B, H, K, D}); }
    if (K > 256 || D > 256) raise(PyExc_ValueError, "decay_attention: heads of " + std::to_string(K) + " and " + std::to_string(D) + " (at most 256)");
    q = unit_last(q_); k = unit_last(k_); v = unit_last(v_);
    log_decay = g_;
    s = packed(s_);
    mask = mask_of(what, mask_, B, T, q_);
    c.T = T; c.B = as_int(what, B); c.H = as_int(what, H); c.K = static_cast<int>(K); c.D = static_cast<int>(D);
    c.scale = static_cast<float>(scale_of(scale, K));
    if (empty()) return;
    c.q = q.data_ptr(); c.k = k.data_ptr(); c.v = v.data_ptr(); c.log_decay = log_decay.data_ptr();
    c.q_t = q.stride(0); c.q_b = q.stride(1); c.q_h = q.stride(2);
    c.k_t = k.stride(0); c.k_b = k.stride(1); c.k_h = k.stride(2);
    c.v_t = v.stride(0); c.v_b = v.stride(1); c.v_h = v.stride(2);
    c.g_h = log_decay.stride(-1);
    if (!c.per_head) { c.g_t = log_decay.stride(0); c.g_b = log_decay.stride(1); }
    c.s_in = maybe_f(s);
    c.mask = static_cast<const uint8_t*>(maybe(mask));
  }
  bool empty() const { return c.T == 0 || c.B == 0 || c.H == 0 || c.K == 0 || c.D == 0; }
  bool wants_copies() const {
    return !empty() && copies_pay(q, c.K) && c.D <= 128 && (c.K % 8 || c.D % 8 || !rows_fit(q) || !rows_fit(k) || !rows_fit(v));
  }
  Tensor workspace(bool backward) const { return scratch(rfa_decay_workspace_bytes(c.T, c.B, c.H, c.K, c.D, c.dtype, backward), q); }
};

// -> out; the last state where asked, in place of `s` where that is asked too; with `save` what the backward goes on from, if anything
std::tuple<Tensor, OptTensor, OptTensor> decay_attention_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const OptTensor& s, const OptTensor& mask,
                                                  std::optional<double> scale, bool return_state, bool in_place, bool save) {
  Decay d(q, k, v, log_decay, s, mask, scale);
  if (in_place && s && !s->is_contiguous()) raise(PyExc_ValueError, "decay_attention: the state must be contiguous (it is updated in place)");
  const std::vector<int64_t> state{q.size(1), q.size(2), q.size(3), v.size(3)};
  if (d.empty()) {
    Tensor out = at::zeros(v.sizes(), v.options().requires_grad(false));
    if (!return_state) return {out, std::nullopt, std::nullopt};
    if (in_place && s) return {out, *s, std::nullopt};
    return {out, s ? s->clone() : fresh_zeros(state, q), std::nullopt};
  }
  if (d.wants_copies()) {
    const int64_t K = q.size(3), D = v.size(3);
    auto [out, last, kept] = decay_attention_fwd(filled(q), filled(k), filled(v), log_decay, s ? OptTensor(filled_state(*s)) : s, mask, scale_of(scale, K), return_state, false, save);
    if (last) {
      last = cut_state(*last, K, D);
      if (in_place && s) {
        s->copy_(*last);
        last = s;
      }
    }
    return {cut(out, D), last, kept};
  }
  Tensor out = fresh(v.sizes(), q, q.scalar_type());
  OptTensor last, kept;
  const bool here = in_place && s && d.s->is_same(*s);
  if (d.c.T == 1 && return_state && !save) {           // the state is read and written once
    last = here ? *s : s ? d.s->is_same(*s) || d.s->is_alias_of(*s) ? d.s->clone() : *d.s : fresh_zeros(state, q);
    Call call(q);
    check(rfa_decay_step(&d.c, out.data_ptr(), last->data_ptr<float>(), call.stream), "rfa_decay_step");
  } else {
    if (return_state) last = here ? *s : fresh(state, q, at::kFloat);
    const size_t bytes = save ? rfa_decay_kept_bytes(&d.c) : 0;
    if (bytes) kept = scratch(bytes, q);
    const Tensor ws = d.workspace(false);
    Call call(q);
    check(rfa_decay_fwd(&d.c, out.data_ptr(), last ? last->data_ptr<float>() : nullptr, maybe_out(kept), ws.data_ptr(), ws.numel(), call.stream), "rfa_decay_fwd");
  }
  if (last && here) written(*s);
  if (last && in_place && s && !here) {
    s->copy_(*last);
    last = s;
  }
  return {out, last, kept};
}

// -> gq, gk, gv, g_decay, gs
std::tuple<Tensor, Tensor, Tensor, OptTensor, OptTensor> decay_attention_bwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const OptTensor& s,
                                                                             const OptTensor& mask, std::optional<double> scale, Tensor g, OptTensor g_s, const OptTensor& kept, bool need_decay,
                                                                             bool need_state) {
  Decay d(q, k, v, log_decay, s, mask, scale);
  need_grad("decay_attention", "g", g, v.sizes(), q);
  need_grad("decay_attention", "g_s", g_s, {q.size(1), q.size(2), q.size(3), v.size(3)}, q);
  const auto half = q.scalar_type();
  Tensor gq = fresh(q.sizes(), q, half), gk = fresh(k.sizes(), q, half), gv = fresh(v.sizes(), q, half);
  OptTensor gd, gs;
  if (need_decay) gd = fresh(log_decay.sizes(), q, log_decay.scalar_type());
  if (need_state && s) gs = fresh(s->sizes(), q, at::kFloat);
  if (d.empty()) {
    for (const Tensor& t : {gq, gk, gv}) t.zero_();
    if (gd) gd->zero_();
    if (gs) g_s ? gs->copy_(*g_s) : gs->zero_();
    return {gq, gk, gv, gd, gs};
  }
  if (d.wants_copies()) {
    const int64_t K = q.size(3), D = v.size(3);
    auto [pq, pk, pv, pd, ps] = decay_attention_bwd(filled(q), filled(k), filled(v), log_decay, s ? OptTensor(filled_state(*s)) : s, mask, scale_of(scale, K), filled(g.to(half)),
                                                    g_s ? OptTensor(filled_state(g_s->to(at::kFloat))) : g_s, kept, need_decay, need_state);
    return {cut(pq, K), cut(pk, K), cut(pv, D), pd, ps ? OptTensor(cut_state(*ps, K, D)) : ps};
  }
  if (kept && (!kept->is_contiguous() || kept->nbytes() < rfa_decay_kept_bytes(&d.c))) raise(PyExc_ValueError, "decay_attention: kept is not what this call's forward left");
  if (kept) require_device(q, {&*kept});
  g = packed(g.to(half));
  if (g_s) g_s = packed(g_s->to(at::kFloat));
  const Tensor ws = d.workspace(true);
  Call call(q);
  check(rfa_decay_bwd(&d.c, g.data_ptr(), maybe_f(g_s), maybe(kept), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), maybe_out(gd), gs ? gs->data_ptr<float>() : nullptr, ws.data_ptr(),
                      ws.numel(), call.stream),
        "rfa_decay_bwd");
  return {gq, gk, gv, gd, gs};
}

struct DecayAttentionBackward : torch::autograd::Function<DecayAttentionBackward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const OptTensor& s, const OptTensor& mask,
                               std::optional<double> scale, bool return_state) {
    ctx->set_materialize_grads(false);
    ctx->saved_data["scale"] = scale_of(scale, q.size(3));
    ctx->saved_data["need"] = static_cast<int64_t>(log_decay.requires_grad() | wants(s) << 1);
    auto [out, last, kept] = decay_attention_fwd(q, k, v, log_decay, s, mask, scale, return_state, false, true);
    ctx->save_for_backward({q, k, v, log_decay, plain(s), plain(mask), plain(kept)});
    if (!return_state) return {out};
    return {out, *last};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    once("decay_attention");
    const variable_list t = ctx->get_saved_variables();
    const int64_t need = ctx->saved_data["need"].toInt();
    const Tensor go = g[0].defined() ? g[0] : at::zeros_like(t[2]);
    auto [gq, gk, gv, gd, gs] = decay_attention_bwd(t[0], t[1], t[2], t[3], opt(t[4]), opt(t[5]), ctx->saved_data["scale"].toDouble(), go,
                                                    g.size() > 1 ? opt(g[1]) : OptTensor(), opt(t[6]), need & 1, need & 2);
    return {gq, gk, gv, plain(gd), plain(gs), Tensor(), Tensor(), Tensor()};
  }
};

Tensor decay_attention_node(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const OptTensor& mask, std::optional<double> scale) {
  if (!records(q, k, v, log_decay)) return std::get<0>(decay_attention_fwd(q, k, v, log_decay, std::nullopt, mask, scale, false, false, false));
  return DecayAttentionBackward::apply(q, k, v, log_decay, OptTensor(), mask, scale, false)[0];
}
std::tuple<Tensor, Tensor> incremental_decay_attention_node(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const OptTensor& s,
                                                            const OptTensor& mask, std::optional<double> scale) {
  if (!records(q, k, v, log_decay, s)) {
    auto [out, last, kept] = decay_attention_fwd(q, k, v, log_decay, s, mask, scale, true, true, false);
    return {out, *last};
  }
  const variable_list r = DecayAttentionBackward::apply(q, k, v, log_decay, s, mask, scale, true);
  return {r[0], r[1]};
}

// ---- sliding-window attention -------------------------------------------------------------------------------------------------
struct Window {
  rfa_window_t c{};
  Tensor q, k, v;
  OptTensor mask;
  Window(const Tensor& q_, const Tensor& k_, const Tensor& v_, int64_t window, int64_t sinks, const OptTensor& mask_, const std::optional<double>& scale) {
    const char* what = "window_attention";
    require_cuda(q_);
    rank(q_, 4);
    rank(k_, 4);
    const int64_t T = q_.size(0), B = q_.size(1), H = q_.size(2), D = q_.size(3), G = k_.size(2);
    c.dtype = float_code(q_);
    same_dtype(what, q_, {&k_, &v_});
    require_device(q_, {&k_, &v_});
    need_shape(what, "k", k_, {T, B, G, D});
    need_shape(what, "v", v_, {T, B, G, D});
    if (G == 0 ? H != 0 : H % G != 0) raise(PyExc_ValueError, "window_attention: " + std::to_string(H) + " heads share " + std::to_string(G) + " key heads");
    if (D > 256) raise(PyExc_ValueError, "window_attention: heads of " + std::to_string(D) + " (at most 256)");
    if (window < 1 || sinks < 0 || window >= 1 << 30 || sinks >= 1 << 30 || window + sinks >= 1 << 30)
      raise(PyExc_ValueError, "window_attention: a window of " + std::to_string(window) + " and " + std::to_string(sinks) + " first tokens");
    q = unit_last(q_); k = unit_last(k_); v = unit_last(v_);
    mask = mask_of(what, mask_, B, T, q_);
    c.T = T; c.B = as_int(what, B); c.H = as_int(what, H); c.G = as_int(what, G); c.D = static_cast<int>(D);
    c.window = static_cast<int>(window); c.sinks = static_cast<int>(sinks);
    c.scale = static_cast<float>(scale_of(scale, D));
    if (empty()) return;
    c.q = q.data_ptr(); c.k = k.data_ptr(); c.v = v.data_ptr();
    c.q_t = q.stride(0); c.q_b = q.stride(1); c.q_h = q.stride(2);
    c.k_t = k.stride(0); c.k_b = k.stride(1); c.k_h = k.stride(2);
    c.v_t = v.stride(0); c.v_b = v.stride(1); c.v_h = v.stride(2);
    c.mask = static_cast<const uint8_t*>(maybe(mask));
  }
  bool empty() const { return c.T == 0 || c.B == 0 || c.H == 0 || c.D == 0; }
  bool wants_copies() const { return !empty() && copies_pay(q, c.D) && c.scale > 0.f && (c.D % 8 || !rows_fit(q) || !rows_fit(k) || !rows_fit(v)); }
  Tensor workspace(bool backward) const {
    return scratch(rfa_window_workspace_bytes(c.T, c.B, c.H, c.G, c.D, c.dtype, c.window, c.sinks, backward), q);
  }
};

// -> out, and where asked what the backward wants of the softmax
std::tuple<Tensor, OptTensor> window_attention_fwd(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, const OptTensor& mask,
                                                   std::optional<double> scale, bool save) {
  Window w(q, k, v, window, sinks, mask, scale);
  if (w.wants_copies()) {
    auto [out, lse] = window_attention_fwd(filled(q), filled(k), filled(v), window, sinks, mask, scale_of(scale, q.size(3)), save);
    return {cut(out, q.size(3)), lse};
  }
  Tensor out = fresh(q.sizes(), q, q.scalar_type());
  OptTensor lse;
  if (save) lse = fresh({q.size(1), q.size(2), q.size(0)}, q, at::kFloat);
  if (w.empty()) return {out, lse};
  const Tensor ws = w.workspace(false);
  Call call(q);
  check(rfa_window_fwd(&w.c, out.data_ptr(), lse ? lse->data_ptr<float>() : nullptr, ws.data_ptr(), ws.numel(), call.stream), "rfa_window_fwd");
  return {out, lse};
}

// -> gq, gk, gv
std::tuple<Tensor, Tensor, Tensor> window_attention_bwd(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, const OptTensor& mask,
                                                        std::optional<double> scale, const Tensor& out, const Tensor& lse, Tensor g) {
  Window w(q, k, v, window, sinks, mask, scale);
  need_grad("window_attention", "g", g, q.sizes(), q);
  need_grad("window_attention", "out", out, q.sizes(), q);
  need_grad("window_attention", "lse", lse, {q.size(1), q.size(2), q.size(0)}, q);
  same_dtype("window_attention", q, {&out});
  need_f32("window_attention", "lse", lse);
  const auto half = q.scalar_type();
  if (w.wants_copies()) {
    const int64_t D = q.size(3);
    auto [pq, pk, pv] = window_attention_bwd(filled(q), filled(k), filled(v), window, sinks, mask, scale_of(scale, D), filled(out), lse, filled(g.to(half)));
    return {cut(pq, D), cut(pk, D), cut(pv, D)};
  }
  Tensor gq = fresh(q.sizes(), q, half), gk = fresh(k.sizes(), q, half), gv = fresh(v.sizes(), q, half);
  if (w.empty()) {
    gk.zero_();
    gv.zero_();
    return {gq, gk, gv};
  }
  g = packed(g.to(half));
  const Tensor o = packed(out), l = packed(lse), ws = w.workspace(true);
  Call call(q);
  check(rfa_window_bwd(&w.c, o.data_ptr(), l.data_ptr<float>(), g.data_ptr(), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), ws.data_ptr(), ws.numel(), call.stream),
        "rfa_window_bwd");
  return {gq, gk, gv};
}

struct WindowAttentionBackward : torch::autograd::Function<WindowAttentionBackward> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, const OptTensor& mask,
                        std::optional<double> scale) {
    auto [out, lse] = window_attention_fwd(q, k, v, window, sinks, mask, scale, true);
    ctx->save_for_backward({q, k, v, plain(mask), out, *lse});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale_of(scale, q.size(3));
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    once("window_attention");
    const variable_list t = ctx->get_saved_variables();
    auto [gq, gk, gv] = window_attention_bwd(t[0], t[1], t[2], ctx->saved_data["window"].toInt(), ctx->saved_data["sinks"].toInt(), opt(t[3]),
                                             ctx->saved_data["scale"].toDouble(), t[4], t[5], g[0]);
    return {gq, gk, gv, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor window_attention_node(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks, const OptTensor& mask, std::optional<double> scale) {
  if (!records(q, k, v)) return std::get<0>(window_attention_fwd(q, k, v, window, sinks, mask, scale, false));
  return WindowAttentionBackward::apply(q, k, v, window, sinks, mask, scale);
}

// -> out, prev_k, prev_v, prev_len, updated in place where they are given
std::tuple<Tensor, Tensor, Tensor, Tensor> window_attention_append(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks,
                                                                   const OptTensor& prev_k, const OptTensor& prev_v, const OptTensor& prev_len, const OptTensor& mask,
                                                                   std::optional<double> scale) {
  const char* what = "window_attention";
  if (records(q, k, v, prev_k, prev_v)) raise(PyExc_RuntimeError, "incremental_window_attention is for decoding: no gradient goes through its cache (call it under no_grad)");
  Window w(q, k, v, window, sinks, mask, scale);
  if (prev_k.has_value() != prev_v.has_value() || prev_k.has_value() != prev_len.has_value())
    raise(PyExc_ValueError, "window_attention: prev_k, prev_v and prev_len come together");
  const std::vector<int64_t> shape{q.size(1), k.size(2), window + sinks, q.size(3)};
  Tensor ck, cv, len;
  if (prev_k) {
    ck = *prev_k; cv = *prev_v; len = *prev_len;
    same_dtype(what, q, {&ck, &cv});
    require_device(q, {&ck, &cv, &len});
    need_shape(what, "prev_k", ck, shape);
    need_shape(what, "prev_v", cv, shape);
    need_shape(what, "prev_len", len, {q.size(1)});
    if (len.scalar_type() != at::kLong) raise(PyExc_TypeError, "window_attention: prev_len must be int64, got " + dtype_name(len));
    if (!ck.is_contiguous() || !cv.is_contiguous() || !len.is_contiguous())
      raise(PyExc_ValueError, "window_attention: prev_k, prev_v and prev_len must be contiguous (they are updated in place)");
    const auto *k0 = static_cast<const char*>(ck.data_ptr()), *v0 = static_cast<const char*>(cv.data_ptr());
    if (ck.numel() && k0 < v0 + cv.nbytes() && v0 < k0 + ck.nbytes()) raise(PyExc_ValueError, "window_attention: prev_k and prev_v share memory");
  } else {                                             // slots that no token reaches are zero, so that a copy of the cache is a number
    ck = at::zeros(shape, q.options().requires_grad(false));
    cv = at::zeros(shape, q.options().requires_grad(false));
    len = at::zeros({q.size(1)}, q.options().dtype(at::kLong).requires_grad(false));
  }
  Tensor out = fresh(q.sizes(), q, q.scalar_type());
  if (w.empty()) return {out, ck, cv, len};
  const bool empty = !prev_k;
  const Tensor ka = packed(ck), va = packed(cv);      // a copy where a view starts off a 16-byte boundary
  {
    const Tensor ws = scratch(rfa_window_append_workspace_bytes(w.c.T, w.c.B, w.c.H, w.c.G, w.c.D, w.c.dtype, w.c.window, w.c.sinks, empty), q);
    Call call(q);
    check(rfa_window_append(&w.c, ka.data_ptr(), va.data_ptr(), len.data_ptr<int64_t>(), empty, out.data_ptr(), ws.data_ptr(), ws.numel(), call.stream),
          "rfa_window_append");
  }
  for (const auto& [kept, used] : {std::pair<const Tensor&, const Tensor&>(ck, ka), std::pair<const Tensor&, const Tensor&>(cv, va)})
    used.is_same(kept) ? written(kept) : static_cast<void>(kept.copy_(used));
  written(len);
  return {out, ck, cv, len};
}

}  // namespace

void def_attention(py::module_& m) {
  const auto def = [&](const char* name, auto* f) { m.def(name, f, py::call_guard<py::gil_scoped_release>()); };
  def("decay_attention_fwd", &decay_attention_fwd);
  def("decay_attention_bwd", &decay_attention_bwd);
  def("decay_attention_node", &decay_attention_node);
  def("incremental_decay_attention_node", &incremental_decay_attention_node);
  def("window_attention_fwd", &window_attention_fwd);
  def("window_attention_bwd", &window_attention_bwd);
  def("window_attention_node", &window_attention_node);
  def("window_attention_append", &window_attention_append);
}
