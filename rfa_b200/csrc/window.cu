// Sliding-window attention: the C entry points.
#include "window.cuh"

namespace rfa {

namespace {

int window_check(const rfa_window_t* c, const char* what) {
  RFA_REQUIRE(c, RFA_EINVAL, "%s: null argument", what);
  RFA_REQUIRE(c->q && c->k && c->v, RFA_EINVAL, "%s: null pointer", what);
  RFA_REQUIRE(c->T > 0 && c->B > 0 && c->H > 0 && c->G > 0 && c->D > 0, RFA_EINVAL, "%s: empty or negative size", what);
  RFA_REQUIRE(c->dtype == RFA_F16 || c->dtype == RFA_F32 || c->dtype == RFA_BF16, RFA_EUNSUPPORTED, "%s: dtype %d", what, c->dtype);
  RFA_REQUIRE(c->H % c->G == 0, RFA_EUNSUPPORTED, "%s: %d heads share %d key heads", what, c->H, c->G);
  RFA_REQUIRE(c->D <= kWindowMaxWidth, RFA_EUNSUPPORTED, "%s: heads of %d (at most %d)", what, c->D, kWindowMaxWidth);
  RFA_REQUIRE(c->window >= 1 && c->sinks >= 0 && (int64_t)c->window + c->sinks < (1 << 30), RFA_EUNSUPPORTED, "%s: window %d, sinks %d", what, c->window, c->sinks);
  RFA_REQUIRE(c->T < ((int64_t)1 << 30) && c->B <= 65535 && c->H <= 65535 && (int64_t)c->B * c->H < (1 << 24), RFA_EUNSUPPORTED, "%s: T %lld, B %d, H %d", what,
              (long long)c->T, c->B, c->H);
  return 0;
}

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }
size_t order_bytes(int64_t S, int B) { return round256(4 * (size_t)S * B) + round256(4 * (size_t)(S + 1) * B); }

// Parts that the queries of first tokens' keys are split in, 1 where these take no longer than other work does: a part is as long as what another tile of keys
// goes through, half of what an SM does in all, or 8 tiles of 64 queries, whichever is most.  Training, 8192 tokens, 8 heads of 128 that share one key head,
// window 64 + 4, bf16: 108 us, in one piece 1147; 1 x 4096 x 4 heads of 64 that share one, window 128 + 4, fp32: 412 us and 4401.
int window_splits(int64_t T, int B, int H, int G, int window, int sinks) {
  if (sinks <= 0 || T <= window) return 1;
  const double group = H / G, far = group * (double)(T - window) / 64, near = group * ((double)window + 128) / 64;
  const double all = (double)B * G * ((double)((T + 127) / 128) * near + (double)((std::min<int64_t>(sinks, T) + 127) / 128) * far);
  const double unit = std::max(std::max(near, all / 148 / 2), 8.0);
  return far * 2 <= unit ? 1 : 1 + (int)std::min(63.0, far / unit + 1);
}
size_t parts_bytes(int64_t T, int B, int H, int G, int D, int window, int sinks) {
  const int n = window_splits(T, B, H, G, window, sinks);
  return n > 1 ? round256(sizeof(float) * n * B * G * (size_t)std::min<int64_t>(sinks, T) * 2 * D) : 0;
}

WindowArgs window_args(const rfa_window_t& c) {
  WindowArgs a{};
  a.q = {c.q, c.q_t, c.q_b, c.q_h};
  a.k = {c.k, c.k_t, c.k_b, c.k_h};
  a.v = {c.v, c.v_t, c.v_b, c.v_h};
  a.T = a.S = c.T;
  a.B = c.B; a.H = c.H; a.G = c.G; a.D = c.D; a.window = c.window; a.sinks = c.sinks; a.dtype = c.dtype;
  a.scale = c.scale;
  a.splits = 1;
  return a;
}
// numbers of the places, at the workspace's start
int number(WindowArgs& a, const rfa_window_t& c, const int64_t* length, int cap, void* workspace, cudaStream_t stream) {
  int32_t* order = static_cast<int32_t*>(workspace);
  int32_t* pos = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + round256(4 * (size_t)a.S * c.B));
  a.order = order;
  a.pos = pos;
  return launch_window_order(c.mask, length, cap, order, pos, c.T, c.B, stream);
}

int forward(const WindowArgs& a, cudaStream_t stream) { return window_tc_ok(a) ? launch_window_fwd_tc(a, stream) : launch_window_fwd_tiles(a, stream); }

}  // namespace
}  // namespace rfa

extern "C" size_t rfa_window_workspace_bytes(int64_t T, int B, int H, int G, int D, int dtype, int window, int sinks, int backward) {
  using namespace rfa;
  if (T <= 0 || B <= 0 || H <= 0 || G <= 0 || D <= 0) return 0;
  return order_bytes(T, B) + (backward ? round256(4 * (size_t)T * B * H) + parts_bytes(T, B, H, G, D, window, sinks) : 0);
}

extern "C" int rfa_window_fwd(const rfa_window_t* c, void* out, float* lse, void* workspace, size_t workspace_bytes, rfa_stream_t stream) {
  using namespace rfa;
  if (int r = window_check(c, "window_fwd")) return r;
  RFA_REQUIRE(out, RFA_EINVAL, "window_fwd: null pointer");
  RFA_REQUIRE(aligned16(lse) && aligned16(workspace), RFA_EALIGN, "window_fwd: lse or workspace is not 16-byte aligned");
  const size_t need = rfa_window_workspace_bytes(c->T, c->B, c->H, c->G, c->D, c->dtype, c->window, c->sinks, 0);
  RFA_REQUIRE(workspace && workspace_bytes >= need, RFA_EWORKSPACE, "window_fwd: workspace %zu bytes, %zu needed", workspace_bytes, need);
  WindowArgs a = window_args(*c);
  a.out = out;
  a.lse = lse;
  if (c->mask)
    if (int r = number(a, *c, nullptr, 0, workspace, as_stream(stream))) return r;
  return forward(a, as_stream(stream));
}

extern "C" int rfa_window_bwd(const rfa_window_t* c, const void* out, const float* lse, const void* g, void* gq, void* gk, void* gv, void* workspace, size_t workspace_bytes,
                              rfa_stream_t stream) {
  using namespace rfa;
  if (int r = window_check(c, "window_bwd")) return r;
  RFA_REQUIRE(out && lse && g && gq && gk && gv, RFA_EINVAL, "window_bwd: null pointer");
  RFA_REQUIRE(aligned16(lse) && aligned16(workspace), RFA_EALIGN, "window_bwd: lse or workspace is not 16-byte aligned");
  const size_t need = rfa_window_workspace_bytes(c->T, c->B, c->H, c->G, c->D, c->dtype, c->window, c->sinks, 1);
  RFA_REQUIRE(workspace && workspace_bytes >= need, RFA_EWORKSPACE, "window_bwd: workspace %zu bytes, %zu needed", workspace_bytes, need);
  WindowArgs a = window_args(*c);
  const int64_t row = (int64_t)c->H * c->D;
  a.o = {out, c->B * row, row, c->D};
  a.g = {g, c->B * row, row, c->D};
  a.lse = const_cast<float*>(lse);
  a.delta = reinterpret_cast<float*>(static_cast<char*>(workspace) + order_bytes(c->T, c->B));
  a.gq = gq; a.gk = gk; a.gv = gv;
  a.splits = window_splits(c->T, c->B, c->H, c->G, c->window, c->sinks);
  a.parts = a.delta + round256(4 * (size_t)c->T * c->B * c->H) / 4;
  if (c->mask)
    if (int r = number(a, *c, nullptr, 0, workspace, as_stream(stream))) return r;
  bool tc = window_tc_ok(a);
  for (const void* p : {out, g, static_cast<const void*>(gq), static_cast<const void*>(gk), static_cast<const void*>(gv)}) tc = tc && aligned16(p);
  return tc ? launch_window_bwd_tc(a, c->mask, as_stream(stream)) : launch_window_bwd_tiles(a, as_stream(stream));
}

extern "C" size_t rfa_window_append_workspace_bytes(int64_t T, int B, int H, int G, int D, int dtype, int window, int sinks, int empty) {
  using namespace rfa;
  if (T <= 0 || B <= 0 || H <= 0 || G <= 0 || D <= 0 || window < 1 || sinks < 0) return 0;
  if (T == 1 && !empty) return 0;
  const int64_t S = T + (empty ? 0 : (int64_t)window + sinks);
  return order_bytes(S, B) + (empty ? 0 : 2 * round256((size_t)S * B * G * D * (dtype == RFA_F32 ? 4 : 2)));
}

extern "C" int rfa_window_append(const rfa_window_t* c, void* cache_k, void* cache_v, int64_t* length, int empty, void* out, void* workspace, size_t workspace_bytes,
                                 rfa_stream_t stream) {
  using namespace rfa;
  if (int r = window_check(c, "window_append")) return r;
  RFA_REQUIRE(cache_k && cache_v && length && out, RFA_EINVAL, "window_append: null pointer");
  RFA_REQUIRE(aligned16(cache_k) && aligned16(cache_v) && aligned16(workspace), RFA_EALIGN, "window_append: cache or workspace is not 16-byte aligned");
  const size_t need = rfa_window_append_workspace_bytes(c->T, c->B, c->H, c->G, c->D, c->dtype, c->window, c->sinks, empty);
  RFA_REQUIRE(!need || (workspace && workspace_bytes >= need), RFA_EWORKSPACE, "window_append: workspace %zu bytes, %zu needed", workspace_bytes, need);
  const cudaStream_t st = as_stream(stream);
  if (c->T == 1 && !empty) return launch_window_step(*c, cache_k, cache_v, length, out, st);
  WindowArgs a = window_args(*c);
  a.out = out;
  const int cap = empty ? 0 : c->sinks + c->window;
  a.S = cap + c->T;
  if (c->mask || !empty)
    if (int r = number(a, *c, empty ? nullptr : length, cap, workspace, st)) return r;
  if (!empty) {
    char* keys = static_cast<char*>(workspace) + order_bytes(a.S, c->B);
    char* values = keys + round256((size_t)a.S * c->B * c->G * c->D * (c->dtype == RFA_F32 ? 4 : 2));
    if (int r = launch_window_gather(*c, cache_k, cache_v, length, keys, values, st)) return r;
    const int64_t row = (int64_t)c->G * c->D;
    a.k = {keys, c->B * row, row, c->D};
    a.v = {values, c->B * row, row, c->D};
  }
  if (int r = forward(a, st)) return r;
  return launch_window_keep(*c, cache_k, cache_v, length, a.order, empty != 0, st);
}
