// Linear attention with a decay: the C entry points.  Which kernels a call takes is decided here, from its sizes, type and alignment.
#include <algorithm>

#include "decay.cuh"

namespace rfa {

namespace {

int decay_check(const rfa_decay_t* c, const char* what) {
  RFA_REQUIRE(c, RFA_EINVAL, "%s: null argument", what);
  RFA_REQUIRE(c->q && c->k && c->v && c->log_decay, RFA_EINVAL, "%s: null pointer", what);
  RFA_REQUIRE(c->T > 0 && c->B > 0 && c->H > 0 && c->K > 0 && c->D > 0, RFA_EINVAL, "%s: empty or negative size", what);
  for (const int t : {c->dtype, c->decay_dtype})
    RFA_REQUIRE(t == RFA_F16 || t == RFA_F32 || t == RFA_BF16, RFA_EUNSUPPORTED, "%s: dtype %d", what, t);
  RFA_REQUIRE(c->K <= kDecayMaxWidth && c->D <= kDecayMaxWidth, RFA_EUNSUPPORTED, "%s: heads of %d and %d (at most %d)", what, c->K, c->D, kDecayMaxWidth);
  RFA_REQUIRE(c->T < ((int64_t)1 << 31) - 256 && c->B <= 65535 && c->H <= 65535 && (int64_t)c->B * c->H < (1 << 24), RFA_EUNSUPPORTED, "%s: T %lld, B %d, H %d", what,
              (long long)c->T, c->B, c->H);
  RFA_REQUIRE(aligned16(c->s_in), RFA_EALIGN, "%s: s_in is not 16-byte aligned", what);
  return 0;
}

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// Workspace of a backward pass: the arrays of the largest sweep, then what the decays' gradient is made of.
struct BwdPlan {
  SweepPlan sweeps;
  size_t dots, front, sums;   // bytes; dots: each of two
  explicit BwdPlan(const rfa_decay_t& c) {
    const int64_t BH = (int64_t)c.B * c.H;
    sweeps = sweep_plan(c.T, BH, 2 * sweep_tiles(c.K) + sweep_tiles(c.D), 3, c.K, c.D);
    dots = round256(2 * sizeof(float) * sweep_tiles(c.K) * BH * c.T);
    front = round256(sizeof(float) * BH * c.K * c.D);
    sums = round256(sizeof(float) * BH);
  }
  size_t sweep() const { return round256(sweeps.totals) + round256(sweeps.seg_decay); }
  size_t bytes() const { return sweep() + 2 * dots + front + sums; }
};
size_t bwd_bytes(const rfa_decay_t& c) {
  const size_t tc = c.dtype != RFA_F32 && c.K <= 128 && c.D <= 128 && c.K % 8 == 0 && c.D % 8 == 0 ? decay_tc_bwd_bytes(c) : 0;
  return std::max(BwdPlan(c).bytes(), tc);
}

// sweep `i` of `n` in a launch
SweepArgs sweep_args(const rfa_decay_t& c, int A, int W, bool rev, char* ws, const SweepPlan& plan, int i, int n) {
  SweepArgs a{};
  a.decay = {c.log_decay, c.g_t, c.g_b, c.g_h};
  a.mask = c.mask;
  a.T = c.T; a.B = c.B; a.H = c.H; a.A = A; a.W = W;
  a.dtype = c.dtype; a.decay_dtype = c.decay_dtype; a.rev = rev;
  a.in_scale = rev ? c.scale : 1.f;
  a.out_scale = rev ? 1.f : c.scale;
  a.totals = reinterpret_cast<float*>(ws) + plan.totals / sizeof(float) / n * i;
  a.seg_decay = reinterpret_cast<double*>(ws + round256(plan.totals)) + plan.seg_decay / sizeof(double) / n * i;
  return a;
}

}  // namespace
}  // namespace rfa

extern "C" size_t rfa_decay_workspace_bytes(int64_t T, int B, int H, int K, int D, int dtype, int backward) {
  using namespace rfa;
  if (T <= 0 || B <= 0 || H <= 0 || K <= 0 || D <= 0) return 0;
  rfa_decay_t c{};
  c.T = T; c.B = B; c.H = H; c.K = K; c.D = D; c.dtype = dtype;
  if (backward) return bwd_bytes(c);
  size_t most = 0;
  for (const SweepPlan& p : {sweep_plan(T, (int64_t)B * H, sweep_tiles(D), 1, K, D), decay_tc_plan(T, (int64_t)B * H, K, D)}) most = std::max(most, round256(p.totals) + round256(p.seg_decay));
  return most;
}

extern "C" size_t rfa_decay_kept_bytes(const rfa_decay_t* c) {
  using namespace rfa;
  if (!c || c->T <= 0 || c->B <= 0 || c->H <= 0 || c->K <= 0 || c->D <= 0 || !decay_tc_ok(*c)) return 0;
  return decay_tc_kept_bytes(c->T, (int64_t)c->B * c->H, c->K, c->D);
}

extern "C" int rfa_decay_fwd(const rfa_decay_t* c, void* out, float* s_out, void* kept, void* workspace, size_t workspace_bytes, rfa_stream_t stream) {
  using namespace rfa;
  if (int r = decay_check(c, "decay_fwd")) return r;
  RFA_REQUIRE(out, RFA_EINVAL, "decay_fwd: null pointer");
  RFA_REQUIRE(aligned16(s_out) && aligned16(kept) && aligned16(workspace), RFA_EALIGN, "decay_fwd: s_out, kept or workspace is not 16-byte aligned");
  const size_t need = rfa_decay_workspace_bytes(c->T, c->B, c->H, c->K, c->D, c->dtype, 0);
  RFA_REQUIRE(!need || (workspace && workspace_bytes >= need), RFA_EWORKSPACE, "decay_fwd: workspace %zu bytes, %zu needed", workspace_bytes, need);
  RFA_REQUIRE(!decay_tc_ok(*c) || aligned16(out), RFA_EALIGN, "decay_fwd: out is not 16-byte aligned");
  if (decay_tc_ok(*c)) return launch_decay_tc(*c, decay_tc_plan(c->T, (int64_t)c->B * c->H, c->K, c->D), static_cast<char*>(workspace), out, s_out, kept, as_stream(stream));
  const SweepPlan plan = sweep_plan(c->T, (int64_t)c->B * c->H, sweep_tiles(c->D), 1, c->K, c->D);
  SweepBatch batch{};
  batch.count = 1;
  SweepArgs& a = batch.sweep[0];
  a = sweep_args(*c, c->K, c->D, false, static_cast<char*>(workspace), plan, 0, 1);
  a.x1 = {c->q, c->q_t, c->q_b, c->q_h};
  a.x2 = {c->k, c->k_t, c->k_b, c->k_h};
  a.x3 = {c->v, c->v_t, c->v_b, c->v_h};
  a.out = out;
  a.s_in = {const_cast<float*>(c->s_in), c->D, 1};
  a.s_out = {s_out, c->D, 1};
  return launch_sweeps(batch, plan, as_stream(stream));
}

extern "C" int rfa_decay_bwd(const rfa_decay_t* c, const void* g, const float* g_s, const void* kept, void* gq, void* gk, void* gv, void* g_decay, float* gs_in, void* workspace,
                             size_t workspace_bytes, rfa_stream_t stream) {
  using namespace rfa;
  if (int r = decay_check(c, "decay_bwd")) return r;
  RFA_REQUIRE(g && gq && gk && gv, RFA_EINVAL, "decay_bwd: null pointer");
  RFA_REQUIRE(aligned16(g_s) && aligned16(gs_in) && aligned16(kept) && aligned16(workspace), RFA_EALIGN, "decay_bwd: g_s, gs_in, kept or workspace is not 16-byte aligned");
  const size_t need = bwd_bytes(*c);
  RFA_REQUIRE(workspace && workspace_bytes >= need, RFA_EWORKSPACE, "decay_bwd: workspace %zu bytes, %zu needed", workspace_bytes, need);
  const cudaStream_t st = as_stream(stream);
  if (decay_tc_ok(*c)) RFA_REQUIRE(aligned16(g) && aligned16(gq) && aligned16(gk) && aligned16(gv), RFA_EALIGN, "decay_bwd: g or a gradient is not 16-byte aligned");
  if (decay_tc_ok(*c))
    return launch_decay_tc_bwd(*c, static_cast<char*>(workspace), kept, g, g_s, gq, gk, gv, g_decay, gs_in, st);
  const BwdPlan plan(*c);
  char *ws = static_cast<char*>(workspace), *rest = ws + plan.sweep();
  float* q_dots = reinterpret_cast<float*>(rest);
  float* k_dots = reinterpret_cast<float*>(rest + plan.dots);
  float* front = reinterpret_cast<float*>(rest + 2 * plan.dots);
  float* sums = reinterpret_cast<float*>(rest + 2 * plan.dots + plan.front);
  const DecayRows q{c->q, c->q_t, c->q_b, c->q_h}, k{c->k, c->k_t, c->k_b, c->k_h}, v{c->v, c->v_t, c->v_b, c->v_h};
  const DecayRows gr{g, (int64_t)c->B * c->H * c->D, (int64_t)c->H * c->D, c->D};
  float *s_in = const_cast<float*>(c->s_in), *g_last = const_cast<float*>(g_s);
  SweepBatch batch{};
  batch.count = 3;
  SweepArgs& a = batch.sweep[0];
  a = sweep_args(*c, c->D, c->K, false, ws, plan.sweeps, 0, 3);
  a.x1 = gr; a.x2 = v; a.x3 = k; a.out = gq;
  a.s_in = {s_in, 1, c->D};
  SweepArgs& ak = batch.sweep[1];
  ak = sweep_args(*c, c->D, c->K, true, ws, plan.sweeps, 1, 3);
  ak.x1 = v; ak.x2 = gr; ak.x3 = q; ak.out = gk;
  ak.s_in = {g_last, 1, c->D};
  SweepArgs& av = batch.sweep[2];
  av = sweep_args(*c, c->K, c->D, true, ws, plan.sweeps, 2, 3);
  av.x1 = k; av.x2 = q; av.x3 = gr; av.out = gv;
  av.s_in = {g_last, c->D, 1};
  av.s_out = {gs_in, c->D, 1};
  if (g_decay) {
    a.x4 = q; a.dots = q_dots;
    ak.x4 = k; ak.dots = k_dots;
    if (g_s) {
      a.s_out = {front, 1, c->D};
      a.front_out = true;
    }
  }
  if (int r = launch_sweeps(batch, plan.sweeps, st)) return r;

  if (!g_decay) return 0;
  const int tiles = sweep_tiles(c->K);
  return launch_decay_grad(q_dots, tiles, k_dots, tiles, g_s, front, c->K * c->D, c->mask, a.decay, g_decay, c->decay_dtype, c->per_head != 0, !c->s_in, sums, c->T, c->B, c->H, st);
}

extern "C" int rfa_decay_step(const rfa_decay_t* c, void* out, float* s, rfa_stream_t stream) {
  using namespace rfa;
  if (int r = decay_check(c, "decay_step")) return r;
  RFA_REQUIRE(out && s, RFA_EINVAL, "decay_step: null pointer");
  RFA_REQUIRE(c->T == 1, RFA_EINVAL, "decay_step: %lld tokens", (long long)c->T);
  RFA_REQUIRE(aligned16(s), RFA_EALIGN, "decay_step: s is not 16-byte aligned");
  return launch_decay_step(*c, out, s, as_stream(stream));
}
