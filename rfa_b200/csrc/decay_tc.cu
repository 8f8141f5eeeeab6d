// Linear attention with a decay on the tensor cores: plans and launches (the kernel: decay_tc.cuh).
#define RFA_TC_FAMILY 10
#include <cmath>

#include "decay_tc.cuh"

namespace rfa {

namespace {

template <typename T, int KB, int DB, bool OUT, bool EXACT>
int launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const DecayTcArgs& a, bool totals_only, cudaStream_t stream) {
  constexpr uint32_t smem = DecLayout<KB, DB, OUT, EXACT>::bytes;
  cudaError_t e = cudaFuncSetAttribute(decay_tc_kernel<T, KB, DB, OUT, EXACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return fail((int)e, "decay: cannot reserve %u bytes of shared memory: %s", smem, cudaGetErrorString(e));
  e = launch_pdl(decay_tc_kernel<T, KB, DB, OUT, EXACT>, dim3((unsigned)((int64_t)a.B * a.H), a.nseg), dim3(kDecThreads), smem, stream, q, k, v, a, totals_only);
  if (e != cudaSuccess) return fail((int)e, "rfa_decay: launch failed: %s", cudaGetErrorString(e));
  return check_launch("rfa_decay");
}
template <bool OUT, bool EXACT>
int launch_sizes(bool bf16, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const DecayTcArgs& a, bool totals_only, cudaStream_t stream) {
  const int at = (bf16 ? 4 : 0) + (a.K > 64 ? 2 : 0) + (a.D > 64 ? 1 : 0);
  switch (at) {
    case 0: return launch<__half, 1, 1, OUT, EXACT>(q, k, v, a, totals_only, stream);
    case 1: return launch<__half, 1, 2, OUT, EXACT>(q, k, v, a, totals_only, stream);
    case 2: return launch<__half, 2, 1, OUT, EXACT>(q, k, v, a, totals_only, stream);
    case 3: return launch<__half, 2, 2, OUT, EXACT>(q, k, v, a, totals_only, stream);
    case 4: return launch<__nv_bfloat16, 1, 1, OUT, EXACT>(q, k, v, a, totals_only, stream);
    case 5: return launch<__nv_bfloat16, 1, 2, OUT, EXACT>(q, k, v, a, totals_only, stream);
    case 6: return launch<__nv_bfloat16, 2, 1, OUT, EXACT>(q, k, v, a, totals_only, stream);
    default: return launch<__nv_bfloat16, 2, 2, OUT, EXACT>(q, k, v, a, totals_only, stream);
  }
}

}  // namespace

bool decay_tc_ok(const rfa_decay_t& c) {
  return c.dtype != RFA_F32 && c.K <= 128 && c.D <= 128 && tmap_rows_ok(c.q, c.T, c.B, c.H, c.K, c.q_t, c.q_b, c.q_h) &&
         tmap_rows_ok(c.k, c.T, c.B, c.H, c.K, c.k_t, c.k_b, c.k_h) && tmap_rows_ok(c.v, c.T, c.B, c.H, c.D, c.v_t, c.v_b, c.v_h);
}

SweepPlan decay_tc_plan(int64_t T, int64_t BH, int K, int D) {
  const int64_t chunks = (T + kTC - 1) / kTC;
  // Chunks that an SM goes through one after the other, the reading of keys and values for the segments' own states counted as 0.6 of a chunk, and a few chunks'
  // time for two more launches
  int64_t best = (BH + 147) / 148 * chunks * 10, best_n = 1;
  for (int64_t n = 2; n <= 64 && n * 2 <= chunks && BH <= 148; ++n) {
    const int64_t cost = (BH * n + 147) / 148 * ((chunks + n - 1) / n) * 16 + 60;
    if (cost < best) { best = cost; best_n = n; }
  }
  SweepPlan p{1, T, 0, 0};
  if (best_n == 1) return p;
  p.tseg = (chunks + best_n - 1) / best_n * kTC;
  p.nseg = (int)((T + p.tseg - 1) / p.tseg);
  p.totals = sizeof(float) * p.nseg * BH * K * D;
  p.seg_decay = sizeof(double) * p.nseg * BH;
  return p;
}

namespace {

// the sweep over segments where there are several: their own states, the states in front of each, then the sweep itself
template <bool OUT>
int sweep(bool bf16, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const DecayTcArgs& a, bool exact, cudaStream_t stream) {
  if (a.nseg > 1) {
    DecayTcArgs own = a;
    own.kept = nullptr;
    if (int r = exact ? launch_sizes<false, true>(bf16, q, k, v, own, true, stream) : launch_sizes<false, false>(bf16, q, k, v, own, true, stream)) return r;
    if (int r = launch_decay_combine(a.totals, a.seg_decay, a.s_in, a.nseg, (int64_t)a.B * a.H, a.K, a.D, stream)) return r;
  }
  return exact ? launch_sizes<OUT, true>(bf16, q, k, v, a, false, stream) : launch_sizes<OUT, false>(bf16, q, k, v, a, false, stream);
}
DecayTcArgs sweep_args(const rfa_decay_t& c, const SweepPlan& plan, char* workspace) {
  DecayTcArgs a{};
  a.decay = {c.log_decay, c.g_t, c.g_b, c.g_h};
  a.mask = c.mask;
  a.totals = reinterpret_cast<float*>(workspace);
  a.seg_decay = reinterpret_cast<double*>(workspace + ((plan.totals + 255) & ~(size_t)255));
  a.T = c.T; a.tseg = plan.tseg;
  a.B = c.B; a.H = c.H; a.K = c.K; a.D = c.D; a.nseg = plan.nseg; a.decay_dtype = c.decay_dtype;
  return a;
}
size_t kept_bytes(int64_t T, int64_t BH, int K, int D) { return (size_t)((T + kTC - 1) / kTC) * BH * (K > 64 ? 2 : 1) * (D > 64 ? 2 : 1) * 64 * 128; }

}  // namespace

size_t decay_tc_bwd_bytes(const rfa_decay_t& c) {
  const int64_t BH = (int64_t)c.B * c.H;
  const SweepPlan plan = decay_tc_plan(c.T, BH, c.K, c.D);
  return ((plan.totals + 255) & ~(size_t)255) + ((plan.seg_decay + 255) & ~(size_t)255) + 2 * kept_bytes(c.T, BH, c.K, c.D) + sizeof(float) * BH * ((c.T + kTC - 1) / kTC);
}

size_t decay_tc_kept_bytes(int64_t T, int64_t BH, int K, int D) { return kept_bytes(T, BH, K, D); }

int launch_decay_tc_bwd(const rfa_decay_t& c, char* workspace, const void* kept, const void* g, const float* g_s, void* gq, void* gk, void* gv, void* g_decay, float* gs_in, cudaStream_t stream) {
  const bool bf16 = c.dtype == RFA_BF16;
  const int64_t BH = (int64_t)c.B * c.H, row = (int64_t)c.H * c.D, chunks = (c.T + kTC - 1) / kTC;
  CUtensorMap q, k, v, gm;
  if (make_tmap_heads(&q, c.q, bf16, c.T, c.B, c.H, c.K, c.q_t, c.q_b, c.q_h, kTC) || make_tmap_heads(&k, c.k, bf16, c.T, c.B, c.H, c.K, c.k_t, c.k_b, c.k_h, kTC) ||
      make_tmap_heads(&v, c.v, bf16, c.T, c.B, c.H, c.D, c.v_t, c.v_b, c.v_h, kTC) || make_tmap_heads(&gm, g, bf16, c.T, c.B, c.H, c.D, c.B * row, row, c.D, kTC))
    return fail(RFA_EDEVICE, "decay_bwd: cuTensorMapEncodeTiled failed or is unavailable");
  const SweepPlan plan = decay_tc_plan(c.T, BH, c.K, c.D);
  char* states = workspace + ((plan.totals + 255) & ~(size_t)255) + ((plan.seg_decay + 255) & ~(size_t)255);
  char* grads = states + kept_bytes(c.T, BH, c.K, c.D);
  float* sums = reinterpret_cast<float*>(grads + kept_bytes(c.T, BH, c.K, c.D));
  DecayTcArgs a = sweep_args(c, plan, workspace);
  if (!kept) {      // the states in front of the chunks once more
    a.in_scale = 1.f;
    a.s_in = {const_cast<float*>(c.s_in), c.D, 1};
    a.kept = states;
    if (int r = sweep<false>(bf16, q, k, v, a, false, stream)) return r;
  }
  a.in_scale = c.scale;
  a.rev = 1;
  a.s_in = {const_cast<float*>(g_s), c.D, 1};
  a.s_out = {gs_in, c.D, 1};
  a.kept = grads;
  if (int r = sweep<false>(bf16, q, q, gm, a, gs_in != nullptr, stream)) return r;
  if (int r = launch_decay_grad_tc(c, q, k, v, gm, kept ? kept : states, grads, gq, gk, gv, g_decay && c.per_head ? sums : g_decay, stream)) return r;
  if (!g_decay || !c.per_head) return 0;
  const SumJob job{sums, g_decay, c.H, (int)(c.B * chunks), c.decay_dtype};
  return sum_parts(&job, 1, stream);
}

int launch_decay_tc(const rfa_decay_t& c, const SweepPlan& plan, char* workspace, void* out, float* s_out, void* kept, cudaStream_t stream) {
  const bool bf16 = c.dtype == RFA_BF16;
  CUtensorMap q, k, v;
  if (make_tmap_heads(&q, c.q, bf16, c.T, c.B, c.H, c.K, c.q_t, c.q_b, c.q_h, kTC) || make_tmap_heads(&k, c.k, bf16, c.T, c.B, c.H, c.K, c.k_t, c.k_b, c.k_h, kTC) ||
      make_tmap_heads(&v, c.v, bf16, c.T, c.B, c.H, c.D, c.v_t, c.v_b, c.v_h, kTC))
    return fail(RFA_EDEVICE, "decay: cuTensorMapEncodeTiled failed or is unavailable");
  DecayTcArgs a = sweep_args(c, plan, workspace);
  a.out = out;
  a.kept = kept;
  a.s_in = {const_cast<float*>(c.s_in), c.D, 1};
  a.s_out = {s_out, c.D, 1};
  a.in_scale = 1.f;
  a.out_scale = c.scale;
  a.p_scale = std::fabs(c.scale) <= 1.f ? c.scale : 1.f;
  a.o_scale = std::fabs(c.scale) <= 1.f ? 1.f : c.scale;
  return sweep<true>(bf16, q, k, v, a, s_out != nullptr, stream);
}

RFA_TC_UNIT(decay)

}  // namespace rfa
