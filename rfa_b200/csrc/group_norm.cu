// Group norm of rows with SiLU on a gate or on itself: each run of C / groups adjacent channels of a row is brought to mean 0 and variance 1,
// n = xhat w + bias, y = n silu(gate) or silu(n); and its gradients
//   gx = rstd (h - mean(h) - xhat mean(h xhat)), h = gn w,  gw = sum over rows of gn xhat,  gbias = sum of gn,  ggate = g n silu'(gate).
//
// Bound by memory: x and gate once, y once (backward: x, gate, g; gx, ggate).  A group stays in the registers of 1 to 512 threads, with 16-byte
// words where the sizes allow; mean and variance are two passes over registers (no difference of squares), joined by
// shuffles, beyond a warp through shared memory.  The backward forms the statistics again rather than reading them; its threads keep
// their channels over many rows, so that the weights' gradients stay in registers until a CTA's end, and sum_parts adds the CTAs' up.
#include "state_space.cuh"

namespace rfa {
namespace {

struct NormArgs {
  rfa_group_norm_t p;
  void* y;
  const void* g;
  int64_t g_r;
  void *gx, *g_gate;
  float *part_w, *part_b;      // [gridDim.y][C] each
  int size, groups_here, rows_here;      // channels of a group; groups and rows side by side in a CTA of the backward
  bool wide;
};

// Sum over the `TPG` threads of a group; K values at once.
template <int TPG, int K> __device__ __forceinline__ void group_sum(float* v, float (*red)[K]) {
#pragma unroll
  for (int o = (TPG < 32 ? TPG : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (TPG > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();                                   // the last sum's reads
    if (lane == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) red[warp][k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int i = 0; i < TPG / 32; ++i) v[k] += red[i][k];
    }
  }
}

constexpr int norm_threads(int tpg) { return tpg > 256 ? tpg : tpg > 32 ? tpg : 256; }

// A thread's elements of a group: vectors first + i * TPG of NV elements.
template <typename T, int NV, int V, int TPG> struct NormPart {
  int first;
  __device__ NormPart() : first(threadIdx.x % TPG) {}
  __device__ __forceinline__ int at(int i) const { return (first + i * TPG) * NV; }
  __device__ __forceinline__ void load(const T* p, int size, bool wide, Raw<T, NV>* r) const {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i].load(p + at(i), size - at(i), wide);
  }
  __device__ __forceinline__ void floats(const T* p, int size, bool wide, float none, float* v) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (p) {
        Raw<T, NV> r;
        r.load(p + at(i), size - at(i), wide);
#pragma unroll
        for (int c = 0; c < NV; ++c) v[i * NV + c] = r.get(c);
      } else {
#pragma unroll
        for (int c = 0; c < NV; ++c) v[i * NV + c] = none;
      }
    }
  }
};

// x -> x - mean (0 beyond the group's end); returns 1 / sqrt(variance + eps)
template <int NV, int V, int TPG> __device__ __forceinline__ float centre(float* x, int first, int size, float eps, float (*red)[1]) {
  float sum[1] = {0.f};
#pragma unroll
  for (int i = 0; i < V * NV; ++i) sum[0] += x[i];     // zeros beyond the end
  group_sum<TPG, 1>(sum, red);
  const float mean = sum[0] / (float)size;
  float var[1] = {0.f};
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      float& v = x[i * NV + c];
      v = (first + i * TPG) * NV + c < size ? v - mean : 0.f;
      var[0] = fmaf(v, v, var[0]);
    }
  group_sum<TPG, 1>(var, red);
  return rsqrtf(var[0] / (float)size + eps);
}

template <typename T, int NV, int V, int TPG>
__global__ void __launch_bounds__(norm_threads(TPG)) norm_fwd_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[32][1];
  const rfa_group_norm_t& p = a.p;
  const NormPart<T, NV, V, TPG> part;
  const int64_t items = p.rows * p.groups, item = (int64_t)blockIdx.x * (blockDim.x / TPG) + threadIdx.x / TPG;
  const bool there = item < items;
  int64_t row = 0;
  int group = 0;
  if (there) {
    if (items < (int64_t)1 << 31) { row = (uint32_t)item / (uint32_t)p.groups; group = (uint32_t)item % (uint32_t)p.groups; }
    else { row = item / p.groups; group = (int)(item % p.groups); }
  }
  const int c0 = group * a.size, size = there ? a.size : 0;
  Raw<T, NV> rx[V], rg[V];
  part.load(static_cast<const T*>(p.x) + row * p.x_r + c0, size, a.wide, rx);
  if (p.gate) part.load(static_cast<const T*>(p.gate) + row * p.gate_r + c0, size, a.wide, rg);
  float x[V * NV], w[V * NV], bias[V * NV];
  part.floats(p.weight ? static_cast<const T*>(p.weight) + c0 : nullptr, size, a.wide, 1.f, w);
  part.floats(p.bias ? static_cast<const T*>(p.bias) + c0 : nullptr, size, a.wide, 0.f, bias);
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int c = 0; c < NV; ++c) x[i * NV + c] = rx[i].get(c);
  const float rstd = centre<NV, V, TPG>(x, part.first, a.size, p.eps, red);
  T* y = static_cast<T*>(a.y) + row * p.C + c0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    Raw<T, NV> out;
    out.zero();
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int k = i * NV + c;
      const float n = fmaf(x[k] * rstd, w[k], bias[k]), by = p.gate ? rg[i].get(c) : n;
      const float act = p.silu ? by * sigmoid(by) : by;
      out.set(c, from_f<T>(p.gate ? n * act : act));
    }
    out.store(y + part.at(i), size - part.at(i), a.wide);
  }
}

template <typename T, int NV, int V, int TPG>
__global__ void __launch_bounds__(norm_threads(TPG)) norm_bwd_kernel(const __grid_constant__ NormArgs a) {
  constexpr int E = V * NV;
  __shared__ float red[32][1], red2[32][2], over_rows[norm_threads(TPG)];
  const rfa_group_norm_t& p = a.p;
  const NormPart<T, NV, V, TPG> part;
  const int sub = threadIdx.x / TPG, group = blockIdx.x * a.groups_here + sub % a.groups_here, row0 = sub / a.groups_here;
  const bool mine = group < p.groups && row0 < a.rows_here;
  const int c0 = mine ? group * a.size : 0;
  float w[E], dw[E], db[E];
  part.floats(p.weight ? static_cast<const T*>(p.weight) + c0 : nullptr, mine ? a.size : 0, a.wide, 1.f, w);
#pragma unroll
  for (int k = 0; k < E; ++k) dw[k] = db[k] = 0.f;
  const int64_t step = (int64_t)gridDim.y * a.rows_here;
  for (int64_t r0 = (int64_t)blockIdx.y * a.rows_here; r0 < p.rows; r0 += step) {
    const int64_t row = r0 + row0;
    const int size = mine && row < p.rows ? a.size : 0;
    Raw<T, NV> rx[V], rg[V], rz[V];
    part.load(static_cast<const T*>(p.x) + row * p.x_r + c0, size, a.wide, rx);
    part.load(static_cast<const T*>(a.g) + row * a.g_r + c0, size, a.wide, rg);
    if (p.gate) part.load(static_cast<const T*>(p.gate) + row * p.gate_r + c0, size, a.wide, rz);
    float x[E], h[E];
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int c = 0; c < NV; ++c) x[i * NV + c] = rx[i].get(c);
    const float rstd = centre<NV, V, TPG>(x, part.first, a.size, p.eps, red);
    float sums[2] = {};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      Raw<T, NV> bias, out;
      bias.zero();
      out.zero();
      if (p.bias) bias.load(static_cast<const T*>(p.bias) + c0 + part.at(i), size - part.at(i), a.wide);
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const int k = i * NV + c;
        const float xn = x[k] * rstd, n = fmaf(xn, w[k], bias.get(c)), g = rg[i].get(c);
        const float by = p.gate ? rz[i].get(c) : n, sig = p.silu ? sigmoid(by) : 1.f;
        const float slope = p.silu ? fmaf(by * sig, 1.f - sig, sig) : 1.f;      // of the activation
        const float gn = p.gate ? g * (by * sig) : g * slope;
        if (p.gate) out.set(c, from_f<T>(g * n * slope));
        db[k] += gn;
        dw[k] = fmaf(gn, xn, dw[k]);
        x[k] = xn;
        h[k] = gn * w[k];
        sums[0] += h[k];
        sums[1] = fmaf(h[k], xn, sums[1]);
      }
      if (p.gate && a.g_gate) out.store(static_cast<T*>(a.g_gate) + row * p.C + c0 + part.at(i), size - part.at(i), a.wide);
    }
    group_sum<TPG, 2>(sums, red2);
    const float mh = sums[0] / (float)a.size, mhx = sums[1] / (float)a.size;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      Raw<T, NV> out;
      out.zero();
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const int k = i * NV + c;
        out.set(c, from_f<T>(rstd * (h[k] - fmaf(x[k], mhx, mh))));
      }
      out.store(static_cast<T*>(a.gx) + row * p.C + c0 + part.at(i), size - part.at(i), a.wide);
    }
  }
  if (!a.part_w) return;
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int k = 0; k < E; ++k) {
      float v = pass ? db[k] : dw[k];
      if (a.rows_here > 1) {
        __syncthreads();
        over_rows[threadIdx.x] = v;
        __syncthreads();
        if (row0 == 0)
          for (int r = 1; r < a.rows_here; ++r) v += over_rows[threadIdx.x + r * a.groups_here * TPG];
      }
      const int at = part.at(k / NV) + k % NV;
      if (mine && row0 == 0 && at < a.size) (pass ? a.part_b : a.part_w)[(size_t)blockIdx.y * p.C + c0 + at] = v;
    }
  }
}

// The rows that one CTA of the backward takes side by side, and how many CTAs share the rows.
struct NormGrid {
  int nv, tpg, v, groups_here, rows_here, x, y;
};
NormGrid norm_grid(int64_t rows, int C, int groups, int nv) {
  NormGrid s{};
  s.nv = nv;
  const int n = (C / groups + nv - 1) / nv;            // vectors of a group
  s.tpg = 1; s.v = 1;
  if (n <= 32) while (s.tpg < n) s.tpg *= 2;
  else s.tpg = n <= 128 ? 32 : n <= 512 ? 128 : 512;
  while (s.tpg * s.v < n) s.v *= 2;
  const int subs = norm_threads(s.tpg) / s.tpg;
  s.groups_here = groups < subs ? groups : subs;
  s.rows_here = subs / s.groups_here;
  s.x = (groups + s.groups_here - 1) / s.groups_here;
  const int64_t most = (rows + s.rows_here - 1) / s.rows_here, want = 148 * 4 / s.x > 1 ? 148 * 4 / s.x : 1;
  s.y = (int)(most < want ? most : want);
  return s;
}

template <typename T, int NV, int V, int TPG> int norm_launch(const NormArgs& a, const NormGrid& s, cudaStream_t stream) {
  constexpr int threads = norm_threads(TPG);
  if (a.g) {
    norm_bwd_kernel<T, NV, V, TPG><<<dim3(s.x, s.y), threads, 0, stream>>>(a);
    return check_launch("group_norm_bwd");
  }
  const int64_t blocks = (a.p.rows * a.p.groups + threads / TPG - 1) / (threads / TPG);
  RFA_REQUIRE(blocks < (int64_t)1 << 31, RFA_EUNSUPPORTED, "group_norm_fwd: too many rows");
  norm_fwd_kernel<T, NV, V, TPG><<<(unsigned)blocks, threads, 0, stream>>>(a);
  return check_launch("group_norm_fwd");
}
template <typename T, int NV> int norm_shape(const NormArgs& a, const NormGrid& s, cudaStream_t stream) {
  switch (s.tpg * 32 + s.v) {
#define CASE(TPG, V) case TPG * 32 + V: return norm_launch<T, NV, V, TPG>(a, s, stream);
    CASE(1, 1) CASE(2, 1) CASE(4, 1) CASE(8, 1) CASE(16, 1) CASE(32, 1) CASE(32, 2) CASE(32, 4) CASE(128, 2) CASE(128, 4) CASE(512, 2) CASE(512, 4)
#undef CASE
    case 512 * 32 + 8:
      if constexpr (NV <= 4) return norm_launch<T, NV, 8, 512>(a, s, stream);
      break;
    case 512 * 32 + 16:
      if constexpr (NV <= 2) return norm_launch<T, NV, 16, 512>(a, s, stream);
      break;
  }
  return fail(RFA_EUNSUPPORTED, "group_norm: groups of %d channels", a.size);
}

int norm_run(NormArgs a, const char* what, void* workspace, size_t workspace_bytes, void* g_weight, void* g_bias, cudaStream_t stream) {
  const rfa_group_norm_t& p = a.p;
  RFA_REQUIRE(p.x, RFA_EINVAL, "%s: null pointer", what);
  RFA_REQUIRE(p.rows > 0 && p.C > 0 && p.groups > 0, RFA_EINVAL, "%s: empty or negative size", what);
  RFA_REQUIRE(p.dtype == RFA_F16 || p.dtype == RFA_F32 || p.dtype == RFA_BF16, RFA_EUNSUPPORTED, "%s: dtype %d", what, p.dtype);
  RFA_REQUIRE(p.C % p.groups == 0 && p.C / p.groups <= 16384, RFA_EUNSUPPORTED, "%s: %d channels in %d groups (of at most 16384)", what, p.C, p.groups);
  a.size = p.C / p.groups;
  const int bytes = p.dtype == RFA_F32 ? 4 : 2, nv = bytes == 2 ? 8 : 4;
  a.wide = a.size % nv == 0 && wide_ok(p.x, p.x_r, 0, bytes, nv) && wide_ok(p.gate, p.gate ? p.gate_r : 0, 0, bytes, nv) && wide_ok(a.y, 0, 0, bytes, nv) &&
           wide_ok(p.weight, 0, 0, bytes, nv) && wide_ok(p.bias, 0, 0, bytes, nv) && wide_ok(a.g, a.g_r, 0, bytes, nv) && wide_ok(a.gx, 0, 0, bytes, nv) &&
           wide_ok(a.g_gate, 0, 0, bytes, nv);
  const NormGrid s = norm_grid(p.rows, p.C, p.groups, a.wide ? nv : 2);
  a.groups_here = s.groups_here; a.rows_here = s.rows_here;
  if (g_weight || g_bias) {
    const size_t need = rfa_group_norm_workspace_bytes(p.rows, p.C, p.groups);
    RFA_REQUIRE(workspace && workspace_bytes >= need, RFA_EWORKSPACE, "%s: workspace %zu bytes, %zu needed", what, workspace_bytes, need);
    a.part_w = static_cast<float*>(workspace);
    a.part_b = a.part_w + (size_t)s.y * p.C;
  }
  int r;
  if (p.dtype == RFA_F32) r = a.wide ? norm_shape<float, 4>(a, s, stream) : norm_shape<float, 2>(a, s, stream);
  else if (p.dtype == RFA_F16) r = a.wide ? norm_shape<__half, 8>(a, s, stream) : norm_shape<__half, 2>(a, s, stream);
  else r = a.wide ? norm_shape<__nv_bfloat16, 8>(a, s, stream) : norm_shape<__nv_bfloat16, 2>(a, s, stream);
  if (r || !a.part_w) return r;
  const SumJob jobs[2] = {{a.part_w, g_weight, p.C, s.y, p.dtype}, {a.part_b, g_bias, p.C, s.y, p.dtype}};
  return sum_parts(jobs, 2, stream);
}

}  // namespace
}  // namespace rfa

extern "C" int rfa_group_norm_fwd(const rfa_group_norm_t* norm, void* y, rfa_stream_t stream) {
  using namespace rfa;
  RFA_REQUIRE(norm && y, RFA_EINVAL, "group_norm_fwd: null pointer");
  NormArgs a{};
  a.p = *norm;
  a.y = y;
  return norm_run(a, "group_norm_fwd", nullptr, 0, nullptr, nullptr, as_stream(stream));
}

extern "C" size_t rfa_group_norm_workspace_bytes(int64_t rows, int C, int groups) {
  using namespace rfa;
  if (rows <= 0 || C <= 0 || groups <= 0 || C % groups) return 0;
  int y = 1;
  for (int nv : {2, 4, 8}) {
    const NormGrid s = norm_grid(rows, C, groups, nv);
    y = s.y > y ? s.y : y;
  }
  return (size_t)2 * y * C * 4;
}

extern "C" int rfa_group_norm_bwd(const rfa_group_norm_t* norm, const void* g, int64_t g_r, void* gx, void* g_gate, void* g_weight, void* g_bias,
                                  void* workspace, size_t workspace_bytes, rfa_stream_t stream) {
  using namespace rfa;
  RFA_REQUIRE(norm && g && gx, RFA_EINVAL, "group_norm_bwd: null pointer");
  RFA_REQUIRE(aligned16(workspace), RFA_EALIGN, "group_norm_bwd: the workspace is not 16-byte aligned");
  NormArgs a{};
  a.p = *norm;
  a.g = g; a.g_r = g_r; a.gx = gx; a.g_gate = g_gate;
  return norm_run(a, "group_norm_bwd", workspace, workspace_bytes, g_weight, g_bias, as_stream(stream));
}
