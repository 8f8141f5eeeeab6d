// Group norm of rows with SiLU on a gate or on itself: each run of C / groups adjacent channels of a row is brought to mean 0 and variance 1,
// n = xhat w + bias, y = n silu(gate) or silu(n); and its gradients
//   gx = rstd (h - mean(h) - xhat mean(h xhat)), h = gn w,  gw = sum over rows of gn xhat,  gbias = sum of gn,  ggate = g n silu'(gate).
//
// Bound by memory: x and gate once, y once (backward: x, gate, g; gx, ggate); 8 x 2048 tokens x 2048 channels in groups of 64, bf16, forward:
// 41 us, 4.9 TB/s of 6.5 (issue slots are 73 % busy; a launch of one row per thread, with weight and bias read for each, took 60 us).
// Backward, 16 x 1531 x 2048: 113 us, 77 of memory for its five passes (issue slots 72 %, two CTAs an SM by registers).
// A group stays in the registers of 1 to 512 threads, with 16-byte
// words where the sizes allow; threads keep their channels, and weight and bias, over many rows, the next of which is on the way; mean and variance are two passes over registers (no difference of squares), joined by
// shuffles, beyond a warp through shared memory.  The backward forms the statistics again rather than reading them; the
// weights' gradients stay in registers until a CTA's end, and sum_parts adds the CTAs' up.
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
  int size, groups_here, rows_here;      // channels of a group; groups and rows side by side in a CTA
  float over_size;                       // 1 / size
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

// A thread's elements of a group: vectors first + i * TPG of NV elements; NV > 2: in wide accesses, and whole (NV divides the group).
template <typename T, int NV, int V, int TPG> struct NormPart {
  static constexpr bool kWide = NV > 2;
  int first;
  __device__ NormPart() : first(threadIdx.x % TPG) {}
  __device__ __forceinline__ int at(int i) const { return (first + i * TPG) * NV; }
  __device__ __forceinline__ void load(const T* p, int size, Raw<T, NV>* r) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (kWide) {
        r[i].zero();
        if (at(i) < size) r[i].load(p + at(i), NV, true);
      } else {
        r[i].load(p + at(i), size - at(i), false);
      }
    }
  }
  __device__ __forceinline__ void store(T* p, int i, int size, const Raw<T, NV>& r) const {
    if (!kWide) r.store(p + at(i), size - at(i), false);
    else if (at(i) < size) r.store(p + at(i), NV, true);
  }
  __device__ __forceinline__ void floats(const T* p, int size, float none, float* v) const {
    Raw<T, NV> r[V];
    if (p) load(p, size, r);
#pragma unroll
    for (int k = 0; k < V * NV; ++k) v[k] = p ? r[k / NV].get(k % NV) : none;
  }
};

// x -> x - mean (0 beyond the group's end); returns 1 / sqrt(variance + eps)
template <int NV, int V, int TPG> __device__ __forceinline__ float centre(float* x, int first, int size, float over_size, float eps, float (*red)[1]) {
  const bool full = size == TPG * V * NV;              // for all threads: nothing lies beyond the end
  float sum[1] = {0.f};
#pragma unroll
  for (int i = 0; i < V * NV; ++i) sum[0] += x[i];     // zeros beyond the end
  group_sum<TPG, 1>(sum, red);
  const float mean = sum[0] * over_size;
  float var[1] = {0.f};
#pragma unroll
  for (int k = 0; k < V * NV; ++k) x[k] -= mean;
  if (!full) {
#pragma unroll
    for (int k = 0; k < V * NV; ++k)
      if ((first + k / NV * TPG) * NV + k % NV >= size) x[k] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < V * NV; ++k) var[0] = fmaf(x[k], x[k], var[0]);
  group_sum<TPG, 1>(var, red);
  return rsqrtf(fmaf(var[0], over_size, eps));
}

// Rows r0 + row0, r0 + row0 + step ... of one group: what a thread of either kernel walks, the next row on the way while one is worked on.
struct NormPlace {
  int group, row0, c0;
  bool mine;
  __device__ NormPlace(const NormArgs& a, int tpg) {
    const int sub = threadIdx.x / tpg;
    group = blockIdx.x * a.groups_here + sub % a.groups_here;
    row0 = sub / a.groups_here;
    mine = group < a.p.groups && row0 < a.rows_here;
    c0 = mine ? group * a.size : 0;
  }
};

template <typename T, int NV, int V, int TPG>
__global__ void __launch_bounds__(norm_threads(TPG)) norm_fwd_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[32][1];
  const rfa_group_norm_t& p = a.p;
  const NormPart<T, NV, V, TPG> part;
  const NormPlace at(a, TPG);
  float w[V * NV], bias[V * NV];
  part.floats(p.weight ? static_cast<const T*>(p.weight) + at.c0 : nullptr, at.mine ? a.size : 0, 1.f, w);
  part.floats(p.bias ? static_cast<const T*>(p.bias) + at.c0 : nullptr, at.mine ? a.size : 0, 0.f, bias);
  const int64_t step = (int64_t)gridDim.y * a.rows_here;
  int64_t row = (int64_t)blockIdx.y * a.rows_here + at.row0;
  const T* px = static_cast<const T*>(p.x) + row * p.x_r + at.c0;
  const T* pg = p.gate ? static_cast<const T*>(p.gate) + row * p.gate_r + at.c0 : nullptr;
  T* py = static_cast<T*>(a.y) + row * p.C + at.c0;
  Raw<T, NV> next_x[V], next_g[V];
  int next_size = 0;
  const auto ask = [&]() {
    next_size = at.mine && row < p.rows ? a.size : 0;
    part.load(px, next_size, next_x);
    if (p.gate) part.load(pg, next_size, next_g);
    px += step * p.x_r;
    if (p.gate) pg += step * p.gate_r;
    row += step;
  };
  ask();
  for (int64_t r0 = (int64_t)blockIdx.y * a.rows_here; r0 < p.rows; r0 += step, py += step * p.C) {
    const int size = next_size;
    float x[V * NV];
    Raw<T, NV> rg[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      rg[i] = next_g[i];
#pragma unroll
      for (int c = 0; c < NV; ++c) x[i * NV + c] = next_x[i].get(c);
    }
    ask();
    const float rstd = centre<NV, V, TPG>(x, part.first, a.size, a.over_size, p.eps, red);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float n[NV], v[NV];                              // v: what the activation is of, then the result (branches that a call takes one way)
#pragma unroll
      for (int c = 0; c < NV; ++c) n[c] = fmaf(x[i * NV + c] * rstd, w[i * NV + c], bias[i * NV + c]);
      if (p.gate) {
#pragma unroll
        for (int c = 0; c < NV; ++c) v[c] = rg[i].get(c);
      } else {
#pragma unroll
        for (int c = 0; c < NV; ++c) v[c] = n[c];
      }
      if (p.silu) {
#pragma unroll
        for (int c = 0; c < NV; ++c) v[c] *= sigmoid(v[c]);
      }
      if (p.gate) {
#pragma unroll
        for (int c = 0; c < NV; ++c) v[c] *= n[c];
      }
      Raw<T, NV> out;
#pragma unroll
      for (int c = 0; c < NV; c += 2) out.set2(c / 2, v[c], v[c + 1]);
      part.store(py, i, size, out);
    }
  }
}

template <typename T, int NV, int V, int TPG>
__global__ void __launch_bounds__(norm_threads(TPG)) norm_bwd_kernel(const __grid_constant__ NormArgs a) {
  constexpr int E = V * NV;
  __shared__ float red[32][1], red2[32][2], over_rows[norm_threads(TPG)];
  const rfa_group_norm_t& p = a.p;
  const NormPart<T, NV, V, TPG> part;
  const NormPlace at(a, TPG);
  float w[E], dw[E], db[E];
  part.floats(p.weight ? static_cast<const T*>(p.weight) + at.c0 : nullptr, at.mine ? a.size : 0, 1.f, w);
  Raw<T, NV> bias[V];
#pragma unroll
  for (int i = 0; i < V; ++i) bias[i].zero();
  if (p.bias) part.load(static_cast<const T*>(p.bias) + at.c0, at.mine ? a.size : 0, bias);
#pragma unroll
  for (int k = 0; k < E; ++k) dw[k] = db[k] = 0.f;
  const int64_t step = (int64_t)gridDim.y * a.rows_here;
  int64_t row = (int64_t)blockIdx.y * a.rows_here + at.row0;
  const T* px = static_cast<const T*>(p.x) + row * p.x_r + at.c0;
  const T* pu = static_cast<const T*>(a.g) + row * a.g_r + at.c0;
  const T* pg = p.gate ? static_cast<const T*>(p.gate) + row * p.gate_r + at.c0 : nullptr;
  int64_t out = row * p.C + at.c0;
  Raw<T, NV> next_x[V], next_u[V], next_g[V];
  int next_size = 0;
  const auto ask = [&]() {
    next_size = at.mine && row < p.rows ? a.size : 0;
    part.load(px, next_size, next_x);
    part.load(pu, next_size, next_u);
    if (p.gate) part.load(pg, next_size, next_g);
    px += step * p.x_r;
    pu += step * a.g_r;
    if (p.gate) pg += step * p.gate_r;
    row += step;
  };
  ask();
  for (int64_t r0 = (int64_t)blockIdx.y * a.rows_here; r0 < p.rows; r0 += step, out += step * p.C) {
    const int size = next_size;
    float x[E], h[E];
    Raw<T, NV> ru[V], rz[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      ru[i] = next_u[i];
      rz[i] = next_g[i];
#pragma unroll
      for (int c = 0; c < NV; ++c) x[i * NV + c] = next_x[i].get(c);
    }
    ask();
    float rstd = centre<NV, V, TPG>(x, part.first, a.size, a.over_size, p.eps, red);
    if (!size) rstd = 0.f;                             // no such row: without a variance, and eps may be 0
    float sums[2] = {};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float n[NV], act[NV], slope[NV], gn[NV];         // act, slope: the activation and its derivative (branches that a call takes one way)
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        x[i * NV + c] *= rstd;
        n[c] = fmaf(x[i * NV + c], w[i * NV + c], bias[i].get(c));
        gn[c] = ru[i].get(c);
      }
      if (p.gate) {
#pragma unroll
        for (int c = 0; c < NV; ++c) act[c] = rz[i].get(c);
      } else {
#pragma unroll
        for (int c = 0; c < NV; ++c) act[c] = n[c];
      }
      if (p.silu) {
#pragma unroll
        for (int c = 0; c < NV; ++c) {
          const float sig = sigmoid(act[c]);
          act[c] *= sig;
          slope[c] = fmaf(act[c], 1.f - sig, sig);
        }
      } else {
#pragma unroll
        for (int c = 0; c < NV; ++c) slope[c] = 1.f;
      }
      if (p.gate) {
        if (a.g_gate) {
          Raw<T, NV> o;
#pragma unroll
          for (int c = 0; c < NV; c += 2) o.set2(c / 2, gn[c] * n[c] * slope[c], gn[c + 1] * n[c + 1] * slope[c + 1]);
          part.store(static_cast<T*>(a.g_gate) + out, i, size, o);
        }
#pragma unroll
        for (int c = 0; c < NV; ++c) gn[c] *= act[c];
      } else {
#pragma unroll
        for (int c = 0; c < NV; ++c) gn[c] *= slope[c];
      }
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const int k = i * NV + c;
        db[k] += gn[c];
        dw[k] = fmaf(gn[c], x[k], dw[k]);
        h[k] = gn[c] * w[k];
        sums[0] += h[k];
        sums[1] = fmaf(h[k], x[k], sums[1]);
      }
    }
    group_sum<TPG, 2>(sums, red2);
    const float mh = sums[0] * a.over_size, mhx = sums[1] * a.over_size;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      Raw<T, NV> o;
#pragma unroll
      for (int c = 0; c < NV; c += 2) {
        const int k = i * NV + c;
        o.set2(c / 2, rstd * (h[k] - fmaf(x[k], mhx, mh)), rstd * (h[k + 1] - fmaf(x[k + 1], mhx, mh)));
      }
      part.store(static_cast<T*>(a.gx) + out, i, size, o);
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
        if (at.row0 == 0)
          for (int r = 1; r < a.rows_here; ++r) v += over_rows[threadIdx.x + r * a.groups_here * TPG];
      }
      const int c = part.at(k / NV) + k % NV;
      if (at.mine && at.row0 == 0 && c < a.size) (pass ? a.part_b : a.part_w)[(size_t)blockIdx.y * p.C + at.c0 + c] = v;
    }
  }
}

// The groups and rows that a CTA takes side by side, and how many CTAs share the rows.
//
// Threads of a group: as many as it has vectors up to 32, then 32 for up to 128 vectors (2 or 4 a thread), 128 for up to 512, 512 beyond.
// us forward / backward of 16 x 1531 x 2048 elements, the rule and (in brackets) other threads, vectors of 8 elements in bf16:
//   512 channels, 64 vectors     32 threads 68 / 160 (128: 128 / 247)      2048, 256 vectors    128 threads 69 / 144 (32: 103 / 613, 512: 144 / 338)
//   1024, 128 vectors            32 threads 81 / 220 (128: 68 / 134)       4096, 512 vectors    128 threads 77 / 195 (512: 78 / 193)
//   256: 65 / 133    64: 63 / 130    8192: 87 / 239    16384: 100 / 763
// and of 4 elements in fp32:
//   512, 128 vectors             32 threads 99 / 200 (128: 105 / 213)      1024, 256 vectors    128 threads 118 / 175 (32: 104 / 405)
//   2048, 512 vectors            128 threads 99 / 189 (512: 127 / 273)     64: 105 / 214    4096: 128 / 201    16384: 220 / 1232
// What a thread holds decides: up to 16 elements stay in 255 registers; with 32 the backward spills (in 16 bits 168 bytes for 513 to 1024 channels,
// where 128 threads would be the better rule, 160 for 2049 to 4096).  512 threads have 128 registers: 250 bytes above 4096 channels, 2 KB above
// 8192; fp32 0.6 and 2.9 KB.
struct NormGrid {
  int nv, tpg, v, groups_here, rows_here, x, y;
};
NormGrid norm_grid(int64_t rows, int C, int groups, int nv, bool backward) {
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
  const int64_t most = (rows + s.rows_here - 1) / s.rows_here, ctas = 148 * (backward ? 4 : 8), want = ctas / s.x > 1 ? ctas / s.x : 1;
  s.y = (int)(most < want ? most : want);
  return s;
}

template <typename T, int NV, int V, int TPG> int norm_launch(const NormArgs& a, const NormGrid& s, cudaStream_t stream) {
  constexpr int threads = norm_threads(TPG);
  if (a.g) norm_bwd_kernel<T, NV, V, TPG><<<dim3(s.x, s.y), threads, 0, stream>>>(a);
  else norm_fwd_kernel<T, NV, V, TPG><<<dim3(s.x, s.y), threads, 0, stream>>>(a);
  return check_launch(a.g ? "group_norm_bwd" : "group_norm_fwd");
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
  RFA_REQUIRE(p.C <= kMaxChannels, RFA_EUNSUPPORTED, "%s: %d channels", what, p.C);
  a.size = p.C / p.groups;
  const int bytes = p.dtype == RFA_F32 ? 4 : 2, nv = bytes == 2 ? 8 : 4;
  a.over_size = 1.f / (float)a.size;
  const bool wide = a.size % nv == 0 && wide_ok(p.x, p.x_r, p.C, bytes, nv) && wide_ok(p.gate, p.gate ? p.gate_r : 0, 0, bytes, nv) && wide_ok(a.y, 0, 0, bytes, nv) &&
           wide_ok(p.weight, 0, 0, bytes, nv) && wide_ok(p.bias, 0, 0, bytes, nv) && wide_ok(a.g, a.g_r, 0, bytes, nv) && wide_ok(a.gx, 0, 0, bytes, nv) &&
           wide_ok(a.g_gate, 0, 0, bytes, nv);
  const NormGrid s = norm_grid(p.rows, p.C, p.groups, wide ? nv : 2, a.g);
  a.groups_here = s.groups_here; a.rows_here = s.rows_here;
  if (g_weight || g_bias) {
    const size_t need = rfa_group_norm_workspace_bytes(p.rows, p.C, p.groups);
    RFA_REQUIRE(workspace && workspace_bytes >= need, RFA_EWORKSPACE, "%s: workspace %zu bytes, %zu needed", what, workspace_bytes, need);
    a.part_w = static_cast<float*>(workspace);
    a.part_b = a.part_w + (size_t)s.y * p.C;
  }
  int r;
  if (p.dtype == RFA_F32) r = wide ? norm_shape<float, 4>(a, s, stream) : norm_shape<float, 2>(a, s, stream);
  else if (p.dtype == RFA_F16) r = wide ? norm_shape<__half, 8>(a, s, stream) : norm_shape<__half, 2>(a, s, stream);
  else r = wide ? norm_shape<__nv_bfloat16, 8>(a, s, stream) : norm_shape<__nv_bfloat16, 2>(a, s, stream);
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
    const NormGrid s = norm_grid(rows, C, groups, nv, true);
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
