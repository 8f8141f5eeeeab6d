// Sliding-window attention, any sizes and types: fp32 multiply-adds on tiles in shared memory, forward and backward.
//
// 64 rows (queries; in the keys' pass keys) against tiles of 32 of the other side, 256 threads as 16 x 16, a thread 4 rows by 2 columns of a tile of scores and 4
// rows by every 16th column of the results.  Softmax with a running maximum and sum; the backward recomputes the weights from their logarithms' sums, with
// one pass over keys for gq and one over queries for gk and gv, so that no result is added up by two CTAs.  Bound by shared memory's reads.
#include "window.cuh"

namespace rfa {

namespace {

constexpr int kRows = 64, kOther = 32, kThreads = 256;

// `n` rows of a head into shared memory, ld apart; rows that hold no token are zero, whatever stands there
template <typename T>
__device__ __forceinline__ void load_tile(float* dst, int ld, const WindowRows& x, int b, int h, int64_t t0, int n, int64_t T_, int D, const int* num) {
  const T* base = static_cast<const T*>(x.p) + b * x.b + h * x.h;
  for (int i = threadIdx.x; i < n * D; i += kThreads) {
    const int r = i / D, c = i - r * D;
    dst[r * ld + c] = t0 + r < T_ && num[r] >= 0 ? to_f<T>(base[(t0 + r) * x.t + c]) : 0.f;
  }
}

__device__ __forceinline__ float row_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// x rows (4 a thread, 16 apart) times y rows (2, 16 apart)
__device__ __forceinline__ void tile_products(const float* x, const float* y, int ld, int D, int ty, int tx, float (&s)[4][2]) {
#pragma unroll 4
  for (int d = 0; d < D; ++d) {
    const float y0 = y[tx * ld + d], y1 = y[(tx + 16) * ld + d];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float q = x[(ty + 16 * i) * ld + d];
      s[i][0] = fmaf(q, y0, s[i][0]);
      s[i][1] = fmaf(q, y1, s[i][1]);
    }
  }
}
// acc[i][c] += sum_j w[row i][j] y[j][tx + 16 c]
template <int NC>
__device__ __forceinline__ void tile_add(const float* w, const float* y, int ld, int D, int ty, int tx, float (&acc)[4][NC]) {
  for (int j = 0; j < kOther; ++j) {
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = w[(ty + 16 * i) * (kOther + 1) + j];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float v = tx + 16 * c < D ? y[j * ld + tx + 16 * c] : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][c] = fmaf(p[i], v, acc[i][c]);
    }
  }
}

template <typename T, int NC>
__global__ void __launch_bounds__(kThreads) window_fwd_kernel(const __grid_constant__ WindowArgs a) {
  extern __shared__ float tiles_smem[];
  __shared__ int nq[kRows], nk[kOther];
  const int D = a.D, ld = D | 1, tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  float *Q = tiles_smem, *K = Q + kRows * ld, *V = K + kOther * ld, *P = V + kOther * ld;
  const int64_t tiles = (a.T + kRows - 1) / kRows, bh = blockIdx.x / tiles, i0 = blockIdx.x % tiles * kRows, at = a.S - a.T;
  const int b = (int)(bh / a.H), h = (int)(bh % a.H), kv = h / (a.H / a.G);
  const WindowNumbers num(a, b);
  const int rows = (int)min((int64_t)kRows, a.T - i0);
  if (tid < kRows) nq[tid] = tid < rows ? num.at(at + i0 + tid) : -1;
  __syncthreads();
  load_tile<T>(Q, ld, a.q, b, h, i0, kRows, a.T, D, nq);
  const int64_t first = num.first_key(at + i0) / kOther, sink_tiles = (num.first_end() + kOther - 1) / kOther, end = (at + i0 + rows + kOther - 1) / kOther;
  float acc[4][NC] = {}, top[4], sum[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { top[i] = -INFINITY; sum[i] = 0.f; }
  for (int64_t kt = sink_tiles > 0 ? 0 : first; kt < end; kt = kt + 1 < sink_tiles ? kt + 1 : max(kt + 1, first)) {
    __syncthreads();
    if (tid < kOther) nk[tid] = num.at(kt * kOther + tid);
    __syncthreads();
    load_tile<T>(K, ld, a.k, b, kv, kt * kOther, kOther, a.S, D, nk);
    load_tile<T>(V, ld, a.v, b, kv, kt * kOther, kOther, a.S, D, nk);
    __syncthreads();
    float s[4][2] = {};
    tile_products(Q, K, ld, D, ty, tx, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = nq[ty + 16 * i];
#pragma unroll
      for (int c = 0; c < 2; ++c) s[i][c] = window_sees(n, nk[tx + 16 * c], a.window, a.sinks) ? s[i][c] * a.scale : -INFINITY;
      const float now = fmaxf(top[i], row_max(fmaxf(s[i][0], s[i][1]))), ref = now == -INFINITY ? 0.f : now;
      const float keep = expf(top[i] - ref);            // 0 where nothing was seen before
      const float p0 = expf(s[i][0] - ref), p1 = expf(s[i][1] - ref);
      sum[i] = sum[i] * keep + row_sum(p0 + p1);
      top[i] = now;
      P[(ty + 16 * i) * (kOther + 1) + tx] = p0;
      P[(ty + 16 * i) * (kOther + 1) + tx + 16] = p1;
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[i][c] *= keep;
    }
    __syncthreads();
    tile_add<NC>(P, V, ld, D, ty, tx, acc);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty + 16 * i;
    if (r >= rows) continue;
    const float inv = sum[i] > 0.f ? 1.f / sum[i] : 0.f;       // a query that sees nothing (a padded one) has 0
    T* o = static_cast<T*>(a.out) + (((i0 + r) * a.B + b) * a.H + h) * D;
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (tx + 16 * c < D) o[tx + 16 * c] = from_f<T>(nq[r] >= 0 ? acc[i][c] * inv : 0.f);
    if (a.lse && tx == 0) a.lse[bh * a.T + i0 + r] = sum[i] > 0.f ? top[i] + logf(sum[i]) : 0.f;
  }
}

// gq_i = scale sum_j ds_ij k_j, ds = p (g . v - delta), delta_i = g_i . out_i, which is left for the keys' pass
template <typename T, int NC>
__global__ void __launch_bounds__(kThreads) window_gq_kernel(const __grid_constant__ WindowArgs a) {
  extern __shared__ float tiles_smem[];
  __shared__ int nq[kRows], nk[kOther];
  __shared__ float lse[kRows], delta[kRows];
  const int D = a.D, ld = D | 1, tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  float *Q = tiles_smem, *Gr = Q + kRows * ld, *K = Gr + kRows * ld, *V = K + kOther * ld, *P = V + kOther * ld;
  const int64_t tiles = (a.T + kRows - 1) / kRows, bh = blockIdx.x / tiles, i0 = blockIdx.x % tiles * kRows;
  const int b = (int)(bh / a.H), h = (int)(bh % a.H), kv = h / (a.H / a.G);
  const WindowNumbers num(a, b);
  const int rows = (int)min((int64_t)kRows, a.T - i0);
  if (tid < kRows) {
    nq[tid] = tid < rows ? num.at(i0 + tid) : -1;
    lse[tid] = tid < rows ? a.lse[bh * a.T + i0 + tid] : 0.f;
  }
  __syncthreads();
  load_tile<T>(Q, ld, a.q, b, h, i0, kRows, a.T, D, nq);
  load_tile<T>(Gr, ld, a.g, b, h, i0, kRows, a.T, D, nq);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty + 16 * i;
    float d = 0.f;
    if (nq[r] >= 0) {
      const T* o = static_cast<const T*>(a.o.p) + b * a.o.b + h * a.o.h + (i0 + r) * a.o.t;
      for (int c = tx; c < D; c += 16) d = fmaf(Gr[r * ld + c], to_f<T>(o[c]), d);
    }
    d = row_sum(d);
    if (tx == 0) {
      delta[r] = d;
      if (r < rows) a.delta[bh * a.T + i0 + r] = d;
    }
  }
  const int64_t first = num.first_key(i0) / kOther, sink_tiles = (num.first_end() + kOther - 1) / kOther, end = (i0 + rows + kOther - 1) / kOther;
  float acc[4][NC] = {};
  for (int64_t kt = sink_tiles > 0 ? 0 : first; kt < end; kt = kt + 1 < sink_tiles ? kt + 1 : max(kt + 1, first)) {
    __syncthreads();
    if (tid < kOther) nk[tid] = num.at(kt * kOther + tid);
    __syncthreads();
    load_tile<T>(K, ld, a.k, b, kv, kt * kOther, kOther, a.S, D, nk);
    load_tile<T>(V, ld, a.v, b, kv, kt * kOther, kOther, a.S, D, nk);
    __syncthreads();
    float s[4][2] = {}, gp[4][2] = {};
    tile_products(Q, K, ld, D, ty, tx, s);
    tile_products(Gr, V, ld, D, ty, tx, gp);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = ty + 16 * i;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float p = window_sees(nq[r], nk[tx + 16 * c], a.window, a.sinks) ? expf(s[i][c] * a.scale - lse[r]) : 0.f;
        P[r * (kOther + 1) + tx + 16 * c] = p * (gp[i][c] - delta[r]) * a.scale;
      }
    }
    __syncthreads();
    tile_add<NC>(P, K, ld, D, ty, tx, acc);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty + 16 * i;
    if (r >= rows) continue;
    T* o = static_cast<T*>(a.gq) + (((i0 + r) * a.B + b) * a.H + h) * D;
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (tx + 16 * c < D) o[tx + 16 * c] = from_f<T>(acc[i][c]);
  }
}

// gv_j = sum_i p_ij g_i, gk_j = scale sum_i ds_ij q_i, over the queries and heads that see the key
template <typename T, int NC>
__global__ void __launch_bounds__(kThreads) window_gkv_kernel(const __grid_constant__ WindowArgs a) {
  extern __shared__ float tiles_smem[];
  __shared__ int nq[kOther], nk[kRows];
  __shared__ float lse[kOther], delta[kOther];
  const int D = a.D, ld = D | 1, tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  float *K = tiles_smem, *V = K + kRows * ld, *Q = V + kRows * ld, *Gr = Q + kOther * ld, *P = Gr + kOther * ld, *dS = P + kRows * (kOther + 1);
  const int64_t tiles = (a.S + kRows - 1) / kRows, bg = blockIdx.x / tiles, j0 = blockIdx.x % tiles * kRows;
  const int b = (int)(bg / a.G), kv = (int)(bg % a.G), group = a.H / a.G;
  const WindowNumbers num(a, b);
  const int rows = (int)min((int64_t)kRows, a.S - j0);
  if (tid < kRows) nk[tid] = tid < rows ? num.at(j0 + tid) : -1;
  __syncthreads();
  load_tile<T>(K, ld, a.k, b, kv, j0, kRows, a.S, D, nk);
  load_tile<T>(V, ld, a.v, b, kv, j0, kRows, a.S, D, nk);
  const int64_t first = j0 / kOther, end = (num.last_query(j0, j0 + rows) + kOther - 1) / kOther;
  float gk[4][NC] = {}, gv[4][NC] = {};
  for (int h = kv * group; h < (kv + 1) * group; ++h)
    for (int64_t qt = first; qt < end; ++qt) {
      __syncthreads();
      if (tid < kOther) {
        const int64_t i = qt * kOther + tid;
        nq[tid] = num.at(i);
        lse[tid] = i < a.T ? a.lse[((int64_t)b * a.H + h) * a.T + i] : 0.f;
        delta[tid] = i < a.T ? a.delta[((int64_t)b * a.H + h) * a.T + i] : 0.f;
      }
      __syncthreads();
      load_tile<T>(Q, ld, a.q, b, h, qt * kOther, kOther, a.T, D, nq);
      load_tile<T>(Gr, ld, a.g, b, h, qt * kOther, kOther, a.T, D, nq);
      __syncthreads();
      float s[4][2] = {}, gp[4][2] = {};
      tile_products(K, Q, ld, D, ty, tx, s);
      tile_products(V, Gr, ld, D, ty, tx, gp);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = ty + 16 * i;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int q = tx + 16 * c;
          const float p = window_sees(nq[q], nk[r], a.window, a.sinks) ? expf(s[i][c] * a.scale - lse[q]) : 0.f;
          P[r * (kOther + 1) + q] = p;
          dS[r * (kOther + 1) + q] = p * (gp[i][c] - delta[q]) * a.scale;
        }
      }
      __syncthreads();
      tile_add<NC>(P, Gr, ld, D, ty, tx, gv);
      tile_add<NC>(dS, Q, ld, D, ty, tx, gk);
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty + 16 * i;
    if (r >= rows) continue;
    const int64_t at = (((j0 + r) * a.B + b) * a.G + kv) * D;
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (tx + 16 * c < D) {
        static_cast<T*>(a.gk)[at + tx + 16 * c] = from_f<T>(gk[i][c]);
        static_cast<T*>(a.gv)[at + tx + 16 * c] = from_f<T>(gv[i][c]);
      }
  }
}

size_t tile_bytes(int rows, int others, int scores, int D) {
  return sizeof(float) * ((size_t)rows * kRows * (D | 1) + (size_t)others * kOther * (D | 1) + (size_t)scores * kRows * (kOther + 1));
}
int run(void (*kernel)(const WindowArgs), const WindowArgs& a, int64_t places, int heads, size_t smem, cudaStream_t stream, const char* what) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return fail((int)e, "%s: cannot reserve %zu bytes of shared memory: %s", what, smem, cudaGetErrorString(e));
  const int64_t ctas = (places + kRows - 1) / kRows * a.B * heads;
  RFA_REQUIRE(ctas < (int64_t)1 << 31, RFA_EUNSUPPORTED, "%s: %lld tiles", what, (long long)ctas);
  kernel<<<(unsigned)ctas, kThreads, smem, stream>>>(a);
  return check_launch(what);
}
template <typename T, int NC>
int fwd(const WindowArgs& a, cudaStream_t stream) {
  return run(window_fwd_kernel<T, NC>, a, a.T, a.H, tile_bytes(1, 2, 1, a.D), stream, "rfa_window_fwd");
}
template <typename T, int NC>
int bwd(const WindowArgs& a, cudaStream_t stream) {
  if (int r = run(window_gq_kernel<T, NC>, a, a.T, a.H, tile_bytes(2, 2, 1, a.D), stream, "rfa_window_bwd (q)")) return r;
  return run(window_gkv_kernel<T, NC>, a, a.S, a.G, tile_bytes(2, 2, 2, a.D), stream, "rfa_window_bwd (k, v)");
}
#define RFA_WINDOW_TILES(CALL)                                                                                       \
  do {                                                                                                               \
    if (a.dtype == RFA_F32) return a.D <= 64 ? CALL<float, 4>(a, stream) : a.D <= 128 ? CALL<float, 8>(a, stream) : CALL<float, 16>(a, stream);       \
    if (a.dtype == RFA_F16) return a.D <= 64 ? CALL<__half, 4>(a, stream) : a.D <= 128 ? CALL<__half, 8>(a, stream) : CALL<__half, 16>(a, stream);    \
    return a.D <= 64 ? CALL<__nv_bfloat16, 4>(a, stream) : a.D <= 128 ? CALL<__nv_bfloat16, 8>(a, stream) : CALL<__nv_bfloat16, 16>(a, stream);       \
  } while (0)

}  // namespace

int launch_window_fwd_tiles(const WindowArgs& a, cudaStream_t stream) { RFA_WINDOW_TILES(fwd); }
int launch_window_bwd_tiles(const WindowArgs& a, cudaStream_t stream) { RFA_WINDOW_TILES(bwd); }

}  // namespace rfa
