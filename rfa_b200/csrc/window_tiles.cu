// Sliding-window attention, any sizes and types: fp32 multiply-adds on tiles in shared memory, forward and backward.
//
// 64 rows (queries; in the keys' pass keys) against tiles of 32 of the other side, 256 threads as 16 x 16: of a tile of scores a thread has 4 adjacent rows by 2
// columns, of the results 4 rows by runs of 4 columns, so that both products read shared memory 16 bytes at a time (32 multiply-adds for 6 reads, 16 for 2).  Rows lie an odd
// number of 16 bytes apart: neighbours' reads fall in different banks.  Softmax with a running maximum and sum; the backward recomputes the weights from their
// logarithms' sums, with one pass over keys for gq and one over queries for gk and gv, so that no result is added up by two CTAs.
//
// Bound by issue slots: 4 x 16 heads x 1024 x 64, window 256, fp32: forward 280 us, forward + backward 1.36 ms (4-byte reads and rows dealt out by divisions 366 and 1.68).
// What is 16 bits, up to 128 wide and starts on 16 bytes goes to window_tc.cu from the first token on: 8 x 16 heads of 64, bf16, there / here, us: 2 tokens 5 / 10, 64 5 / 27,
// 1024 45 / 710.
#include "window.cuh"

namespace rfa {

namespace {

constexpr int kRows = 64, kOther = 32, kThreads = 256;

__host__ __device__ constexpr int row_floats(int D) { return 4 * (((D + 3) / 4) | 1); }
constexpr int kLdP = kRows + 4;      // weights lie column by column

// N rows of a head into shared memory; rows that hold no token are zero, whatever stands there, and so is what fills a row up to a multiple of 4.  A thread takes
// runs of 4 numbers, all of a 64-wide block on the way together.
template <typename T, int N>
__device__ __forceinline__ void load_tile(float* dst, int ld, const WindowRows& x, int b, int h, int64_t t0, int64_t T_, int D, const int* num) {
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const T* base = static_cast<const T*>(x.p) + b * x.b + h * x.h + t0 * x.t;
  const bool wide = D % 4 == 0 && x.t % 4 == 0 && reinterpret_cast<uintptr_t>(base) % (4 * sizeof(T)) == 0;
  for (int c = 4 * tx; c < D; c += 64) {
    Raw<T, 4> v[N / 16];
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const int r = ty + 16 * i;
      v[i].zero();
      if (t0 + r < T_ && num[r] >= 0) v[i].load(base + r * x.t + c, D - c, wide);
    }
#pragma unroll
    for (int i = 0; i < N / 16; ++i) {
      const float2 lo = v[i].get2(0), hi = v[i].get2(1);
      *reinterpret_cast<float4*>(dst + (ty + 16 * i) * ld + c) = make_float4(lo.x, lo.y, hi.x, hi.y);
    }
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

// x rows 4 ty + i times y rows tx + 16 j
__device__ __forceinline__ void tile_products(const float* x, const float* y, int ld, int D, int ty, int tx, float (&s)[4][2]) {
#pragma unroll 2
  for (int d = 0; d < D; d += 4) {
    float4 u[4], w[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = *reinterpret_cast<const float4*>(x + (4 * ty + i) * ld + d);
#pragma unroll
    for (int j = 0; j < 2; ++j) w[j] = *reinterpret_cast<const float4*>(y + (tx + 16 * j) * ld + d);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) s[i][j] = fmaf(u[i].x, w[j].x, fmaf(u[i].y, w[j].y, fmaf(u[i].z, w[j].z, fmaf(u[i].w, w[j].w, s[i][j]))));
  }
}
// weights of rows 4 ty + i and column j of a tile
__device__ __forceinline__ void put_weights(float* w, int j, int ty, float a, float b, float c, float d) {
  *reinterpret_cast<float4*>(w + j * kLdP + 4 * ty) = make_float4(a, b, c, d);
}
// acc[i][c] += sum_j w[row 4 ty + i][j] y[j][4 tx + 64 c ...]
template <int NC>
__device__ __forceinline__ void tile_add(const float* w, const float* y, int ld, int D, int ty, int tx, float (&acc)[4][NC][4]) {
#pragma unroll 4
  for (int j = 0; j < kOther; ++j) {
    const float4 p4 = *reinterpret_cast<const float4*>(w + j * kLdP + 4 * ty);
    const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (4 * tx + 64 * c >= D) continue;
      const float4 v = *reinterpret_cast<const float4*>(y + j * ld + 4 * tx + 64 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[i][c][0] = fmaf(p[i], v.x, acc[i][c][0]); acc[i][c][1] = fmaf(p[i], v.y, acc[i][c][1]);
        acc[i][c][2] = fmaf(p[i], v.z, acc[i][c][2]); acc[i][c][3] = fmaf(p[i], v.w, acc[i][c][3]);
      }
    }
  }
}
// a thread's part of a row of results
template <typename T, int NC>
__device__ __forceinline__ void store_part(T* o, const float (&acc)[NC][4], int D, int tx, float f) {
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (4 * tx + 64 * c + e < D) o[4 * tx + 64 * c + e] = from_f<T>(f * acc[c][e]);
}

template <typename T, int NC>
__global__ void __launch_bounds__(kThreads, NC == 1 ? 3 : 1) window_fwd_kernel(const __grid_constant__ WindowArgs a) {
  extern __shared__ __align__(16) float tiles_smem[];
  __shared__ int nq[kRows], nk[kOther];
  const int D = a.D, ld = row_floats(D), tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  float *Q = tiles_smem, *K = Q + kRows * ld, *V = K + kOther * ld, *P = V + kOther * ld;
  const int64_t tiles = (a.T + kRows - 1) / kRows, bh = blockIdx.x / tiles, i0 = blockIdx.x % tiles * kRows, at = a.S - a.T;
  const int b = (int)(bh / a.H), h = (int)(bh % a.H), kv = h / (a.H / a.G);
  const WindowNumbers num(a, b);
  const int rows = (int)min((int64_t)kRows, a.T - i0);
  if (tid < kRows) nq[tid] = tid < rows ? num.at(at + i0 + tid) : -1;
  __syncthreads();
  load_tile<T, kRows>(Q, ld, a.q, b, h, i0, a.T, D, nq);
  const int64_t first = num.first_key(at + i0) / kOther, sink_tiles = (num.first_end() + kOther - 1) / kOther, end = (num.last_key(at + i0, at + i0 + rows) + kOther - 1) / kOther;
  float acc[4][NC][4] = {}, top[4], sum[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { top[i] = -INFINITY; sum[i] = 0.f; }
  for (int64_t kt = sink_tiles > 0 ? num.front() / kOther : first; kt < end; kt = kt + 1 < sink_tiles ? kt + 1 : max(kt + 1, first)) {
    __syncthreads();
    if (tid < kOther) nk[tid] = num.key_of_tile(kt * kOther + tid, kt < first);
    __syncthreads();
    load_tile<T, kOther>(K, ld, a.k, b, kv, kt * kOther, a.S, D, nk);
    load_tile<T, kOther>(V, ld, a.v, b, kv, kt * kOther, a.S, D, nk);
    __syncthreads();
    float s[4][2] = {};
    tile_products(Q, K, ld, D, ty, tx, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = nq[4 * ty + i];
#pragma unroll
      for (int c = 0; c < 2; ++c) s[i][c] = window_sees(n, nk[tx + 16 * c], a.window, a.sinks) ? s[i][c] * a.scale : -INFINITY;
      const float now = fmaxf(top[i], row_max(fmaxf(s[i][0], s[i][1]))), ref = now == -INFINITY ? 0.f : now;
      const float keep = expf(top[i] - ref);            // 0 where nothing was seen before
      s[i][0] = expf(s[i][0] - ref);
      s[i][1] = expf(s[i][1] - ref);
      sum[i] = sum[i] * keep + row_sum(s[i][0] + s[i][1]);
      top[i] = now;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][c][e] *= keep;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) put_weights(P, tx + 16 * c, ty, s[0][c], s[1][c], s[2][c], s[3][c]);
    __syncthreads();
    tile_add<NC>(P, V, ld, D, ty, tx, acc);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * ty + i;
    if (r >= rows) continue;
    const bool real = nq[r] >= 0;                       // sees itself at least; a padded query has 0
    const float inv = real ? 1.f / sum[i] : 0.f;        // whatever the sum is: a NaN score makes the row NaN
    if (!real)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][c][e] = 0.f;
    store_part<T, NC>(static_cast<T*>(a.out) + (((i0 + r) * a.B + b) * a.H + h) * D, acc[i], D, tx, inv);
    if (a.lse && tx == 0) a.lse[bh * a.T + i0 + r] = real ? top[i] + logf(sum[i]) : 0.f;
  }
}

// gq_i = scale sum_j ds_ij k_j, ds = p (g . v - delta), delta_i = g_i . out_i, which is left for the keys' pass
template <typename T, int NC>
__global__ void __launch_bounds__(kThreads, NC <= 2 ? 2 : 1) window_gq_kernel(const __grid_constant__ WindowArgs a) {
  extern __shared__ __align__(16) float tiles_smem[];
  __shared__ int nq[kRows], nk[kOther];
  __shared__ float lse[kRows], delta[kRows];
  const int D = a.D, ld = row_floats(D), tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
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
  load_tile<T, kRows>(Q, ld, a.q, b, h, i0, a.T, D, nq);
  load_tile<T, kRows>(Gr, ld, a.g, b, h, i0, a.T, D, nq);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * ty + i;
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
  const int64_t first = num.first_key(i0) / kOther, sink_tiles = (num.first_end() + kOther - 1) / kOther, end = (num.last_key(i0, i0 + rows) + kOther - 1) / kOther;
  float acc[4][NC][4] = {};
  for (int64_t kt = sink_tiles > 0 ? num.front() / kOther : first; kt < end; kt = kt + 1 < sink_tiles ? kt + 1 : max(kt + 1, first)) {
    __syncthreads();
    if (tid < kOther) nk[tid] = num.key_of_tile(kt * kOther + tid, kt < first);
    __syncthreads();
    load_tile<T, kOther>(K, ld, a.k, b, kv, kt * kOther, a.S, D, nk);
    load_tile<T, kOther>(V, ld, a.v, b, kv, kt * kOther, a.S, D, nk);
    __syncthreads();
    float s[4][2] = {}, gp[4][2] = {};
    tile_products(Q, K, ld, D, ty, tx, s);
    tile_products(Gr, V, ld, D, ty, tx, gp);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * ty + i;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float p = window_sees(nq[r], nk[tx + 16 * c], a.window, a.sinks) ? expf(s[i][c] * a.scale - lse[r]) : 0.f;
        s[i][c] = p * (gp[i][c] - delta[r]) * a.scale;
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) put_weights(P, tx + 16 * c, ty, s[0][c], s[1][c], s[2][c], s[3][c]);
    __syncthreads();
    tile_add<NC>(P, K, ld, D, ty, tx, acc);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * ty + i;
    if (r < rows) store_part<T, NC>(static_cast<T*>(a.gq) + (((i0 + r) * a.B + b) * a.H + h) * D, acc[i], D, tx, num.query_factor(nq[r]));
  }
}

// gv_j = sum_i p_ij g_i, gk_j = scale sum_i ds_ij q_i, over the queries and heads that see the key
template <typename T, int NC>
__global__ void __launch_bounds__(kThreads, NC == 1 ? 2 : 1) window_gkv_kernel(const __grid_constant__ WindowArgs a) {
  extern __shared__ __align__(16) float tiles_smem[];
  __shared__ int nq[kOther], nk[kRows];
  __shared__ float lse[kOther], delta[kOther];
  const int D = a.D, ld = row_floats(D), tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  float *K = tiles_smem, *V = K + kRows * ld, *Q = V + kRows * ld, *Gr = Q + kOther * ld, *P = Gr + kOther * ld, *dS = P + kOther * kLdP;
  const int64_t tiles = (a.S + kRows - 1) / kRows, normal = tiles * a.B * a.G;
  int64_t bg = blockIdx.x / tiles, j0 = blockIdx.x % tiles * kRows;
  int split = 0, far = a.splits - 1;
  if (blockIdx.x >= normal) {      // a part of the queries that see a tile of first tokens
    const int64_t x = blockIdx.x - normal, y = x / far;
    const int count = WindowNumbers(a, 0).first_tiles(kRows);
    split = 1 + (int)(x % far);
    bg = y / count;
    const WindowNumbers num(a, (int)(bg / a.G));
    j0 = (num.front() / kRows + y % count) * kRows;
    if (j0 >= num.first_end()) return;
  }
  const int b = (int)(bg / a.G), kv = (int)(bg % a.G), group = a.H / a.G;
  const WindowNumbers num(a, b);
  const bool part = num.is_split(j0, kRows, a.splits);
  const int rows = (int)min((int64_t)kRows, a.S - j0);
  if (tid < kRows) nk[tid] = tid < rows ? num.at(j0 + tid) : -1;
  __syncthreads();
  load_tile<T, kRows>(K, ld, a.k, b, kv, j0, a.S, D, nk);
  load_tile<T, kRows>(V, ld, a.v, b, kv, j0, a.S, D, nk);
  int64_t first = j0 / kOther, end = (num.last_query(j0, j0 + rows) + kOther - 1) / kOther;
  if (part) {
    const int64_t near = (num.near_query(j0, j0 + rows) + kOther - 1) / kOther, all = end - near;
    if (split == 0) end = near;
    else { first = near + all * (split - 1) / far; end = near + all * split / far; }
  }
  float gk[4][NC][4] = {}, gv[4][NC][4] = {};
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
      load_tile<T, kOther>(Q, ld, a.q, b, h, qt * kOther, a.T, D, nq);
      load_tile<T, kOther>(Gr, ld, a.g, b, h, qt * kOther, a.T, D, nq);
      __syncthreads();
      float s[4][2] = {}, gp[4][2] = {};
      tile_products(K, Q, ld, D, ty, tx, s);
      tile_products(V, Gr, ld, D, ty, tx, gp);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int q = tx + 16 * c;
          s[i][c] = window_sees(nq[q], nk[4 * ty + i], a.window, a.sinks) ? expf(s[i][c] * a.scale - lse[q]) : 0.f;
          gp[i][c] = s[i][c] * (gp[i][c] - delta[q]) * a.scale;
        }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        put_weights(P, tx + 16 * c, ty, s[0][c], s[1][c], s[2][c], s[3][c]);
        put_weights(dS, tx + 16 * c, ty, gp[0][c], gp[1][c], gp[2][c], gp[3][c]);
      }
      __syncthreads();
      tile_add<NC>(P, Gr, ld, D, ty, tx, gv);
      tile_add<NC>(dS, Q, ld, D, ty, tx, gk);
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * ty + i;
    if (r >= rows) continue;
    if (part && nk[r] >= 0 && nk[r] < a.sinks) {
      float* parts = a.parts + ((bg * a.splits + split) * min((int64_t)a.sinks, a.T) + nk[r]) * 2 * D;
      store_part<float, NC>(parts, gk[i], D, tx, 1.f);
      store_part<float, NC>(parts + D, gv[i], D, tx, 1.f);
      continue;
    }
    if (split > 0) continue;
    const int64_t at = (((j0 + r) * a.B + b) * a.G + kv) * D;
    store_part<T, NC>(static_cast<T*>(a.gk) + at, gk[i], D, tx, num.key_factor());
    store_part<T, NC>(static_cast<T*>(a.gv) + at, gv[i], D, tx, 1.f);
  }
}

// gk and gv of the first tokens from their parts, in the parts' order: one CTA per (row, head, token)
template <typename T>
__global__ void __launch_bounds__(128) window_parts_kernel(const __grid_constant__ WindowArgs a, int rows, float scale) {
  const int64_t firsts = min((int64_t)a.sinks, a.T), bg = blockIdx.x / firsts, m = blockIdx.x % firsts;
  const int b = (int)(bg / a.G), kv = (int)(bg % a.G);
  const WindowNumbers num(a, b);
  const int64_t j = num.place(m);
  if (j >= a.S || !num.is_split(j / rows * rows, rows, a.splits)) return;
  const int64_t at = ((j * a.B + b) * a.G + kv) * a.D;
  const float* parts = a.parts + (bg * a.splits * firsts + m) * 2 * a.D;
  for (int c = threadIdx.x; c < 2 * a.D; c += 128) {
    float sum = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) sum += parts[s * firsts * 2 * a.D + c];
    if (c < a.D) static_cast<T*>(a.gk)[at + c] = from_f<T>(scale * num.key_factor() * sum);
    else static_cast<T*>(a.gv)[at + c - a.D] = from_f<T>(sum);
  }
}

size_t tile_bytes(int rows, int others, int scores, int D) {
  return sizeof(float) * ((size_t)rows * kRows * row_floats(D) + (size_t)others * kOther * row_floats(D) + (size_t)scores * kOther * kLdP);
}
int run(void (*kernel)(const WindowArgs), const WindowArgs& a, int64_t places, int heads, size_t smem, cudaStream_t stream, const char* what, int64_t more = 0) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return fail((int)e, "%s: cannot reserve %zu bytes of shared memory: %s", what, smem, cudaGetErrorString(e));
  const int64_t ctas = (places + kRows - 1) / kRows * a.B * heads + more;
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
  const int64_t parts = a.splits > 1 ? ((std::min<int64_t>(a.sinks, a.T) + kRows - 1) / kRows + (a.order ? 1 : 0)) * (a.splits - 1) * a.B * a.G : 0;
  if (int r = run(window_gkv_kernel<T, NC>, a, a.S, a.G, tile_bytes(2, 2, 2, a.D), stream, "rfa_window_bwd (k, v)", parts)) return r;
  return a.splits > 1 ? launch_window_parts(a, kRows, 1.f, stream) : 0;
}
#define RFA_WINDOW_TILES(CALL)                                                                                       \
  do {                                                                                                               \
    if (a.dtype == RFA_F32) return a.D <= 64 ? CALL<float, 1>(a, stream) : a.D <= 128 ? CALL<float, 2>(a, stream) : CALL<float, 4>(a, stream);       \
    if (a.dtype == RFA_F16) return a.D <= 64 ? CALL<__half, 1>(a, stream) : a.D <= 128 ? CALL<__half, 2>(a, stream) : CALL<__half, 4>(a, stream);    \
    return a.D <= 64 ? CALL<__nv_bfloat16, 1>(a, stream) : a.D <= 128 ? CALL<__nv_bfloat16, 2>(a, stream) : CALL<__nv_bfloat16, 4>(a, stream);       \
  } while (0)

}  // namespace

int launch_window_parts(const WindowArgs& a, int rows, float scale, cudaStream_t stream) {
  const int64_t ctas = std::min<int64_t>(a.sinks, a.T) * a.B * a.G;
  RFA_REQUIRE(ctas < (int64_t)1 << 31, RFA_EUNSUPPORTED, "window_bwd: %lld first tokens", (long long)ctas);
  if (a.dtype == RFA_F32) window_parts_kernel<float><<<(unsigned)ctas, 128, 0, stream>>>(a, rows, scale);
  else if (a.dtype == RFA_F16) window_parts_kernel<__half><<<(unsigned)ctas, 128, 0, stream>>>(a, rows, scale);
  else window_parts_kernel<__nv_bfloat16><<<(unsigned)ctas, 128, 0, stream>>>(a, rows, scale);
  return check_launch("rfa_window_bwd (first tokens)");
}
int launch_window_fwd_tiles(const WindowArgs& a, cudaStream_t stream) { RFA_WINDOW_TILES(fwd); }
int launch_window_bwd_tiles(const WindowArgs& a, cudaStream_t stream) { RFA_WINDOW_TILES(bwd); }

}  // namespace rfa
