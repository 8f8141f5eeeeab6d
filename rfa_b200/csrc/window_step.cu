// Sliding-window attention, one token against the cache; and what moves whole runs of tokens into and out of the cache.
//
// The step is bound by memory: every slot that holds a token is read once.  The kernel for any widths and types: a CTA takes a (batch row, key head), the query heads that share it (up to kHeads, more
// in further CTAs) and a part of the slots; where there are few (row, head)s the parts of one are a cluster, joined through distributed shared
// memory.  kLanes lanes take a slot, 8 of its numbers each, kFlight slots of a warp's lane group on the way at a time.  Scores are in units of log 2, the running
// maximum moves only when it is exceeded.  The token's own key and value are taken from the call's inputs, never from the cache, which one CTA writes meanwhile.
//
// A row's length is read by all its CTAs and is to grow by one when all have: each adds 2^40 to it when it is done, and the one that finds the others there
// takes these marks off and adds the token.  A length stays below 2^40.
#include <cooperative_groups.h>

#include <algorithm>

#include "window.cuh"

namespace rfa {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kFlight = 4, kMost = 8;      // kMost: CTAs of a cluster
constexpr unsigned long long kMark = 1ull << 40;

struct StepArgs {
  WindowRows q, k, v;
  const uint8_t* mask;
  void *cache_k, *cache_v, *out;
  unsigned long long* length;
  int H, G, D, window, sinks, passes, parts;
  float scale;
};

// A CTA's warps, then its cluster's CTAs: each has sums of weighted values, the reference of the weights and their sum for each head.
template <typename T, int kThreads, int kWarps, int kHeads, int kWidth>
__device__ __forceinline__ void join_parts(const StepArgs& a, float (&red)[kWarps][kHeads][kWidth + 2], float (&whole)[kHeads][kWidth + 2], T* out, int heads, int part, int tid) {
  namespace cg = cooperative_groups;
  __syncthreads();
  for (int i = tid; i < kHeads * kWidth; i += kThreads) {
    const int h = i / kWidth, c = i % kWidth;
    float t = kLowest, n = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t = fmaxf(t, red[w][h][kWidth]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(red[w][h][kWidth] - t);
      n = fmaf(f, red[w][h][kWidth + 1], n);
      o = fmaf(f, red[w][h][c], o);
    }
    if (a.parts == 1) {
      if (h < heads && c < a.D) out[h * a.D + c] = from_f<T>(o / n);
    } else {
      whole[h][c] = o;
      if (c == 0) {
        whole[h][kWidth] = t;
        whole[h][kWidth + 1] = n;
      }
    }
  }
  if (a.parts > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int i = part * kThreads + tid; i < kHeads * kWidth; i += a.parts * kThreads) {
      const int h = i / kWidth, c = i % kWidth;
      float t = kLowest, n = 0.f, o = 0.f;
      for (int r = 0; r < a.parts; ++r) t = fmaxf(t, cluster.map_shared_rank(&whole[h][0], r)[kWidth]);
      for (int r = 0; r < a.parts; ++r) {
        const float* w = cluster.map_shared_rank(&whole[h][0], r);
        const float f = ex2(w[kWidth] - t);
        n = fmaf(f, w[kWidth + 1], n);
        o = fmaf(f, w[c], o);
      }
      if (h < heads && c < a.D) out[h * a.D + c] = from_f<T>(o / n);
    }
    cluster.sync();                              // nobody's shared memory goes while it is read
  }
}

template <typename T, bool WIDE, int kLanes, int kHeads>
__global__ void __launch_bounds__(kThreads) window_step_kernel(const __grid_constant__ StepArgs a) {
  constexpr int kVec = WIDE ? 16 / (int)sizeof(T) : 1, kVecs = 8 / kVec, kSlots = 32 / kLanes, kWidth = kLanes * 8;
  __shared__ float red[kWarps][kHeads][kWidth + 2];
  __shared__ float whole[kHeads][kWidth + 2];
  __shared__ unsigned long long age;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, sub = lane / kLanes, at = lane % kLanes;
  const int part = blockIdx.x % a.parts;
  const int64_t unit = blockIdx.x / a.parts;
  const int pass = (int)(unit % a.passes);
  const int64_t bg = unit / a.passes;
  const int b = (int)(bg / a.G), kv = (int)(bg % a.G), group = a.H / a.G, h0 = kv * group + pass * kHeads, heads = min(kHeads, group - pass * kHeads);
  T* out = static_cast<T*>(a.out) + ((int64_t)b * a.H + h0) * a.D;
  if (a.mask && a.mask[b]) {
    if (part == 0)
      for (int i = tid; i < heads * a.D; i += kThreads) out[i] = from_f<T>(0.f);
    return;
  }
  if (tid == 0) age = a.length[b] & (kMark - 1);
  __syncthreads();
  const unsigned long long L = age;
  const int cap = a.sinks + a.window;
  const int have = L + 1 < (unsigned long long)cap ? (int)L + 1 : cap;
  const int slot = L < (unsigned long long)a.sinks ? (int)L : a.sinks + (int)((L - a.sinks) % a.window);
  const int per = (have + a.parts - 1) / a.parts, lo = min(have, part * per), hi = min(have, lo + per);
  const T* kn = static_cast<const T*>(a.k.p) + b * a.k.b + kv * a.k.h;
  const T* vn = static_cast<const T*>(a.v.p) + b * a.v.b + kv * a.v.h;
  T* ck = static_cast<T*>(a.cache_k) + bg * cap * a.D;
  T* cv = static_cast<T*>(a.cache_v) + bg * cap * a.D;
  int col[kVecs];      // the first of each run of adjacent numbers of this lane
#pragma unroll
  for (int i = 0; i < kVecs; ++i) col[i] = (i * kLanes + at) * kVec;

  const auto load = [&](const T* row, Raw<T, 8>& r) {
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (col[i] < a.D) w = *reinterpret_cast<const uint4*>(row + col[i]);      // the width is a multiple of a run
        r.w[4 * i] = w.x; r.w[4 * i + 1] = w.y; r.w[4 * i + 2] = w.z; r.w[4 * i + 3] = w.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.put_bits(i, col[i] < a.D ? row[col[i]] : from_f<T>(0.f));
    }
  };
  float q[kHeads][8], acc[kHeads][8] = {}, top[kHeads], sum[kHeads] = {};
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    Raw<T, 8> r;
    r.zero();
    if (h < heads) load(static_cast<const T*>(a.q.p) + b * a.q.b + (h0 + h) * a.q.h, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) q[h][e] = r.get(e) * (a.scale * kLog2e);
    top[h] = kLowest;
  }
  const int step = kWarps * kSlots;
  for (int j0 = lo + warp * kSlots; j0 < hi; j0 += kFlight * step) {      // the same number of times for a warp's lanes
    Raw<T, 8> kr[kFlight], vr[kFlight];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int j = j0 + f * step + sub;
      kr[f].zero();
      vr[f].zero();
      if (j < hi) {
        load(j == slot ? kn : ck + (int64_t)j * a.D, kr[f]);
        load(j == slot ? vn : cv + (int64_t)j * a.D, vr[f]);
      }
    }
    float s[kFlight][kHeads];
#pragma unroll
    for (int f = 0; f < kFlight; ++f)
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = kr[f].get2(e);
          d = fmaf(q[h][2 * e], x.x, d);
          d = fmaf(q[h][2 * e + 1], x.y, d);
        }
        s[f][h] = d;
      }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
      for (int f = 0; f < kFlight; ++f)
#pragma unroll
        for (int h = 0; h < kHeads; ++h) s[f][h] += __shfl_xor_sync(0xffffffffu, s[f][h], o);
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      float now = top[h];
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        if (j0 + f * step + sub >= hi) s[f][h] = -INFINITY;
        now = fmaxf(now, s[f][h]);
      }
      if (now > top[h]) {
        const float keep = ex2(top[h] - now);
        sum[h] *= keep;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[h][e] *= keep;
        top[h] = now;
      }
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        const float p = ex2(s[f][h] - top[h]);
        sum[h] += p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = vr[f].get2(e);
          acc[h][2 * e] = fmaf(p, x.x, acc[h][2 * e]);
          acc[h][2 * e + 1] = fmaf(p, x.y, acc[h][2 * e + 1]);
        }
      }
    }
  }
  // the warp's lane groups, then the CTA's warps, then the cluster's CTAs
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1) {
      const float t = __shfl_xor_sync(0xffffffffu, top[h], o), now = fmaxf(t, top[h]), mine = ex2(top[h] - now), other = ex2(t - now);
      sum[h] = sum[h] * mine + __shfl_xor_sync(0xffffffffu, sum[h], o) * other;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[h][e] = acc[h][e] * mine + __shfl_xor_sync(0xffffffffu, acc[h][e], o) * other;
      top[h] = now;
    }
    if (sub == 0) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i)
#pragma unroll
        for (int e = 0; e < kVec; ++e) red[warp][h][col[i] + e] = acc[h][i * kVec + e];
      if (at == 0) {
        red[warp][h][kWidth] = top[h];
        red[warp][h][kWidth + 1] = sum[h];
      }
    }
  }
  if (lo <= slot && slot < hi && pass == 0)      // the token takes its place
    for (int i = tid; i < a.D; i += kThreads) {
      ck[(int64_t)slot * a.D + i] = kn[i];
      cv[(int64_t)slot * a.D + i] = vn[i];
    }
  join_parts<T, kThreads, kWarps, kHeads, kWidth>(a, red, whole, out, heads, part, tid);
  if (tid == 0) {
    const unsigned long long all = (unsigned long long)a.G * a.passes * a.parts;
    const unsigned long long before = atomicAdd((a.length + b), kMark);
    if (before / kMark == all - 1) atomicAdd((a.length + b), 1ull - all * kMark);
  }
}

// ---- the step for fp16 and bf16, widths that are multiples of 8 up to 128 --------------------------------------------------------
// The same split of the work with warp-wide matrix products (16 x 8 x 16): up to 8 query heads that share a key head are rows, 16 slots of a warp's step are first the
// columns of the scores, then the depth of the sums.  Both operands come straight from memory in 16-byte pieces: the order of a product's depth is free, so that a
// lane's 8 adjacent numbers of a key are its operands of two depth steps, and so is the order of the columns, so that its 8 adjacent numbers of four values
// are, halves of two put together, its operands of 8 column tiles.  32 products stand for 16 slots of 128, where the lanes' own multiply-adds take about 1000
// instructions for 4 heads: 256 x 8 key heads x 1028 slots x 128 (4 heads each) take 194 us, 5.6 TB/s, where the lanes took 418; 8 x 16 x 516 x 64 with one head 8.4 where
// they took 11.9.  Weights are rounded to the type for the second product, each off by half a step of itself.
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1, __half) {      // rows 8..15 of A are zero
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(0u), "r"(a2), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(0u), "r"(a2), "r"(b0), "r"(b1));
}

constexpr int kMmaThreads = 128, kMmaWarps = kMmaThreads / 32, kMmaHeads = 8;

template <typename T, int DB>      // DB: 64-wide blocks of a head
__global__ void __launch_bounds__(kMmaThreads, DB == 1 ? 5 : 3) window_step_mma_kernel(const __grid_constant__ StepArgs a) {
  namespace cg = cooperative_groups;
  constexpr int kWidth = DB * 64;
  __shared__ float red[kMmaWarps][kMmaHeads][kWidth + 2];
  __shared__ float whole[kMmaHeads][kWidth + 2];
  __shared__ unsigned long long age;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int part = blockIdx.x % a.parts;
  const int64_t unit = blockIdx.x / a.parts;
  const int pass = (int)(unit % a.passes);
  const int64_t bg = unit / a.passes;
  const int b = (int)(bg / a.G), kv = (int)(bg % a.G), group = a.H / a.G, h0 = kv * group + pass * kMmaHeads, heads = min(kMmaHeads, group - pass * kMmaHeads);
  T* out = static_cast<T*>(a.out) + ((int64_t)b * a.H + h0) * a.D;
  if (a.mask && a.mask[b]) {
    if (part == 0)
      for (int i = tid; i < heads * a.D; i += kMmaThreads) out[i] = from_f<T>(0.f);
    return;
  }
  if (tid == 0) age = a.length[b] & (kMark - 1);
  const T* qh = static_cast<const T*>(a.q.p) + b * a.q.b + (h0 + g) * a.q.h;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 q[2 * DB];      // the lane's pieces of head g
#pragma unroll
  for (int x = 0; x < 2 * DB; ++x) q[x] = g < heads && (x * 4 + t) * 8 < a.D ? *reinterpret_cast<const uint4*>(qh + (x * 4 + t) * 8) : zero;
  __syncthreads();
  const unsigned long long L = age;
  const int cap = a.sinks + a.window;
  const int have = L + 1 < (unsigned long long)cap ? (int)L + 1 : cap;
  const int slot = L < (unsigned long long)a.sinks ? (int)L : a.sinks + (int)((L - a.sinks) % a.window);
  const int per = ((have + a.parts - 1) / a.parts + 15) / 16 * 16, lo = min(have, part * per), hi = min(have, lo + per);
  const T* kn = static_cast<const T*>(a.k.p) + b * a.k.b + kv * a.k.h;
  const T* vn = static_cast<const T*>(a.v.p) + b * a.v.b + kv * a.v.h;
  T* ck = static_cast<T*>(a.cache_k) + bg * cap * a.D;
  T* cv = static_cast<T*>(a.cache_v) + bg * cap * a.D;
  const float scale = a.scale * kLog2e;
  float o[8 * DB][4] = {}, top = kLowest, sum = 0.f;      // column tile 8 y + j, columns 2 t and 2 t + 1: numbers 64 y + 16 t + j and + 8 of head g
  const auto piece = [&](const T* row, int at) { return at < a.D ? *reinterpret_cast<const uint4*>(row + at) : zero; };
  for (int j0 = lo + warp * 16; j0 < hi; j0 += kMmaWarps * 16) {
    uint4 k[2][2 * DB], v[4][DB];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int j = j0 + 8 * n + g;
      const T* row = j == slot ? kn : ck + (int64_t)j * a.D;
#pragma unroll
      for (int x = 0; x < 2 * DB; ++x) k[n][x] = j < hi ? piece(row, (x * 4 + t) * 8) : zero;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = j0 + 2 * t + (e & 1) + 8 * (e >> 1);
      const T* row = j == slot ? vn : cv + (int64_t)j * a.D;
#pragma unroll
      for (int y = 0; y < DB; ++y) v[e][y] = j < hi ? piece(row, (8 * y + g) * 8) : zero;
    }
    float s[2][4] = {};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int x = 0; x < 2 * DB; ++x) {
        mma16816(s[n], q[x].x, q[x].y, k[n][x].x, k[n][x].y, T());
        mma16816(s[n], q[x].z, q[x].w, k[n][x].z, k[n][x].w, T());
      }
    float p[4], now = top;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = j0 + 2 * t + (e & 1) + 8 * (e >> 1);
      p[e] = j < hi ? s[e >> 1][e & 1] * scale : -INFINITY;
      now = fmaxf(now, p[e]);
    }
    now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 1));
    now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, 2));
    if (__any_sync(0xffffffffu, now > top)) {
      const float keep = ex2(top - now);
      sum *= keep;
#pragma unroll
      for (int n = 0; n < 8 * DB; ++n) { o[n][0] *= keep; o[n][1] *= keep; }
      top = now;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      p[e] = ex2(p[e] - top);
      sum += p[e];
    }
    Raw<T, 2> a0, a2;      // weights of heads as rows, slots as depth
    a0.set2(0, p[0], p[1]);
    a2.set2(0, p[2], p[3]);
#pragma unroll
    for (int y = 0; y < DB; ++y) {
      const uint32_t *v0 = reinterpret_cast<const uint32_t*>(&v[0][y]), *v1 = reinterpret_cast<const uint32_t*>(&v[1][y]), *v2 = reinterpret_cast<const uint32_t*>(&v[2][y]),
                     *v3 = reinterpret_cast<const uint32_t*>(&v[3][y]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t pick = j & 1 ? 0x7632u : 0x5410u;      // the upper or the lower halves of two words
        mma16816(o[8 * y + j], a0.w[0], a2.w[0], __byte_perm(v0[j / 2], v1[j / 2], pick), __byte_perm(v2[j / 2], v3[j / 2], pick), T());
      }
    }
  }
  sum += __shfl_xor_sync(0xffffffffu, sum, 1);
  sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
  for (int y = 0; y < DB; ++y)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      red[warp][g][64 * y + 16 * t + j] = o[8 * y + j][0];
      red[warp][g][64 * y + 16 * t + 8 + j] = o[8 * y + j][1];
    }
  if (t == 0) {
    red[warp][g][kWidth] = top;
    red[warp][g][kWidth + 1] = sum;
  }
  if (lo <= slot && slot < hi && pass == 0)      // the token takes its place
    for (int i = tid; i < a.D / 8; i += kMmaThreads) {
      reinterpret_cast<uint4*>(ck + (int64_t)slot * a.D)[i] = reinterpret_cast<const uint4*>(kn)[i];
      reinterpret_cast<uint4*>(cv + (int64_t)slot * a.D)[i] = reinterpret_cast<const uint4*>(vn)[i];
    }
  join_parts<T, kMmaThreads, kMmaWarps, kMmaHeads, kWidth>(a, red, whole, out, heads, part, tid);
  if (tid == 0) {
    const unsigned long long all = (unsigned long long)a.G * a.passes * a.parts;
    const unsigned long long before = atomicAdd(a.length + b, kMark);
    if (before / kMark == all - 1) atomicAdd(a.length + b, 1ull - all * kMark);
  }
}

int step_launch(void (*kernel)(const StepArgs), StepArgs a, int kernel_heads, int threads, int resident, int64_t rows, int group, cudaStream_t stream) {
  a.passes = (group + kernel_heads - 1) / kernel_heads;
  const int64_t units = rows * a.passes;
  a.parts = 1;
  // parts of at least 64 slots, as long as there are fewer CTAs than the SMs hold
  while (a.parts < kMost && units * a.parts * 2 <= resident * 148 && (a.sinks + a.window) / (2 * a.parts) >= 64) a.parts *= 2;
  RFA_REQUIRE(units * a.parts < (int64_t)1 << 31, RFA_EUNSUPPORTED, "window_append: %lld parts", (long long)(units * a.parts));
  RFA_REQUIRE((int64_t)a.G * a.passes * a.parts < (1 << 23), RFA_EUNSUPPORTED, "window_append: %d key heads", a.G);      // marks of a length
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * a.parts));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) return fail((int)e, "rfa_window_append: launch failed: %s", cudaGetErrorString(e));
  return check_launch("rfa_window_append");
}
template <typename T, bool WIDE, int kLanes>
int step_heads(const StepArgs& a, int64_t rows, int group, cudaStream_t stream) {
  if (group == 1) return step_launch(window_step_kernel<T, WIDE, kLanes, 1>, a, 1, kThreads, 4, rows, group, stream);
  if (group == 2) return step_launch(window_step_kernel<T, WIDE, kLanes, 2>, a, 2, kThreads, 4, rows, group, stream);
  if constexpr (kLanes < 32) {
    if (group > 4) return step_launch(window_step_kernel<T, WIDE, kLanes, 8>, a, 8, kThreads, 4, rows, group, stream);
  }
  return step_launch(window_step_kernel<T, WIDE, kLanes, 4>, a, 4, kThreads, 4, rows, group, stream);
}
template <typename T>
int step_type(const StepArgs& a, int64_t rows, int group, bool wide, cudaStream_t stream) {
  if (!wide) return step_heads<T, false, 32>(a, rows, group, stream);
  if constexpr (sizeof(T) == 2) {
    if (a.D <= 64) return step_launch(window_step_mma_kernel<T, 1>, a, kMmaHeads, kMmaThreads, 5, rows, group, stream);
    if (a.D <= 128) return step_launch(window_step_mma_kernel<T, 2>, a, kMmaHeads, kMmaThreads, 3, rows, group, stream);
    return step_heads<T, true, 32>(a, rows, group, stream);
  }
  if (a.D <= 64) return step_heads<T, true, 8>(a, rows, group, stream);
  if (a.D <= 128) return step_heads<T, true, 16>(a, rows, group, stream);
  return step_heads<T, true, 32>(a, rows, group, stream);
}

// ---- runs of tokens -------------------------------------------------------------------------------------------------------
// Slot of the i-th of the `have` tokens that a cache holds, oldest first, `age` tokens after its sequence's start.
__device__ __forceinline__ int cache_slot(int64_t number, int window, int sinks) {
  return number < sinks ? (int)number : sinks + (int)((number - sinks) % window);
}

// Numbers of the places: `cap` of the cache (the last min(length, cap) of them hold its tokens, which are numbered from 0 without those that were pushed out), then the
// call's tokens.  One CTA per batch row.
constexpr int kOrderThreads = 1024;
__global__ void __launch_bounds__(kOrderThreads) window_order_kernel(const uint8_t* mask, const int64_t* length, int cap, int32_t* order, int32_t* pos, int64_t T) {
  __shared__ int counts[kOrderThreads / 32];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int64_t S = cap + T;
  const int have = length ? (int)min((int64_t)cap, length[b]) : 0;
  order += b * S;
  pos += b * (S + 1);
  int carry = 0;
  for (int64_t s0 = 0; s0 < S; s0 += kOrderThreads) {
    const int64_t s = s0 + tid;
    const bool real = s < S && (s < cap ? s >= cap - have : !(mask && mask[b * T + s - cap]));
    const unsigned ballot = __ballot_sync(0xffffffffu, real);
    if (lane == 0) counts[warp] = __popc(ballot);
    __syncthreads();
    int before = carry + __popc(ballot & ((1u << lane) - 1));
    for (int w = 0; w < kOrderThreads / 32; ++w) {
      if (w < warp) before += counts[w];
      carry += counts[w];
    }
    __syncthreads();
    if (s < S) {
      order[s] = real ? before : ~before;
      if (real) pos[before] = (int32_t)s;
    }
  }
  for (int64_t n = carry + tid; n <= S; n += kOrderThreads) pos[n] = (int32_t)S;
}

template <typename U>
__global__ void __launch_bounds__(256) window_gather_kernel(const U* src, const U* cache, const int64_t* length, U* dst, int64_t s_t, int64_t s_b, int64_t s_h, int64_t S,
                                                            int cap, int G, int n, int window, int sinks, int64_t total) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {      // [S][B][G][n]
    const int c = (int)(i % n), g = (int)(i / n % G);
    const int64_t row = i / n / G, B = total / n / G / S, b = row % B, s = row / B;
    U v{};
    if (s >= cap) {
      v = src[(s - cap) * s_t + b * s_b + g * s_h + c];
    } else {
      const int64_t L = length[b];
      const int have = (int)min((int64_t)cap, L), k = (int)s - (cap - have);
      if (k >= 0) v = cache[((b * G + g) * cap + cache_slot(k < sinks ? k : L - have + k, window, sinks)) * n + c];
    }
    dst[i] = v;
  }
}

// The call's tokens that the cache keeps.  `order` null: all are real and the cache was empty.
template <typename U>
__global__ void __launch_bounds__(256) window_keep_kernel(const U* src, U* cache, const int64_t* length, const int32_t* order, int64_t s_t, int64_t s_b, int64_t s_h, int64_t T,
                                                          int front, int G, int n, int window, int sinks, int64_t total) {
  const int cap = sinks + window;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {      // [T][B][G][n]
    const int c = (int)(i % n), g = (int)(i / n % G);
    const int64_t row = i / n / G, B = total / n / G / T, b = row % B, t = row / B;
    int64_t number = t, end = T;
    if (order) {
      const int64_t L = front ? length[b] : 0, gone = L - min((int64_t)front, L), S = front + T;      // `gone` tokens have left the numbering
      const int32_t mine = order[b * S + front + t], last = order[b * S + S - 1];
      if (mine < 0) continue;
      number = mine + gone;
      end = (last < 0 ? ~last : last + 1) + gone;
    }
    if (number < sinks || number >= end - window) cache[((b * G + g) * cap + cache_slot(number, window, sinks)) * n + c] = src[t * s_t + b * s_b + g * s_h + c];
  }
}
__global__ void window_length_kernel(int64_t* length, const int32_t* order, int64_t T, int front, int B) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b >= B) return;
  const int64_t L = front ? length[b] : 0, S = front + T;
  int64_t all = T;
  if (order) {
    const int32_t last = order[b * S + S - 1];
    all = (last < 0 ? ~last : last + 1) - min((int64_t)front, L);
  }
  length[b] = L + all;
}

unsigned blocks_for(int64_t n) { return (unsigned)std::min<int64_t>((n + 255) / 256, 148 * 32); }
// units of 16 bytes where every row starts and ends on one
bool rows_wide(const void* p, int64_t t, int64_t b, int64_t h, int D, int size) {
  return aligned16(p) && t * size % 16 == 0 && b * size % 16 == 0 && h * size % 16 == 0 && D * size % 16 == 0;
}

template <typename U>
void gather(const rfa_window_t& c, const void* src, int64_t s_t, int64_t s_b, int64_t s_h, const void* cache, const int64_t* length, void* dst, int per, cudaStream_t stream) {
  const int cap = c.sinks + c.window, n = c.D / per;
  const int64_t total = (cap + c.T) * c.B * c.G * n;
  window_gather_kernel<U><<<blocks_for(total), 256, 0, stream>>>(static_cast<const U*>(src), static_cast<const U*>(cache), length, static_cast<U*>(dst), s_t / per, s_b / per,
                                                                 s_h / per, cap + c.T, cap, c.G, n, c.window, c.sinks, total);
}
template <typename U>
void keep(const rfa_window_t& c, const void* src, int64_t s_t, int64_t s_b, int64_t s_h, void* cache, const int64_t* length, const int32_t* order, int front, int per,
          cudaStream_t stream) {
  const int n = c.D / per;
  const int64_t total = c.T * c.B * c.G * n;
  window_keep_kernel<U><<<blocks_for(total), 256, 0, stream>>>(static_cast<const U*>(src), static_cast<U*>(cache), length, order, s_t / per, s_b / per, s_h / per, c.T, front,
                                                               c.G, n, c.window, c.sinks, total);
}

}  // namespace

int launch_window_order(const uint8_t* mask, const int64_t* length, int cap, int32_t* order, int32_t* pos, int64_t T, int B, cudaStream_t stream) {
  window_order_kernel<<<B, kOrderThreads, 0, stream>>>(mask, length, cap, order, pos, T);
  return check_launch("rfa_window (order)");
}

int launch_window_gather(const rfa_window_t& c, const void* cache_k, const void* cache_v, const int64_t* length, void* keys, void* values, cudaStream_t stream) {
  const int size = c.dtype == RFA_F32 ? 4 : 2;
  const bool wide = rows_wide(c.k, c.k_t, c.k_b, c.k_h, c.D, size) && rows_wide(c.v, c.v_t, c.v_b, c.v_h, c.D, size);
#define GATHER(U, per)                                                              \
  gather<U>(c, c.k, c.k_t, c.k_b, c.k_h, cache_k, length, keys, per, stream);       \
  gather<U>(c, c.v, c.v_t, c.v_b, c.v_h, cache_v, length, values, per, stream)
  if (wide) { GATHER(uint4, 16 / size); }
  else if (size == 4) { GATHER(uint32_t, 1); }
  else { GATHER(uint16_t, 1); }
#undef GATHER
  return check_launch("rfa_window_append (gather)");
}

int launch_window_keep(const rfa_window_t& c, void* cache_k, void* cache_v, int64_t* length, const int32_t* order, bool empty, cudaStream_t stream) {
  const int size = c.dtype == RFA_F32 ? 4 : 2, front = empty ? 0 : c.sinks + c.window;
  const bool wide = rows_wide(c.k, c.k_t, c.k_b, c.k_h, c.D, size) && rows_wide(c.v, c.v_t, c.v_b, c.v_h, c.D, size);
#define KEEP(U, per)                                                                       \
  keep<U>(c, c.k, c.k_t, c.k_b, c.k_h, cache_k, length, order, front, per, stream);        \
  keep<U>(c, c.v, c.v_t, c.v_b, c.v_h, cache_v, length, order, front, per, stream)
  if (wide) { KEEP(uint4, 16 / size); }
  else if (size == 4) { KEEP(uint32_t, 1); }
  else { KEEP(uint16_t, 1); }
#undef KEEP
  if (int r = check_launch("rfa_window_append (keep)")) return r;
  window_length_kernel<<<(c.B + 255) / 256, 256, 0, stream>>>(length, order, c.T, front, c.B);
  return check_launch("rfa_window_append (length)");
}

int launch_window_step(const rfa_window_t& c, void* cache_k, void* cache_v, int64_t* length, void* out, cudaStream_t stream) {
  StepArgs a{};
  a.q = {c.q, c.q_t, c.q_b, c.q_h};
  a.k = {c.k, c.k_t, c.k_b, c.k_h};
  a.v = {c.v, c.v_t, c.v_b, c.v_h};
  a.mask = c.mask;
  a.cache_k = cache_k; a.cache_v = cache_v; a.out = out;
  a.length = reinterpret_cast<unsigned long long*>(length);
  a.H = c.H; a.G = c.G; a.D = c.D; a.window = c.window; a.sinks = c.sinks; a.scale = c.scale;
  const int size = c.dtype == RFA_F32 ? 4 : 2;
  const bool wide = rows_wide(c.q, 0, c.q_b, c.q_h, c.D, size) && rows_wide(c.k, 0, c.k_b, c.k_h, c.D, size) && rows_wide(c.v, 0, c.v_b, c.v_h, c.D, size);
  const int64_t rows = (int64_t)c.B * c.G;
  const int group = c.H / c.G;
  if (c.dtype == RFA_F32) return step_type<float>(a, rows, group, wide, stream);
  if (c.dtype == RFA_F16) return step_type<__half>(a, rows, group, wide, stream);
  return step_type<__nv_bfloat16>(a, rows, group, wide, stream);
}

}  // namespace rfa
