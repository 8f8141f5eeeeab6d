// Linear attention with a decay, any sizes and types: the sweep of decay.cuh in fp32 multiply-adds, the joining of its segments, and the gradient
// of the decays.
//
// One CTA takes a (batch row, head), a tile of x3's columns and a segment of the tokens, in chunks of 32.  The tile's columns of the state stay in shared
// memory.  Sums of log decays are 64 bits: what is subtracted from each other there is the sum over a chunk, and the difference may be that of
// two neighbours.  Bound by shared memory's reads (a thread's 8 multiply-adds take one 16-byte and two 4-byte reads).  Where there are
// few (row, head, tile)s the tokens are cut into segments: each one's own state first, then the states in front of each (combine), then the sweep proper.
#include <algorithm>

#include "decay.cuh"

namespace rfa {

namespace {

constexpr int kC = 32, kThreads = 256, DT = 32;
constexpr int kCols = DT / 4, kRowGroups = kThreads / kCols, kRows = kC / kRowGroups;     // a thread: kRows rows of 4 columns
size_t sweep_smem_bytes(int A) {
  return sizeof(float) * ((size_t)2 * kC * (A + 1) + kC * DT + (size_t)A * DT + kC * (kC + 1) + 2 * kC) + sizeof(double) * kC;
}

template <typename T>
__device__ __forceinline__ void load_rows(float* dst, int ld, const DecayRows& x, int64_t base, int64_t t0, int n, int c0, int width, const uint8_t* mask, int tid) {
  for (int i = tid; i < kC * width; i += kThreads) {
    const int r = i / width, c = i - r * width;
    const bool there = r < n && !(mask && mask[t0 + r]);
    dst[r * ld + c] = there ? to_f<T>(static_cast<const T*>(x.p)[base + (t0 + r) * x.t + c0 + c]) : 0.f;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) decay_sweep_kernel(const __grid_constant__ SweepArgs a, bool state_only) {
  extern __shared__ double sweep_smem[];
  double* L = sweep_smem;
  float* x1 = reinterpret_cast<float*>(L + kC);
  const int A = a.A, ld = A + 1, tid = threadIdx.x;
  float *x2 = x1 + kC * ld, *x3 = x2 + kC * ld, *S = x3 + kC * DT, *P = S + (size_t)A * DT, *fa = P + kC * (kC + 1), *fb = fa + kC;
  // x1, x2 rows are A + 1 apart (a bank more each); x3 and S rows are read 16 bytes at a time (kC * (A + 1) floats are a multiple of that)
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / a.H), h = (int)(bh % a.H), c0 = blockIdx.y * DT, W = min(DT, a.W - c0), seg = blockIdx.z;
  const int64_t BH = (int64_t)a.B * a.H;
  const int place = a.rev ? a.nseg - 1 - seg : seg;                 // segments are counted in the order of the sweep
  const int64_t t_begin = place * a.tseg, t_end = min(a.T, t_begin + a.tseg);
  const int nchunk = (int)((t_end - t_begin + kC - 1) / kC);
  const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.T : nullptr;
  const int64_t b1 = b * a.x1.b + h * a.x1.h, b2 = b * a.x2.b + h * a.x2.h, b3 = b * a.x3.b + h * a.x3.h, bd = b * a.decay.b + h * a.decay.h;
  const int64_t slot = ((int64_t)seg * BH + bh) * A * a.W;

  for (int i = tid; i < A * DT; i += kThreads) {
    const int r = i / DT, c = i % DT;
    float v = 0.f;
    if (c < W && !state_only) {
      if (a.nseg > 1) v = a.totals[slot + (int64_t)r * a.W + c0 + c];
      else if (a.s_in.p) v = a.s_in.p[bh * A * a.W + r * a.s_in.row + (c0 + c) * a.s_in.col];
    }
    S[i] = v;
  }
  const int col = (tid % kCols) * 4, rg = tid / kCols;
  double run = 0.0;
  for (int k = 0; k < nchunk; ++k) {
    const int64_t t0 = t_begin + (int64_t)(a.rev ? nchunk - 1 - k : k) * kC;
    const int n = (int)min((int64_t)kC, t_end - t0);
    __syncthreads();
    if (!state_only) load_rows<T>(x1, ld, a.x1, b1, t0, n, 0, A, mask, tid);
    load_rows<T>(x2, ld, a.x2, b2, t0, n, 0, A, mask, tid);
    for (int i = tid; i < kC * DT; i += kThreads) {
      const int r = i / DT, c = i % DT;
      x3[i] = c < W && r < n && !(mask && mask[t0 + r]) ? to_f<T>(static_cast<const T*>(a.x3.p)[b3 + (t0 + r) * a.x3.t + c0 + c]) : 0.f;
    }
    if (tid < kC) {
      double g = tid < n && !(mask && mask[t0 + tid]) ? log_decay_at(a.decay.p, a.decay_dtype, bd + (t0 + tid) * a.decay.t) : 0.0;
#pragma unroll
      for (int o = 1; o < kC; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, g, o);
        if (tid >= o) g += up;
      }
      const double end = __shfl_sync(0xffffffffu, g, kC - 1);
      L[tid] = g;
      const float in = expf((float)g), rest = expf((float)(end - g));
      fa[tid] = a.rev ? rest : in;
      fb[tid] = a.in_scale * (a.rev ? in : rest);
    }
    __syncthreads();
    run += L[kC - 1];
    const Factor decay((float)L[kC - 1]);
    if (!state_only) {
      for (int i = tid; i < kC * kC; i += kThreads) {
        const int r = i / kC, c = i % kC;
        float p = 0.f;
        if (a.rev ? c >= r : c <= r) {
          for (int d = 0; d < A; ++d) p = fmaf(x1[r * ld + d], x2[c * ld + d], p);
          p *= a.in_scale * expf((float)(a.rev ? L[c] - L[r] : L[r] - L[c]));
        }
        P[r * (kC + 1) + c] = p;
      }
      __syncthreads();
      float acc[kRows][4] = {};
#pragma unroll 4
      for (int d = 0; d < A; ++d) {
        const float4 s = *reinterpret_cast<const float4*>(S + (size_t)d * DT + col);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const float q = x1[(rg + i * kRowGroups) * ld + d];
          acc[i][0] = fmaf(q, s.x, acc[i][0]); acc[i][1] = fmaf(q, s.y, acc[i][1]);
          acc[i][2] = fmaf(q, s.z, acc[i][2]); acc[i][3] = fmaf(q, s.w, acc[i][3]);
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] *= fa[rg + i * kRowGroups];
#pragma unroll 4
      for (int j = 0; j < kC; ++j) {
        const float4 s = *reinterpret_cast<const float4*>(x3 + j * DT + col);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const float p = P[(rg + i * kRowGroups) * (kC + 1) + j];
          acc[i][0] = fmaf(p, s.x, acc[i][0]); acc[i][1] = fmaf(p, s.y, acc[i][1]);
          acc[i][2] = fmaf(p, s.z, acc[i][2]); acc[i][3] = fmaf(p, s.w, acc[i][3]);
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int r = rg + i * kRowGroups;
        const int64_t t = t0 + r;
        float dot = 0.f;
        if (r < n) {
          T* o = static_cast<T*>(a.out) + ((t * a.B + b) * a.H + h) * a.W + c0;
          const bool gone = mask && mask[t];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col + e < W) {
              const float v = a.out_scale * acc[i][e];
              o[col + e] = from_f<T>(v);
              if (a.x4.p && !gone) dot = fmaf(v, to_f<T>(static_cast<const T*>(a.x4.p)[b * a.x4.b + h * a.x4.h + t * a.x4.t + c0 + col + e]), dot);
            }
        }
        if (a.x4.p) {
#pragma unroll
          for (int s = kCols / 2; s > 0; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
          if (col == 0 && r < n) a.dots[((int64_t)blockIdx.y * BH + bh) * a.T + t] = dot;
        }
      }
      __syncthreads();      // the state is read by all before it changes
    }
    for (int d0 = 0; d0 < A; d0 += 4 * kRowGroups) {
      float u[4][4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int d = d0 + rg + m * kRowGroups;
        const float4 s = d < A ? *reinterpret_cast<const float4*>(S + (size_t)d * DT + col) : make_float4(0.f, 0.f, 0.f, 0.f);
        u[m][0] = decay.times(s.x); u[m][1] = decay.times(s.y); u[m][2] = decay.times(s.z); u[m][3] = decay.times(s.w);
      }
#pragma unroll 4
      for (int j = 0; j < kC; ++j) {
        const float4 s = *reinterpret_cast<const float4*>(x3 + j * DT + col);
        const float f = fb[j];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const int d = d0 + rg + m * kRowGroups;
          const float kk = d < A ? f * x2[j * ld + d] : 0.f;
          u[m][0] = fmaf(kk, s.x, u[m][0]); u[m][1] = fmaf(kk, s.y, u[m][1]); u[m][2] = fmaf(kk, s.z, u[m][2]); u[m][3] = fmaf(kk, s.w, u[m][3]);
        }
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int d = d0 + rg + m * kRowGroups;
        if (d < A) *reinterpret_cast<float4*>(S + (size_t)d * DT + col) = make_float4(u[m][0], u[m][1], u[m][2], u[m][3]);
      }
    }
  }
  __syncthreads();
  if (state_only) {
    for (int i = tid; i < A * DT; i += kThreads)
      if (i % DT < W) a.totals[slot + (int64_t)(i / DT) * a.W + c0 + i % DT] = S[i];
    if (tid == 0 && blockIdx.y == 0) a.seg_decay[(int64_t)seg * BH + bh] = run;
  } else if (a.s_out.p && seg == a.nseg - 1) {
    for (int i = tid; i < A * DT; i += kThreads)
      if (i % DT < W) a.s_out.p[bh * A * a.W + (i / DT) * a.s_out.row + (c0 + i % DT) * a.s_out.col] = S[i];
  }
}

// What each segment adds becomes the state in front of it, in the order of the sweep.  Bound by memory; a thread takes one element along all segments, eight of
// them on the way at a time.
__global__ void __launch_bounds__(256) decay_combine_kernel(float* totals, const double* seg_decay, DecayState s_in, int nseg, int64_t BH, int A, int W) {
  constexpr int kFlight = 8;
  const int64_t bh = blockIdx.y;
  const int i = blockIdx.x * 256 + threadIdx.x, n = A * W;
  if (i >= n) return;
  float s = s_in.p ? s_in.p[bh * n + (i / W) * s_in.row + (i % W) * s_in.col] : 0.f;
  for (int k0 = 0; k0 < nseg; k0 += kFlight) {
    float own[kFlight];
    double log[kFlight];
#pragma unroll
    for (int f = 0; f < kFlight; ++f)
      if (k0 + f < nseg) {
        own[f] = totals[((k0 + f) * BH + bh) * n + i];
        log[f] = seg_decay[(k0 + f) * BH + bh];
      }
#pragma unroll
    for (int f = 0; f < kFlight; ++f)
      if (k0 + f < nseg) {
        totals[((k0 + f) * BH + bh) * n + i] = s;
        s = Factor((float)log[f]).times(s) + own[f];
      }
  }
}

// g_decay_t = sum over i >= t of (q_i . gq_i - k_i . gk_i) + g_s . s_last.  One CTA per (batch row, head), from the last token to the first; sums in 64 bits,
// because near numbers are subtracted.
constexpr int kGradThreads = 512;
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < kGradThreads / 32; ++w) s += red[w];
  __syncthreads();
  return s;
}
__global__ void __launch_bounds__(kGradThreads) decay_grad_kernel(const float* q_dots, int q_tiles, const float* k_dots, int k_tiles, const float* g_s, const float* s_last,
                                                                  int KD, const uint8_t* mask, void* g_decay, int dtype, bool per_head, float* sums, int64_t T, int B, int H) {
  __shared__ double red[kGradThreads / 32];
  const int64_t bh = blockIdx.x, BH = (int64_t)B * H;
  const int b = (int)(bh / H), h = (int)(bh % H), tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  double carry = 0.0, all = 0.0;
  if (g_s) {
    double v = 0.0;
    for (int i = tid; i < KD; i += kGradThreads) v += (double)g_s[bh * KD + i] * (double)s_last[bh * KD + i];
    carry = block_sum(v, red);
  }
  for (int64_t p0 = 0; p0 < T; p0 += kGradThreads) {
    const int64_t t = T - 1 - p0 - tid;
    double v = 0.0;
    if (t >= 0) {
      for (int i = 0; i < q_tiles; ++i) v += (double)q_dots[((int64_t)i * BH + bh) * T + t];
      for (int i = 0; i < k_tiles; ++i) v -= (double)k_dots[((int64_t)i * BH + bh) * T + t];
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    if (lane == 31) red[warp] = v;
    __syncthreads();
    double before = carry;
    for (int w = 0; w < warp; ++w) before += red[w];
    for (int w = 0; w < kGradThreads / 32; ++w) carry += red[w];
    __syncthreads();
    if (t >= 0) {
      const double r = mask && mask[(int64_t)b * T + t] ? 0.0 : before + v;
      all += r;
      if (!per_head) {
        const int64_t i = (t * B + b) * H + h;
        if (dtype == RFA_F32) static_cast<float*>(g_decay)[i] = (float)r;
        else if (dtype == RFA_F16) static_cast<__half*>(g_decay)[i] = __float2half_rn((float)r);
        else static_cast<__nv_bfloat16*>(g_decay)[i] = __float2bfloat16_rn((float)r);
      }
    }
  }
  if (per_head) {
    const double s = block_sum(all, red);
    if (tid == 0) sums[(int64_t)b * H + h] = (float)s;
  }
}

}  // namespace

int launch_decay_combine(float* totals, const double* seg_decay, DecayState s_in, int nseg, int64_t BH, int A, int W, cudaStream_t stream) {
  decay_combine_kernel<<<dim3((A * W + 255) / 256, (unsigned)BH), 256, 0, stream>>>(totals, seg_decay, s_in, nseg, BH, A, W);
  return check_launch("rfa_decay (combine)");
}

namespace {

template <typename T>
int sweep_launches(const SweepArgs& a, const SweepPlan& plan, cudaStream_t stream) {
  const size_t smem = sweep_smem_bytes(a.A);
  cudaError_t e = cudaFuncSetAttribute(decay_sweep_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return fail((int)e, "decay: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
  const int64_t BH = (int64_t)a.B * a.H;
  const dim3 grid((unsigned)BH, (a.W + DT - 1) / DT, plan.nseg);
  if (plan.nseg > 1) {
    decay_sweep_kernel<T><<<grid, kThreads, smem, stream>>>(a, true);
    if (int r = check_launch("rfa_decay (segments)")) return r;
    if (int r = launch_decay_combine(a.totals, a.seg_decay, a.s_in, plan.nseg, BH, a.A, a.W, stream)) return r;
  }
  decay_sweep_kernel<T><<<grid, kThreads, smem, stream>>>(a, false);
  return check_launch("rfa_decay");
}

}  // namespace

int sweep_tiles(int W) { return (W + DT - 1) / DT; }

SweepPlan sweep_plan(int64_t T, int64_t BH, int A, int W) {
  SweepPlan p{1, T, 0, 0};
  const int64_t ctas = BH * sweep_tiles(W), chunks = (T + kC - 1) / kC;
  // Segments cost a second reading of two operands.  Wanted: two CTAs an SM; at least 4 chunks a segment.
  const int64_t want = std::min<int64_t>({(2 * 148 + ctas - 1) / ctas, chunks / 4, 64});
  if (ctas < 148 && want > 1) {
    const int64_t per = (chunks + want - 1) / want;
    p.tseg = per * kC;
    p.nseg = (int)((T + p.tseg - 1) / p.tseg);
  }
  if (p.nseg <= 1) return {1, T, 0, 0};
  p.totals = sizeof(float) * p.nseg * BH * A * W;
  p.seg_decay = sizeof(double) * p.nseg * BH;
  return p;
}

int launch_sweep(SweepArgs a, const SweepPlan& plan, cudaStream_t stream) {
  a.nseg = plan.nseg;
  a.tseg = plan.tseg;
  if (a.dtype == RFA_F32) return sweep_launches<float>(a, plan, stream);
  if (a.dtype == RFA_F16) return sweep_launches<__half>(a, plan, stream);
  return sweep_launches<__nv_bfloat16>(a, plan, stream);
}

int launch_decay_grad(const float* q_dots, int q_tiles, const float* k_dots, int k_tiles, const float* g_s, const float* s_last, int KD, const uint8_t* mask,
                      void* g_decay, int decay_dtype, bool per_head, float* sums, int64_t T, int B, int H, cudaStream_t stream) {
  decay_grad_kernel<<<(unsigned)((int64_t)B * H), kGradThreads, 0, stream>>>(q_dots, q_tiles, k_dots, k_tiles, g_s, s_last, KD, mask, g_decay, decay_dtype, per_head,
                                                                            sums, T, B, H);
  if (int r = check_launch("rfa_decay_bwd (decays)")) return r;
  if (!per_head) return 0;
  const SumJob job{sums, g_decay, H, B, decay_dtype};
  return sum_parts(&job, 1, stream);
}

}  // namespace rfa
