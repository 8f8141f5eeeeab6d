// Linear attention with a decay, any sizes and types: the sweep of decay.cuh in fp32 multiply-adds, the joining of its segments, and the gradient
// of the decays.
//
// One CTA takes a (batch row, head), a tile of 32 or 64 of x3's columns and a segment of the tokens, in chunks of 32.  The tile's columns of the state stay in shared
// memory.  Sums of log decays are 64 bits: what is subtracted from each other there is the sum over a chunk, and the difference may be that of
// two neighbours.  Bound by shared memory's reads (a thread's 8 multiply-adds of out take one 16-byte and two 4-byte reads).  Where there are
// few (row, head, tile)s the tokens are cut into segments: each one's own state first, then the states in front of each (combine), then the sweep proper.
// 4 x 16 heads x 1024 x 64, fp32: forward 156 us, forward + backward 567; 3 x 4 x 531 x 40 x 52, padded, forward + backward 100 (126 with the calls).
#include <algorithm>

#include "decay.cuh"

namespace rfa {

namespace {

constexpr int kC = 32, kThreads = 256;
constexpr int tile_of(int W) { return W <= 32 ? 32 : 64; }      // columns of x3 that a CTA takes
size_t sweep_smem_bytes(int A, int DT) {
  return sizeof(float) * ((size_t)2 * kC * (A + 1) + kC * DT + (size_t)A * DT + kC * (kC + 1) + 3 * kC) + sizeof(double) * kC;
}

// kC rows of `width` numbers, `cols` of a row in shared memory, ld apart; rows from n on and padded ones are zero, whatever stands there.  A thread takes runs of 4 numbers of
// two rows.
template <typename T>
__device__ __forceinline__ void load_rows(float* dst, int ld, int cols, const T* src, int64_t s_t, int n, int width, const uint8_t* mask, int tid) {
  static_assert(kC == 32 && kThreads == 256, "two rows a thread");
  const int tx = tid % 16, ty = tid / 16;
  const bool wide = width % 4 == 0 && s_t % 4 == 0 && reinterpret_cast<uintptr_t>(src) % (4 * sizeof(T)) == 0;
  for (int c = 4 * tx; c < cols; c += 64) {
    Raw<T, 4> v[2];
    uint8_t gone[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = ty + 16 * i;
      v[i].zero();
      gone[i] = 0;
      if (r < n && c < width) {
        v[i].load(src + r * s_t + c, width - c, wide);
        if (mask) gone[i] = mask[r];
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < cols) dst[(ty + 16 * i) * ld + c + e] = gone[i] ? 0.f : v[i].get(e);
  }
}

template <typename T, int DT>
__device__ __forceinline__ void decay_sweep(const SweepArgs& a, int tile, bool state_only) {
  constexpr int kCols = DT / 4, kRowGroups = kThreads / kCols, kRows = kC / kRowGroups;     // a thread: kRows rows of 4 columns of out
  constexpr int kStateRows = DT == 64 ? 4 : 2;
  extern __shared__ double sweep_smem[];
  double* L = sweep_smem;
  float* x1 = reinterpret_cast<float*>(L + kC);
  const int A = a.A, ld = A + 1, tid = threadIdx.x;
  float *x2 = x1 + kC * ld, *x3 = x2 + kC * ld, *S = x3 + kC * DT, *P = S + (size_t)A * DT, *fa = P + kC * (kC + 1), *fb = fa + kC, *own = fb + kC;
  // x1, x2 rows are A + 1 apart (a bank more each); x3 and S rows are read 16 bytes at a time (kC * (A + 1) floats are a multiple of that)
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / a.H), h = (int)(bh % a.H), c0 = tile * DT, W = min(DT, a.W - c0), seg = blockIdx.z;
  const int64_t BH = (int64_t)a.B * a.H;
  const int place = a.rev ? a.nseg - 1 - seg : seg;                 // segments are counted in the order of the sweep
  const int64_t t_begin = place * a.tseg, t_end = min(a.T, t_begin + a.tseg);
  const int nchunk = (int)((t_end - t_begin + kC - 1) / kC);
  const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.T : nullptr;
  const int64_t b1 = b * a.x1.b + h * a.x1.h, b2 = b * a.x2.b + h * a.x2.h, b3 = b * a.x3.b + h * a.x3.h, bd = b * a.decay.b + h * a.decay.h;
  const int64_t slot = ((int64_t)seg * BH + bh) * A * a.W;

  const float* start = state_only ? nullptr : a.nseg > 1 ? a.totals + slot + c0 : a.s_in.p ? a.s_in.p + bh * A * a.W + c0 * a.s_in.col : nullptr;
  const int64_t start_r = a.nseg > 1 ? a.W : a.s_in.row, start_c = a.nseg > 1 ? 1 : a.s_in.col;
  for (int i0 = tid; i0 < A * DT; i0 += 8 * kThreads) {
    float v[8];
#pragma unroll
    for (int f = 0; f < 8; ++f) {
      const int i = i0 + f * kThreads;
      v[f] = start && i < A * DT && i % DT < W ? start[(i / DT) * start_r + (i % DT) * start_c] : 0.f;
    }
#pragma unroll
    for (int f = 0; f < 8; ++f)
      if (i0 + f * kThreads < A * DT) S[i0 + f * kThreads] = v[f];
  }
  const int col = (tid % kCols) * 4, rg = tid / kCols;
  const bool dots = a.x4.p != nullptr;
  double run = 0.0;
  for (int k = 0; k < nchunk; ++k) {
    const int64_t t0 = t_begin + (int64_t)(a.rev ? nchunk - 1 - k : k) * kC;
    const int n = (int)min((int64_t)kC, t_end - t0);
    __syncthreads();
    const uint8_t* gone = mask ? mask + t0 : nullptr;
    if (!state_only) load_rows<T>(x1, ld, A, static_cast<const T*>(a.x1.p) + b1 + t0 * a.x1.t, a.x1.t, n, A, gone, tid);
    load_rows<T>(x2, ld, A, static_cast<const T*>(a.x2.p) + b2 + t0 * a.x2.t, a.x2.t, n, A, gone, tid);
    load_rows<T>(x3, DT, DT, static_cast<const T*>(a.x3.p) + b3 + t0 * a.x3.t + c0, a.x3.t, n, W, gone, tid);
    if (tid < kC) {
      double g = tid < n && !(gone && gone[tid]) ? log_decay_at(a.decay.p, a.decay_dtype, bd + (t0 + tid) * a.decay.t) : 0.0;
#pragma unroll
      for (int o = 1; o < kC; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, g, o);
        if (tid >= o) g += up;
      }
      const double end = __shfl_sync(0xffffffffu, g, kC - 1);
      L[tid] = g;
      const float in = expf((float)g), rest = expf((float)(end - g));
      fa[tid] = a.rev ? rest : in;
      fb[tid] = a.front_out && seg == a.nseg - 1 && k == nchunk - 1 ? 0.f : a.in_scale * (a.rev ? in : rest);
    }
    __syncthreads();
    run += L[kC - 1];
    const Factor decay((float)L[kC - 1]);
    if (!state_only) {
      {      // 2 x 2 scores a thread, one of them beyond the diagonal
        const int ty = tid / 16, tx = tid % 16;
        float p[2][2] = {};
        const float *y0 = x1 + ty * ld, *y1 = y0 + 16 * ld, *z0 = x2 + tx * ld, *z1 = z0 + 16 * ld;
#pragma unroll 4
        for (int d = 0; d < A; ++d) {
          const float u0 = y0[d], u1 = y1[d], w0 = z0[d], w1 = z1[d];
          p[0][0] = fmaf(u0, w0, p[0][0]);
          p[1][1] = fmaf(u1, w1, p[1][1]);
          p[1][0] = fmaf(a.rev ? u0 : u1, a.rev ? w1 : w0, p[1][0]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int r = ty + 16 * i, c = tx + 16 * j;
            const float dot = i == j ? p[i][i] : p[1][0];      // that of rows behind 16 and columns before, or backwards the other one
            float w = (a.rev ? c >= r : c <= r) ? dot * a.in_scale * expf((float)(a.rev ? L[c] - L[r] : L[r] - L[c])) : 0.f;
            if (dots && r == c) {      // a token with itself is in no sum of the dots
              own[r] = w;
              w = 0.f;
            }
            P[r * (kC + 1) + c] = w;
          }
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
      float near[kRows][4];      // of the chunk's own tokens, apart from the state's where dots are wanted
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) near[i][e] = dots ? 0.f : acc[i][e];
#pragma unroll 4
      for (int j = 0; j < kC; ++j) {
        const float4 s = *reinterpret_cast<const float4*>(x3 + j * DT + col);
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const float p = P[(rg + i * kRowGroups) * (kC + 1) + j];
          near[i][0] = fmaf(p, s.x, near[i][0]); near[i][1] = fmaf(p, s.y, near[i][1]);
          near[i][2] = fmaf(p, s.z, near[i][2]); near[i][3] = fmaf(p, s.w, near[i][3]);
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int r = rg + i * kRowGroups;
        const int64_t t = t0 + r;
        float far_dot = 0.f, near_dot = 0.f;
        if (r < n) {
          T* o = static_cast<T*>(a.out) + ((t * a.B + b) * a.H + h) * a.W + c0;
          const bool padded = gone && r < n && gone[r];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col + e < W) {
              o[col + e] = from_f<T>(a.out_scale * (dots ? acc[i][e] + fmaf(own[r], x3[r * DT + col + e], near[i][e]) : near[i][e]));
              if (dots && !padded) {
                const float y = a.out_scale * to_f<T>(static_cast<const T*>(a.x4.p)[b * a.x4.b + h * a.x4.h + t * a.x4.t + c0 + col + e]);
                far_dot = fmaf(acc[i][e], y, far_dot);
                near_dot = fmaf(near[i][e], y, near_dot);
              }
            }
        }
        if (dots) {
#pragma unroll
          for (int s = kCols / 2; s > 0; s >>= 1) {
            far_dot += __shfl_xor_sync(0xffffffffu, far_dot, s);
            near_dot += __shfl_xor_sync(0xffffffffu, near_dot, s);
          }
          if (col == 0 && r < n) reinterpret_cast<float2*>(a.dots)[((int64_t)tile * BH + bh) * a.T + t] = make_float2(far_dot, near_dot);
        }
      }
      __syncthreads();      // the state is read by all before it changes
    }
    for (int d0 = rg; d0 < A; d0 += kStateRows * kRowGroups) {
      float u[kStateRows][4];
      const float* row[kStateRows];      // rows beyond the last read the last key's number, and are not written
#pragma unroll
      for (int m = 0; m < kStateRows; ++m) {
        const int d = min(d0 + m * kRowGroups, A - 1);
        row[m] = x2 + d;
        const float4 s = d0 + m * kRowGroups < A ? *reinterpret_cast<const float4*>(S + (size_t)d * DT + col) : make_float4(0.f, 0.f, 0.f, 0.f);
        u[m][0] = decay.times(s.x); u[m][1] = decay.times(s.y); u[m][2] = decay.times(s.z); u[m][3] = decay.times(s.w);
      }
#pragma unroll 4
      for (int j = 0; j < kC; ++j) {
        float4 s = *reinterpret_cast<const float4*>(x3 + j * DT + col);
        const float f = fb[j];
        s.x *= f; s.y *= f; s.z *= f; s.w *= f;
#pragma unroll
        for (int m = 0; m < kStateRows; ++m) {
          const float kk = row[m][j * ld];
          u[m][0] = fmaf(kk, s.x, u[m][0]); u[m][1] = fmaf(kk, s.y, u[m][1]); u[m][2] = fmaf(kk, s.z, u[m][2]); u[m][3] = fmaf(kk, s.w, u[m][3]);
        }
      }
#pragma unroll
      for (int m = 0; m < kStateRows; ++m) {
        const int d = d0 + m * kRowGroups;
        if (d < A) *reinterpret_cast<float4*>(S + (size_t)d * DT + col) = make_float4(u[m][0], u[m][1], u[m][2], u[m][3]);
      }
    }
  }
  __syncthreads();
  if (state_only) {
    for (int i = tid; i < A * DT; i += kThreads)
      if (i % DT < W) a.totals[slot + (int64_t)(i / DT) * a.W + c0 + i % DT] = S[i];
    if (tid == 0 && tile == 0) a.seg_decay[(int64_t)seg * BH + bh] = run;
  } else if (a.s_out.p && seg == a.nseg - 1) {
    for (int i = tid; i < A * DT; i += kThreads)
      if (i % DT < W) a.s_out.p[bh * A * a.W + (i / DT) * a.s_out.row + (c0 + i % DT) * a.s_out.col] = S[i];
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) decay_sweep_kernel(const __grid_constant__ SweepBatch batch, bool state_only) {
  int tile = blockIdx.y, which = 0;
  while (which + 1 < batch.count && tile >= batch.tiles[which]) tile -= batch.tiles[which++];
  const SweepArgs& a = batch.sweep[which];
  if (tile_of(a.W) == 32) decay_sweep<T, 32>(a, tile, state_only);
  else decay_sweep<T, 64>(a, tile, state_only);
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

// The gradient of the log decay at t is the sum over all pairs of a query i >= t and a key j < t (the end's gradient counts as a query behind all, a first state as a key in
// front of all).  Of a query's and of a key's pairs the sweeps give two sums each, `far` over those outside its chunk and `near` over those with other tokens of
// it: q_i . gq_i and k_j . gk_j without the token itself.  With across_c the pairs with a query behind the chunk c of t and a key in front of it,
//     g_t = across_c + sum over i >= t in c of (far_q + near_q - near_k) + sum over j < t in c of far_k
//     across_(c - 1) = across_c + sum over c of far_q - sum over c - 1 of far_k
// from the last chunk to the first, where across is g_s . s_front (the state in front of the last chunk, times its decay).  What does not straddle t is left out wherever
// it can be, rather than added and subtracted: a token with itself, pairs within other chunks, and where a chunk fades by e^-16 and more all that would cross it.
// These are of the size of a gradient without decay, and what their roundings leave grows with the sequence while the rest shrinks with the decay: as one
// difference of q_i . gq_i and k_j . gk_j over all tokens, 1000 tokens that fade by e^-3 each had 3e-3 of their gradient wrong.
// One CTA per (batch row, head), a warp to a chunk; sums in 64 bits, because near numbers are subtracted.  The sequence's first token decays nothing where no state
// is in front (`from_zero`): exactly 0, not the rounding that the sum over all tokens leaves.
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
__global__ void __launch_bounds__(kGradThreads) decay_grad_kernel(const float* q_dots, int q_tiles, const float* k_dots, int k_tiles, const float* g_s, const float* s_front,
                                                                  int KD, const uint8_t* mask, DecayRows decay, void* g_decay, int dtype, bool per_head, bool from_zero, float* sums, int64_t T, int B,
                                                                  int H) {
  __shared__ int head;
  __shared__ double red[kGradThreads / 32], from_keys[kGradThreads / 32];
  __shared__ bool faded[kGradThreads / 32];
  const int64_t bh = blockIdx.x, BH = (int64_t)B * H;
  const int b = (int)(bh / H), h = (int)(bh % H), tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  double carry = 0.0, all = 0.0;
  int64_t first = from_zero ? 0 : -1;
  if (from_zero && mask) {
    if (tid == 0) head = kGradThreads;
    while (first < T && !__syncthreads_or(first + tid < T && !mask[(int64_t)b * T + first + tid])) first += kGradThreads;
    if (first + tid < T && !mask[(int64_t)b * T + first + tid]) atomicMin(&head, tid);
    __syncthreads();
    first += head;
  }
  if (g_s) {
    double v = 0.0;
    for (int i = tid; i < KD; i += kGradThreads) v += (double)g_s[bh * KD + i] * (double)s_front[bh * KD + i];
    carry = block_sum(v, red);
  }
  static_assert(kC == 32, "a warp to a chunk");
  constexpr float kFaded = -16.f;
  const int64_t places = (T + kC - 1) / kC * kC;
  const float2 *qd = reinterpret_cast<const float2*>(q_dots), *kd = reinterpret_cast<const float2*>(k_dots);
  for (int64_t p0 = 0; p0 < places; p0 += kGradThreads) {
    const int64_t t = places - 1 - p0 - tid;
    const bool there = t >= 0 && t < T, gone = there && mask && mask[(int64_t)b * T + t];
    double far_q = 0.0, far_k = 0.0, v = 0.0;
    float fade = there && !gone ? (float)log_decay_at(decay.p, dtype, b * decay.b + h * decay.h + t * decay.t) : 0.f;
    if (there) {
      for (int i = 0; i < q_tiles; ++i) {
        const float2 d = qd[((int64_t)i * BH + bh) * T + t];
        far_q += (double)d.x;
        v += (double)d.y;
      }
      for (int i = 0; i < k_tiles; ++i) {
        const float2 d = kd[((int64_t)i * BH + bh) * T + t];
        far_k += (double)d.x;
        v -= (double)d.y;
      }
    }
    v += far_q;
    double keys = far_k;      // of this token and the ones before
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, v, o), down = __shfl_down_sync(0xffffffffu, keys, o);
      if (lane >= o) v += up;
      if (lane + o < 32) keys += down;
      far_q += __shfl_xor_sync(0xffffffffu, far_q, o);
      fade += __shfl_xor_sync(0xffffffffu, fade, o);
    }
    const double before = __shfl_down_sync(0xffffffffu, keys, 1);
    if (lane < 31) v += before;
    if (lane == 0) {
      red[warp] = far_q;
      from_keys[warp] = keys;
      faded[warp] = fade < kFaded;
    }
    __syncthreads();
    double across = 0.0;
    for (int w = 0; w < kGradThreads / 32; ++w) {
      if (p0 > 0 || w > 0) carry = (carry - from_keys[w]) * (faded[w] ? 0.0 : 1.0);      // times zero, so that what is no number stays none
      if (w == warp) across = carry;
      carry += red[w];
    }
    __syncthreads();
    if (there) {
      const double r = t == first || gone ? 0.0 : across + v;
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
int sweep_launches(const SweepBatch& batch, const SweepPlan& plan, cudaStream_t stream) {
  size_t smem = 0;
  int tiles = 0;
  for (int i = 0; i < batch.count; ++i) {
    smem = std::max(smem, sweep_smem_bytes(batch.sweep[i].A, tile_of(batch.sweep[i].W)));
    tiles += batch.tiles[i];
  }
  cudaError_t e = cudaFuncSetAttribute(decay_sweep_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return fail((int)e, "decay: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
  const int64_t BH = (int64_t)batch.sweep[0].B * batch.sweep[0].H;
  const dim3 grid((unsigned)BH, tiles, plan.nseg);
  if (plan.nseg > 1) {
    decay_sweep_kernel<T><<<grid, kThreads, smem, stream>>>(batch, true);
    if (int r = check_launch("rfa_decay (segments)")) return r;
    for (int i = 0; i < batch.count; ++i) {
      const SweepArgs& a = batch.sweep[i];
      if (int r = launch_decay_combine(a.totals, a.seg_decay, a.s_in, plan.nseg, BH, a.A, a.W, stream)) return r;
    }
  }
  decay_sweep_kernel<T><<<grid, kThreads, smem, stream>>>(batch, false);
  return check_launch("rfa_decay");
}

}  // namespace

int sweep_tiles(int W) { return (W + tile_of(W) - 1) / tile_of(W); }

SweepPlan sweep_plan(int64_t T, int64_t BH, int tiles, int states, int A, int W) {
  SweepPlan p{1, T, 0, 0};
  const int64_t ctas = BH * tiles, chunks = (T + kC - 1) / kC;
  // Segments cost a second pass over the keys' side, which idle SMs take.  Wanted: two CTAs an SM, down to a chunk a segment.
  const int64_t want = std::min<int64_t>({(2 * 148 + ctas - 1) / ctas, chunks, 64});
  if (ctas < 148 && want > 1) {
    const int64_t per = (chunks + want - 1) / want;
    p.tseg = per * kC;
    p.nseg = (int)((T + p.tseg - 1) / p.tseg);
  }
  if (p.nseg <= 1) return {1, T, 0, 0};
  p.totals = sizeof(float) * states * p.nseg * BH * A * W;
  p.seg_decay = sizeof(double) * states * p.nseg * BH;
  return p;
}

int launch_sweeps(SweepBatch batch, const SweepPlan& plan, cudaStream_t stream) {
  for (int i = 0; i < batch.count; ++i) {
    SweepArgs& a = batch.sweep[i];
    a.nseg = plan.nseg;
    a.tseg = plan.tseg;
    batch.tiles[i] = sweep_tiles(a.W);
  }
  const int dtype = batch.sweep[0].dtype;
  if (dtype == RFA_F32) return sweep_launches<float>(batch, plan, stream);
  if (dtype == RFA_F16) return sweep_launches<__half>(batch, plan, stream);
  return sweep_launches<__nv_bfloat16>(batch, plan, stream);
}

int launch_decay_grad(const float* q_dots, int q_tiles, const float* k_dots, int k_tiles, const float* g_s, const float* s_front, int KD, const uint8_t* mask, const DecayRows& decay,
                      void* g_decay, int decay_dtype, bool per_head, bool from_zero, float* sums, int64_t T, int B, int H, cudaStream_t stream) {
  decay_grad_kernel<<<(unsigned)((int64_t)B * H), kGradThreads, 0, stream>>>(q_dots, q_tiles, k_dots, k_tiles, g_s, s_front, KD, mask, decay, g_decay, decay_dtype, per_head,
                                                                            from_zero, sums, T, B, H);
  if (int r = check_launch("rfa_decay_bwd (decays)")) return r;
  if (!per_head) return 0;
  const SumJob job{sums, g_decay, H, B, decay_dtype};
  return sum_parts(&job, 1, stream);
}

}  // namespace rfa
