// Linear attention with a decay, one token: s = e^g s + k (x) v in place, out = scale q . s, per (batch row, head).
//
// Bound by memory: the fp32 state is read and written once.  A CTA takes a (row, head) and up to 128 columns; a thread four adjacent columns
// (one where the width is no multiple of 4) of every n-th row, kFlight rows on the way at a time; its parts of out are summed over the rows' threads
// through shared memory.  256 x 16 x 128 x 128: 84 us, 6.4 TB/s; 8 x 16 x 64 x 64: 2.7 us.
#include "decay.cuh"

namespace rfa {

namespace {

constexpr int kThreads = 256, kFlight = 4;

template <typename T, int VEC, int LANES>
__global__ void __launch_bounds__(kThreads) decay_step_kernel(const __grid_constant__ rfa_decay_t c, void* out, float* state) {
  constexpr int kTile = LANES * VEC, kGroups = kThreads / LANES;
  __shared__ float ks[kDecayMaxWidth], qs[kDecayMaxWidth], red[kGroups][kTile];
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / c.H), h = (int)(bh % c.H), tid = threadIdx.x, lane = tid % LANES, group = tid / LANES;
  const int col = blockIdx.y * kTile + lane * VEC;
  const bool in = col < c.D, gone = c.mask && c.mask[b];
  T* o = static_cast<T*>(out) + bh * c.D;
  if (gone) {
    if (group == 0 && in)
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[col + e] = from_f<T>(0.f);
    return;
  }
  float* s = state + bh * c.K * c.D + col;
  float v[VEC], acc[VEC] = {}, st[kFlight][VEC];
  // the first rows of the state are asked for before the token's own numbers
  const auto load = [&](int k, float (&r)[VEC]) {
    if (!in || k >= c.K) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) r[e] = 0.f;
    } else if constexpr (VEC == 4) {
      const float4 f = *reinterpret_cast<const float4*>(s + (int64_t)k * c.D);
      r[0] = f.x; r[1] = f.y; r[2] = f.z; r[3] = f.w;
    } else {
      r[0] = s[(int64_t)k * c.D];
    }
  };
#pragma unroll
  for (int f = 0; f < kFlight; ++f) load(group + f * kGroups, st[f]);
  for (int i = tid; i < c.K; i += kThreads) {
    ks[i] = to_f<T>(static_cast<const T*>(c.k)[b * c.k_b + h * c.k_h + i]);
    qs[i] = to_f<T>(static_cast<const T*>(c.q)[b * c.q_b + h * c.q_h + i]);
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) v[e] = in ? to_f<T>(static_cast<const T*>(c.v)[b * c.v_b + h * c.v_h + col + e]) : 0.f;
  const Factor decay((float)log_decay_at(c.log_decay, c.decay_dtype, b * c.g_b + h * c.g_h));
  __syncthreads();
  for (int k0 = group; k0 < c.K; k0 += kFlight * kGroups) {
    float next[kFlight][VEC];
    if (k0 + kFlight * kGroups < c.K)
#pragma unroll
      for (int f = 0; f < kFlight; ++f) load(k0 + (kFlight + f) * kGroups, next[f]);
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int k = k0 + f * kGroups;
      if (k >= c.K) break;
      const float kk = ks[k], qq = qs[k];
      float r[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        r[e] = fmaf(kk, v[e], decay.times(st[f][e]));
        acc[e] = fmaf(qq, r[e], acc[e]);
      }
      if (in) {
        if constexpr (VEC == 4) *reinterpret_cast<float4*>(s + (int64_t)k * c.D) = make_float4(r[0], r[1], r[2], r[3]);
        else s[(int64_t)k * c.D] = r[0];
      }
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f)
#pragma unroll
      for (int e = 0; e < VEC; ++e) st[f][e] = next[f][e];
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) red[group][lane * VEC + e] = acc[e];
  __syncthreads();
  for (int i = tid; i < kTile; i += kThreads) {
    if (blockIdx.y * kTile + i >= c.D) continue;
    float sum = 0.f;
    for (int g = 0; g < kGroups; ++g) sum += red[g][i];
    o[blockIdx.y * kTile + i] = from_f<T>(c.scale * sum);
  }
}

template <typename T>
int step_launch(const rfa_decay_t& c, void* out, float* s, cudaStream_t stream) {
  const unsigned BH = (unsigned)((int64_t)c.B * c.H);
  // lanes of a row: as few as hold the width, so that narrow states keep all threads busy
  if (c.D % 4) decay_step_kernel<T, 1, 32><<<dim3(BH, (c.D + 31) / 32), kThreads, 0, stream>>>(c, out, s);
  else if (c.D <= 32) decay_step_kernel<T, 4, 8><<<dim3(BH, 1), kThreads, 0, stream>>>(c, out, s);
  else if (c.D <= 64) decay_step_kernel<T, 4, 16><<<dim3(BH, 1), kThreads, 0, stream>>>(c, out, s);
  else decay_step_kernel<T, 4, 32><<<dim3(BH, (c.D + 127) / 128), kThreads, 0, stream>>>(c, out, s);
  return check_launch("rfa_decay_step");
}

}  // namespace

int launch_decay_step(const rfa_decay_t& c, void* out, float* s, cudaStream_t stream) {
  if (c.dtype == RFA_F32) return step_launch<float>(c, out, s, stream);
  if (c.dtype == RFA_F16) return step_launch<__half>(c, out, s, stream);
  return step_launch<__nv_bfloat16>(c, out, s, stream);
}

}  // namespace rfa
