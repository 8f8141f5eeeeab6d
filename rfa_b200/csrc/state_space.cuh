// Shared by the state-space operators (causal_conv.cu, selective_scan.cu, selective_scan_bwd.cu, group_norm.cu): element types, runs of
// eight adjacent channels, and the sums of partial results.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"
#include "wide.h"

namespace rfa {

template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// NV adjacent elements as they stand in memory: asked for early, converted when they are needed.
template <typename T, int NV>
struct Raw {
  static constexpr int kWords = NV * (int)sizeof(T) / 4;
  static_assert(kWords > 0, "whole words");
  uint32_t w[kWords];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  static constexpr int kStep = kWords % 4 == 0 ? 4 : kWords % 2 == 0 ? 2 : 1;      // words of a wide access
  static_assert(kStep * 4 == access_bytes(NV * (int)sizeof(T)), "what wide_ok asks for");
  // `wide`: the address is a multiple of a wide access; n elements are there.  kConst: nobody writes to them during the launch, so that the
  // read-only path may be taken; a state that is updated in place is not constant.
  template <bool kConst = true> __device__ __forceinline__ void load(const T* p, int n, bool wide) {
    const auto get = [](const auto* at) {
      if constexpr (kConst) return __ldg(at);
      else return *at;
    };
    if (wide && n >= NV) {
#pragma unroll
      for (int i = 0; i < kWords; i += kStep) {
        const uint32_t* at = reinterpret_cast<const uint32_t*>(p) + i;
        if constexpr (kStep == 4) {
          const uint4 v = get(reinterpret_cast<const uint4*>(at));
          w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        } else if constexpr (kStep == 2) {
          const uint2 v = get(reinterpret_cast<const uint2*>(at));
          w[i] = v.x; w[i + 1] = v.y;
        } else {
          w[i] = get(at);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) put_bits(i, i < n ? p[i] : from_f<T>(0.f));
    }
  }
  // Elements in pairs: a conversion of one alone goes to the special function unit, which has enough to do.
  __device__ __forceinline__ float2 get2(int k) const {
    if constexpr (sizeof(T) == 4) {
      return make_float2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
    } else if constexpr (std::is_same_v<T, __half>) {
      return __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
    } else {
      return make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
    }
  }
  __device__ __forceinline__ void set2(int k, float a, float b) {
    if constexpr (sizeof(T) == 4) {
      w[2 * k] = __float_as_uint(a);
      w[2 * k + 1] = __float_as_uint(b);
    } else if constexpr (std::is_same_v<T, __half>) {
      const __half2 h = __floats2half2_rn(a, b);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  __device__ __forceinline__ float get(int i) const { return i & 1 ? get2(i / 2).y : get2(i / 2).x; }
  // element i as it stands in memory
  __device__ __forceinline__ T bits(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else {
      const uint16_t h = i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffff;
      return *reinterpret_cast<const T*>(&h);
    }
  }
  __device__ __forceinline__ void put_bits(int i, T v) {
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(v);
    } else {
      const uint32_t h = *reinterpret_cast<const uint16_t*>(&v);
      w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | h << 16 : (w[i / 2] & 0xffff0000u) | h;
    }
  }
  __device__ __forceinline__ void store(T* p, int n, bool wide) const {
    if (wide && n >= NV) {
#pragma unroll
      for (int i = 0; i < kWords; i += kStep) {
        uint32_t* at = reinterpret_cast<uint32_t*>(p) + i;
        if constexpr (kStep == 4) *reinterpret_cast<uint4*>(at) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        else if constexpr (kStep == 2) *reinterpret_cast<uint2*>(at) = make_uint2(w[i], w[i + 1]);
        else *at = w[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i < n) p[i] = bits(i);
    }
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;

// 1 / (1 + exp(-x)); exp's overflow gives 0.  Relative error: 5e-7 (the unit's 2^-22, a reciprocal and an addition), and where x < 0 7.3e-8 |x|
// more: the argument's product is rounded by 2^-24 and the constant by 1.3e-8.  For x sigmoid(x) that is at most 2e-8 |x|, because
// |x| sigmoid (1 - sigmoid) is below 0.23; at -12, where the result is 7e-5, it is 9e-7 of it.
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-kLog2e * x)); }

// log(1 + exp(v)) = max(v, 0) + log1p(z), z = exp(-|v|) in (0, 1]; log1p(z) = 2 atanh(w), w = z / (2 + z) in (0, 1/3]: an odd polynomial in w,
// interpolated at Chebyshev nodes of w^2 in [0, 1/9] (4.1e-9 relative).  No difference of near numbers: small steps are
// off by 7e-7 (the unit, the reciprocal, roundings) and 7.3e-8 |v| (the argument's product, as above), 1.2e-6 at most at 1e-3.  The product's rest
// handed on by two multiply-adds brings that to 7e-7, takes 2 % of a prompt's time (8 x 2048 x 2048 x 16: 236 us beside 230) and 1 to 3 % of its outputs'
// errors, which are the decays'.  16 instructions, where log1pf(expf(v)) takes about 45.  `sig`: its derivative.
__device__ __forceinline__ float softplus(float v, float& sig) {
  const float z = ex2(-kLog2e * fabsf(v)), w = z * rcp(2.f + z), s = w * w, r = rcp(1.f + z);
  sig = v >= 0.f ? r : z * r;
  const float q = fmaf(fmaf(fmaf(fmaf(0.281577788f, s, 0.279651582f), s, 0.400245965f), s, 0.666663229f), s, 2.f);
  return fmaxf(v, 0.f) + w * q;
}

constexpr int kMaxChannels = 1 << 24;     // a call: with 64 states or 8 taps a channel, their indexes and thread numbers stay below 2^31

// ---- sums of partial results: dst[i] = sum over p of src[p * n + i], in a fixed order ----------------------------------------
struct SumJob {
  const float* src;
  void* dst;
  int64_t n;
  int parts, dtype;
};
constexpr int kSumJobs = 5;
int sum_parts(const SumJob* jobs, int count, cudaStream_t stream);      // state_space.cu

}  // namespace rfa
