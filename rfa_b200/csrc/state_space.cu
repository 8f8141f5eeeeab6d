// The last step of the state-space operators' backward passes: sums of the partial gradients that their CTAs left, in a fixed order (no
// atomics: the same call gives the same bits).
//
// Bound by latency and then by memory.  A CTA takes 32 adjacent results and deals the parts to 16 rows of threads, four loads on the way per
// thread; all gradients of a call go in one launch.
#include "state_space.cuh"

namespace rfa {

constexpr int kSpRows = 16, kSpFlight = 4;
struct SumArgs {
  SumJob job[kSumJobs];
  int64_t first[kSumJobs + 1];      // the first CTA of each job
  int count;
};

__global__ void __launch_bounds__(32 * kSpRows) sum_parts_kernel(const __grid_constant__ SumArgs a) {
  __shared__ float red[kSpRows][32];
  int k = 0;
  while (k + 1 < a.count && (int64_t)blockIdx.x >= a.first[k + 1]) ++k;
  const SumJob& job = a.job[k];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int64_t i = ((int64_t)blockIdx.x - a.first[k]) * 32 + lane;
  float acc = 0.f;
  if (i < job.n) {
    for (int p = row; p < job.parts; p += kSpRows * kSpFlight) {
      float v[kSpFlight];
#pragma unroll
      for (int f = 0; f < kSpFlight; ++f) v[f] = p + f * kSpRows < job.parts ? job.src[(size_t)(p + f * kSpRows) * job.n + i] : 0.f;
#pragma unroll
      for (int f = 0; f < kSpFlight; ++f) acc += v[f];
    }
  }
  red[row][lane] = acc;
  __syncthreads();
  if (row == 0 && i < job.n) {
    const int rows = job.parts < kSpRows ? job.parts : kSpRows;
    for (int r = 1; r < rows; ++r) acc += red[r][lane];
    if (job.dtype == RFA_F32) static_cast<float*>(job.dst)[i] = acc;
    else if (job.dtype == RFA_F16) static_cast<__half*>(job.dst)[i] = from_f<__half>(acc);
    else static_cast<__nv_bfloat16*>(job.dst)[i] = from_f<__nv_bfloat16>(acc);
  }
}

int sum_parts(const SumJob* jobs, int count, cudaStream_t stream) {
  SumArgs a{};
  for (int k = 0; k < count; ++k) {
    if (!jobs[k].dst) continue;
    a.job[a.count] = jobs[k];
    a.first[a.count + 1] = a.first[a.count] + (jobs[k].n + 31) / 32;
    ++a.count;
  }
  if (!a.count) return 0;
  RFA_REQUIRE(a.first[a.count] < (int64_t)1 << 31, RFA_EUNSUPPORTED, "sum_parts: too many results");
  sum_parts_kernel<<<(unsigned)a.first[a.count], 32 * kSpRows, 0, stream>>>(a);
  return check_launch("sum_parts");
}

}  // namespace rfa
