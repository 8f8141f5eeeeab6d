// Shared by the kernels of linear attention with a decay (decay.cu, decay_sweep.cu, decay_step.cu).
//
// One sweep serves the forward pass and, with its operands exchanged, each of the gradients:
//   out_i = out_scale (sum_j w_ij (x1_i . x2_j) x3_j + a_i x1_i . S)       S' = e^(L_end) S + sum_j b_j x2_j (x) x3_j
// over chunks of tokens, L_i the sum of the log decays up to and with token i of its chunk, S the state that the chunks
// before it left.  Forwards j <= i, w_ij = e^(L_i - L_j), a_i = e^(L_i), b_j = e^(L_end - L_j); backwards, from the last
// chunk to the first, j >= i, w_ij = e^(L_j - L_i), a_i = e^(L_end - L_i), b_j = e^(L_j); w and b times in_scale.  With (x1, x2, x3):
//   out = forwards (q, k, v),  gq = forwards (g, v, k),  gv = backwards (k, q, g),  gk = backwards (v, g, q),
// the scale of the scores in out_scale forwards and in in_scale backwards, where S is the gradient of the state.
#pragma once

#include "state_space.cuh"

namespace rfa {

// rows [T][B][H] of n adjacent elements, strides in elements
struct DecayRows {
  const void* p;
  int64_t t, b, h;
};
struct DecayState {      // fp32 [B * H] of [x2's width][x3's width], strides in elements: a transposed state is read and written in place
  float* p;
  int64_t row, col;
};
struct SweepArgs {
  DecayRows x1, x2, x3;       // x1.p null: the state alone
  DecayRows x4;               // null, or: dots[tile][b * H + h][t] = (far, near), out_t . x4_t over a tile's columns, of the state and of the chunk's other tokens
  DecayRows decay;            // of decay_dtype, strides of 0 where it does not depend on the token or the batch row
  const uint8_t* mask;        // [B][T]
  void* out;                  // [T][B][H][width3], x1's type
  float* dots;
  DecayState s_in, s_out;     // p null: zeros, nowhere
  bool front_out;             // s_out is the state without the last chunk's tokens, times that chunk's decay
  float* totals;              // segments: what each adds [segment][b * H + h][width2][width3], then the state in front of each
  double* seg_decay;          // [segment][b * H + h]
  int64_t T, tseg;
  int B, H, A, W, nseg, dtype, decay_dtype, rev;     // A: width of x1 and x2, W: of x3
  float in_scale, out_scale;
};

// Sweeps that do not depend on each other, in one launch: the same tokens, rows and heads
struct SweepBatch {
  SweepArgs sweep[3];
  int tiles[3], count;
};

// decay_sweep.cu: any sizes up to kDecayMaxWidth, any types
constexpr int kDecayMaxWidth = 256;
struct SweepPlan {
  int nseg;
  int64_t tseg;
  size_t totals, seg_decay;      // workspace bytes of the two arrays, for all of a launch's sweeps
};
SweepPlan sweep_plan(int64_t T, int64_t BH, int tiles, int states, int A, int W);      // tiles: of all sweeps together; `states` of A x W
int sweep_tiles(int W);
int launch_sweeps(SweepBatch batch, const SweepPlan& plan, cudaStream_t stream);
// totals: what each segment adds -> the state in front of it; at most 65535 (row, head)s
int launch_decay_combine(float* totals, const double* seg_decay, DecayState s_in, int nseg, int64_t BH, int A, int W, cudaStream_t stream);
int launch_decay_grad(const float* q_dots, int q_tiles, const float* k_dots, int k_tiles, const float* g_s, const float* s_front, int KD, const uint8_t* mask, const DecayRows& decay,
                      void* g_decay, int decay_dtype, bool per_head, bool from_zero, float* sums, int64_t T, int B, int H, cudaStream_t stream);

// decay_tc.cu: fp16 and bf16, heads of up to 128 in rows that a tensor map can describe
bool decay_tc_ok(const rfa_decay_t& c);
SweepPlan decay_tc_plan(int64_t T, int64_t BH, int K, int D);
int launch_decay_tc(const rfa_decay_t& c, const SweepPlan& plan, char* workspace, void* out, float* s_out, void* kept, cudaStream_t stream);
size_t decay_tc_kept_bytes(int64_t T, int64_t BH, int K, int D);      // what a forward pass leaves for the backward
size_t decay_tc_bwd_bytes(const rfa_decay_t& c);
int launch_decay_tc_bwd(const rfa_decay_t& c, char* workspace, const void* kept, const void* g, const float* g_s, void* gq, void* gk, void* gv, void* g_decay, float* gs_in, cudaStream_t stream);

int launch_decay_step(const rfa_decay_t& c, void* out, float* s, cudaStream_t stream);      // decay_step.cu

#ifdef __CUDACC__
// A log decay as it is taken: below -1e4 it is that (e^-1e4 is nothing beside any state), so that the differences of sums that cross a reset
// are numbers.
__device__ __forceinline__ uint32_t log_decay_bits(const void* p, int dtype, int64_t i) {      // as it stands in memory, to be asked for early
  return dtype == RFA_F32 ? static_cast<const uint32_t*>(p)[i] : static_cast<const uint16_t*>(p)[i];
}
__device__ __forceinline__ float log_decay_number(uint32_t bits, int dtype) {
  return dtype == RFA_F32 ? __uint_as_float(bits) : dtype == RFA_F16 ? __half2float(__ushort_as_half((uint16_t)bits)) : __uint_as_float(bits << 16);
}
__device__ __forceinline__ double log_decay_of(uint32_t bits, int dtype) {
  const float g = log_decay_number(bits, dtype);
  return (double)(g < -1e4f ? -1e4f : g);
}
__device__ __forceinline__ double log_decay_at(const void* p, int dtype, int64_t i) { return log_decay_of(log_decay_bits(p, dtype, i), dtype); }
// The factor e^x as whole + part, so that e^x times state is fma(state, part, state * whole): a slow decay is taken as one and what it lacks, whose error
// is 2^-24 of that and not of one.  The factors of a fixed decay are the same for every chunk or token, and an error of theirs adds up along a sequence.
struct Factor {
  float whole, part;
  __device__ __forceinline__ explicit Factor(float x) : whole(x > -0.5f && x < 0.5f ? 1.f : expf(x)), part(x > -0.5f && x < 0.5f ? expm1f(x) : 0.f) {}
  __device__ __forceinline__ float times(float s) const { return fmaf(s, part, s * whole); }
};
#endif

}  // namespace rfa
