// Shared by the selective scan's forward and backward: the work of a CTA, its tiles in shared memory, how inputs are staged.
//
// A state element (channel i, state n) evolves alone, so a thread holds 2 adjacent channels x 4 adjacent states in registers and walks the
// tokens; LN = 2, 4, 8 or 16 neighbouring lanes hold a channel's up to 4 LN states.  A CTA of four warps has 256 / LN channels
// of one group and one batch row, and a segment of the tokens; tiles of 16 tokens go through shared memory: inputs are asked for a
// tile ahead as wide loads along the channels, turned into fp32 (delta = softplus(dt + bias) once per channel) by the thread that
// loaded them, and read by the scan as one 16-byte word per token (both channels' delta and x, broadcast to the LN lanes) and one each of b, c.
#pragma once

#include "state_space.cuh"

namespace rfa {

constexpr int kScanThreads = 128, kScanTile = 16;      // tokens of a tile, and of a checkpoint

struct ScanShape {
  int64_t T;
  int B, D, N, G, heads;          // heads = D / G channels share b and c
  int per_group, tiles, seg_tiles, segs, n4;      // CTAs per group, tiles of the sequence, tiles per segment, segments; states rounded up to 4
};

template <int LN> struct ScanTile {
  static constexpr int kChannels = 256 / LN, kN = 4 * LN, kPairs = kChannels / 2;
  static constexpr int kVecs = kChannels / 8;                       // runs of eight channels
  static constexpr int kRows = kScanThreads / kVecs;                // tokens that the CTA loads side by side
  static constexpr int kPasses = kRows >= kScanTile ? 1 : kScanTile / kRows;
  static constexpr int kBc = kScanTile * kN / kScanThreads;         // elements of b (and of c) per thread and tile
  static_assert(kBc >= 1, "a tile of b");
};

// What a thread of the CTA is.
template <int LN> struct ScanThread {
  int group, c0, nch, b;          // the CTA's group, first channel, channels (<= kChannels), batch row
  int lane, warp, ln, pair;       // this thread's place in the scan: lane of the channel, pair of channels in the CTA
  int vec, row;                   // and when it loads: run of eight channels, first token
  __device__ ScanThread(const ScanShape& s) {
    using Tile = ScanTile<LN>;
    group = blockIdx.x / s.per_group;
    const int in_group = (blockIdx.x % s.per_group) * Tile::kChannels;
    c0 = group * s.heads + in_group;
    nch = min(Tile::kChannels, s.heads - in_group);
    b = blockIdx.y;
    lane = threadIdx.x & 31; warp = threadIdx.x >> 5;
    ln = lane % LN;
    pair = warp * (32 / LN) + lane / LN;
    vec = threadIdx.x % Tile::kVecs;
    row = threadIdx.x / Tile::kVecs;
  }
  __device__ int first_channel() const { return 2 * pair; }      // in the CTA
};

// One tile's raw b or c: element e = thread + i * 128 of [token][state].
template <typename T, int LN> struct RawStates {
  T v[ScanTile<LN>::kBc];
  __device__ __forceinline__ void load(const T* p, int64_t stride, int tokens, int N, const uint8_t* gone) {
#pragma unroll
    for (int i = 0; i < ScanTile<LN>::kBc; ++i) {
      const int e = threadIdx.x + i * kScanThreads, t = e / ScanTile<LN>::kN, n = e % ScanTile<LN>::kN;
      v[i] = t < tokens && n < N && !(gone && gone[t]) ? p[(int64_t)t * stride + n] : from_f<T>(0.f);
    }
  }
  __device__ __forceinline__ void store(float* smem) const {
#pragma unroll
    for (int i = 0; i < ScanTile<LN>::kBc; ++i) smem[threadIdx.x + i * kScanThreads] = to_f(v[i]);
  }
};

__device__ __forceinline__ void load4f(const float* p, int n, float* v) {      // n of 4, the rest 0; 16 | p's address
  if (n >= 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.f;
  }
}
__device__ __forceinline__ void load4u(const float* p, int n, float* v) {      // any address
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.f;
}
__device__ __forceinline__ void store4u(float* p, int n, const float* v, bool wide) {
  if (wide && n >= 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = v[i];
  }
}

// Sums `K` values over LN lanes, dealing the results out: afterwards v[0 .. max(1, K / LN)) of lane l are the totals of values
// l * K / LN ... (K >= LN), or of value l * K / LN in every lane (K < LN).  K / 2 + K / 4 + ... exchanges instead of K log LN.
template <int K, int LN, int W = LN> __device__ __forceinline__ void lanes_sum(float* v, int ln, int stride = 1) {
  if constexpr (W > 1) {
    const bool upper = ln & (W / 2);
    if constexpr (K > 1) {
#pragma unroll
      for (int i = 0; i < K / 2; ++i) {
        const float give = upper ? v[i] : v[i + K / 2], keep = upper ? v[i + K / 2] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, give, (W / 2) * stride);
      }
      lanes_sum<K / 2, LN, W / 2>(v, ln, stride);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], (W / 2) * stride);
      lanes_sum<1, LN, W / 2>(v, ln, stride);
    }
  }
}

// The segments a call is cut into: see scan_shape in selective_scan.cu.
ScanShape scan_shape(int64_t T, int B, int D, int N, int G, bool backward);
int scan_lanes(int N);
int scan_check(const rfa_scan_t* s, const char* what);

#define RFA_SCAN_DISPATCH(dtype, lanes, CALL)                                  \
  do {                                                                         \
    if ((dtype) == RFA_F16) { RFA_SCAN_LANES(__half, lanes, CALL); }           \
    else if ((dtype) == RFA_BF16) { RFA_SCAN_LANES(__nv_bfloat16, lanes, CALL); } \
    else { RFA_SCAN_LANES(float, lanes, CALL); }                               \
  } while (0)
#define RFA_SCAN_LANES(T, lanes, CALL)          \
  switch (lanes) {                              \
    case 2: CALL(T, 2); break;                  \
    case 4: CALL(T, 4); break;                  \
    case 8: CALL(T, 8); break;                  \
    default: CALL(T, 16); break;                \
  }

}  // namespace rfa
