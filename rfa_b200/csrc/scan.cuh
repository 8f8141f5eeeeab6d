// Shared by the selective scan's forward and backward: the work of a CTA, its tiles in shared memory, how inputs are staged.
//
// A state element (channel i, state n) evolves alone, so a thread holds 2 adjacent channels x 4 states in registers and walks the
// tokens; LN = 2, 4, 8 or 16 neighbouring lanes hold a channel's up to 4 LN states, lane l the states l, LN + l, 2 LN + l, 3 LN + l.  A CTA
// has 256 / LN channels of one group and one batch row, and a segment of the tokens.  Some of its warps scan; others bring tiles of
// inputs and take results away meanwhile, so that a scheduler with few CTAs still has work while one warp waits.
//
// Exponentials are what bounds it: 16 a clock and SM come from the special function unit.  The first of a thread's four states -- the first
// quarter of a channel's -- takes a polynomial on the FMA units instead (`decays`), at which both are busy equally long.  Issue slots come
// next: all arithmetic is packed, both channels in one instruction (`fma.rn.f32x2`; 68 instructions a token and warp, 96 without).
//
// Tiles of 16 tokens go through shared memory, two of them by turns: a thread asks for a pair of channels' inputs a tile ahead (a
// warp's loads are whole 128-byte rows), turns them into delta and delta x and leaves them as one 16-byte word, which the scan's lanes read.  Shared memory hands a
// warp 128 bytes a clock whether lanes read the same words or not: 48 bytes a lane and token (b and c as pairs of equal
// values were 80, and bound the forward at 245 us for 8 x 2048 x 2048).
#pragma once

#include "state_space.cuh"

namespace rfa {

constexpr int kScanTile = 16;      // tokens of a forward's tile
// Tokens of a backward's tile, in front of each of which the forward leaves the states: fewer where a CTA has 128 channels, so that two CTAs' tiles
// fit an SM (8 states, 8 x 2048 tokens x 2048 channels: 1215 us a training step with tiles of 16, one CTA per SM)
__host__ __device__ constexpr int kept_tokens(int lanes) { return lanes == 2 ? 8 : 16; }

struct ScanShape {
  int64_t T;
  int B, D, N, G, heads;          // heads = D / G channels share b and c
  int per_group, tiles, seg_tiles, segs, kn;      // CTAs per group, tiles of the sequence, tiles per segment, segments; states of a kept row (4 LN)
};

// The two halves of a CTA meet at named barriers: a tile is there (kFull + buffer), a tile has been scanned (kDone + buffer).  Every tile
// passes both once, on each side, in one order: no wait is left over.
enum { kFull = 1, kDone = 3 };
template <int kThreads> __device__ __forceinline__ void meet_wait(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kThreads) : "memory"); }
template <int kThreads> __device__ __forceinline__ void meet_go(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kThreads) : "memory"); }

template <int LN> struct ScanTile {
  static constexpr int kChannels = 256 / LN, kN = 4 * LN, kPairs = kChannels / 2;
};

// ---- two floats in one instruction -------------------------------------------------------------------------------------------
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split2(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 both(float v) { return pack2(v, v); }

__device__ __forceinline__ f32x2 exp2_unit(f32x2 u) {
  const float2 v = split2(u);
  return pack2(ex2(v.x), ex2(v.y));
}
// The first state's on the FMA units, -126 <= u < 128 (below: 2^-126): u = k + r with k whole (the addition of 1.5 * 2^23 rounds) and
// |r| <= 1/2, 2^r by a polynomial of degree 5 with 1 + r log 2 in front (least maximum of the relative error, by Lawson's iteration:
// 1.1e-7, and 2.3e-7 |r| near 0, so that a decay near 1 is as near as its argument is), k added to the exponent.
//
// R of them side by side: few warps share an SM's scheduler, and a chain alone would wait for itself.
template <int R> struct Poly {
  f32x2 t[R], r[R], p[R];
  // kMost: what overflows is inf, for two instructions (of a prompt's 230 us 6; a single token has them to spare).  Without: not defined.
  template <bool kMost = false> __device__ __forceinline__ void begin(int i, f32x2 u) {
    const float2 v = split2(u);
    const auto most = [](float f) { return kMost ? fminf(f, 128.f) : f; };
    r[i] = pack2(most(fmaxf(v.x, -126.f)), most(fmaxf(v.y, -126.f)));
  }
  __device__ __forceinline__ void run() {
#pragma unroll
    for (int i = 0; i < R; ++i) t[i] = add2(r[i], both(12582912.f));
#pragma unroll
    for (int i = 0; i < R; ++i) r[i] = fma2(add2(t[i], both(-12582912.f)), both(-1.f), r[i]);
#pragma unroll
    for (int i = 0; i < R; ++i) p[i] = fma2(both(1.33006054e-3f), r[i], both(9.66969132e-3f));
#pragma unroll
    for (int i = 0; i < R; ++i) p[i] = fma2(p[i], r[i], both(5.55055849e-2f));
#pragma unroll
    for (int i = 0; i < R; ++i) p[i] = fma2(p[i], r[i], both(2.40222827e-1f));
#pragma unroll
    for (int i = 0; i < R; ++i) p[i] = fma2(p[i], r[i], both(kLn2));
#pragma unroll
    for (int i = 0; i < R; ++i) p[i] = fma2(p[i], r[i], both(1.f));
  }
  __device__ __forceinline__ f32x2 end(int i) const {
    const float2 q = split2(p[i]), k = split2(t[i]);
    return pack2(__int_as_float(__float_as_int(q.x) + (__float_as_int(k.x) << 23)), __int_as_float(__float_as_int(q.y) + (__float_as_int(k.y) << 23)));
  }
};
// exp(delta a) of both channels for R tokens and the thread's four states, a in units of log 2; kPoly: the first one's as above
template <int R, bool kPoly> __device__ __forceinline__ void decays(const f32x2* delta, const f32x2* a2, f32x2 (*e)[4]) {
  Poly<R> poly;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (kPoly) poly.begin(i, mul2(delta[i], a2[0]));
#pragma unroll
    for (int j = kPoly; j < 4; ++j) e[i][j] = exp2_unit(mul2(delta[i], a2[j]));
  }
  if (!kPoly) return;
  poly.run();
#pragma unroll
  for (int i = 0; i < R; ++i) e[i][0] = poly.end(i);
}

// ---- the work of a thread ----------------------------------------------------------------------------------------------------
// Of kScan threads that scan and kBring that bring and take, a pair of adjacent channels each.
template <int LN, int kScan, int kBring, int kTokens> struct ScanThread {
  using Tile = ScanTile<LN>;
  static constexpr int kRows = kBring / Tile::kPairs;            // tokens that are brought side by side
  static constexpr int kPasses = kTokens / kRows;
  static constexpr int kStep = kBring / Tile::kN;                // tokens whose b (and c) are
  static constexpr int kBc = kTokens > kStep ? kTokens / kStep : 1;
  // whether the thread's elements of b and c are of the tile's tokens
  __device__ __forceinline__ bool has_states() const { return kBc * kStep == kTokens || tid / Tile::kN < kTokens; }
  static_assert(kScan == LN * Tile::kPairs && kPasses >= 1 && kStep >= 1, "work for every thread");
  int group, c0, nch, b;          // the CTA's group, first channel, channels (<= kChannels), batch row
  bool scans;                     // or brings and takes
  int tid, ln, pair;              // of its kind; in the scan: lane of the channels, pair in the CTA
  int vpair, row, vn;             // when it brings: pair of channels, first token, how many of the two channels there are
  __device__ ScanThread(const ScanShape& s) {
    group = blockIdx.x / s.per_group;
    const int in_group = (blockIdx.x % s.per_group) * Tile::kChannels;
    c0 = group * s.heads + in_group;
    nch = min(Tile::kChannels, s.heads - in_group);
    b = blockIdx.y;
    scans = threadIdx.x < kScan;
    tid = scans ? threadIdx.x : threadIdx.x - kScan;
    ln = tid % LN;
    pair = tid / LN;
    vpair = tid % Tile::kPairs;
    row = tid / Tile::kPairs;
    vn = max(0, min(2, nch - 2 * vpair));
  }
  // n of the thread's state j; channel h of its pair, and whether it is there
  __device__ __forceinline__ int state(int j) const { return j * LN + ln; }
  __device__ __forceinline__ int channel(int h) const { return c0 + 2 * pair + h; }
  __device__ __forceinline__ bool has(int h) const { return 2 * pair + h < nch; }
  // rows [D][N] of fp32 at p, both channels' state j; 0 where there is none
  __device__ __forceinline__ f32x2 get(const float* p, int j, int N) const {
    const bool n = state(j) < N;
    return pack2(n && has(0) ? p[(size_t)channel(0) * N + state(j)] : 0.f, n && has(1) ? p[(size_t)channel(1) * N + state(j)] : 0.f);
  }
  __device__ __forceinline__ void put(float* p, int j, int N, f32x2 v) const {
    const float2 f = split2(v);
    if (state(j) < N && has(0)) p[(size_t)channel(0) * N + state(j)] = f.x;
    if (state(j) < N && has(1)) p[(size_t)channel(1) * N + state(j)] = f.y;
  }
  __device__ __forceinline__ f32x2 get1(const float* p) const {      // [D]
    return pack2(has(0) ? p[channel(0)] : 0.f, has(1) ? p[channel(1)] : 0.f);
  }
  __device__ __forceinline__ void put1(float* p, f32x2 v) const {
    const float2 f = split2(v);
    if (ln == 0 && has(0)) p[channel(0)] = f.x;
    if (ln == 0 && has(1)) p[channel(1)] = f.y;
  }
  // kept rows [D][kN], a lane's four states adjacent
  __device__ __forceinline__ void load_kept(const float* p, f32x2* v) const {
    float4 f[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      f[h] = has(h) ? *reinterpret_cast<const float4*>(p + (size_t)channel(h) * Tile::kN + 4 * ln) : make_float4(0.f, 0.f, 0.f, 0.f);
    v[0] = pack2(f[0].x, f[1].x); v[1] = pack2(f[0].y, f[1].y); v[2] = pack2(f[0].z, f[1].z); v[3] = pack2(f[0].w, f[1].w);
  }
  __device__ __forceinline__ void store_kept(float* p, const f32x2* v) const {
    const float2 a = split2(v[0]), b = split2(v[1]), c = split2(v[2]), d = split2(v[3]);
    if (has(0)) *reinterpret_cast<float4*>(p + (size_t)channel(0) * Tile::kN + 4 * ln) = make_float4(a.x, b.x, c.x, d.x);
    if (has(1)) *reinterpret_cast<float4*>(p + (size_t)channel(1) * Tile::kN + 4 * ln) = make_float4(a.y, b.y, c.y, d.y);
  }
  // Which of a bringing thread's tokens of a tile are there: bit i of pass i.  A plain tile is full, of a full CTA, without a mask and in wide
  // words: nothing is asked about its elements (the questions were a quarter of the forward's instructions).
  __device__ __forceinline__ uint32_t tokens_here(const uint8_t* mask, int64_t t0, int64_t T) const {
    uint32_t here = 0;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int64_t t = t0 + row + i * kRows;
      if (t < T && !(mask && mask[t])) here |= 1u << i;
    }
    return here;
  }
};

// Both channels of a bringing thread's tokens, as they stand in memory; p: at the thread's first token of the tile.
template <typename T, class Thread> struct RawPairs {
  Raw<T, 2> v[Thread::kPasses];
  template <bool kPlain> __device__ __forceinline__ void load(const T* p, int64_t stride, uint32_t here, int vn, bool wide) {
#pragma unroll
    for (int i = 0; i < Thread::kPasses; ++i) {
      const T* at = p + i * Thread::kRows * stride;
      if (kPlain) {
        v[i].load(at, 2, true);
      } else {
        v[i].zero();
        if (here >> i & 1) v[i].load(at, vn, wide);
      }
    }
  }
};
// One tile's b or c, as they stand in memory, n = tid % kN of tokens tid / kN + i * kStep; in shared memory a lane's four states are adjacent.
template <typename T, int LN, class Thread> struct RawStates {
  static constexpr int kN = ScanTile<LN>::kN, kStep = Thread::kStep;
  T v[Thread::kBc];
  template <bool kPlain> __device__ __forceinline__ void load(const Thread& th, const T* p, int64_t stride, int64_t t0, int64_t T_, int N, const uint8_t* mask) {
    const int n = th.tid % kN;
    const T* at = p + (t0 + th.tid / kN) * stride + n;
#pragma unroll
    for (int i = 0; i < Thread::kBc; ++i) {
      const int64_t t = t0 + th.tid / kN + i * kStep;
      const bool there = n < N && th.has_states() && (kPlain || (t < T_ && !(mask && mask[t])));
      v[i] = there ? at[i * kStep * stride] : from_f<T>(0.f);
    }
  }
  __device__ __forceinline__ void store(const Thread& th, float (*smem)[kN]) const {
    const int n = th.tid % kN, t = th.tid / kN;
    if (!th.has_states()) return;
#pragma unroll
    for (int i = 0; i < Thread::kBc; ++i) smem[t + i * kStep][(n % LN) * 4 + n / LN] = to_f(v[i]);
  }
};
struct Plain { static constexpr bool value = true; };
struct Ragged { static constexpr bool value = false; };

// softplus of both channels, and with `kSlope` its derivatives (state_space.cuh has one alone)
template <bool kSlope> __device__ __forceinline__ f32x2 softplus2(float2 v, float2& sig) {
  const float2 z = make_float2(ex2(-kLog2e * fabsf(v.x)), ex2(-kLog2e * fabsf(v.y)));
  const f32x2 z2 = pack2(z.x, z.y);
  const float2 d = split2(add2(z2, both(2.f)));
  const f32x2 w = mul2(z2, pack2(rcp(d.x), rcp(d.y))), s = mul2(w, w);
  f32x2 q = fma2(both(0.281577788f), s, both(0.279651582f));
  q = fma2(q, s, both(0.400245965f));
  q = fma2(q, s, both(0.666663229f));
  q = fma2(q, s, both(2.f));
  if (kSlope) {
    const float r0 = rcp(1.f + z.x), r1 = rcp(1.f + z.y);
    sig = make_float2(v.x >= 0.f ? r0 : z.x * r0, v.y >= 0.f ? r1 : z.y * r1);
  }
  return fma2(w, q, pack2(fmaxf(v.x, 0.f), fmaxf(v.y, 0.f)));
}
__device__ __forceinline__ void lane_states(const float* row, int ln, float* v) {
  const float4 f = *reinterpret_cast<const float4*>(row + 4 * ln);
  v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
}
// Sums `K` values over LN lanes, dealing the results out: afterwards v[0 .. max(1, K / LN)) of lane l are the totals of values
// l * K / LN ... (K >= LN), or of value l * K / LN in every lane (K < LN).  K / 2 + K / 4 + ... exchanges instead of K log LN.
template <int K, int LN, int W = LN> __device__ __forceinline__ void lanes_sum(float* v, int ln) {
  if constexpr (W > 1) {
    if constexpr (K > 1) {
      const bool upper = ln & (W / 2);
#pragma unroll
      for (int i = 0; i < K / 2; ++i) {
        const float give = upper ? v[i] : v[i + K / 2], keep = upper ? v[i + K / 2] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, give, W / 2);
      }
      lanes_sum<K / 2, LN, W / 2>(v, ln);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], W / 2);
      lanes_sum<1, LN, W / 2>(v, ln);
    }
  }
}

// s -> 2^(sum a) s + v over `count` segments, the first at `at`: a thread's states in front of its own segment (or gradients behind it), from the
// others' states and sums of deltas.  The decays may be growth that overflows by itself where the state does not (one that is still zero stays
// so).  A call that meets such a power, beyond 2^126, goes over its segments once more with what is beyond it apart from the rest; beyond
// 2^252 every state but a subnormal one is inf.
template <class Thread>
__device__ __forceinline__ void join_segments(const Thread& th, const ScanShape& sh, const float* states, const float* sums, int at, int count, int step,
                                              const f32x2* a2, f32x2* s) {
  const f32x2 start[4] = {s[0], s[1], s[2], s[3]};
  float most = 0.f;
  const auto segment = [&](int i, f32x2* u, f32x2* v) {
    const size_t row = ((size_t)(at + i * step) * sh.B + th.b) * sh.D;
    th.load_kept(states + row * sh.kn, v);
    const f32x2 over = th.get1(sums + row);
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = mul2(over, a2[j]);
  };
  for (int i = 0; i < count; ++i) {
    f32x2 u[4], v[4];
    segment(i, u, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = split2(u[j]);
      most = fmaxf(most, fmaxf(f.x, f.y));
      s[j] = fma2(exp2_unit(u[j]), s[j], v[j]);
    }
  }
  if (most <= 126.f) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) s[j] = start[j];
#pragma unroll 1
  for (int i = 0; i < count; ++i) {
    f32x2 u[4], v[4];
    segment(i, u, v);
    const auto low = [](float u) { return u > 126.f ? 126.f : u; };                        // NaN stays
    const auto high = [](float u) { return u > 126.f ? fminf(u - 126.f, 126.f) : 0.f; };
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = split2(u[j]);
      s[j] = fma2(exp2_unit(pack2(low(f.x), low(f.y))), mul2(exp2_unit(pack2(high(f.x), high(f.y))), s[j]), v[j]);
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
