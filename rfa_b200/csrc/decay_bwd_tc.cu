// Linear attention with a decay on the tensor cores: the gradients of a chunk, fp16 and bf16, heads of up to 128.
//
// The states in front of each chunk (S) and their gradients behind it (dS, scaled) have been left by two sweeps of decay_tc.cuh as 16-bit tiles.  Then
// the chunks do not depend on each other, and a CTA takes one chunk of 128 tokens of a (batch row, head) after the other.  With w_ij = scale 2^(L_i - L_j), j <= i:
//     T0 = Q K^T, T1 = G V^T          -> P = T0 o w, D = T1 o w      16 bits, in shared memory
//     gq_i = (D K)_i + scale 2^(L_i) (G S^T)_i
//     gk_j = (D^T Q)_j + 2^(L_end - L_j) (V dS^T)_j
//     gv_j = (P^T G)_j + 2^(L_end - L_j) (K dS)_j
// The gradient of the log decay at t is the sum over all pairs of a query i >= t and a key j < t.  With D as it is rounded, M_ij = D_ij q_i . k_j: its rows' sums are
// q_i . (D K)_i and its columns' k_j . (D^T Q)_j, both in fp32 and of one and the same matrix, so that little more than fp32's roundings is left of pairs that
// do not straddle t when they are subtracted.  A token's pair with itself straddles none and does not shrink with the decays: D's diagonal is kept out of the products and
// sums and its part added to gq and gk by itself (where decays of -10 are a head's, it left 10 to 40 % of their gradient wrong; 2 % of a training step).
//     g_t = sum_(i >= t) q_i . gq_i - sum_(j >= t) k_j . (D^T Q)_j + sum_(j < t) 2^(L_end - L_j) k_j . (V dS^T)_j + 2^(L_end) S . dS
//
// Warp roles (608 threads): warp 0 TMA producer, warp 1 MMA issuer, warp 2 the decays, warps 3..18 four groups that share the rows' columns 16 by 16: clear padded
// rows, T0, T1 -> P, D, then the gradients straight from registers.  P takes the place of S.  TMEM: four regions of 128 columns, T0 / T1 / G S^T / V dS^T, the first three
// of them used again.  All waits are bounded.
//
// 8 x 16 heads x 2048 x 128, bf16: 141 us, 149 under the profiler (the whole forward and backward 264 to 287, by the machine), 580 MB of memory traffic (4.1 TB/s); a chunk's chain of loads and products is what the rest waits for.
#define RFA_TC_FAMILY 11
#include <algorithm>

#include "decay_tc.cuh"

namespace rfa {

constexpr int kDgThreads = 608, kDgGroups = 4, kDgRows = kDgGroups * 128;

struct DecayGradArgs {
  DecayRows decay;
  const uint8_t* mask;
  const void *states, *grads;      // [B H][chunks][copy]
  void *gq, *gk, *gv;
  void* g_decay;                   // null; [T][B][H] of decay_dtype, or per_head: fp32 [B][chunks][H]
  int64_t T;
  int B, H, K, D, decay_dtype, per_head;
  bool from_zero;                  // no state in front of the first token
  float scale;
};

template <int KB, int DB>
struct GradLayout {
  static constexpr uint32_t kCopyBytes = KB * DB * 64 * 128;
  static constexpr uint32_t q = 0, k = KB * kBox, v = 2 * KB * kBox, g = v + DB * kBox, s = g + DB * kBox;      // s: S, then P [128][128]
  static constexpr uint32_t d = s + 2 * kBox, ds = d + 2 * kBox, l = ds + (kCopyBytes + 1023) / 1024 * 1024, own = l + 128 * 4, bar = own + 128 * 4, bytes = bar + 160;
  static_assert(bytes <= 227 * 1024, "shared memory");
};
enum { gQK = 0, gVG, gS, gDS, gL, gClean, gT, gN1, gN2, gX, gP, gO1, gO2, gE1, gE2, gO3, gE3, gAll, gSum, gNum };
// Each but gSum completes once a chunk, so that a chunk's parity is every wait's.  gE1, gE2, gE3: gq, gk and gv have been read, with the rows of Q and K.

template <typename T, int KB, int DB>
__global__ void __launch_bounds__(kDgThreads, 1)
decay_grad_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ CUtensorMap tm_g, const __grid_constant__ DecayGradArgs a, int64_t works) {
  using Lay = GradLayout<KB, DB>;
  constexpr int KP = KB * 64, DP = DB * 64;
  extern __shared__ __align__(1024) unsigned char sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Lay::bar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + gNum);
  float *L = reinterpret_cast<float*>(sm + Lay::l), *own = reinterpret_cast<float*>(sm + Lay::own);      // own: D's diagonal
  const uint32_t sbase = smem_u32(sm);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t chunks = (a.T + kTC - 1) / kTC;
  struct Work {
    int64_t bh, chunk, t0;
    int b, h;
    const uint8_t* mask;
  };
  const auto work_of = [&](int64_t w) {
    Work k;
    k.bh = w / chunks;
    k.chunk = w % chunks;
    k.t0 = k.chunk * kTC;
    k.b = (int)(k.bh / a.H);
    k.h = (int)(k.bh % a.H);
    k.mask = a.mask ? a.mask + (int64_t)k.b * a.T : nullptr;
    return k;
  };
  if (tid == 0) {
    for (int i = 0; i < gNum; ++i) mbar_init(&bars[i], i == gL ? 32 : i == gClean || i == gX || i == gP || (i >= gE1 && i <= gE3 && i != gO3) || i == gAll ? kDgRows : i == gSum ? 128 : 1);
    mbar_fence_init();
    tma_prefetch_desc(&tm_q); tma_prefetch_desc(&tm_k); tma_prefetch_desc(&tm_v); tma_prefetch_desc(&tm_g);
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      uint32_t ph = 0;
      for (int64_t w = blockIdx.x; w < works; w += gridDim.x, ph ^= 1) {
        const Work k = work_of(w);
        const int t0 = (int)k.t0;
        if (w != blockIdx.x && (!mbar_wait(&bars[gE2], ph ^ 1) || !mbar_wait(&bars[gO3], ph ^ 1))) { tc_fail(1); break; }
        mbar_arrive_expect_tx(&bars[gQK], 2 * KB * kBox);
        for (int x = 0; x < KB; ++x) tma_load_4d(sm + Lay::q + x * kBox, &tm_q, &bars[gQK], x * 64, k.h, k.b, t0);
        for (int x = 0; x < KB; ++x) tma_load_4d(sm + Lay::k + x * kBox, &tm_k, &bars[gQK], x * 64, k.h, k.b, t0);
        mbar_arrive_expect_tx(&bars[gVG], 2 * DB * kBox);
        for (int x = 0; x < DB; ++x) tma_load_4d(sm + Lay::g + x * kBox, &tm_g, &bars[gVG], x * 64, k.h, k.b, t0);
        for (int x = 0; x < DB; ++x) tma_load_4d(sm + Lay::v + x * kBox, &tm_v, &bars[gVG], x * 64, k.h, k.b, t0);
        const int64_t at = (k.bh * chunks + k.chunk) * Lay::kCopyBytes;
        mbar_arrive_expect_tx(&bars[gS], Lay::kCopyBytes);
        bulk_load(sm + Lay::s, static_cast<const unsigned char*>(a.states) + at, Lay::kCopyBytes, &bars[gS]);
        mbar_arrive_expect_tx(&bars[gDS], Lay::kCopyBytes);
        bulk_load(sm + Lay::ds, static_cast<const unsigned char*>(a.grads) + at, Lay::kCopyBytes, &bars[gDS]);
        if (!mbar_wait(&bars[gDS], ph)) { tc_fail(20); break; }
        if (w + gridDim.x < works) {      // the next chunk on its way to L2 while this one, which has come, is worked on: its tiles have no room here yet
          const Work n = work_of(w + gridDim.x);
          for (int x = 0; x < KB; ++x) {
            tma_prefetch_4d(&tm_q, x * 64, n.h, n.b, (int)n.t0);
            tma_prefetch_4d(&tm_k, x * 64, n.h, n.b, (int)n.t0);
          }
          for (int x = 0; x < DB; ++x) {
            tma_prefetch_4d(&tm_g, x * 64, n.h, n.b, (int)n.t0);
            tma_prefetch_4d(&tm_v, x * 64, n.h, n.b, (int)n.t0);
          }
          const int64_t at = (n.bh * chunks + n.chunk) * Lay::kCopyBytes;
          bulk_prefetch(static_cast<const unsigned char*>(a.states) + at, Lay::kCopyBytes);
          bulk_prefetch(static_cast<const unsigned char*>(a.grads) + at, Lay::kCopyBytes);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t lead = 1u;
      constexpr uint32_t idT = umma_idesc<T>(128, 128, false, false);                                                    // Q K^T, G V^T
      constexpr uint32_t idKK = umma_idesc<T>(128, KP, false, false);                                                   // G S^T, V dS^T
      constexpr uint32_t idD = umma_idesc<T>(128, DP, false, true), idTD = umma_idesc<T>(128, DP, true, true);          // K dS; P^T G
      constexpr uint32_t idK = umma_idesc<T>(128, KP, false, true), idTK = umma_idesc<T>(128, KP, true, true);          // D K; D^T Q
      constexpr uint32_t kCopyBlock = (KP * 128) >> 4;
      const auto rows = [&](uint32_t at) { return umma_smem_desc(sbase + at, 0, 1024, kSwizzle128B); };                 // K-major
      const auto columns = [&](uint32_t at, uint32_t block) { return umma_smem_desc(sbase + at, block, 1024, kSwizzle128B); };      // MN-major
      const uint32_t R0 = tmem, R1 = tmem + 128, R2 = tmem + 256, R3 = tmem + 384;
      uint32_t ph = 0;
      for (int64_t w = blockIdx.x; w < works; w += gridDim.x, ph ^= 1) {
        if (w != blockIdx.x && !mbar_wait(&bars[gE3], ph ^ 1)) { tc_fail(18); break; }
        if (a.mask && !mbar_wait(&bars[gClean], ph)) { tc_fail(1); break; }
        if (!mbar_wait(&bars[gQK], ph)) { tc_fail(2); break; }
        tc_fence_after_sync();
        umma_chain_ss<4 * KB, kStepK, kBlockK, kStepK, kBlockK>(lead, R0, rows(Lay::q), rows(Lay::k), idT, 0);
        if (!mbar_wait(&bars[gVG], ph)) { tc_fail(3); break; }
        umma_chain_ss<4 * DB, kStepK, kBlockK, kStepK, kBlockK>(lead, R1, rows(Lay::g), rows(Lay::v), idT, 0);
        umma_commit(&bars[gT]);
        if (!mbar_wait(&bars[gS], ph)) { tc_fail(4); break; }
        umma_chain_ss<4 * DB, kStepK, kBlockK, kStepK, kCopyBlock>(lead, R2, rows(Lay::g), rows(Lay::s), idKK, 0);
        umma_commit(&bars[gN1]);
        if (!mbar_wait(&bars[gDS], ph)) { tc_fail(5); break; }
        umma_chain_ss<4 * DB, kStepK, kBlockK, kStepK, kCopyBlock>(lead, R3, rows(Lay::v), rows(Lay::ds), idKK, 0);
        umma_commit(&bars[gN2]);
        if (!mbar_wait(&bars[gP], ph)) { tc_fail(6); break; }
        tc_fence_after_sync();
        umma_chain_ss<8, kStepK, kBlockK, kStepMN, kBlockMN>(lead, R0, rows(Lay::d), columns(Lay::k, kBox), idK, 0);
        umma_commit(&bars[gO1]);
        umma_chain_ss<8, kStepMN, kBlockMN, kStepMN, kBlockMN>(lead, R1, columns(Lay::d, kBox), columns(Lay::q, kBox), idTK, 0);
        umma_commit(&bars[gO2]);
        if (!mbar_wait(&bars[gE1], ph)) { tc_fail(7); break; }
        tc_fence_after_sync();
        umma_chain_ss<8, kStepMN, kBlockMN, kStepMN, kBlockMN>(lead, R0, columns(Lay::s, kBox), columns(Lay::g, kBox), idTD, 0);
        umma_chain_ss<4 * KB, kStepK, kBlockK, kStepMN, kBlockMN>(lead, R2, rows(Lay::k), columns(Lay::ds, KP * 128), idD, 0);
        umma_commit(&bars[gO3]);
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ decays: a lane takes four adjacent tokens
    // Sums of 40 bits behind the point: as exact as 64-bit floats' for this and several times as fast; L itself is stored in 32 bits, as in the sweep
    uint32_t ph = 0;
    for (int64_t w = blockIdx.x; w < works; w += gridDim.x, ph ^= 1) {
      const Work k = work_of(w);
      uint32_t bits[4];
      bool real[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t t = k.t0 + lane * 4 + e;
        real[e] = t < a.T;
        bits[e] = real[e] ? log_decay_bits(a.decay.p, a.decay_dtype, k.b * a.decay.b + k.h * a.decay.h + t * a.decay.t) : 0u;
        if (real[e] && k.mask) real[e] = !k.mask[t];
      }
      // Growth beyond 2^32768 (e^22713) is taken as that: an infinite weight still, and 128 of them fit 64 bits.  What is no number makes L none from its token on.
      long long sum[4], all = 0;
      bool none[4], any = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (real[e]) {
          const float g = log_decay_number(bits[e], a.decay_dtype);
          any |= g != g;
          all += __double2ll_rn((double)fminf(fmaxf(g, kDecayFloor), 22713.f) * (kLog2eD * 1099511627776.0));
        }
        sum[e] = all;
        none[e] = any;
      }
      const bool behind = (__ballot_sync(0xffffffffu, any) & ((1u << lane) - 1)) != 0;
      long long before = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
      }
      before -= all;
      if (w != blockIdx.x && !mbar_wait(&bars[gP], ph ^ 1)) { tc_fail(19); break; }      // the last chunk's have been read
#pragma unroll
      for (int e = 0; e < 4; ++e) L[lane * 4 + e] = none[e] || behind ? __int_as_float(0x7fffffff) : __ll2float_rn(sum[e] + before) * 0x1p-40f;
      mbar_arrive(&bars[gL]);
    }
  } else {
    // ------------------------------------------------------------------ four groups of 128: rows of the chunk, every fourth 16 columns
    const int group = (warp - 3) >> 2, quarter = warp & 3, row = quarter * 32 + lane, wtid = tid - 96;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t R0 = tmem + lane_addr, R1 = R0 + 128, R2 = R0 + 256, R3 = R0 + 384;
    const bool want = a.g_decay != nullptr;
    const auto sectors = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; };
    const bool wide_q = a.K % 16 == 0 && sectors(a.gq), wide_k = a.K % 16 == 0 && sectors(a.gk), wide_d = a.D % 16 == 0 && sectors(a.gv);
    uint32_t ph = 0, sum_phase = 0;
    for (int64_t w = blockIdx.x; w < works; w += gridDim.x, ph ^= 1) {
      const Work k = work_of(w);
      const uint8_t* mask = k.mask;
      const int64_t t = k.t0 + row;
      const bool there = t < a.T;
      float x = 0.f, rows_sum = 0.f, cols_sum = 0.f, keys_sum = 0.f;      // S . dS; q . gq; k . (D^T Q), both without the token itself; k . (V dS^T)
      if (mask) {      // padded rows may hold anything: zero before a product reads them
        if (!mbar_wait(&bars[gQK], ph) || !mbar_wait(&bars[gVG], ph)) { tc_fail(8); break; }
        if (there && mask[t]) {
          const uint4 zero = make_uint4(0, 0, 0, 0);
          if (group == 0) {
#pragma unroll 1
            for (int ch = 0; ch < 8 * KB; ++ch) {
              *reinterpret_cast<uint4*>(sm + Lay::q + row_chunk2(row, ch)) = zero;
              *reinterpret_cast<uint4*>(sm + Lay::k + row_chunk2(row, ch)) = zero;
            }
          } else if (group == 1) {
#pragma unroll 1
            for (int ch = 0; ch < 8 * DB; ++ch) {
              *reinterpret_cast<uint4*>(sm + Lay::v + row_chunk2(row, ch)) = zero;
              *reinterpret_cast<uint4*>(sm + Lay::g + row_chunk2(row, ch)) = zero;
            }
          }
        }
        fence_async_smem();
        mbar_arrive(&bars[gClean]);
      }
      if (!mbar_wait(&bars[gS], ph) || !mbar_wait(&bars[gDS], ph)) { tc_fail(9); break; }
      if (want) {
#pragma unroll 1
        for (uint32_t i = wtid * 16; i < Lay::kCopyBytes; i += kDgRows * 16) {
          const uint4 u = *reinterpret_cast<const uint4*>(sm + Lay::s + i), w = *reinterpret_cast<const uint4*>(sm + Lay::ds + i);
          const uint32_t us[4] = {u.x, u.y, u.z, u.w}, ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack2h<T>(us[e]), g = unpack2h<T>(ws[e]);
            x = fmaf(f.x, g.x, fmaf(f.y, g.y, x));
          }
        }
      }
      mbar_release_stage(&bars[gX]);      // S has been read
      if (!mbar_wait(&bars[gX], ph) || !mbar_wait(&bars[gL], ph)) { tc_fail(10); break; }
      const float mine = L[row], end = L[127];
      if (!mbar_wait(&bars[gT], ph) || !mbar_wait(&bars[gN1], ph)) { tc_fail(11); break; }
      tc_fence_after_sync();
      const int pieces = 2 * quarter + 2;      // of 16 columns, that reach up to the diagonal
#pragma unroll 1
      for (int p = group; p < 8; p += kDgGroups) {
        uint32_t pw[8], dw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) pw[i] = dw[i] = 0u;
        if (p < pieces) {
          uint32_t s0[16], s1[16];
          tmem_ld16(R0 + p * 16, s0);
          tmem_ld16(R1 + p * 16, s1);
          float f[16];
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const float4 l = *reinterpret_cast<const float4*>(L + p * 16 + i);
            f[i] = a.scale * ex2(mine - l.x); f[i + 1] = a.scale * ex2(mine - l.y); f[i + 2] = a.scale * ex2(mine - l.z); f[i + 3] = a.scale * ex2(mine - l.w);
          }
          tmem_ld_wait();
          if (p >= 2 * quarter) {      // the diagonal's
            const int last = row - p * 16, self = want ? last : -1;
            float with_itself = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              f[i] = i > last ? 0.f : f[i];
              with_itself = i == self ? __uint_as_float(s1[i]) * f[i] : with_itself;
              s1[i] = i == self ? 0u : s1[i];      // the token with itself: apart, see the decays below
            }
            if (self >= 0 && self < 16) own[row] = with_itself;
          }
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            pw[i >> 1] = pack2h<T>(__uint_as_float(s0[i]) * f[i], __uint_as_float(s0[i + 1]) * f[i + 1]);
            dw[i >> 1] = pack2h<T>(__uint_as_float(s1[i]) * f[i], __uint_as_float(s1[i + 1]) * f[i + 1]);
          }
        }
        *reinterpret_cast<uint4*>(sm + Lay::s + row_chunk2(row, 2 * p)) = make_uint4(pw[0], pw[1], pw[2], pw[3]);
        *reinterpret_cast<uint4*>(sm + Lay::s + row_chunk2(row, 2 * p + 1)) = make_uint4(pw[4], pw[5], pw[6], pw[7]);
        *reinterpret_cast<uint4*>(sm + Lay::d + row_chunk2(row, 2 * p)) = make_uint4(dw[0], dw[1], dw[2], dw[3]);
        *reinterpret_cast<uint4*>(sm + Lay::d + row_chunk2(row, 2 * p + 1)) = make_uint4(dw[4], dw[5], dw[6], dw[7]);
      }
      fence_async_smem();
      tc_fence_before_sync();
      mbar_arrive(&bars[gP]);

      const float fq = a.scale * ex2(mine), fk = ex2(end - mine);
      const int64_t at = (t * a.B + k.b) * a.H + k.h;
      // ---- gq, gk
      const auto grad = [&](uint32_t main, uint32_t side, float f, void* out, uint32_t tile, uint32_t other, float& inside, float& across, bool wide) {
        T* o = static_cast<T*>(out) + at * a.K;
        const float self = want ? own[row] : 0.f;
#pragma unroll 1
        for (int c0 = group * 16; c0 < KP; c0 += kDgGroups * 16) {
          uint32_t u[16], n[16];
          tmem_ld16(main + c0, u);
          tmem_ld16(side + c0, n);
          tmem_ld_wait();
          float v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float s = f * __uint_as_float(n[i]);
            v[i] = __uint_as_float(u[i]) + s;
            n[i] = __float_as_uint(s);
          }
          if (want) {
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
              const uint4 y = *reinterpret_cast<const uint4*>(sm + tile + row_chunk2(row, (c0 >> 3) + ch));
              const uint32_t ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 z = unpack2h<T>(ys[e]);
                inside = fmaf(__uint_as_float(u[8 * ch + 2 * e]), z.x, fmaf(__uint_as_float(u[8 * ch + 2 * e + 1]), z.y, inside));
                across = fmaf(__uint_as_float(n[8 * ch + 2 * e]), z.x, fmaf(__uint_as_float(n[8 * ch + 2 * e + 1]), z.y, across));
              }
              const uint4 y2 = *reinterpret_cast<const uint4*>(sm + other + row_chunk2(row, (c0 >> 3) + ch));
              const uint32_t y2s[4] = {y2.x, y2.y, y2.z, y2.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 z = unpack2h<T>(y2s[e]);
                v[8 * ch + 2 * e] = fmaf(self, z.x, v[8 * ch + 2 * e]);
                v[8 * ch + 2 * e + 1] = fmaf(self, z.y, v[8 * ch + 2 * e + 1]);
              }
            }
          }
          if (there && c0 < a.K) store_row16(o + c0, v, a.K - c0, wide);
        }
      };
      if ((want && !mbar_wait(&bars[gP], ph)) || !mbar_wait(&bars[gO1], ph)) { tc_fail(12); break; }      // gP: `own` is there
      tc_fence_after_sync();
      grad(R0, R2, fq, a.gq, Lay::q, Lay::k, rows_sum, rows_sum, wide_q);
      tc_fence_before_sync();
      mbar_arrive(&bars[gE1]);
      if (!mbar_wait(&bars[gN2], ph) || !mbar_wait(&bars[gO2], ph)) { tc_fail(13); break; }
      tc_fence_after_sync();
      grad(R1, R3, fk, a.gk, Lay::k, Lay::q, cols_sum, keys_sum, wide_k);
      mbar_release_stage(&bars[gE2]);
      // ---- gv
      if (!mbar_wait(&bars[gO3], ph)) { tc_fail(14); break; }
      tc_fence_after_sync();
      T* o = static_cast<T*>(a.gv) + at * a.D;
#pragma unroll 1
      for (int c0 = group * 16; c0 < DP; c0 += kDgGroups * 16) {
        uint32_t u[16], n[16];
        tmem_ld16(R0 + c0, u);
        tmem_ld16(R2 + c0, n);
        tmem_ld_wait();
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = fmaf(fk, __uint_as_float(n[i]), __uint_as_float(u[i]));
        if (there && c0 < a.D) store_row16(o + c0, v, a.D - c0, wide_d);
      }
      tc_fence_before_sync();
      mbar_arrive(&bars[gE3]);
      // ---- the decays: D has been read by its products (gO1, gO2), so that its place serves the exchange
      if (want) {
        // [group][128] rows less columns, [group][128] keys of the other groups, a sum of S . dS for each warp, the first group's warps' sums
        float* ex = reinterpret_cast<float*>(sm + Lay::d);
        float *ex_x = ex + 2 * kDgRows, *ex_down = ex_x + 16, *ex_up = ex_down + 4, *ex_all = ex_up + 4;
        x = warp_sum(x);
        if (lane == 0) ex_x[warp - 3] = x;
        if (group > 0) {
          ex[group * 128 + row] = rows_sum - cols_sum;
          ex[kDgRows + group * 128 + row] = keys_sum;
        }
        mbar_arrive(&bars[gAll]);
        if (!mbar_wait(&bars[gAll], ph)) { tc_fail(15); break; }
        // suffix sums of rows less columns, prefix sums of keys, by the first group: within a warp, then across
        if (group == 0) {
          float down = rows_sum - cols_sum, up = keys_sum;
#pragma unroll
          for (int i = 1; i < kDgGroups; ++i) {
            down += ex[i * 128 + row];
            up += ex[kDgRows + i * 128 + row];
          }
          const float own_up = up;
#pragma unroll
          for (int o2 = 1; o2 < 32; o2 <<= 1) {
            const float d = __shfl_down_sync(0xffffffffu, down, o2), u = __shfl_up_sync(0xffffffffu, up, o2);
            if (lane + o2 < 32) down += d;
            if (lane >= o2) up += u;
          }
          if (lane == 0) ex_down[quarter] = down;
          if (lane == 31) ex_up[quarter] = up;
          if (!epi_sync(&bars[gSum], sum_phase)) { tc_fail(16); break; }
          float g = 0.f;
#pragma unroll
          for (int i = 0; i < 4 * kDgGroups; ++i) g += ex_x[i];
          g = ex2(end) * g + down + up - own_up;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i > quarter) g += ex_down[i];
            if (i < quarter) g += ex_up[i];
          }
          const bool real = there && !(mask && mask[t]);
          // The first token with nothing in front decays nothing: 0, not the rounding of sums that cancel.  It is a warp's first one, if padding or nothing is right in
          // front of that and in all places before, which the warp looks at 128 at a time.
          const bool edge = lane > 0 || t == 0 || (there && mask && mask[t - 1]);
          const unsigned reals = __ballot_sync(0xffffffffu, real), edges = __ballot_sync(0xffffffffu, edge);
          const int lead = __ffs(reals) - 1;
          bool first = a.from_zero && reals && (lead > 0 || (edges & 1u));
          if (first)
            for (int64_t p = k.t0 + quarter * 32 + lead - 1 - lane; __any_sync(0xffffffffu, p >= 0); p -= 128) {
              bool found = false;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (p - 32 * i >= 0) found |= !mask[p - 32 * i];
              if (__any_sync(0xffffffffu, found)) {
                first = false;
                break;
              }
            }
          first = first && lane == lead;
          if (!real || first) g = 0.f;
          if (!a.per_head) {
            if (there) {
              if (a.decay_dtype == RFA_F32) static_cast<float*>(a.g_decay)[at] = g;
              else if (a.decay_dtype == RFA_F16) static_cast<__half*>(a.g_decay)[at] = __float2half_rn(g);
              else static_cast<__nv_bfloat16*>(a.g_decay)[at] = __float2bfloat16_rn(g);
            }
          } else {
            g = warp_sum(g);
            if (lane == 0) ex_all[quarter] = g;
            if (!epi_sync(&bars[gSum], sum_phase)) { tc_fail(17); break; }
            if (row == 0) static_cast<float*>(a.g_decay)[(k.b * chunks + k.chunk) * a.H + k.h] = ex_all[0] + ex_all[1] + ex_all[2] + ex_all[3];
          }
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

namespace {

template <typename T, int KB, int DB>
int launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& g, const DecayGradArgs& a, cudaStream_t stream) {
  constexpr uint32_t smem = GradLayout<KB, DB>::bytes;
  cudaError_t e = cudaFuncSetAttribute(decay_grad_tc_kernel<T, KB, DB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return fail((int)e, "decay_bwd: cannot reserve %u bytes of shared memory: %s", smem, cudaGetErrorString(e));
  const int64_t ctas = (int64_t)a.B * a.H * ((a.T + kTC - 1) / kTC);
  e = launch_pdl(decay_grad_tc_kernel<T, KB, DB>, dim3((unsigned)std::min<int64_t>(ctas, 148)), dim3(kDgThreads), smem, stream, q, k, v, g, a, ctas);
  if (e != cudaSuccess) return fail((int)e, "rfa_decay_bwd: launch failed: %s", cudaGetErrorString(e));
  return check_launch("rfa_decay_bwd");
}

}  // namespace

int launch_decay_grad_tc(const rfa_decay_t& c, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& g, const void* states, const void* grads,
                         void* gq, void* gk, void* gv, void* g_decay, cudaStream_t stream) {
  DecayGradArgs a{};
  a.decay = {c.log_decay, c.g_t, c.g_b, c.g_h};
  a.mask = c.mask;
  a.states = states; a.grads = grads;
  a.gq = gq; a.gk = gk; a.gv = gv; a.g_decay = g_decay;
  a.T = c.T; a.B = c.B; a.H = c.H; a.K = c.K; a.D = c.D; a.decay_dtype = c.decay_dtype; a.per_head = c.per_head != 0;
  a.from_zero = !c.s_in;
  a.scale = c.scale;
  switch ((c.dtype == RFA_BF16 ? 4 : 0) + (c.K > 64 ? 2 : 0) + (c.D > 64 ? 1 : 0)) {
    case 0: return launch<__half, 1, 1>(q, k, v, g, a, stream);
    case 1: return launch<__half, 1, 2>(q, k, v, g, a, stream);
    case 2: return launch<__half, 2, 1>(q, k, v, g, a, stream);
    case 3: return launch<__half, 2, 2>(q, k, v, g, a, stream);
    case 4: return launch<__nv_bfloat16, 1, 1>(q, k, v, g, a, stream);
    case 5: return launch<__nv_bfloat16, 1, 2>(q, k, v, g, a, stream);
    case 6: return launch<__nv_bfloat16, 2, 1>(q, k, v, g, a, stream);
    default: return launch<__nv_bfloat16, 2, 2>(q, k, v, g, a, stream);
  }
}

RFA_TC_UNIT(decay_bwd)

}  // namespace rfa
