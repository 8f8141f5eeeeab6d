// Linear attention with a decay on the 5th-generation tensor cores (tcgen05 + TMEM + TMA), fp16 and bf16, heads of up to 128: the sweep over the
// tokens that gives the outputs, or the states alone.
//
// One CTA walks a (batch row, head[, segment]) in chunks of 128 tokens.  With L_i the sum of the log decays up to and with token i of the chunk (in units of
// log 2), w_ij = 2^(L_i - L_j), K'_j = 2^(L_end - L_j) k_j, S the running state [key dim][head dim], fp32 in TMEM:
//     A  = Q K^T             -> P = A o w for j <= i, 16 bits, over A
//     N  = Q S                  (S's 16-bit copy in shared memory)
//     O  = P V
//     S  = 2^(L_end) S + K'^T V
//     out_i = scale (2^(L_i) N_i + O_i)
// A scale of at most one goes into P, a larger one to what comes of it: fp16 then holds scores that fit with the scale or without it.
// L_i - L_j is at most 0 in a model, so that nothing overflows whatever the decays are.  S is exact where it leaves the call (EXACT): K' goes in as two 16-bit
// parts then (bf16's hold 16 bits: the products are off by 2^-17, the state by 3e-6 of its norm).  Where only outputs are wanted its first part is as
// good as the 16-bit copies of S and P.  A log decay below -64 (in units of log 2) is taken as that.
// L is summed in 64 bits and stored in 32: its rounding, 2^-24 |L|, is a weight's error.  That is 1e-6 for gates whose chunk fades by e^-10, and with resets, each worth
// 64, 3e-6 apiece: up to what fp16 rounds a weight by (2^-11) where a chunk is nothing but resets, and between these no weight is left.  A pair of floats would
// take one more instruction and read a score.
//
// Backwards (states alone), from the last chunk to the first: S = 2^(L_end) S + scale Q'^T G, Q'_i = 2^(L_i) q_i: the gradient of the state.  `kept`: the
// 16-bit copy of the state in front of each chunk (behind it, backwards) goes to memory as it stands in shared memory, for decay_bwd_tc.cu.
//
// Warp roles (768 threads): warp 0 TMA producer; warps 1 and 18 MMA issuers (A: Q K^T, P V; B: Q S, the state: issuing one costs the issuing thread about 70
// cycles, and a chunk has 20 to 40); warps 2..5 score group (A -> P); warps 6..9 and 20..23 state groups, half of the columns each (state -> 16-bit copy,
// state times the next chunk's decay); warps 14..17 output group; warp 19 the decays (64-bit sums); warps 10..13 key group (states alone: with 2..5): K' in place of K once A is complete,
// zeros over the rows of padded tokens.  Per chunk the serial chain is  state MMA -> copy and decay -> next state MMA.  All waits are bounded.
//
// 8 x 16 heads x 2048, bf16: 64 wide with an exact state 45 us (3.0 TB/s of what it cannot do without), 128 wide with states kept 62 us, states alone 36 us (5.6 TB/s).  It takes
// every length: 8 x 16 heads of 64, here / the sweep for any sizes (decay_sweep.cu), us, 2 tokens 6 / 11, 64 6 / 35, 1024 22 / 385.  Many narrow heads of a few tokens would be faster
// there (168 x 16 x 2 tokens x 8 x 32: 111 / 52), because a chunk takes its 6 us however little is in it.
#pragma once

#include "decay.cuh"
#include "tc_rows.cuh"

namespace rfa {

constexpr int kDecThreads = 768;
constexpr double kLog2eD = 1.4426950408889634;
constexpr float kDecayFloor = -44.3614196f;      // -64 in units of log 2

struct DecayTcArgs {
  DecayRows decay;
  const uint8_t* mask;
  void *out, *kept;              // kept: [B H][chunks][copy]
  DecayState s_in, s_out;
  float* totals;
  double* seg_decay;
  int64_t T, tseg;
  int B, H, K, D, nseg, decay_dtype, rev;
  float in_scale, out_scale;     // of the scores; out_scale = p_scale o_scale: in P, of its products
  float p_scale, o_scale;
};

// Offsets in shared memory, from a 1024-aligned base, and TMEM columns.  KB, DB: 64-wide boxes of a key, of a value.  As many stages as there is room for: a load
// takes 2 to 3 us when all SMs load, a chunk of narrow heads about one.
constexpr int kDecMaxStages = 5;
template <int KB, int DB, bool OUT, bool EXACT>
struct DecLayout {
  static constexpr uint32_t kCopyBytes = KB * DB * 64 * 128;            // S's copy: DB boxes of [KB 64][64]
  static constexpr uint32_t kCopyRoom = KB == 1 ? kBox : kCopyBytes;    // an operand's second 64-block may be read past a single box
  static constexpr int kCopies = OUT ? 1 : 2;                           // one on its way to memory while the next is written
  static constexpr uint32_t kFixed = (EXACT ? KB * kBox : 0) + kCopies * kCopyRoom, kStage = (KB + DB) * kBox, kTail = 8 * 128 * 4 + 32 + 400;
  static constexpr int kFit = (int)((227 * 1024 - kTail - kFixed) / (kStage + (OUT ? KB * kBox : 0)));
  static constexpr int kStages = kFit >= 2 ? (kFit < kDecMaxStages ? kFit : kDecMaxStages) : 2, kQStages = OUT ? kStages : 0;
  // Where two whole stages have no room it is V that has one place: its load runs beside the key group's work, Q's would run in front of it.
  static constexpr int kVStages = OUT && kFit < 2 ? 1 : kStages;
  static constexpr int kL = kFit >= 2 ? 4 : 2;                          // chunks' decays at a time: they run ahead of what waits for the state
  static constexpr uint32_t q = 0, k = q + kQStages * KB * kBox, v = k + kStages * KB * kBox, low = v + kVStages * DB * kBox, copy = low + (EXACT ? KB * kBox : 0);
  static constexpr uint32_t l = copy + kCopies * kCopyRoom;
  static constexpr uint32_t key_fac = l + kL * 128 * 4, fac = key_fac + kL * 128 * 4, bar = fac + 8 * kL, bytes = bar + 400;
  static constexpr int kA = OUT && DB == 1 ? 2 : 1;                     // buffers of A
  static constexpr uint32_t colS = 0, colN = DB * 64, colO = 2 * DB * 64, colA = 3 * DB * 64, cols = 512;
  static_assert(colA + kA * 128 <= 512, "TMEM");
  static_assert(bytes <= 227 * 1024, "shared memory");
};
enum { dFull = 0, dFree = 5, dFullV = 10, dFreeV, dL = 12, dLFree = 16, dA = 20, dP = 22, dKp = 24, dClean = 28, dS = 32, dSt, dNFree, dKept, dNum };
static_assert(dNum * 8 + 4 <= 400, "barriers");
// dFull, dFree: a stage's tiles have come, all products of its chunk are complete (out may be read); dFullV, dFreeV: the same of V where it has one place only.
// dL / dLFree: a chunk's L and factors are there, have been used.  dClean: the rows of padded tokens are zero (waited for where there is a mask).  dKp: K' stands in
// place of K.  dS: the state's MMAs of a chunk are complete.  dSt: the copy of the state and the decayed state are there.  Barriers in pairs alternate with the
// chunk where their waiter could otherwise be two phases behind (the decays, and so the key group, are at most kL chunks ahead, by dLFree).

template <typename T, int KB, int DB, bool OUT, bool EXACT>
__global__ void __launch_bounds__(kDecThreads, 1)
decay_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const __grid_constant__ DecayTcArgs a, bool totals_only) {
  using Lay = DecLayout<KB, DB, OUT, EXACT>;
  constexpr int KP = KB * 64, DP = DB * 64;
  constexpr bool kOneV = Lay::kVStages == 1;
  extern __shared__ __align__(1024) unsigned char sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Lay::bar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + dNum);
  float* Ls = reinterpret_cast<float*>(sm + Lay::l);
  float* key_fac = reinterpret_cast<float*>(sm + Lay::key_fac);
  Factor* fac = reinterpret_cast<Factor*>(sm + Lay::fac);
  const uint32_t sbase = smem_u32(sm);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t bh = blockIdx.x, BH = (int64_t)a.B * a.H;
  const int b = (int)(bh / a.H), h = (int)(bh % a.H), seg = blockIdx.y, place = a.rev ? a.nseg - 1 - seg : seg;
  const int64_t t_begin = place * a.tseg, t_end = min(a.T, t_begin + a.tseg);
  const int nchunk = (int)((t_end - t_begin + kTC - 1) / kTC);
  const uint8_t* mask = a.mask ? a.mask + (int64_t)b * a.T : nullptr;
  const auto chunk_t0 = [&](int c) { return t_begin + (int64_t)(a.rev ? nchunk - 1 - c : c) * kTC; };

  if (tid == 0) {
    for (int i = 0; i < dL; ++i) mbar_init(&bars[i], OUT && (i >= dFree && i != dFullV) ? 2 : 1);      // both issuers
    for (int i = 0; i < Lay::kL; ++i) {
      mbar_init(&bars[dL + i], 32); mbar_init(&bars[dLFree + i], OUT ? 128 : 256);
      mbar_init(&bars[dKp + i], OUT ? 128 : 256); mbar_init(&bars[dClean + i], 128);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[dA + i], 1); mbar_init(&bars[dP + i], 128);
    }
    mbar_init(&bars[dS], 1); mbar_init(&bars[dSt], 256); mbar_init(&bars[dNFree], 128); mbar_init(&bars[dKept], 1);
    mbar_fence_init();
    if (OUT) tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k); tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) { tmem_alloc(tmem_slot, Lay::cols); tmem_relinquish(); }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      for (int c = 0; c < nchunk; ++c) {
        const int st = c % Lay::kStages, n = c / Lay::kStages, t0 = (int)chunk_t0(c);
        if (n >= 1 && !mbar_wait(&bars[dFree + st], (n + 1) & 1)) { tc_fail(1); break; }
        mbar_arrive_expect_tx(&bars[dFull + st], (KB + (OUT ? KB : 0) + (kOneV ? 0 : DB)) * kBox);
        for (int x = 0; x < KB; ++x) tma_load_4d(sm + Lay::k + (st * KB + x) * kBox, &tm_k, &bars[dFull + st], x * 64, h, b, t0);
        if constexpr (OUT)
          for (int x = 0; x < KB; ++x) tma_load_4d(sm + Lay::q + (st * KB + x) * kBox, &tm_q, &bars[dFull + st], x * 64, h, b, t0);
        uint64_t* full = &bars[kOneV ? dFullV : dFull + st];
        if (kOneV) {
          if (c >= 1 && !mbar_wait(&bars[dFreeV], (c + 1) & 1)) { tc_fail(2); break; }
          mbar_arrive_expect_tx(full, DB * kBox);
        }
        for (int x = 0; x < DB; ++x) tma_load_4d(sm + Lay::v + ((kOneV ? 0 : st) * DB + x) * kBox, &tm_v, full, x * 64, h, b, t0);
      }
    }
  } else if (warp == 1 || warp == 18) {
    // ------------------------------------------------------------------ MMA issuers
    if (lane == 0) {
      constexpr uint32_t lead = 1u;
      constexpr uint32_t idA = umma_idesc<T>(128, 128, false, false);    // Q K^T
      constexpr uint32_t idN = umma_idesc<T>(128, DP, false, true);      // Q S; P V   (B MN-major)
      constexpr uint32_t idS = umma_idesc<T>(128, DP, true, true);       // K'^T V     (A, B MN-major; with 64 keys the rows behind them are not used)
      const uint64_t dQ = umma_smem_desc(sbase + Lay::q, 0, 1024, kSwizzle128B), dK = umma_smem_desc(sbase + Lay::k, 0, 1024, kSwizzle128B);
      const uint64_t dKt = umma_smem_desc(sbase + Lay::k, kBox, 1024, kSwizzle128B), dLow = umma_smem_desc(sbase + Lay::low, kBox, 1024, kSwizzle128B);
      const uint64_t dV = umma_smem_desc(sbase + Lay::v, kBox, 1024, kSwizzle128B), dC = umma_smem_desc(sbase + Lay::copy, KP * 128, 1024, kSwizzle128B);
      constexpr uint64_t kK = (KB * kBox) >> 4, kV = (DB * kBox) >> 4;
      if (warp == 1) {
        // ---- issuer A: the scores of the next chunk as early as they can be, O = P V
        if constexpr (OUT) {
          const auto issue_A = [&](int c) {
            const int before = c - Lay::kA;      // the key group has seen this buffer's last completion
            if (before >= 0 && !mbar_wait(&bars[dKp + before % Lay::kL], (before / Lay::kL) & 1)) { tc_fail(27); return false; }
            const int ab = Lay::kA == 2 ? c & 1 : 0, st = c % Lay::kStages;
            if (!mbar_wait(&bars[dFull + st], (c / Lay::kStages) & 1)) { tc_fail(4); return false; }
            if (mask && !mbar_wait(&bars[dClean + c % Lay::kL], (c / Lay::kL) & 1)) { tc_fail(5); return false; }
            tc_fence_after_sync();
            umma_chain_ss<4 * KB, kStepK, kBlockK, kStepK, kBlockK>(lead, tmem + Lay::colA + ab * 128, dQ + st * kK, dK + st * kK, idA, 0);
            umma_commit(&bars[dA + ab]);
            return true;
          };
          bool ok = nchunk > 0 && issue_A(0);
#pragma unroll 1
          for (int c = 0; ok && c < nchunk; ++c) {
            const int st = c % Lay::kStages, ab = Lay::kA == 2 ? c & 1 : 0, an = Lay::kA == 2 ? c >> 1 : c;
            if (Lay::kA == 2 && c + 1 < nchunk && !issue_A(c + 1)) break;
            if (c >= 1 && !mbar_wait(&bars[dNFree], (c + 1) & 1)) { tc_fail(25); break; }
            if (kOneV && !mbar_wait(&bars[dFullV], c & 1)) { tc_fail(24); break; }
            if (!mbar_wait(&bars[dP + ab], an & 1)) { tc_fail(9); break; }
            tc_fence_after_sync();
            umma_chain_ts<8, kStepMN, kBlockMN>(lead, tmem + Lay::colO, tmem + Lay::colA + ab * 128, dV + (kOneV ? 0 : st) * kV, idN, 0);
            umma_commit(&bars[dFree + st]);
            if (kOneV) umma_commit(&bars[dFreeV]);
            if (Lay::kA == 1 && c + 1 < nchunk && !issue_A(c + 1)) break;
          }
        }
      } else {
        // ---- issuer B: S += K'^T V, N = Q S
#pragma unroll 1
        for (int c = 0; c < nchunk; ++c) {
          const int st = c % Lay::kStages;
          if (!mbar_wait(&bars[dFull + st], (c / Lay::kStages) & 1) || !mbar_wait(&bars[dKp + c % Lay::kL], (c / Lay::kL) & 1)) { tc_fail(8); break; }
          if (kOneV && !mbar_wait(&bars[dFullV], c & 1)) { tc_fail(26); break; }
          if (!mbar_wait(&bars[dSt], c & 1)) { tc_fail(6); break; }
          tc_fence_after_sync();
          umma_chain_ss<8, kStepMN, kBlockMN, kStepMN, kBlockMN>(lead, tmem + Lay::colS, dKt + st * kK, dV + (kOneV ? 0 : st) * kV, idS, 1);
          if (EXACT) umma_chain_ss<8, kStepMN, kBlockMN, kStepMN, kBlockMN>(lead, tmem + Lay::colS, dLow, dV + (kOneV ? 0 : st) * kV, idS, 1);
          if (kOneV) umma_commit(&bars[dFreeV]);
          if constexpr (OUT) {
            if (c >= 1 && !mbar_wait(&bars[dNFree], (c + 1) & 1)) { tc_fail(7); break; }
            tc_fence_after_sync();
            umma_chain_ss<4 * KB, kStepK, kBlockK, kStepMN, kBlockMN>(lead, tmem + Lay::colN, dQ + st * kK, dC, idN, 0);
          }
          umma_commit(&bars[dS]);                // the copy has been read, too
          umma_commit(&bars[dFree + st]);
        }
      }
    }
  } else if (OUT && warp < 6) {
    // ------------------------------------------------------------------ score group: P = A o w
    if constexpr (OUT) {
      const int quarter = warp & 3, row = quarter * 32 + lane;
      const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
      for (int c = 0; c < nchunk; ++c) {
        const int ab = Lay::kA == 2 ? c & 1 : 0, an = Lay::kA == 2 ? c >> 1 : c;
        const uint32_t col = tmem + lane_addr + Lay::colA + ab * 128;
        if (!mbar_wait(&bars[dL + c % Lay::kL], (c / Lay::kL) & 1)) { tc_fail(10); break; }
        const float* L = Ls + c % Lay::kL * 128;
        const float mine = L[row];
        if (!mbar_wait(&bars[dA + ab], an & 1)) { tc_fail(11); break; }
        tc_fence_after_sync();
        // 16 columns at a time, the next ones on their way; those that reach the diagonal keep columns up to `last`
        uint32_t next[16];
        tmem_ld16(col, next);
        const auto piece_of = [&](int piece, int last, auto DIAG) {
          uint32_t s[16], p[8];
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = next[i];
          if (piece < 7) tmem_ld16(col + piece * 16 + 16, next);
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const float4 l = *reinterpret_cast<const float4*>(L + piece * 16 + i);
            float x[4] = {__uint_as_float(s[i]) * a.p_scale * ex2(mine - l.x), __uint_as_float(s[i + 1]) * a.p_scale * ex2(mine - l.y),
                          __uint_as_float(s[i + 2]) * a.p_scale * ex2(mine - l.z), __uint_as_float(s[i + 3]) * a.p_scale * ex2(mine - l.w)};
            if constexpr (decltype(DIAG)::value) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (i + e > last) x[e] = 0.f;
            }
            p[i >> 1] = pack2h<T>(x[0], x[1]);
            p[(i >> 1) + 1] = pack2h<T>(x[2], x[3]);
          }
          tmem_st8(col + piece * 8, p);
        };
#pragma unroll 1
        for (int piece = 0; piece < 2 * quarter; ++piece) piece_of(piece, 16, std::false_type{});
#pragma unroll 1
        for (int piece = 2 * quarter; piece < 2 * quarter + 2; ++piece) piece_of(piece, row - piece * 16, std::true_type{});
        tmem_ld_wait();
        uint32_t zero[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) zero[i] = 0u;
#pragma unroll 1
        for (int piece = 2 * quarter + 2; piece < 8; ++piece) tmem_st8(col + piece * 8, zero);
        tmem_st_wait();
        tc_fence_before_sync();
        mbar_arrive(&bars[dP + ab]);
      }
    }
  } else if ((warp >= 6 && warp < 10) || warp >= 20) {
    // ------------------------------------------------------------------ state groups
    const int quarter = warp & 3, row = quarter * 32 + lane;      // a row of the state
    const int col0 = warp >= 20 ? DP / 2 : 0, col1 = col0 + DP / 2;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const int64_t slot = ((int64_t)seg * BH + bh) * a.K * a.D;
    const bool copies = OUT || a.kept;
    // 16 numbers of the state, columns from c0 on -> the copy of chunk c, and times the chunk's decay back to TMEM
    const auto put = [&](uint32_t* r, int c0, int c, const Factor& f) {
      if (copies && (KP == 128 || row < KP)) {
        unsigned char* copy = sm + Lay::copy + (Lay::kCopies == 2 ? (c & 1) * Lay::kCopyRoom : 0);
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
          uint4 p;
          p.x = pack2h<T>(__uint_as_float(r[8 * ch]), __uint_as_float(r[8 * ch + 1]));
          p.y = pack2h<T>(__uint_as_float(r[8 * ch + 2]), __uint_as_float(r[8 * ch + 3]));
          p.z = pack2h<T>(__uint_as_float(r[8 * ch + 4]), __uint_as_float(r[8 * ch + 5]));
          p.w = pack2h<T>(__uint_as_float(r[8 * ch + 6]), __uint_as_float(r[8 * ch + 7]));
          *reinterpret_cast<uint4*>(copy + (c0 >> 6) * (KP * 128) + row_chunk1(row, ((c0 & 63) >> 3) + ch)) = p;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(f.times(__uint_as_float(r[i])));
      tmem_st16(tmem + lane_addr + Lay::colS + c0, r);
    };
    bool ok = nchunk > 0;
    if (ok && !mbar_wait(&bars[dL], 0)) { tc_fail(12); ok = false; }
    if (ok) {
      const Factor f = fac[0];
      const float* src = totals_only ? nullptr : a.nseg > 1 ? a.totals + slot : a.s_in.p ? a.s_in.p + bh * a.K * a.D : nullptr;
      const int64_t rs = a.nseg > 1 ? a.D : a.s_in.row, cs = a.nseg > 1 ? 1 : a.s_in.col;
#pragma unroll 1
      for (int c0 = col0; c0 < col1; c0 += 16) {
        uint32_t r[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = src && row < a.K && c0 + i < a.D ? __float_as_uint(src[row * rs + (c0 + i) * cs]) : 0u;
        put(r, c0, 0, f);
      }
      tmem_st_wait();
      fence_async_smem();
      tc_fence_before_sync();
      mbar_arrive(&bars[dSt]);
    }
    for (int c = 0; ok && c < nchunk; ++c) {
      if (a.kept) {
        if (tid == 6 * 32) {      // the copy of chunk c to memory, once it is whole; the place of the next one has been read then
          if (!mbar_wait(&bars[dSt], c & 1)) { tc_fail(19); ok = false; break; }
          const int64_t chunk = chunk_t0(c) / kTC, chunks = (a.T + kTC - 1) / kTC;
          bulk_store(static_cast<unsigned char*>(a.kept) + (bh * chunks + chunk) * Lay::kCopyBytes, sm + Lay::copy + (Lay::kCopies == 2 ? (c & 1) * Lay::kCopyRoom : 0), Lay::kCopyBytes);
          tma_store_commit();
          tma_store_wait_read<Lay::kCopies - 1>();
          mbar_arrive(&bars[dKept]);
        }
        if (!mbar_wait(&bars[dKept], c & 1)) { tc_fail(20); ok = false; break; }
      }
      if (!mbar_wait(&bars[dS], c & 1)) { tc_fail(13); ok = false; break; }
      tc_fence_after_sync();
      if (c + 1 < nchunk) {
        if (!mbar_wait(&bars[dL + (c + 1) % Lay::kL], ((c + 1) / Lay::kL) & 1)) { tc_fail(14); ok = false; break; }
        const Factor f = fac[(c + 1) % Lay::kL];
        uint32_t next[16];
        tmem_ld16(tmem + lane_addr + Lay::colS + col0, next);
#pragma unroll 1
        for (int c0 = col0; c0 < col1; c0 += 16) {
          uint32_t r[16];
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) r[i] = next[i];
          if (c0 + 16 < col1) tmem_ld16(tmem + lane_addr + Lay::colS + c0 + 16, next);
          put(r, c0, c + 1, f);
        }
        tmem_st_wait();
        fence_async_smem();
        tc_fence_before_sync();
        mbar_arrive(&bars[dSt]);
      }
      if (!OUT) mbar_arrive(&bars[dLFree + c % Lay::kL]);
    }
    // the state behind the last chunk; the last wait on dS ordered it
    float* dst = !ok ? nullptr : totals_only ? a.totals + slot : a.s_out.p && seg == a.nseg - 1 ? a.s_out.p + bh * a.K * a.D : nullptr;
    if (dst) {
      const int64_t rs = totals_only ? a.D : a.s_out.row, cs = totals_only ? 1 : a.s_out.col;
#pragma unroll 1
      for (int c0 = col0; c0 < col1; c0 += 16) {
        uint32_t r[16];
        tmem_ld16(tmem + lane_addr + Lay::colS + c0, r);
        tmem_ld_wait();
        if (row < a.K) {
          if (cs == 1) {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              if (c0 + i < a.D)
                *reinterpret_cast<float4*>(dst + row * rs + c0 + i) = make_float4(__uint_as_float(r[i]), __uint_as_float(r[i + 1]), __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (c0 + i < a.D) dst[row * rs + (c0 + i) * cs] = __uint_as_float(r[i]);
          }
        }
      }
    }
    if (a.kept && tid == 6 * 32) tma_store_wait<0>();
  } else if (warp >= 14 && warp < 18) {
    // ------------------------------------------------------------------ output group
    if constexpr (OUT) {
      const int quarter = warp & 3, row = quarter * 32 + lane;      // a token of the chunk
      const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
      const bool wide = a.D % 16 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
      for (int c = 0; c < nchunk; ++c) {
        if (!mbar_wait(&bars[dL + c % Lay::kL], (c / Lay::kL) & 1) || !mbar_wait(&bars[dFree + c % Lay::kStages], (c / Lay::kStages) & 1)) { tc_fail(15); break; }
        tc_fence_after_sync();
        const int64_t t = chunk_t0(c) + row;
        const bool there = t < t_end, gone = there && mask && mask[t];
        const float f = a.out_scale * ex2(Ls[c % Lay::kL * 128 + row]);
        T* o = static_cast<T*>(a.out) + ((t * a.B + b) * a.H + h) * a.D;
#pragma unroll 1
        for (int c0 = 0; c0 < DP; c0 += 16) {
          uint32_t n[16], p[16];
          tmem_ld16(tmem + lane_addr + Lay::colN + c0, n);
          tmem_ld16(tmem + lane_addr + Lay::colO + c0, p);
          tmem_ld_wait();
          if (c0 + 16 == DP) {
            tc_fence_before_sync();
            mbar_arrive(&bars[dNFree]);
          }
          float v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = gone ? 0.f : fmaf(f, __uint_as_float(n[i]), a.o_scale * __uint_as_float(p[i]));
          if (there && c0 < a.D) store_row16(o + c0, v, a.D - c0, wide);
        }
        mbar_arrive(&bars[dLFree + c % Lay::kL]);
      }
    }
  } else if (warp == 19) {
    // ------------------------------------------------------------------ decays: a lane takes four adjacent tokens
    const int64_t bd = b * a.decay.b + h * a.decay.h;
    double run = 0.0;
    uint32_t bits[4];      // the next chunk's decays as they stand in memory, on their way during this chunk
    bool real[4];
    const auto ask = [&](int c) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t t = chunk_t0(c) + lane * 4 + e;
        real[e] = t < t_end;
        if (real[e]) {
          bits[e] = log_decay_bits(a.decay.p, a.decay_dtype, bd + t * a.decay.t);
          if (mask) real[e] = !mask[t];
        }
      }
    };
    if (nchunk > 0) ask(0);
    for (int c = 0; c < nchunk; ++c) {
      const int lb = c % Lay::kL;
      double L[4], all = 0.0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (real[e]) {      // in units of log 2; NaN stays NaN
          const float g = log_decay_number(bits[e], a.decay_dtype);
          all += (double)(g < kDecayFloor ? kDecayFloor : g) * kLog2eD;
        }
        L[e] = all;
      }
      if (c + 1 < nchunk) ask(c + 1);
      double before = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
      }
      const double end = __shfl_sync(0xffffffffu, before, 31);
      before = __shfl_up_sync(0xffffffffu, before, 1);      // and not less its own sum: a lane's first tokens know nothing of its last
      if (lane == 0) before = 0.0;
      run += end;
      float l[4], f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        L[e] += before;
        l[e] = (float)L[e];
        f[e] = a.in_scale * exp2f((float)(a.rev ? L[e] : end - L[e]));
      }
      const Factor whole((float)(end / kLog2eD));
      if (c >= Lay::kL && !mbar_wait(&bars[dLFree + lb], (c / Lay::kL + 1) & 1)) { tc_fail(17); break; }
      *reinterpret_cast<float4*>(Ls + lb * 128 + lane * 4) = make_float4(l[0], l[1], l[2], l[3]);
      *reinterpret_cast<float4*>(key_fac + lb * 128 + lane * 4) = make_float4(f[0], f[1], f[2], f[3]);
      if (lane == 0) fac[lb] = whole;
      mbar_arrive(&bars[dL + lb]);
    }
    if (totals_only && lane == 0) a.seg_decay[(int64_t)seg * BH + bh] = run / kLog2eD;
  } else {
    // ------------------------------------------------------------------ key group: the token's row of K; with states alone warps 2..5 take half of it
    const bool second = !OUT && warp < 6;
    const int j = second ? tid - 64 : tid - 320;
    uint8_t ahead = mask && nchunk > 0 && chunk_t0(0) + j < t_end ? mask[chunk_t0(0) + j] : 0;
    for (int c = 0; c < nchunk; ++c) {
      const int st = c % Lay::kStages, lb = c % Lay::kL;
      const uint32_t filled = (c / Lay::kStages) & 1;
      unsigned char* krow = sm + Lay::k + st * KB * kBox;
      if (mask && second) {
        if (!mbar_wait(&bars[dClean + lb], (c / Lay::kL) & 1)) { tc_fail(29); break; }
      } else if (mask) {      // padded rows of K and V may hold anything: zero before a product reads them
        const bool gone = ahead;
        if (c + 1 < nchunk) ahead = chunk_t0(c + 1) + j < t_end ? mask[chunk_t0(c + 1) + j] : 0;
        if (!mbar_wait(&bars[dFull + st], filled) || (kOneV && !mbar_wait(&bars[dFullV], c & 1))) { tc_fail(18); break; }
        if (gone) {
#pragma unroll
          for (int ch = 0; ch < 8 * KB; ++ch) *reinterpret_cast<uint4*>(krow + row_chunk2(j, ch)) = make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int ch = 0; ch < 8 * DB; ++ch) *reinterpret_cast<uint4*>(sm + Lay::v + (kOneV ? 0 : st) * DB * kBox + row_chunk2(j, ch)) = make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
        mbar_arrive(&bars[dClean + lb]);
      }
      if (!mbar_wait(&bars[dL + c % Lay::kL], (c / Lay::kL) & 1)) { tc_fail(16); break; }
      const float f = key_fac[c % Lay::kL * 128 + j];
      if (OUT) {
        const int ab = Lay::kA == 2 ? c & 1 : 0, an = Lay::kA == 2 ? c >> 1 : c;
        if (!mbar_wait(&bars[dA + ab], an & 1)) { tc_fail(21); break; }
      } else if (!mbar_wait(&bars[dFull + st], filled)) { tc_fail(22); break; }
      if (EXACT && c >= 1 && !mbar_wait(&bars[dS], (c + 1) & 1)) { tc_fail(23); break; }      // the second part of the chunk before has been read
#pragma unroll 1
      for (int c8 = second ? 4 * KB : 0; c8 < (OUT || second ? 8 : 4) * KB; c8 += 2) {
        uint4 k8[2];
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) k8[ch] = *reinterpret_cast<const uint4*>(krow + row_chunk2(j, c8 + ch));
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
          uint4 low;
          uint32_t *xs = reinterpret_cast<uint32_t*>(&k8[ch]), *ls = reinterpret_cast<uint32_t*>(&low);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float2 v = unpack2h<T>(xs[e]);
            v.x *= f;
            v.y *= f;
            xs[e] = pack2h<T>(v.x, v.y);
            const float2 first = unpack2h<T>(xs[e]);
            ls[e] = pack2h<T>(v.x - first.x, v.y - first.y);
          }
          *reinterpret_cast<uint4*>(krow + row_chunk2(j, c8 + ch)) = k8[ch];
          if (EXACT) *reinterpret_cast<uint4*>(sm + Lay::low + row_chunk2(j, c8 + ch)) = low;
        }
      }
      fence_async_smem();
      mbar_arrive(&bars[dKp + lb]);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, Lay::cols);
}

// decay_bwd_tc.cu
int launch_decay_grad_tc(const rfa_decay_t& c, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& g, const void* states, const void* grads,
                         void* gq, void* gk, void* gv, void* g_decay, cudaStream_t stream);

}  // namespace rfa
