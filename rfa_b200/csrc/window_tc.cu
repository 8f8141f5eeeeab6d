// Sliding-window attention on the 5th-generation tensor cores (tcgen05 + TMEM + TMA), fp16 and bf16, heads of up to 128: the forward pass.
//
// A CTA takes one pair of units after the other, each unit 128 queries of one batch row, that read the same keys -- two heads that share a key head, or else two
// runs of one head -- and goes through the 64-key tiles that either of them sees: those of the first tokens, then from the window's start on.  Per unit and tile
//     S = Q K^T (fp32, TMEM)  ->  P = 2^(scale log2(e) (S - m)), 16 bits, over S  ->  O += P V
// with a thread to each row, whose scores it holds in registers: the row's maximum, then P and the sum.  m moves only when it is exceeded by more than 8 (P is then
// at most 256, which both types hold), and only then O is rescaled, by the row's own thread.  Tiles that every query of the unit sees whole need no mask; in the
// others scores that are not seen are -inf before anything is made of them.  A unit's scores have two places in TMEM, so that the products of the next tile run under the
// exponentials of this one: with tiles of 128 keys and one place a unit's chain of products, maxima, exponentials and products again took 4500 cycles, of which the
// special function unit worked 2048 (16 exponentials a cycle and SM, two units).
//
// Tiles in front of all windows are seen for their first tokens only.  Their values come by a tensor map that ends behind these, so that the rows beside them are
// zero: a weight of nothing times what is not finite is not nothing, and such a tile is seen by every query.
//
// With padded tokens or a cache in front (ORDERED) places are not numbers: warp 3 fetches the numbers of a tile's keys and clears the values of places that hold
// no token, whatever stands there, and those beside first tokens.
//
// Warp roles (384 threads): warp 0 TMA producer, warps 1 and 2 one MMA issuer for each unit, warps 4..7 and 8..11 one softmax group for each unit.  All waits are
// bounded.  Window 256 + 4 of 8 x 16 (4) heads x 2048 x 64, bf16: 77 us; 1024 + 4 of 16 (4) x 32768 x 128: 386 to 395 us (690 TFLOP/s of what is seen).
#define RFA_TC_FAMILY 12
#include <algorithm>

#include "window_tc.cuh"

namespace rfa {

constexpr int kWinThreads = 384;

constexpr int kWinTile = 64;
template <int DB>
struct WinLayout {
  static constexpr int kStages = 4;
  static constexpr uint32_t kHalf = kBox / 2;      // 64 rows of 128 bytes
  static constexpr uint32_t q = 0, k = 2 * DB * kBox, v = k + kStages * DB * kHalf, num = v + kStages * DB * kHalf, bar = num + kStages * kWinTile * 4, bytes = bar + 288;
  static_assert(bytes <= 227 * 1024, "shared memory");
};
// wS, wP, wO: [unit][place of the scores].  wO (a tile's sums are complete) is not waited for at every tile, and the tile before the last may be pending when it is:
// one barrier for both would take the completion before that for the one that is wanted.
enum { wQ = 0, wQEmpty = 2, wFullK = 4, wFullV = 8, wEmpty = 12, wNumbers = 16, wS = 20, wP = 24, wO = 28, wCount = 32 };
static_assert(wCount * 8 + 4 <= 288, "barriers");

template <typename T, int DB, bool ORDERED>
__global__ void __launch_bounds__(kWinThreads, 1)
window_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                 const __grid_constant__ CUtensorMap tm_first, const __grid_constant__ WindowArgs a, bool pair_heads, int works) {
  using Lay = WinLayout<DB>;
  constexpr int DP = DB * 64, kStages = Lay::kStages;
  extern __shared__ __align__(1024) unsigned char sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Lay::bar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + wCount);
  const uint32_t sbase = smem_u32(sm);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t at = a.S - a.T;
  const int runs = (int)((a.T + 127) / 128), per_head = pair_heads ? runs : (runs + 1) / 2, heads = pair_heads ? a.H / 2 : a.H;
  // a work: two units of 128 queries from row[u] on, of heads h0 and h0 + 1 or of one
  struct Work {
    int b, h0, kv;
    int64_t row[2];
    WindowSpan span[2], both;
  };
  const auto work_of = [&](int w, Work& k) {
    const int bh = w / per_head, run = w % per_head;
    k.b = bh / heads;
    k.h0 = bh % heads * (pair_heads ? 2 : 1);
    k.kv = k.h0 / (a.H / a.G);
    k.row[0] = (int64_t)(pair_heads ? run : 2 * run) * 128;
    k.row[1] = pair_heads ? k.row[0] : k.row[0] + 128;
    const WindowNumbers num(a, k.b);
    k.span[0] = window_span<kWinTile>(num, at, k.row[0], a.T);
    k.span[1] = pair_heads ? k.span[0] : window_span<kWinTile>(num, at, k.row[1], a.T);
    k.both = k.span[0];
    if (k.span[1].end > 0) {      // a last run may be without a partner
      k.both.first = min(k.span[0].first, k.span[1].first);
      k.both.front = min(k.span[0].front, k.span[1].front);
      k.both.firsts = max(k.span[0].firsts, k.span[1].firsts);
      k.both.end = max(k.span[0].end, k.span[1].end);
    }
  };
  if (tid == 0) {
    for (int i = 0; i < wCount; ++i) mbar_init(&bars[i], i >= wP && i < wO ? 128 : i >= wNumbers && i < wS ? 32 : i >= wEmpty && i < wNumbers ? (ORDERED ? 2 + 256 : 2) : 1);
    mbar_fence_init();
    tma_prefetch_desc(&tm_q); tma_prefetch_desc(&tm_k); tma_prefetch_desc(&tm_v);
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
      int n = 0, done = 0;
      bool ok = true;
      for (int w = blockIdx.x; ok && w < works; w += gridDim.x, ++done) {
        Work k;
        work_of(w, k);
        for (int u = 0; u < 2; ++u) {
          if (done > 0 && !mbar_wait(&bars[wQEmpty + u], (done + 1) & 1)) { tc_fail(1); ok = false; break; }
          mbar_arrive_expect_tx(&bars[wQ + u], DB * kBox);
          for (int x = 0; x < DB; ++x)
            tma_load_4d(sm + Lay::q + (u * DB + x) * kBox, &tm_q, &bars[wQ + u], x * 64, k.h0 + (pair_heads ? u : 0), k.b, (int)k.row[u]);
        }
        for (int kt = k.both.begin(); ok && kt < k.both.end; kt = k.both.next(kt), ++n) {
          const int st = n % kStages;
          if (n >= kStages && !mbar_wait(&bars[wEmpty + st], (n / kStages + 1) & 1)) { tc_fail(2); ok = false; break; }
          mbar_arrive_expect_tx(&bars[wFullK + st], DB * Lay::kHalf);
          for (int x = 0; x < DB; ++x) tma_load_4d(sm + Lay::k + (st * DB + x) * Lay::kHalf, &tm_k, &bars[wFullK + st], x * 64, k.kv, k.b, kt * kWinTile);
          mbar_arrive_expect_tx(&bars[wFullV + st], DB * Lay::kHalf);
          const CUtensorMap* values = !ORDERED && kt < k.both.first ? &tm_first : &tm_v;
          for (int x = 0; x < DB; ++x) tma_load_4d(sm + Lay::v + (st * DB + x) * Lay::kHalf, values, &bars[wFullV + st], x * 64, k.kv, k.b, kt * kWinTile);
        }
      }
    }
  } else if (warp == 1 || warp == 2) {
    // ------------------------------------------------------------------ MMA issuers
    // The whole warp goes through the loop and one lane issues: descriptors stay in uniform registers (see umma_ss_w).
    {
      const uint32_t lead = lane == 0;
      const int u = warp - 1;
      constexpr uint32_t idS = umma_idesc<T>(128, kWinTile, false, false), idO = umma_idesc<T>(128, DP, false, true);
      constexpr uint32_t kBlockX = Lay::kHalf >> 4;
      const uint64_t dQ = umma_smem_desc(sbase + Lay::q + u * DB * kBox, 0, 1024, kSwizzle128B), dK = umma_smem_desc(sbase + Lay::k, 0, 1024, kSwizzle128B);
      const uint64_t dV = umma_smem_desc(sbase + Lay::v, Lay::kHalf, 1024, kSwizzle128B);
      constexpr uint64_t kStep = (DB * Lay::kHalf) >> 4;
      const uint32_t S = tmem + u * 128, O = tmem + 256 + u * DP;
      int n = 0, is = 0, it = 0, done = 0;      // tiles; of this unit: scores, sums
      bool ok = true;
      for (int w = blockIdx.x; ok && w < works; w += gridDim.x, ++done) {
        Work k;
        work_of(w, k);
        const WindowSpan own = u ? k.span[1] : k.span[0];
        if (!mbar_wait(&bars[wQ + u], done & 1)) { if (lead) tc_fail(3); break; }
        // Scores run up to two of the unit's tiles ahead of the sums.  No tile is waited for whose stage the unit's own sums have yet to give back.
        int kt = k.both.begin();
        int ahead[2] = {0, 0}, pending = 0;      // tiles whose scores have been issued and whose sums have not, the older first
        bool first = true;
        while (ok && (pending > 0 || kt < k.both.end)) {
          while (pending < 2 && kt < k.both.end && (pending == 0 || n - ahead[0] < kStages)) {
            const int st = n % kStages;
            const uint32_t filled = (n / kStages) & 1;
            if (!mbar_wait(&bars[wFullK + st], filled)) { if (lead) tc_fail(4); ok = false; break; }
            if (own.has(kt)) {
              tc_fence_after_sync();
              umma_chain_ss<4 * DB, kStepK, kBlockK, kStepK, kBlockX>(lead, S + (is & 1) * 64, dQ, dK + st * kStep, idS, 0);
              umma_commit_w(lead, &bars[wS + 2 * u + (is & 1)]);
              ++is;
              if (pending == 0) ahead[0] = n;
              else ahead[1] = n;
              ++pending;
            } else {
              if (!mbar_wait(&bars[wFullV + st], filled)) { if (lead) tc_fail(5); ok = false; break; }
              if (lead) mbar_release_stage(&bars[wEmpty + st]);
            }
            kt = k.both.next(kt);
            ++n;
          }
          if (!ok || pending == 0) continue;
          const int st = ahead[0] % kStages;
          const uint32_t filled = (ahead[0] / kStages) & 1;
          if (!mbar_wait(&bars[ORDERED ? wNumbers + st : wFullV + st], filled)) { if (lead) tc_fail(6); ok = false; break; }
          if (!mbar_wait(&bars[wP + 2 * u + (it & 1)], (it >> 1) & 1)) { if (lead) tc_fail(7); ok = false; break; }
          tc_fence_after_sync();
          umma_chain_ts<4, kStepMN, kBlockMN>(lead, O, S + (it & 1) * 64, dV + st * kStep, idO, first ? 0u : 1u);
          umma_commit_w(lead, &bars[wO + 2 * u + (it & 1)]);
          umma_commit_w(lead, &bars[wEmpty + st]);
          first = false;
          ++it;
          ahead[0] = ahead[1];
          --pending;
        }
        if (!ok) break;
        umma_commit_w(lead, &bars[wQEmpty + u]);      // everything that reads Q is complete
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ softmax groups: a thread to each row
    const int u = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t S = tmem + u * 128 + ((uint32_t)(quarter * 32) << 16), O = tmem + 256 + u * DP + ((uint32_t)(quarter * 32) << 16);
    const float scale = a.scale * kLog2e;
    const bool wide = a.D % 16 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
    int n = 0, it = 0;
    bool ok = true;
    for (int w = blockIdx.x; ok && w < works; w += gridDim.x) {
      Work k;
      work_of(w, k);
      const WindowSpan own = u ? k.span[1] : k.span[0];
      const int64_t i0 = u ? k.row[1] : k.row[0], i = i0 + row, place = at + i;
      const int mine = i < a.T ? WindowNumbers(a, k.b).at(place) : -1;
      // The score that weights are taken against.  It is subtracted before the scale, two scores at a time: scaled and subtracted in one, the rest of the product's
      // rounding stays, and from scores of 2^28 on 2 to that is beyond fp16.
      float top = kLowest, sum = 0.f;
      bool first = true;
#pragma unroll 1
      for (int kt = k.both.begin(); kt < k.both.end; kt = k.both.next(kt), ++n) {
        if (ORDERED && !mbar_wait(&bars[wNumbers + n % kStages], (n / kStages) & 1)) { tc_fail(8); ok = false; break; }
        if (!own.has(kt)) {
          if (ORDERED) mbar_release_stage(&bars[wEmpty + n % kStages]);
          continue;
        }
        const int64_t j0 = (int64_t)kt * kWinTile;
        const uint32_t Sp = S + (it & 1) * 64;
        // every query of the unit sees every key of the tile; or else which keys this row sees
        const bool whole = !ORDERED && j0 + kWinTile - 1 <= at + i0 && at + i0 + 127 - j0 < a.window;
        uint32_t seen[2];
        if constexpr (ORDERED) {
          const int* nums = reinterpret_cast<const int*>(sm + Lay::num) + (n % kStages) * kWinTile;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t bits = 0;
#pragma unroll 1
            for (int c = 28; c >= 0; c -= 4) {
              const int4 m = *reinterpret_cast<const int4*>(nums + x * 32 + c);
              bits = bits << 4 | (window_sees(mine, m.x, a.window, a.sinks) ? 1u : 0u) | (window_sees(mine, m.y, a.window, a.sinks) ? 2u : 0u) |
                     (window_sees(mine, m.z, a.window, a.sinks) ? 4u : 0u) | (window_sees(mine, m.w, a.window, a.sinks) ? 8u : 0u);
            }
            seen[x] = bits;
          }
        } else if (!whole) {
          const int hi = (int)min((int64_t)64, place - j0 + 1), lo = (int)min((int64_t)64, max((int64_t)0, place - j0 - a.window + 1)), front = (int)min((int64_t)64, a.sinks - j0);
#pragma unroll
          for (int x = 0; x < 2; ++x) seen[x] = low_bits(hi - 32 * x) & (~low_bits(lo - 32 * x) | low_bits(front - 32 * x));
        }
        if (!mbar_wait(&bars[wS + 2 * u + (it & 1)], (it >> 1) & 1)) { tc_fail(9); ok = false; break; }
        tc_fence_after_sync();
        uint32_t s[64];
        tmem_ld32(Sp, s);
        tmem_ld32(Sp + 32, s + 32);
        tmem_ld_wait();
        if (!whole) {
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (!(seen[c >> 5] >> (c & 31) & 1)) s[c] = 0xff800000u;
        }
        float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 64; c += 2) most[(c >> 1) & 3] = fmaxf(most[(c >> 1) & 3], fmaxf(__uint_as_float(s[c]), __uint_as_float(s[c + 1])));
        const float now = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
        const bool move = scale * (now - top) > 8.f;
        if (__any_sync(0xffffffffu, move)) {
          const float ref = move ? now : top, keep = ex2(scale * (top - ref));
          top = ref;
          sum *= keep;
          if (!first) {      // O of the tiles before has to follow
            if (!mbar_wait(&bars[wO + 2 * u + ((it - 1) & 1)], ((it - 1) >> 1) & 1)) { tc_fail(10); ok = false; break; }
            tc_fence_after_sync();
#pragma unroll 1
            for (int c0 = 0; c0 < DP; c0 += 16) {
              uint32_t o[16];
              tmem_ld16(O + c0, o);
              tmem_ld_wait();
#pragma unroll
              for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * keep);
              tmem_st16(O + c0, o);
            }
          }
        }
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          uint32_t p[16];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float2 e = scaled_rest(__uint_as_float(s[x * 32 + c]), __uint_as_float(s[x * 32 + c + 1]), top, scale);
            const float p0 = ex2(e.x), p1 = ex2(e.y);
            part[(c >> 1) & 1] += p0;
            part[2 + ((c >> 1) & 1)] += p1;
            p[c >> 1] = pack2h<T>(p0, p1);
          }
          tmem_st16(Sp + x * 16, p);
        }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
        tmem_st_wait();
        tc_fence_before_sync();
        mbar_arrive(&bars[wP + 2 * u + (it & 1)]);
        if (ORDERED) mbar_release_stage(&bars[wEmpty + n % kStages]);      // the numbers have been read
        first = false;
        ++it;
      }
      if (!ok || own.end == 0) continue;
      if (!first && !mbar_wait(&bars[wO + 2 * u + ((it - 1) & 1)], ((it - 1) >> 1) & 1)) { tc_fail(11); break; }
      tc_fence_after_sync();
      const int h = k.h0 + (pair_heads ? u : 0);
      const bool real = mine >= 0;                       // sees itself at least; a padded query has 0
      const float inv = real ? 1.f / sum : 0.f;          // whatever the sum is: a NaN score makes the row NaN
      T* out = static_cast<T*>(a.out) + ((i * a.B + k.b) * a.H + h) * a.D;
#pragma unroll 1
      for (int c0 = 0; c0 < DP; c0 += 32) {
        uint32_t o[32];
        tmem_ld16(O + c0, o);
        tmem_ld16(O + c0 + 16, o + 16);
        tmem_ld_wait();
        float v[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = real ? __uint_as_float(o[c]) * inv : 0.f;
        if (i < a.T && c0 < a.D) store_row16(out + c0, v, a.D - c0, wide);
        if (i < a.T && c0 + 16 < a.D) store_row16(out + c0 + 16, v + 16, a.D - c0 - 16, wide);
      }
      tc_fence_before_sync();      // the next weights let the issuer write O again
      if (a.lse && i < a.T) a.lse[((int64_t)k.b * a.H + h) * a.T + i] = real ? kLn2 * fmaf(top, scale, __log2f(sum)) : 0.f;
    }
  } else if (ORDERED) {
    // ------------------------------------------------------------------ warp 3: numbers of a tile's keys; values of places without a token
    int n = 0;
    bool ok = true;
    for (int w = blockIdx.x; ok && w < works; w += gridDim.x) {
      Work k;
      work_of(w, k);
      const WindowNumbers num(a, k.b);
      for (int kt = k.both.begin(); kt < k.both.end; kt = k.both.next(kt), ++n) {
        const int st = n % kStages;
        int number[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) number[e] = num.key_of_tile((int64_t)kt * kWinTile + e * 32 + lane, kt < k.both.first);
        // the stage has been filled again, so that nobody reads its old numbers
        if (!mbar_wait(&bars[wFullV + st], (n / kStages) & 1)) { tc_fail(12); ok = false; break; }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = e * 32 + lane;
          reinterpret_cast<int*>(sm + Lay::num)[st * kWinTile + j] = number[e];
          if (number[e] < 0) {
#pragma unroll 1
            for (int ch = 0; ch < 8 * DB; ++ch)
              *reinterpret_cast<uint4*>(sm + Lay::v + (st * DB + (ch >> 3)) * Lay::kHalf + row_chunk1(j, ch & 7)) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_async_smem();
        mbar_arrive(&bars[wNumbers + st]);
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

namespace {

template <typename T, int DB, bool ORDERED>
int launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& first, const WindowArgs& a, cudaStream_t stream) {
  using Lay = WinLayout<DB>;
  cudaError_t e = cudaFuncSetAttribute(window_tc_kernel<T, DB, ORDERED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Lay::bytes);
  if (e != cudaSuccess) return fail((int)e, "window_fwd: cannot reserve %u bytes of shared memory: %s", Lay::bytes, cudaGetErrorString(e));
  const bool pair_heads = a.H / a.G % 2 == 0;
  const int64_t runs = (a.T + 127) / 128, ctas = pair_heads ? runs * a.B * (a.H / 2) : (runs + 1) / 2 * a.B * a.H;
  RFA_REQUIRE(ctas < (int64_t)1 << 31, RFA_EUNSUPPORTED, "window_fwd: %lld tiles", (long long)ctas);
  e = launch_pdl(window_tc_kernel<T, DB, ORDERED>, dim3((unsigned)std::min<int64_t>(ctas, 148)), dim3(kWinThreads), Lay::bytes, stream, q, k, v, first, a, pair_heads, (int)ctas);
  if (e != cudaSuccess) return fail((int)e, "rfa_window_fwd: launch failed: %s", cudaGetErrorString(e));
  return check_launch("rfa_window_fwd");
}
template <typename T, int DB>
int launch_order(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& first, const WindowArgs& a, cudaStream_t stream) {
  return a.order ? launch<T, DB, true>(q, k, v, first, a, stream) : launch<T, DB, false>(q, k, v, first, a, stream);
}

}  // namespace

bool window_tc_ok(const WindowArgs& a) {
  const auto ok = [&](const WindowRows& x, int64_t T, int heads) { return tmap_rows_ok(x.p, T, a.B, heads, a.D, x.t, x.b, x.h); };
  // a negative scale turns the order of the scores round, which the maximum goes by, and zero makes something of -inf
  return a.dtype != RFA_F32 && a.D <= 128 && a.scale > 0.f && ok(a.q, a.T, a.H) && ok(a.k, a.S, a.G) && ok(a.v, a.S, a.G) && aligned16(a.out);
}

int launch_window_fwd_tc(const WindowArgs& a, cudaStream_t stream) {
  const bool bf16 = a.dtype == RFA_BF16;
  CUtensorMap q, k, v, first;
  if (make_tmap_heads(&q, a.q.p, bf16, a.T, a.B, a.H, a.D, a.q.t, a.q.b, a.q.h, 128) || make_tmap_heads(&k, a.k.p, bf16, a.S, a.B, a.G, a.D, a.k.t, a.k.b, a.k.h, kWinTile) ||
      make_tmap_heads(&v, a.v.p, bf16, a.S, a.B, a.G, a.D, a.v.t, a.v.b, a.v.h, kWinTile))
    return fail(RFA_EDEVICE, "window_fwd: cuTensorMapEncodeTiled failed or is unavailable");
  if (make_tmap_first(&first, v, a, a.v)) return fail(RFA_EDEVICE, "window_fwd: cuTensorMapEncodeTiled failed or is unavailable");
  if (bf16) return a.D <= 64 ? launch_order<__nv_bfloat16, 1>(q, k, v, first, a, stream) : launch_order<__nv_bfloat16, 2>(q, k, v, first, a, stream);
  return a.D <= 64 ? launch_order<__half, 1>(q, k, v, first, a, stream) : launch_order<__half, 2>(q, k, v, first, a, stream);
}

RFA_TC_UNIT(window)

}  // namespace rfa
