// Sliding-window attention on the tensor cores: the backward pass, fp16 and bf16, heads of up to 128.
//
// The weights are recomputed from the forward's log-sums, twice: once beside the queries, for gq, and once beside the keys, for gk and gv, so that no result is
// added up by two CTAs and the same call gives the same bits.  One kernel does both (KEYS).  A CTA keeps 128 rows (of q and g; KEYS: of k and v) in shared memory and
// streams tiles of 64 of the other side past them:
//     S = R1 X1^T, D = R2 X2^T (fp32, TMEM)  ->  P = 2^(S scale log2(e) - lse), dS = P o (D - delta), 16 bits, over S and D
//     gq += dS X1 (X1 = k);   KEYS: gv += P X2 (X2 = g), gk += dS X1 (X1 = q), over all query heads that share the key head
// Scores and their gradients have three places (two where the sums leave no room for a third) and as many groups of warps, which take the tiles in turn, a thread to
// each row.  delta = sum of g o out comes from a
// kernel of its own.  Tiles that are seen whole need no mask.  Padded places and, beside the queries, keys beside first tokens: as in window_tc.cu, warp 3 fetches numbers (and, KEYS, lse and delta of the queries)
// and clears the rows that are summed over.  First tokens' keys: works behind the tiles' take parts of their queries (SPLIT; window.cuh), whose sums stay in 32 bits for
// window_parts_kernel.
//
// Warp roles (512 or 384 threads): warp 0 TMA producer, warp 1 issues S and D, warp 2 the sums, warp 3 columns' data or, where there are none, D, warps 4..7, 8..11, 12..15 the groups.  All
// waits are bounded.
//
// Window 512 + 4 of 8 x 16 heads x 2048 x 64, bf16: queries 120 us, keys 165 us, bound by the issue of products (1350 and 1640 cycles a tile, of which the tensor pipe works 640 and 830).
#define RFA_TC_FAMILY 13
#include <algorithm>

#include "window_tc.cuh"

namespace rfa {

constexpr int kWbTile = 64;

template <int DB, bool KEYS>
struct WbLayout {
  // groups of warps, each with a place for its scores and their gradients: as many as TMEM holds beside the sums
  static constexpr int kGroups = KEYS && DB == 2 ? 2 : 3, kThreads = 128 + kGroups * 128;
  static constexpr uint32_t colAcc = kGroups * 128;
  static_assert(colAcc + DB * 64 * (KEYS ? 2 : 1) <= 512, "TMEM");
  static constexpr int kStages = 4;
  static constexpr uint32_t kHalf = kBox / 2;      // 64 rows of 128 bytes
  static constexpr uint32_t r1 = 0, r2 = DB * kBox, x1 = 2 * DB * kBox, x2 = x1 + kStages * DB * kHalf, num = x2 + kStages * DB * kHalf, lse = num + kStages * kWbTile * 4,
                            delta = lse + kStages * kWbTile * 4, bar = delta + kStages * kWbTile * 4, bytes = bar + 256;
  static_assert(bytes <= 227 * 1024, "shared memory");
};
enum { bR = 0, bREmpty, bFull, bEmpty = bFull + 4, bCols = bEmpty + 4, bColsFree = bCols + 4, bS = bColsFree + 4, bP = bS + 3, bFree = bP + 3, bAcc = bFree + 3, bAccFree, bCount };
static_assert(bCount * 8 + 4 <= 256, "barriers");

// SPLIT: first tokens' queries are split (window.cuh); 4 % slower where they are not, 424 us against 407 with 8 x 16 heads x 2048 x 64, window 512 + 4
template <typename T, int DB, bool KEYS, bool ORDERED, bool SPLIT>
__global__ void __launch_bounds__(WbLayout<DB, KEYS>::kThreads, 1)
window_bwd_tc_kernel(const __grid_constant__ CUtensorMap tm_r1, const __grid_constant__ CUtensorMap tm_r2, const __grid_constant__ CUtensorMap tm_x1,
                     const __grid_constant__ CUtensorMap tm_x2, const __grid_constant__ CUtensorMap tm_first, const __grid_constant__ WindowArgs a, int works) {
  using Lay = WbLayout<DB, KEYS>;
  constexpr int DP = DB * 64, kStages = Lay::kStages, kGroups = Lay::kGroups;
  constexpr bool kColumns = KEYS || ORDERED;
  constexpr bool kApart = !kColumns;      // warp 3 has no columns to fetch: it issues D beside warp 1's S
  extern __shared__ __align__(1024) unsigned char sm[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + Lay::bar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + bCount);
  const uint32_t sbase = smem_u32(sm);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rows_heads = KEYS ? a.G : a.H, group = a.H / a.G;
  struct Work {
    int b, head;
    int64_t row0;
    WindowSpan span;      // of 64-wide tiles of the other side
    int split : 16, part : 8, none : 8;      // KEYS: the part of the queries, where first tokens' are split (part); none: no query
  };
  const auto work_of = [&](int w, Work& k) {      // the first rows first: keys there may be seen by all queries
    const int per = a.B * rows_heads;
    k.row0 = (int64_t)(w / per) * 128;
    k.b = w % per / rows_heads;
    k.head = w % per % rows_heads;
    k.split = 0;
    k.part = k.none = 0;
    if (!KEYS) {
      k.span = window_span<kWbTile>(WindowNumbers(a, k.b), 0, k.row0, a.T);
      return;
    }
    const auto tile_end = [&](int64_t q) { return (max(k.row0 + 1, q) + kWbTile - 1) / kWbTile; };
    if (!SPLIT || k.row0 < a.S) {
      const WindowNumbers num(a, k.b);
      const int64_t p1 = min(a.S, k.row0 + 128);
      k.part = SPLIT && num.is_split(k.row0, 128, a.splits);
      k.span = {0, 0, (int)(k.row0 / kWbTile), (int)tile_end(k.part ? num.near_query(k.row0, p1) : num.last_query(k.row0, p1))};
    } else {      // behind the tiles: the parts
      const int x = w - (int)((a.S + 127) / 128) * per, far = a.splits - 1, y = x / far, tiles = WindowNumbers(a, 0).first_tiles(128);
      k.split = 1 + x % far;
      k.b = y / tiles / a.G;
      k.head = y / tiles % a.G;
      const WindowNumbers num(a, k.b);
      k.row0 = (num.front() / 128 + y % tiles) * 128;
      k.part = k.row0 < num.first_end();
      if (!k.part) k.row0 = 0;
      const int64_t p1 = min(a.S, k.row0 + 128), from = tile_end(num.near_query(k.row0, p1)), all = tile_end(num.last_query(k.row0, p1)) - from;
      const int64_t lo = from + all * (k.split - 1) / far, hi = from + all * k.split / far;
      k.none = !k.part || lo >= hi;
      k.span = k.none ? WindowSpan{0, 0, (int)(k.row0 / kWbTile), (int)(k.row0 / kWbTile) + 1} : WindowSpan{0, 0, (int)lo, (int)hi};
    }
  };
  // heads of the other side that a work goes through, and where
  const auto first_head = [&](const Work& k) { return KEYS ? k.head * group : k.head / group; };
  const int other_heads = KEYS ? group : 1;
  if (tid == 0) {
    for (int i = 0; i < bCount; ++i)
      mbar_init(&bars[i], i >= bCols && i < bColsFree ? 32 : i >= bColsFree && i < bS ? 128 : i >= bP && i < bFree ? 128 : i == bAccFree ? kGroups * 128 : kApart && (i == bREmpty || (i >= bS && i < bP)) ? 2 : 1);
    mbar_fence_init();
    tma_prefetch_desc(&tm_r1); tma_prefetch_desc(&tm_r2); tma_prefetch_desc(&tm_x1); tma_prefetch_desc(&tm_x2);
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
        if (done > 0 && !mbar_wait(&bars[bREmpty], (done + 1) & 1)) { tc_fail(1); break; }
        mbar_arrive_expect_tx(&bars[bR], 2 * DB * kBox);
        for (int x = 0; x < DB; ++x) tma_load_4d(sm + Lay::r1 + x * kBox, &tm_r1, &bars[bR], x * 64, k.head, k.b, (int)k.row0);
        for (int x = 0; x < DB; ++x) tma_load_4d(sm + Lay::r2 + x * kBox, &tm_r2, &bars[bR], x * 64, k.head, k.b, (int)k.row0);
        for (int h = first_head(k); ok && h < first_head(k) + other_heads; ++h)
          for (int t = k.span.begin(); t < k.span.end; t = k.span.next(t), ++n) {
            const int st = n % kStages;
            if (n >= kStages && !mbar_wait(&bars[bEmpty + st], (n / kStages + 1) & 1)) { tc_fail(2); ok = false; break; }
            mbar_arrive_expect_tx(&bars[bFull + st], 2 * DB * Lay::kHalf);
            const CUtensorMap* summed = !KEYS && !ORDERED && t < k.span.first ? &tm_first : &tm_x1;
            for (int x = 0; x < DB; ++x) tma_load_4d(sm + Lay::x1 + (st * DB + x) * Lay::kHalf, summed, &bars[bFull + st], x * 64, h, k.b, t * kWbTile);
            for (int x = 0; x < DB; ++x) tma_load_4d(sm + Lay::x2 + (st * DB + x) * Lay::kHalf, &tm_x2, &bars[bFull + st], x * 64, h, k.b, t * kWbTile);
          }
      }
    }
  } else if (warp == 1 || warp == 2 || (kApart && warp == 3)) {
    // ------------------------------------------------------------------ MMA issuers
    // the whole warp goes through the loop and one lane issues (see umma_ss_w)
    {
      const uint32_t lead = lane == 0;
      constexpr uint32_t idS = umma_idesc<T>(128, kWbTile, false, false), idG = umma_idesc<T>(128, DP, false, true);
      constexpr uint32_t kBlockX = Lay::kHalf >> 4;
      constexpr uint64_t kStep = (DB * Lay::kHalf) >> 4;
      const uint64_t dR1 = umma_smem_desc(sbase + Lay::r1, 0, 1024, kSwizzle128B), dR2 = umma_smem_desc(sbase + Lay::r2, 0, 1024, kSwizzle128B);
      const uint64_t dX1 = umma_smem_desc(sbase + Lay::x1, 0, 1024, kSwizzle128B), dX2 = umma_smem_desc(sbase + Lay::x2, 0, 1024, kSwizzle128B);
      const uint64_t dX1t = umma_smem_desc(sbase + Lay::x1, Lay::kHalf, 1024, kSwizzle128B), dX2t = umma_smem_desc(sbase + Lay::x2, Lay::kHalf, 1024, kSwizzle128B);
      int n = 0, done = 0, buf = 0;      // buf: the tile's place and group; turn: parity of the places' uses
      uint32_t turn = 0;
      bool ok = true;
      for (int w = blockIdx.x; ok && w < works; w += gridDim.x, ++done) {
        Work k;
        work_of(w, k);
        if (warp != 2) {
          if (!mbar_wait(&bars[bR], done & 1)) { if (lead) tc_fail(3); break; }
        } else if (done > 0 && !mbar_wait(&bars[bAccFree], (done + 1) & 1)) { if (lead) tc_fail(4); break; }
        bool first = true;
        for (int h = 0; ok && h < other_heads; ++h)
          for (int t = k.span.begin(); t < k.span.end; t = k.span.next(t), ++n) {
            const int st = n % kStages;
            if (warp != 2) {
              if (!mbar_wait(&bars[ORDERED ? bCols + st : bFull + st], (n / kStages) & 1)) { if (lead) tc_fail(5); ok = false; break; }
              if (n >= kGroups && !mbar_wait(&bars[bFree + buf], turn ^ 1)) { if (lead) tc_fail(6); ok = false; break; }
              tc_fence_after_sync();
              if (!kApart || warp == 1) umma_chain_ss<4 * DB, kStepK, kBlockK, kStepK, kBlockX>(lead, tmem + buf * 128, dR1, dX1 + st * kStep, idS, 0);
              if (!kApart || warp == 3) umma_chain_ss<4 * DB, kStepK, kBlockK, kStepK, kBlockX>(lead, tmem + buf * 128 + 64, dR2, dX2 + st * kStep, idS, 0);
              umma_commit_w(lead, &bars[bS + buf]);      // the stage is given back by the sums, which come after
            } else {
              if (!mbar_wait(&bars[bP + buf], turn)) { if (lead) tc_fail(7); ok = false; break; }
              tc_fence_after_sync();
              if constexpr (KEYS) umma_chain_ts<4, kStepMN, kBlockMN>(lead, tmem + Lay::colAcc + DP, tmem + buf * 128, dX2t + st * kStep, idG, first ? 0u : 1u);
              umma_chain_ts<4, kStepMN, kBlockMN>(lead, tmem + Lay::colAcc, tmem + buf * 128 + 64, dX1t + st * kStep, idG, first ? 0u : 1u);
              umma_commit_w(lead, &bars[bFree + buf]);
              umma_commit_w(lead, &bars[bEmpty + st]);
              first = false;
            }
            if (++buf == kGroups) { buf = 0; turn ^= 1; }
          }
        if (ok) umma_commit_w(lead, &bars[warp != 2 ? bREmpty : bAcc]);
      }
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------------ what the groups want of a tile's columns; rows without a token
    if constexpr (kColumns) {
      int n = 0;
      bool ok = true;
      for (int w = blockIdx.x; ok && w < works; w += gridDim.x) {
        Work k;
        work_of(w, k);
        const WindowNumbers num(a, k.b);
        for (int h = first_head(k); ok && h < first_head(k) + other_heads; ++h)
          for (int t = k.span.begin(); t < k.span.end; t = k.span.next(t), ++n) {
            const int st = n % kStages;
            int number[2] = {0, 0};
            float lse[2] = {0.f, 0.f}, delta[2] = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int64_t i = (int64_t)t * kWbTile + e * 32 + lane;
              if (ORDERED) number[e] = num.key_of_tile(i, !KEYS && t < k.span.first);
              if (KEYS && i < a.T) {
                lse[e] = kLog2e * a.lse[((int64_t)k.b * a.H + h) * a.T + i];
                delta[e] = a.delta[((int64_t)k.b * a.H + h) * a.T + i];
              }
            }
            if (n >= kStages && !mbar_wait(&bars[bColsFree + st], (n / kStages + 1) & 1)) { tc_fail(12); ok = false; break; }
            if (ORDERED && !mbar_wait(&bars[bFull + st], (n / kStages) & 1)) { tc_fail(8); ok = false; break; }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int j = st * kWbTile + e * 32 + lane;
              if (ORDERED) reinterpret_cast<int*>(sm + Lay::num)[j] = number[e];
              if (KEYS) {
                reinterpret_cast<float*>(sm + Lay::lse)[j] = lse[e];
                reinterpret_cast<float*>(sm + Lay::delta)[j] = delta[e];
              }
              if (ORDERED && number[e] < 0) {
#pragma unroll 1
                for (int ch = 0; ch < 8 * DB; ++ch) {
                  const uint32_t at = st * DB * Lay::kHalf + (ch >> 3) * Lay::kHalf + row_chunk1(e * 32 + lane, ch & 7);
                  *reinterpret_cast<uint4*>(sm + Lay::x1 + at) = make_uint4(0, 0, 0, 0);
                  *reinterpret_cast<uint4*>(sm + Lay::x2 + at) = make_uint4(0, 0, 0, 0);
                }
              }
            }
            if (ORDERED) fence_async_smem();
            mbar_arrive(&bars[bCols + st]);
          }
      }
    }
  } else {
    // ------------------------------------------------------------------ groups: a thread to each row, one tile of kGroups
    const int g = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, S = tmem + lanes + g * 128, D = S + 64, acc = tmem + lanes + Lay::colAcc;
    const float scale = a.scale * kLog2e;
    const auto sectors = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; };
    int n = 0, done = 0, buf = 0;
    uint32_t turn = 0;
    bool ok = true;
    for (int w = blockIdx.x; ok && w < works; w += gridDim.x, ++done) {
      Work k;
      work_of(w, k);
      const int64_t i = k.row0 + row;
      const bool there = i < (KEYS ? a.S : a.T);
      const int mine = there && !k.none ? WindowNumbers(a, k.b).at(i) : -1;
      float lse = 0.f, delta = 0.f;
      if (!KEYS && there) {
        lse = kLog2e * a.lse[((int64_t)k.b * a.H + k.head) * a.T + i];
        delta = a.delta[((int64_t)k.b * a.H + k.head) * a.T + i];
      }
      for (int h = 0; ok && h < other_heads; ++h)
        for (int t = k.span.begin(); t < k.span.end; t = k.span.next(t), ++n) {
          const bool ours = buf == g;
          const uint32_t use = turn;
          if (++buf == kGroups) { buf = 0; turn ^= 1; }
          if (!ours) continue;
          const int st = n % kStages;
          const int64_t c0 = (int64_t)t * kWbTile;
          bool whole;
          uint32_t seen[2] = {0u, 0u};
          if constexpr (ORDERED) whole = false;
          else if constexpr (KEYS) whole = c0 >= k.row0 + 127 && c0 + kWbTile - 1 - k.row0 < a.window && c0 + kWbTile <= a.T;      // never where no query is (none): c0 = row0
          else whole = c0 + kWbTile - 1 <= k.row0 && k.row0 + 127 - c0 < a.window;
          if (kColumns && !mbar_wait(&bars[bCols + st], (n / kStages) & 1)) { tc_fail(9); ok = false; break; }
          if constexpr (ORDERED) {
            const int* nums = reinterpret_cast<const int*>(sm + Lay::num) + st * kWbTile;
            const auto bit = [&](int m) { return (KEYS ? window_sees(m, mine, a.window, a.sinks) : window_sees(mine, m, a.window, a.sinks)) ? 1u : 0u; };
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll 1
              for (int c = 28; c >= 0; c -= 4) {
                const int4 m = *reinterpret_cast<const int4*>(nums + x * 32 + c);
                seen[x] = seen[x] << 4 | bit(m.x) | bit(m.y) << 1 | bit(m.z) << 2 | bit(m.w) << 3;
              }
          } else if (!whole) {
            int lo, hi, front = 0;      // columns [lo, hi), and [0, front) of them
            if (KEYS) {
              lo = (int)min((int64_t)64, max((int64_t)0, i - c0));
              hi = (int)min((int64_t)64, (i < a.sinks ? a.T : min(a.T, i + a.window)) - c0);
              if (mine < 0) hi = 0;
            } else {
              hi = (int)min((int64_t)64, i - c0 + 1);
              lo = (int)min((int64_t)64, max((int64_t)0, i - c0 - a.window + 1));
              front = (int)min((int64_t)64, a.sinks - c0);
              if (!there) hi = 0;
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) seen[x] = low_bits(hi - 32 * x) & (~low_bits(lo - 32 * x) | low_bits(front - 32 * x));
          }
          if (!mbar_wait(&bars[bS + g], use)) { tc_fail(10); ok = false; break; }
          tc_fence_after_sync();
          const float* cl = reinterpret_cast<const float*>(sm + Lay::lse) + st * kWbTile;
          const float* cd = reinterpret_cast<const float*>(sm + Lay::delta) + st * kWbTile;
          // 32 columns at a time: P takes the first half of the place of the scores that it is made of
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t s[32], d[32];
            tmem_ld32(S + x * 32, s);
            tmem_ld32(D + x * 32, d);
            tmem_ld_wait();
            uint32_t pw[16], dw[16];
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              float l[4] = {lse, lse, lse, lse}, e[4] = {delta, delta, delta, delta}, p[4], ds[4];
              if constexpr (KEYS) {
                const float4 lv = *reinterpret_cast<const float4*>(cl + x * 32 + c), dv = *reinterpret_cast<const float4*>(cd + x * 32 + c);
                l[0] = lv.x; l[1] = lv.y; l[2] = lv.z; l[3] = lv.w;
                e[0] = dv.x; e[1] = dv.y; e[2] = dv.z; e[3] = dv.w;
              }
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                p[y] = ex2(fmaf(__uint_as_float(s[c + y]), scale, -l[y]));
                ds[y] = p[y] * (__uint_as_float(d[c + y]) - e[y]);
                if (!whole && !(seen[x] >> (c + y) & 1)) p[y] = ds[y] = 0.f;
              }
              pw[c >> 1] = pack2h<T>(p[0], p[1]);
              pw[(c >> 1) + 1] = pack2h<T>(p[2], p[3]);
              dw[c >> 1] = pack2h<T>(ds[0], ds[1]);
              dw[(c >> 1) + 1] = pack2h<T>(ds[2], ds[3]);
            }
            if (KEYS) tmem_st16(S + x * 16, pw);
            tmem_st16(D + x * 16, dw);
          }
          tmem_st_wait();
          tc_fence_before_sync();
          mbar_arrive(&bars[bP + g]);
          if (kColumns) mbar_arrive(&bars[bColsFree + st]);      // warp 3's plain stores come next; the stage itself is given back by the products
        }
      if (!ok) break;
      // ---- the gradients: the groups take 16 columns in turn
      if (!mbar_wait(&bars[bAcc], done & 1)) { tc_fail(11); break; }
      tc_fence_after_sync();
      const int heads = KEYS ? a.G : a.H;
      const int64_t at = ((i * a.B + k.b) * heads + k.head) * a.D;
      const WindowNumbers num(a, k.b);
      const bool real = there && mine >= 0;
      bool whole_row = there;
      float* parts = nullptr;      // where this row's part goes
      if (SPLIT) {
        const int number = there && k.part ? num.at(i) : -1;
        if (number >= 0 && number < a.sinks) parts = a.parts + ((((int64_t)k.b * a.G + k.head) * a.splits + k.split) * min((int64_t)a.sinks, a.T) + number) * 2 * a.D;
        whole_row = there && !parts && k.split == 0;
      }
      const auto store = [&](uint32_t from, void* to, float f) {
        T* out = static_cast<T*>(to) + at;
        const bool wide = a.D % 16 == 0 && sectors(to);
#pragma unroll 1
        for (int c0 = g * 16; c0 < DP; c0 += kGroups * 16) {
          uint32_t u[16];
          tmem_ld16(from + c0, u);
          tmem_ld_wait();
          float v[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) v[c] = real ? f * __uint_as_float(u[c]) : 0.f;
          if (whole_row && c0 < a.D) store_row16(out + c0, v, a.D - c0, wide);
          if (SPLIT && parts) {
            float* to_parts = parts + (to == a.gv ? a.D : 0) + c0;
#pragma unroll
            for (int c = 0; c < 16; ++c)
              if (c0 + c < a.D) to_parts[c] = real ? __uint_as_float(u[c]) : 0.f;
          }
        }
      };
      store(acc, KEYS ? a.gk : a.gq, a.scale * (KEYS ? num.key_factor() : num.query_factor(mine)));
      if (KEYS) store(acc + DP, a.gv, 1.f);
      tc_fence_before_sync();
      mbar_arrive(&bars[bAccFree]);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// delta [B][H][T] = g . out of each query, both contiguous.  Bound by memory; a lane group of 8 or 16 takes a row, 16 bytes each.
template <typename T>
__global__ void __launch_bounds__(256) window_delta_kernel(const T* __restrict__ g, const T* __restrict__ out, float* delta, int64_t T_, int B, int H, int D, int lanes, const uint8_t* mask) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / lanes;      // a row [T][B][H]
  const int lane = threadIdx.x % lanes;
  const int64_t rows = T_ * B * H;
  float d = 0.f;
  if (i < rows && lane * 8 < D) {
    Raw<T, 8> x, y;
    x.load(g + i * D + lane * 8, 8, true);
    y.load(out + i * D + lane * 8, 8, true);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 u = x.get2(e), v = y.get2(e);
      d = fmaf(u.x, v.x, fmaf(u.y, v.y, d));
    }
  }
  for (int o = lanes / 2; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  if (i < rows && lane == 0) {
    const int64_t t = i / ((int64_t)B * H), bh = i % ((int64_t)B * H);
    delta[bh * T_ + t] = mask && mask[bh / H * T_ + t] ? 0.f : d;
  }
}

namespace {

template <typename T, int DB, bool KEYS, bool ORDERED, bool SPLIT = false>
int launch(const CUtensorMap& r1, const CUtensorMap& r2, const CUtensorMap& x1, const CUtensorMap& x2, const CUtensorMap& first, const WindowArgs& a, cudaStream_t stream) {
  using Lay = WbLayout<DB, KEYS>;
  constexpr uint32_t smem = Lay::bytes;
  cudaError_t e = cudaFuncSetAttribute(window_bwd_tc_kernel<T, DB, KEYS, ORDERED, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return fail((int)e, "window_bwd: cannot reserve %u bytes of shared memory: %s", smem, cudaGetErrorString(e));
  int64_t works = (a.T + 127) / 128 * a.B * (KEYS ? a.G : a.H);
  if (SPLIT) works += ((std::min<int64_t>(a.sinks, a.T) + 127) / 128 + (a.order ? 1 : 0)) * (a.splits - 1) * a.B * a.G;
  RFA_REQUIRE(works < (int64_t)1 << 31, RFA_EUNSUPPORTED, "window_bwd: %lld tiles", (long long)works);
  e = launch_pdl(window_bwd_tc_kernel<T, DB, KEYS, ORDERED, SPLIT>, dim3((unsigned)std::min<int64_t>(works, 148)), dim3(Lay::kThreads), smem, stream, r1, r2, x1, x2, first, a, (int)works);
  if (e != cudaSuccess) return fail((int)e, "rfa_window_bwd: launch failed: %s", cudaGetErrorString(e));
  return check_launch("rfa_window_bwd");
}
template <typename T, int DB, bool KEYS>
int launch_order(const CUtensorMap& r1, const CUtensorMap& r2, const CUtensorMap& x1, const CUtensorMap& x2, const CUtensorMap& first, const WindowArgs& a, cudaStream_t stream) {
  if (KEYS && a.splits > 1) return a.order ? launch<T, DB, KEYS, true, KEYS>(r1, r2, x1, x2, first, a, stream) : launch<T, DB, KEYS, false, KEYS>(r1, r2, x1, x2, first, a, stream);
  return a.order ? launch<T, DB, KEYS, true>(r1, r2, x1, x2, first, a, stream) : launch<T, DB, KEYS, false>(r1, r2, x1, x2, first, a, stream);
}
template <typename T>
int launch_delta(const WindowArgs& a, const uint8_t* mask, cudaStream_t stream) {
  const int lanes = a.D <= 64 ? 8 : 16;
  const int64_t ctas = (a.T * a.B * a.H * lanes + 255) / 256;
  RFA_REQUIRE(ctas < (int64_t)1 << 31, RFA_EUNSUPPORTED, "window_bwd: %lld rows", (long long)(a.T * a.B * a.H));
  window_delta_kernel<T><<<(unsigned)ctas, 256, 0, stream>>>(static_cast<const T*>(a.g.p), static_cast<const T*>(a.o.p), a.delta, a.T, a.B, a.H, a.D, lanes, mask);
  return check_launch("rfa_window_bwd (delta)");
}
template <typename T>
int launch_type(const CUtensorMap (&m)[9], const WindowArgs& a, const uint8_t* mask, cudaStream_t stream) {
  if (int r = launch_delta<T>(a, mask, stream)) return r;
  if (a.D <= 64) {
    if (int r = launch_order<T, 1, false>(m[0], m[1], m[6], m[7], m[8], a, stream)) return r;
    if (int r = launch_order<T, 1, true>(m[2], m[3], m[4], m[5], m[4], a, stream)) return r;
  } else {
    if (int r = launch_order<T, 2, false>(m[0], m[1], m[6], m[7], m[8], a, stream)) return r;
    if (int r = launch_order<T, 2, true>(m[2], m[3], m[4], m[5], m[4], a, stream)) return r;
  }
  return a.splits > 1 ? launch_window_parts(a, 128, a.scale, stream) : 0;
}

}  // namespace

int launch_window_bwd_tc(const WindowArgs& a, const uint8_t* mask, cudaStream_t stream) {
  const bool bf16 = a.dtype == RFA_BF16;
  // as resident rows: q, g, k, v; streamed: q, g, k, v
  CUtensorMap m[9];      // and the keys' first tokens, streamed
  const WindowRows* x[4] = {&a.q, &a.g, &a.k, &a.v};
  for (int i = 0; i < 8; ++i) {
    const WindowRows& r = *x[i & 3];
    if (make_tmap_heads(&m[i], r.p, bf16, a.T, a.B, (i & 3) < 2 ? a.H : a.G, a.D, r.t, r.b, r.h, i < 4 ? 128 : kWbTile))
      return fail(RFA_EDEVICE, "window_bwd: cuTensorMapEncodeTiled failed or is unavailable");
  }
  if (make_tmap_first(&m[8], m[6], a, a.k)) return fail(RFA_EDEVICE, "window_bwd: cuTensorMapEncodeTiled failed or is unavailable");
  return bf16 ? launch_type<__nv_bfloat16>(m, a, mask, stream) : launch_type<__half>(m, a, mask, stream);
}

RFA_TC_UNIT(window_bwd)

}  // namespace rfa
