// Selective scan, backward.  With G_t = c_t g_t + exp(delta_(t+1) a) G_(t+1) (the gradient of s_t) and p_t = G_t exp(delta_t a) s_(t-1):
//   gc_t = sum over the group's channels of s_t g_t        gb_t = sum over them of G_t delta_t x_t
//   gx_t = delta_t sum_n G_t b_t + d g_t                   ga = sum_t delta_t p_t,  gd = sum_t x_t g_t
//   gdt_t = softplus'(dt_t + bias) (x_t sum_n G_t b_t + sum_n a p_t),  gbias = sum_t gdt_t.
//
// Layout in scan.cuh; tiles from the last to the first.  The states come back from the forward's checkpoints, one in front of every
// tile (16 tokens: as many bytes as two 16-bit activations at 16 states, instead of all states): a tile is walked forward once for the state
// in front of every second token, then two tokens at a time, from the last, forward with decays, decayed states and states left in
// registers and backward.  Sums over states go over the LN lanes of a channel; sums over channels over a thread's two, then every four tokens
// through shared memory to the warps that bring and take, over the CTA's pairs (12 instructions a token and thread, where exchanging
// them within the warp takes 28), then over CTAs in sum_parts: a fixed order, no atomics.
//
// 8 x 2048 tokens x 2048 channels x 16 states, bf16: about 860 of the 1100 us of a training step.  Bound by issue slots (224 instructions a
// token and warp), shared memory (55 passes of 128 bytes) and the FMA units (190 cycles) together, each 50 to 60 % busy of the 385 cycles that
// a token takes; memory traffic is 5 % of what could be.  Taking away one of its parts (the sums over channels, over states, the walk for
// the states) saves 7 to 9 % each.  Also measured: four channels a thread (one scanning warp per scheduler, 1430 us a step), parts of two
// tokens (1310), mbarriers instead of named barriers (1180), exponentials of the special function unit alone (1120), four tokens in
// registers (1150).
//
// Few rows: segments as in the forward, whose summaries run backward here (the gradient a segment hands to the one before it).
// Their kernel takes 25 us for 1 x 4096 tokens x 1024 channels (special function unit 63 % busy, FMA units 57 %).
#include "scan.cuh"

namespace rfa {
namespace {

constexpr int kRun = 2;       // tokens whose decays and states are in registers at a time
constexpr int kPart = 4;      // tokens after which the scanning warps hand their partial sums over

constexpr int kBwdScan = 128, kBwdBring = 128, kBwdThreads = kBwdScan + kBwdBring;
template <int LN> using BwdThread = ScanThread<LN, kBwdScan, kBwdBring, kept_tokens(LN)>;

template <int LN> struct __align__(16) BwdSmem {
  using Tile = ScanTile<LN>;
  static constexpr int kTokens = kept_tokens(LN);
  float4 in[2][kTokens][Tile::kPairs];               // delta, delta', delta x, delta' x' of two adjacent channels
  float2 g[2][kTokens][Tile::kPairs], slope[2][kTokens][Tile::kPairs];      // g and softplus' of both
  float b[2][kTokens][Tile::kN], c[2][kTokens][Tile::kN];
  float4 res[kTokens][Tile::kPairs];                 // sum_n G b of both channels, sum_n a log2(e) p of both
  ulonglong2 start[kTokens / kRun][2][kBwdScan]; // each thread's states in front of a run
  ulonglong2 da[2][kBwdScan];                          // each thread's ga: tiles are summed apart (one chain of 2048 tokens is 1e-6 off)
  float4 over_ch[2][kPart][2][Tile::kPairs][LN];       // gb and gc of each pair's channels, a lane's four states adjacent; two parts by turns
};
// Further places where the halves of a CTA meet: a part's sums are there, have been taken.
enum { kSums = 5, kTaken = 7 };

template <int LN> struct __align__(16) SummarySmem {
  using Tile = ScanTile<LN>;
  static constexpr int kTokens = kept_tokens(LN);
  float4 in[kTokens][Tile::kPairs];                  // delta, delta', g, g'
  float c[kTokens][Tile::kN];
};

struct BwdArgs {
  ScanShape sh;
  rfa_scan_t p;
  const void* g;
  const float *g_s, *ckpt;
  void *gx, *gdt, *gb, *gc;
  float *gs_in, *part_b, *part_c;           // part_b, part_c [per_group][T][B][G][N], used where per_group > 1
  float *part_a, *part_d, *part_bias;       // [B * segs][D][N], [B * segs][D]
  float *seg_grad, *seg_sum;                // of segments 1 ...: [segs - 1][B][D][kn], [segs - 1][B][D]
  bool wide;
};

constexpr int kSummaryThreads = 128;
// The gradient that the tokens of a segment alone hand to the state in front of it, and the segment's sum of deltas.
template <typename T, int LN>
__global__ void __launch_bounds__(kSummaryThreads) scan_bwd_summary_kernel(const __grid_constant__ BwdArgs A) {
  using Tile = ScanTile<LN>;
  constexpr int kTokens = kept_tokens(LN);
  using Thread = ScanThread<LN, kSummaryThreads, kSummaryThreads, kTokens>;      // each does both
  __shared__ SummarySmem<LN> sm;
  const ScanShape& sh = A.sh;
  const rfa_scan_t& p = A.p;
  const Thread th(sh);
  const int seg = blockIdx.z + 1, tile0 = seg * sh.seg_tiles, tile1 = min(tile0 + sh.seg_tiles, sh.tiles);
  f32x2 a2[4], G[4], sum = both(0.f);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    a2[j] = mul2(th.get(p.a, j, sh.N), both(kLog2e));
    G[j] = both(0.f);
  }
  const int ch = th.c0 + 2 * th.vpair;
  const T* dt = static_cast<const T*>(p.dt) + (int64_t)th.b * p.dt_b + ch;
  const T* g = static_cast<const T*>(A.g) + (int64_t)th.b * sh.D + ch;
  const T* cp = static_cast<const T*>(p.c) + (int64_t)th.b * p.c_b + (int64_t)th.group * p.c_g;
  const int64_t row_stride = (int64_t)sh.B * sh.D;
  const uint8_t* mask = p.mask ? p.mask + (int64_t)th.b * sh.T : nullptr;
  float bias[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) bias[k] = p.dt_bias && k < th.vn ? p.dt_bias[ch + k] : 0.f;

  RawPairs<T, Thread> rd, rg;
  RawStates<T, LN, Thread> rc;
  uint32_t next = 0;
  const int plain = A.wide && !mask && th.nch == Tile::kChannels ? (int)(sh.T / kTokens) : 0;      // tiles in front of it are
  const auto ask = [&](int tile, auto kind) {
    constexpr bool kPlain = decltype(kind)::value;
    const int64_t t0 = (int64_t)tile * kTokens, t = t0 + th.row;
    next = kPlain ? ~0u : th.tokens_here(mask, t0, sh.T);
    rd.template load<kPlain>(dt + t * p.dt_t, p.dt_t, next, th.vn, A.wide);
    rg.template load<kPlain>(g + t * row_stride, row_stride, next, th.vn, A.wide);
    rc.template load<kPlain>(th, cp, p.c_t, t0, sh.T, sh.N, mask);
  };
  const auto ask_tile = [&](int tile) { tile < plain ? ask(tile, Plain()) : ask(tile, Ragged()); };
  const auto put = [&]() {
#pragma unroll
    for (int i = 0; i < Thread::kPasses; ++i) {
      float2 sig;
      const float2 v = make_float2(rd.v[i].get(0) + bias[0], rd.v[i].get(1) + bias[1]);
      const f32x2 delta = p.softplus ? softplus2<false>(v, sig) : pack2(v.x, v.y);
      const bool on = next >> i & 1;
      *reinterpret_cast<ulonglong2*>(&sm.in[th.row + i * Thread::kRows][th.vpair]) = make_ulonglong2(on ? delta : 0, pack2(rg.v[i].get(0), rg.v[i].get(1)));
    }
    rc.store(th, sm.c);
  };
  ask_tile(tile1 - 1);
  for (int tile = tile1 - 1; tile >= tile0; --tile) {
    put();
    __syncthreads();
    if (tile > tile0) ask_tile(tile - 1);
    constexpr int kLook = 4;                           // tokens whose decays are formed side by side
#pragma unroll
    for (int t0 = kTokens - kLook; t0 >= 0; t0 -= kLook) {
      f32x2 delta[kLook], gt[kLook], e[kLook][4];
#pragma unroll
      for (int r = 0; r < kLook; ++r) {
        const ulonglong2 in = *reinterpret_cast<const ulonglong2*>(&sm.in[t0 + r][th.pair]);
        delta[r] = in.x;
        gt[r] = in.y;
      }
      decays<kLook, true>(delta, a2, e);
#pragma unroll
      for (int r = kLook - 1; r >= 0; --r) {
        float ct[4];
        lane_states(sm.c[t0 + r], th.ln, ct);
#pragma unroll
        for (int j = 0; j < 4; ++j) G[j] = mul2(fma2(gt[r], both(ct[j]), G[j]), e[r][j]);
        sum = add2(sum, delta[r]);
      }
    }
    __syncthreads();
  }
  const size_t at = ((size_t)(seg - 1) * sh.B + th.b) * sh.D;
  th.store_kept(A.seg_grad + at * sh.kn, G);
  th.put1(A.seg_sum + at, sum);
}

// Brings the tiles of a segment, from the last to the first, and takes their gradients away.
template <typename T, int LN>
__device__ __forceinline__ void bwd_bring(const BwdArgs& A, BwdSmem<LN>& sm, const BwdThread<LN>& th, int seg, int tile0, int tile1) {
  using Tile = ScanTile<LN>;
  using Thread = BwdThread<LN>;
  constexpr int kTokens = kept_tokens(LN);
  const ScanShape& sh = A.sh;
  const rfa_scan_t& p = A.p;
  const int ch = th.c0 + 2 * th.vpair;
  const T* x = static_cast<const T*>(p.x) + (int64_t)th.b * p.x_b + ch;
  const T* dt = static_cast<const T*>(p.dt) + (int64_t)th.b * p.dt_b + ch;
  const T* g = static_cast<const T*>(A.g) + (int64_t)th.b * sh.D + ch;
  const T* bp = static_cast<const T*>(p.b) + (int64_t)th.b * p.b_b + (int64_t)th.group * p.b_g;
  const T* cp = static_cast<const T*>(p.c) + (int64_t)th.b * p.c_b + (int64_t)th.group * p.c_g;
  const uint8_t* mask = p.mask ? p.mask + (int64_t)th.b * sh.T : nullptr;
  const int64_t row_stride = (int64_t)sh.B * sh.D, out0 = (int64_t)th.b * sh.D + ch;
  float bias[2], skip[2], gd[2] = {}, gbias[2] = {}, tile_gd[2] = {}, tile_gbias[2] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    bias[k] = p.dt_bias && k < th.vn ? p.dt_bias[ch + k] : 0.f;
    skip[k] = p.d && k < th.vn ? p.d[ch + k] : 0.f;
  }
  RawPairs<T, Thread> rx, rd, rg, kept;
  RawStates<T, LN, Thread> rb, rc;
  uint32_t here = 0, next = 0;                         // which of this thread's tokens are there: in the tile that is scanned, in the next one
  const int plain = A.wide && !mask && th.nch == Tile::kChannels ? (int)(sh.T / kTokens) : 0;      // tiles in front of it are
  const auto ask = [&](int tile, auto kind) {
    constexpr bool kPlain = decltype(kind)::value;
    const int64_t t0 = (int64_t)tile * kTokens, t = t0 + th.row;
    next = kPlain ? ~0u : th.tokens_here(mask, t0, sh.T);
    rx.template load<kPlain>(x + t * p.x_t, p.x_t, next, th.vn, A.wide);
    rd.template load<kPlain>(dt + t * p.dt_t, p.dt_t, next, th.vn, A.wide);
    rg.template load<kPlain>(g + t * row_stride, row_stride, next, th.vn, A.wide);
    rb.template load<kPlain>(th, bp, p.b_t, t0, sh.T, sh.N, mask);
    rc.template load<kPlain>(th, cp, p.c_t, t0, sh.T, sh.N, mask);
  };
  const auto ask_tile = [&](int tile) { tile < plain ? ask(tile, Plain()) : ask(tile, Ragged()); };
  const auto put = [&](int buf) {
#pragma unroll
    for (int i = 0; i < Thread::kPasses; ++i) {
      float2 sig = make_float2(1.f, 1.f);
      const float2 v = make_float2(rd.v[i].get(0) + bias[0], rd.v[i].get(1) + bias[1]);
      const f32x2 delta = p.softplus ? softplus2<true>(v, sig) : pack2(v.x, v.y);
      const f32x2 dx = mul2(delta, pack2(rx.v[i].get(0), rx.v[i].get(1)));
      const bool on = next >> i & 1;
      *reinterpret_cast<ulonglong2*>(&sm.in[buf][th.row + i * Thread::kRows][th.vpair]) = make_ulonglong2(on ? delta : 0, on ? dx : 0);
      sm.g[buf][th.row + i * Thread::kRows][th.vpair] = make_float2(rg.v[i].get(0), rg.v[i].get(1));
      sm.slope[buf][th.row + i * Thread::kRows][th.vpair] = sig;
    }
    rb.store(th, sm.b[buf]);
    rc.store(th, sm.c[buf]);
  };
  // gx and gdt of a part's tokens
  const auto take = [&](int64_t t0, int buf, int part) {
#pragma unroll
    for (int i = 0; i < Thread::kPasses; ++i) {
      const int t = th.row + i * Thread::kRows;
      if (t / kPart != part || t0 + t >= sh.T) continue;
      Raw<T, 2> ox, od;
      ox.zero(); od.zero();
      if (here >> i & 1) {
        const float4 in = sm.in[buf][t][th.vpair], res = sm.res[t][th.vpair];
        const float2 gv = sm.g[buf][t][th.vpair], sv = sm.slope[buf][t][th.vpair];
        const float delta[2] = {in.x, in.y}, gt[2] = {gv.x, gv.y}, sig[2] = {sv.x, sv.y}, gu[2] = {res.x, res.y}, gp[2] = {res.z, res.w};
        float v[2], vx[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float xv = kept.v[i].get(k);
          v[k] = fmaf(xv, gu[k], kLn2 * gp[k]) * sig[k];
          vx[k] = fmaf(delta[k], gu[k], skip[k] * gt[k]);
          tile_gd[k] = fmaf(xv, gt[k], tile_gd[k]);
          tile_gbias[k] += v[k];
        }
        ox.set2(0, vx[0], vx[1]);
        od.set2(0, v[0], v[1]);
      }
      ox.store(static_cast<T*>(A.gx) + (t0 + t) * row_stride + out0, th.vn, A.wide);
      od.store(static_cast<T*>(A.gdt) + (t0 + t) * row_stride + out0, th.vn, A.wide);
    }
  };
  // gb and gc of a part's tokens over the CTA's channels: kEach threads share the sum of one token's and lane's four states
  const auto sum = [&](int64_t t0, int part, int w) {
    constexpr int kOut = kPart * 2 * LN, kEach = kOut < kBwdBring ? kBwdBring / kOut : 1;
#pragma unroll
    for (int o = 0; o < kOut * kEach; o += kBwdBring) {
      const int at = o + th.tid, l = at % LN, share = at / LN % kEach, which = at / (LN * kEach) % 2, t = at / (LN * kEach * 2);
      ulonglong2 f = make_ulonglong2(0, 0);
#pragma unroll
      for (int r = 0; r < Tile::kPairs / kEach; ++r) {
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.over_ch[w][t][which][r * kEach + share][l]);
        f.x = add2(f.x, v.x);
        f.y = add2(f.y, v.y);
      }
      const float2 lo = split2(f.x), hi = split2(f.y);
      float v[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
      for (int s = kEach / 2; s > 0; s >>= 1)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += __shfl_xor_sync(0xffffffffu, v[j], s * LN);
      const int64_t token = t0 + part * kPart + t;
      if (token >= sh.T || share) continue;
      const bool gone = mask && mask[token];
      const int64_t to = ((token * sh.B + th.b) * sh.G + th.group) * sh.N;
      const int64_t to_part = (int64_t)(blockIdx.x % sh.per_group) * sh.T * sh.B * sh.G * sh.N + to;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = j * LN + l;
        if (n >= sh.N) continue;
        const float out = gone ? 0.f : v[j];
        if (sh.per_group == 1) static_cast<T*>(which ? A.gc : A.gb)[to + n] = from_f<T>(out);
        else (which ? A.part_c : A.part_b)[to_part + n] = out;
      }
    }
  };

  ask_tile(tile1 - 1);
  put(0);
  meet_go<kBwdThreads>(kFull);
  kept = rx;
  here = next;
  if (tile1 - 1 > tile0) ask_tile(tile1 - 2);
  for (int tile = tile1 - 1; tile >= tile0; --tile) {
    const int buf = (tile1 - 1 - tile) & 1;
    RawPairs<T, Thread> x_next = rx;
    const uint32_t here_next = next;
    if (tile > tile0) {                                // its last tile has been scanned and taken
      put(buf ^ 1);
      meet_go<kBwdThreads>(kFull + (buf ^ 1));
      if (tile - 1 > tile0) ask_tile(tile - 2);
    }
    const int64_t t0 = (int64_t)tile * kTokens;
#pragma unroll 1
    for (int part = kTokens / kPart - 1; part >= 0; --part) {
      const int w = part & 1;
      meet_wait<kBwdThreads>(kSums + w);
      // The part's place is given back, where somebody waits for it, before its gradients are stored: the scanning warps come to its rows of
      // res a tile on, and wait for another part's place in between -- unless a tile is two parts.
      constexpr bool kEarly = kTokens > 2 * kPart;
      const bool wanted = tile > tile0 || part > 1;
      sum(t0, part, w);
      if (kEarly && wanted) meet_go<kBwdThreads>(kTaken + w);
      take(t0, buf, part);
      if (!kEarly && wanted) meet_go<kBwdThreads>(kTaken + w);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      gd[k] += tile_gd[k];
      gbias[k] += tile_gbias[k];
      tile_gd[k] = tile_gbias[k] = 0.f;
    }
    kept = x_next;
    here = here_next;
  }

  const size_t row = (size_t)th.b * sh.segs + seg;
  // gd and gbias over the rows of bringing threads, where the scanning warps, done with their last part, kept their states
  float4* over_rows = reinterpret_cast<float4*>(&sm.start[0][0][0]);
  over_rows[th.tid] = make_float4(gd[0], gd[1], gbias[0], gbias[1]);
  asm volatile("bar.sync 9, %0;" ::"n"(kBwdBring) : "memory");
  if (th.row == 0) {
    float4 v = over_rows[th.tid];
    for (int r = 1; r < Thread::kRows; ++r) {
      const float4 w = over_rows[r * Tile::kPairs + th.tid];
      v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (k < th.vn) {
        A.part_d[row * sh.D + ch + k] = k ? v.y : v.x;
        A.part_bias[row * sh.D + ch + k] = k ? v.w : v.z;
      }
  }
}

template <typename T, int LN>
__global__ void __launch_bounds__(kBwdThreads, 2) scan_bwd_kernel(const __grid_constant__ BwdArgs A) {
  using Smem = BwdSmem<LN>;
  constexpr int kTokens = kept_tokens(LN);
  extern __shared__ char smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const ScanShape& sh = A.sh;
  const rfa_scan_t& p = A.p;
  const BwdThread<LN> th(sh);
  const int seg = blockIdx.z, tile0 = seg * sh.seg_tiles, tile1 = min(tile0 + sh.seg_tiles, sh.tiles);
  if (!th.scans) {
    bwd_bring<T, LN>(A, sm, th, seg, tile0, tile1);
    return;
  }

  f32x2 a2[4], G[4], da[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    a2[j] = mul2(th.get(p.a, j, sh.N), both(kLog2e));
    G[j] = A.g_s ? th.get(A.g_s + (size_t)th.b * sh.D * sh.N, j, sh.N) : both(0.f);
    da[j] = both(0.f);
  }
  sm.da[0][th.tid] = sm.da[1][th.tid] = make_ulonglong2(0, 0);
  join_segments(th, sh, A.seg_grad, A.seg_sum, sh.segs - 2, sh.segs - 1 - seg, -1, a2, G);      // the segments behind this one

  f32x2 s[4];                                          // the state in front of the tile
  const float* ckpt = A.ckpt + (size_t)th.b * sh.tiles * sh.D * sh.kn;
  th.load_kept(ckpt + (size_t)(tile1 - 1) * sh.D * sh.kn, s);
  for (int tile = tile1 - 1; tile >= tile0; --tile) {
    const int buf = (tile1 - 1 - tile) & 1;
    const auto inputs = [&](int base, f32x2* delta, f32x2* dx) {
#pragma unroll
      for (int r = 0; r < kRun; ++r) {
        const ulonglong2 in = *reinterpret_cast<const ulonglong2*>(&sm.in[buf][base + r][th.pair]);
        delta[r] = in.x;
        dx[r] = in.y;
      }
    };
    meet_wait<kBwdThreads>(kFull + buf);
    // The states in front of each run of the tile, then run by run from the last: forward with what the way back needs, and back.
#pragma unroll 1
    for (int run = 0;; ++run) {
      sm.start[run][0][th.tid] = make_ulonglong2(s[0], s[1]);
      sm.start[run][1][th.tid] = make_ulonglong2(s[2], s[3]);
      if (run == kTokens / kRun - 1) break;
      f32x2 delta[kRun], dx[kRun], e[kRun][4];
      inputs(run * kRun, delta, dx);
      decays<kRun, false>(delta, a2, e);               // over at most 15 tokens: the special function unit's own error does not add up
#pragma unroll
      for (int r = 0; r < kRun; ++r) {
        float bt[4];
        lane_states(sm.b[buf][run * kRun + r], th.ln, bt);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = fma2(e[r][j], s[j], mul2(dx[r], both(bt[j])));
      }
    }
    if (tile > tile0) th.load_kept(ckpt + (size_t)(tile - 1) * sh.D * sh.kn, s);      // asked for early
#pragma unroll 2
    for (int run = kTokens / kRun - 1; run >= 0; --run) {
      const int base = run * kRun, w = base / kPart & 1;
      f32x2 delta[kRun], dx[kRun], e[kRun][4], q[kRun][4], st[kRun][4];      // decays, decayed states, states
      float bt[kRun][4];
      inputs(base, delta, dx);
      const ulonglong2 lo = sm.start[run][0][th.tid], hi = sm.start[run][1][th.tid];
      const f32x2 first[4] = {lo.x, lo.y, hi.x, hi.y};
      decays<kRun, true>(delta, a2, e);
#pragma unroll
      for (int r = 0; r < kRun; ++r) {
        lane_states(sm.b[buf][base + r], th.ln, bt[r]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          q[r][j] = mul2(e[r][j], r ? st[r - 1][j] : first[j]);
          st[r][j] = fma2(dx[r], both(bt[r][j]), q[r][j]);
        }
      }
      // the part's place is free
      if (base % kPart == kPart - kRun && (tile < tile1 - 1 || base < kTokens - 2 * kPart)) meet_wait<kBwdThreads>(kTaken + w);
#pragma unroll
      for (int r = kRun - 1; r >= 0; --r) {
        const f32x2 gt = *reinterpret_cast<const f32x2*>(&sm.g[buf][base + r][th.pair]);
        f32x2 over_b, over_p;                          // sum_n G b, sum_n a2 p
        float ct[4], gb[4], gc[4];                     // gb, gc: of the four states, over both channels
        lane_states(sm.c[buf][base + r], th.ln, ct);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x2 Gt = fma2(gt, both(ct[j]), G[j]), pt = mul2(Gt, q[r][j]);
          const float2 vb = split2(mul2(Gt, dx[r])), vc = split2(mul2(st[r][j], gt));
          gb[j] = vb.x + vb.y;
          gc[j] = vc.x + vc.y;
          over_b = j ? fma2(Gt, both(bt[r][j]), over_b) : mul2(Gt, both(bt[r][j]));
          over_p = j ? fma2(pt, a2[j], over_p) : mul2(pt, a2[j]);
          da[j] = fma2(pt, delta[r], da[j]);
          G[j] = mul2(Gt, e[r][j]);
        }
        const int t = base % kPart + r;
        sm.over_ch[w][t][0][th.pair][th.ln] = make_float4(gb[0], gb[1], gb[2], gb[3]);
        sm.over_ch[w][t][1][th.pair][th.ln] = make_float4(gc[0], gc[1], gc[2], gc[3]);
        const float2 ob = split2(over_b), op = split2(over_p);
        float over_n[4] = {ob.x, ob.y, op.x, op.y};    // as a row of res
        lanes_sum<4, LN>(over_n, th.ln);
        float* res = reinterpret_cast<float*>(&sm.res[base + r][th.pair]);
        if constexpr (LN == 2) *reinterpret_cast<float2*>(res + 2 * th.ln) = make_float2(over_n[0], over_n[1]);
        else if (th.ln % (LN / 4) == 0) res[th.ln / (LN / 4)] = over_n[0];
      }
      if (base % kPart == 0) meet_go<kBwdThreads>(kSums + w);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      ulonglong2& total = sm.da[h][th.tid];
      total = make_ulonglong2(add2(total.x, da[2 * h]), add2(total.y, da[2 * h + 1]));
      da[2 * h] = da[2 * h + 1] = both(0.f);
    }
  }

  const size_t row = (size_t)th.b * sh.segs + seg;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const ulonglong2 total = sm.da[j / 2][th.tid];
    th.put(A.part_a + row * sh.D * sh.N, j, sh.N, j % 2 ? total.y : total.x);
    if (seg == 0 && A.gs_in) th.put(A.gs_in + (size_t)th.b * sh.D * sh.N, j, sh.N, G[j]);
  }
}

template <typename T, int LN> int launch_bwd(const BwdArgs& a, cudaStream_t stream) {
  constexpr int bytes = (int)sizeof(BwdSmem<LN>);
  const dim3 grid(a.sh.per_group * a.sh.G, a.sh.B, a.sh.segs);
  const cudaError_t err = cudaFuncSetAttribute(scan_bwd_kernel<T, LN>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  RFA_REQUIRE(err == cudaSuccess, (int)err, "selective_scan_bwd: %s", cudaGetErrorString(err));
  if (a.sh.segs > 1) {
    scan_bwd_summary_kernel<T, LN><<<dim3(grid.x, grid.y, a.sh.segs - 1), kSummaryThreads, 0, stream>>>(a);
    if (int r = check_launch("selective_scan_bwd (segments)")) return r;
  }
  scan_bwd_kernel<T, LN><<<grid, kBwdThreads, bytes, stream>>>(a);
  return check_launch("selective_scan_bwd");
}

// The parts of the backward's workspace, in floats (each a multiple of four).
struct BwdSpace {
  size_t bc, a, d, grad, sum, total;
  explicit BwdSpace(const ScanShape& s) {
    const auto four = [](size_t n) { return (n + 3) / 4 * 4; };
    bc = s.per_group > 1 ? four((size_t)s.per_group * s.T * s.B * s.G * s.N) : 0;
    a = four((size_t)s.B * s.segs * s.D * s.N);
    d = four((size_t)s.B * s.segs * s.D);
    grad = (size_t)(s.segs - 1) * s.B * s.D * s.kn;
    sum = four((size_t)(s.segs - 1) * s.B * s.D);
    total = 2 * bc + a + 2 * d + grad + sum;
  }
};

}  // namespace
}  // namespace rfa

extern "C" size_t rfa_selective_scan_workspace_bytes(int64_t T, int B, int D, int N, int G, int backward) {
  using namespace rfa;
  if (T <= 0 || B <= 0 || D <= 0 || N <= 0 || N > 64 || G <= 0 || D % G || T >= ((int64_t)1 << 31) - 64) return 0;
  const ScanShape s = scan_shape(T, B, D, N, G, backward != 0);
  if (backward) return BwdSpace(s).total * 4;
  return (size_t)(s.segs - 1) * B * D * (s.kn + 1) * 4;
}

extern "C" int rfa_selective_scan_bwd(const rfa_scan_t* scan, const void* g, const float* g_s, const float* checkpoints, void* gx, void* gdt, float* ga,
                                      void* gb, void* gc, float* gd, float* g_dt_bias, float* gs_in, void* workspace, size_t workspace_bytes,
                                      rfa_stream_t stream) {
  using namespace rfa;
  if (int r = scan_check(scan, "selective_scan_bwd")) return r;
  RFA_REQUIRE(g && checkpoints && gx && gdt && ga && gb && gc, RFA_EINVAL, "selective_scan_bwd: null pointer");
  RFA_REQUIRE(aligned16(checkpoints) && aligned16(workspace), RFA_EALIGN, "selective_scan_bwd: checkpoints or workspace is not 16-byte aligned");
  const size_t need = rfa_selective_scan_workspace_bytes(scan->T, scan->B, scan->D, scan->N, scan->G, 1);
  RFA_REQUIRE(workspace && workspace_bytes >= need, RFA_EWORKSPACE, "selective_scan_bwd: workspace %zu bytes, %zu needed", workspace_bytes, need);
  // every segment's CTAs read g_s, the first one's write gs_in
  RFA_REQUIRE(!gs_in || gs_in != g_s, RFA_EINVAL, "selective_scan_bwd: gs_in is g_s");
  BwdArgs a{};
  a.sh = scan_shape(scan->T, scan->B, scan->D, scan->N, scan->G, true);
  const BwdSpace space(a.sh);
  a.p = *scan;
  a.g = g; a.g_s = g_s; a.ckpt = checkpoints;
  a.gx = gx; a.gdt = gdt; a.gb = gb; a.gc = gc; a.gs_in = gs_in;
  a.part_b = static_cast<float*>(workspace);
  a.part_c = a.part_b + space.bc;
  a.part_a = a.part_c + space.bc;
  a.part_d = a.part_a + space.a;
  a.part_bias = a.part_d + space.d;
  a.seg_grad = a.part_bias + space.d;
  a.seg_sum = a.seg_grad + space.grad;
  const int size = scan->dtype == RFA_F32 ? 4 : 2;
  a.wide = wide_ok(scan->x, scan->x_t, scan->x_b, size, 2) && wide_ok(scan->dt, scan->dt_t, scan->dt_b, size, 2) &&
           wide_ok(g, scan->D, a.sh.heads, size, 2) && wide_ok(gx, 0, 0, size, 2) && wide_ok(gdt, 0, 0, size, 2);
  int r = 0;
#define CALL(T, LN) r = launch_bwd<T, LN>(a, as_stream(stream))
  RFA_SCAN_DISPATCH(scan->dtype, scan_lanes(scan->N), CALL);
#undef CALL
  if (r) return r;
  const int rows = scan->B * a.sh.segs;
  const int64_t states = (int64_t)scan->T * scan->B * scan->G * scan->N;
  SumJob jobs[kSumJobs] = {{a.part_a, ga, (int64_t)scan->D * scan->N, rows, RFA_F32},
                           {a.part_d, gd, scan->D, rows, RFA_F32},
                           {a.part_bias, g_dt_bias, scan->D, rows, RFA_F32},
                           {a.part_b, gb, states, a.sh.per_group, scan->dtype},
                           {a.part_c, gc, states, a.sh.per_group, scan->dtype}};
  return sum_parts(jobs, a.sh.per_group > 1 ? 5 : 3, as_stream(stream));
}
