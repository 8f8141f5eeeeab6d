// Selective scan, backward.  With G_t = c_t g_t + exp(delta_(t+1) a) G_(t+1) (the gradient of s_t) and p_t = G_t exp(delta_t a) s_(t-1):
//   gc_t = sum over the group's channels of s_t g_t        gb_t = sum over them of G_t delta_t x_t
//   gx_t = delta_t sum_n G_t b_t + d g_t                   ga = sum_t delta_t p_t,  gd = sum_t x_t g_t
//   gdt_t = softplus'(dt_t + bias) (x_t sum_n G_t b_t + sum_n a p_t),  gbias = sum_t gdt_t.
//
// Layout in scan.cuh; tiles from the last to the first.  The states come back from the forward's checkpoints, one in front of every
// 16 tokens (as many bytes as two 16-bit activations at 16 states, instead of all states): a half of 8 tokens is walked forward with
// its decays and decayed states left in registers (128 of them), then backward; the first half's walk is made twice.
// Sums over states go over the LN lanes of a channel; sums over channels over a thread's two, then through shared memory over the CTA's
// pairs (12 instructions a token and thread, where exchanging them within the warp takes 28), then over CTAs in sum_parts: a fixed
// order, no atomics.
//
// Few rows: segments as in the forward, whose summaries run backward here (the gradient a segment hands to the one before it).
#include "scan.cuh"

namespace rfa {
namespace {

constexpr int kRun = 4;      // tokens whose decays and decayed states are in registers at a time

template <int LN> struct __align__(16) BwdSmem {
  using Tile = ScanTile<LN>;
  static constexpr int kParts = 4 * (32 / LN);         // pairs of channels in a CTA: partial sums over channels
  float4 in[kScanTile][Tile::kPairs];                  // delta, delta', delta x, delta' x' of two adjacent channels
  float4 up[kScanTile][Tile::kPairs];                  // g, g', and softplus' of both
  float4 res[kScanTile][Tile::kPairs];                 // sum_n G b of both channels, sum_n a log2(e) p of both
  float b[kScanTile][Tile::kN], c[kScanTile][Tile::kN];
  ulonglong2 start[kScanTile / kRun][2][kScanThreads]; // each thread's states in front of a part of the tile
  float4 part[kScanTile][2][kParts][LN];               // gb and gc of each pair's channels, a lane's four states adjacent
};
template <int LN> struct __align__(16) SummarySmem {
  using Tile = ScanTile<LN>;
  float4 in[kScanTile][Tile::kPairs];                  // delta, delta', g, g'
  float c[kScanTile][Tile::kN];
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

// The gradient that the tokens of a segment alone hand to the state in front of it, and the segment's sum of deltas.
template <typename T, int LN>
__global__ void __launch_bounds__(kScanThreads) scan_bwd_summary_kernel(const __grid_constant__ BwdArgs A) {
  using Tile = ScanTile<LN>;
  __shared__ SummarySmem<LN> sm;
  const ScanShape& sh = A.sh;
  const rfa_scan_t& p = A.p;
  const ScanThread<LN> th(sh);
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

  RawPairs<T, LN> rd, rg;
  RawStates<T, LN> rc;
  uint32_t next = 0;
  const int plain = A.wide && !mask && th.nch == Tile::kChannels && sh.N == Tile::kN ? (int)(sh.T / kScanTile) : 0;      // tiles in front of it are
  const auto ask = [&](int tile, auto kind) {
    constexpr bool kPlain = decltype(kind)::value;
    const int64_t t0 = (int64_t)tile * kScanTile, t = t0 + th.row;
    next = kPlain ? ~0u : tokens_here<LN>(th, mask, t0, sh.T);
    rd.template load<kPlain>(dt + t * p.dt_t, p.dt_t, next, th.vn, A.wide);
    rg.template load<kPlain>(g + t * row_stride, row_stride, next, th.vn, A.wide);
    rc.template load<kPlain>(cp, p.c_t, t0, sh.T, sh.N, mask);
  };
  const auto ask_tile = [&](int tile) { tile < plain ? ask(tile, Plain()) : ask(tile, Ragged()); };
  const auto put = [&]() {
#pragma unroll
    for (int i = 0; i < Tile::kPasses; ++i) {
      float2 sig;
      const float2 v = make_float2(rd.v[i].get(0) + bias[0], rd.v[i].get(1) + bias[1]);
      const f32x2 delta = p.softplus ? softplus2<false>(v, sig) : pack2(v.x, v.y);
      const bool on = next >> i & 1;
      *reinterpret_cast<ulonglong2*>(&sm.in[th.row + i * Tile::kRows][th.vpair]) = make_ulonglong2(on ? delta : 0, pack2(rg.v[i].get(0), rg.v[i].get(1)));
    }
    rc.store(sm.c);
  };
  ask_tile(tile1 - 1);
  for (int tile = tile1 - 1; tile >= tile0; --tile) {
    put();
    __syncthreads();
    if (tile > tile0) ask_tile(tile - 1);
#pragma unroll
    for (int t0 = kScanTile - kRun; t0 >= 0; t0 -= kRun) {
      f32x2 delta[kRun], gt[kRun], e[kRun][4];
#pragma unroll
      for (int r = 0; r < kRun; ++r) {
        const ulonglong2 in = *reinterpret_cast<const ulonglong2*>(&sm.in[t0 + r][th.pair]);
        delta[r] = in.x;
        gt[r] = in.y;
      }
      decays<kRun>(delta, a2, e);
#pragma unroll
      for (int r = kRun - 1; r >= 0; --r) {
        float ct[4];
        lane_states(sm.c[t0 + r], th.ln, ct);
#pragma unroll
        for (int j = 0; j < 4; ++j) G[j] = mul2(scale_add(split2(gt[r]), ct[j], G[j]), e[r][j]);
        sum = add2(sum, delta[r]);
      }
    }
    __syncthreads();
  }
  const size_t at = ((size_t)(seg - 1) * sh.B + th.b) * sh.D;
  th.store_kept(A.seg_grad + at * sh.kn, G);
  const float2 f = split2(sum);
  if (th.ln == 0 && 2 * th.pair < th.nch) A.seg_sum[at + th.channel(0)] = f.x;
  if (th.ln == 0 && 2 * th.pair + 1 < th.nch) A.seg_sum[at + th.channel(1)] = f.y;
}

template <typename T, int LN>
__global__ void __launch_bounds__(kScanThreads, 2) scan_bwd_kernel(const __grid_constant__ BwdArgs A) {
  using Tile = ScanTile<LN>;
  using Smem = BwdSmem<LN>;
  extern __shared__ char smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const ScanShape& sh = A.sh;
  const rfa_scan_t& p = A.p;
  const ScanThread<LN> th(sh);
  const int seg = blockIdx.z, tile0 = seg * sh.seg_tiles, tile1 = min(tile0 + sh.seg_tiles, sh.tiles);

  f32x2 a2[4], G[4], da[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    a2[j] = mul2(th.get(p.a, j, sh.N), both(kLog2e));
    G[j] = A.g_s ? th.get(A.g_s + (size_t)th.b * sh.D * sh.N, j, sh.N) : both(0.f);
    da[j] = both(0.f);
  }
  for (int i = sh.segs - 2; i >= seg; --i) {           // the segments behind this one
    const size_t at = ((size_t)i * sh.B + th.b) * sh.D;
    f32x2 v[4];
    th.load_kept(A.seg_grad + at * sh.kn, v);
    const float* total = A.seg_sum + at + th.channel(0);
    const f32x2 over = pack2(2 * th.pair < th.nch ? total[0] : 0.f, 2 * th.pair + 1 < th.nch ? total[1] : 0.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) G[j] = fma2(exp2_unit(mul2(over, a2[j])), G[j], v[j]);
  }

  const int ch = th.c0 + 2 * th.vpair;
  const T* x = static_cast<const T*>(p.x) + (int64_t)th.b * p.x_b + ch;
  const T* dt = static_cast<const T*>(p.dt) + (int64_t)th.b * p.dt_b + ch;
  const T* g = static_cast<const T*>(A.g) + (int64_t)th.b * sh.D + ch;
  const T* bp = static_cast<const T*>(p.b) + (int64_t)th.b * p.b_b + (int64_t)th.group * p.b_g;
  const T* cp = static_cast<const T*>(p.c) + (int64_t)th.b * p.c_b + (int64_t)th.group * p.c_g;
  const uint8_t* mask = p.mask ? p.mask + (int64_t)th.b * sh.T : nullptr;
  const int64_t row_stride = (int64_t)sh.B * sh.D, out0 = (int64_t)th.b * sh.D + ch;
  float bias[2], skip[2], gd[2] = {}, gbias[2] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    bias[k] = p.dt_bias && k < th.vn ? p.dt_bias[ch + k] : 0.f;
    skip[k] = p.d && k < th.vn ? p.d[ch + k] : 0.f;
  }

  RawPairs<T, LN> rx, rd, rg, kept;
  RawStates<T, LN> rb, rc;
  f32x2 first[4];                                      // the state in front of the tile
  uint32_t here = 0, next = 0;
  const int plain = A.wide && !mask && th.nch == Tile::kChannels && sh.N == Tile::kN ? (int)(sh.T / kScanTile) : 0;      // tiles in front of it are
  const auto ask = [&](int tile, auto kind) {
    constexpr bool kPlain = decltype(kind)::value;
    const int64_t t0 = (int64_t)tile * kScanTile, t = t0 + th.row;
    next = kPlain ? ~0u : tokens_here<LN>(th, mask, t0, sh.T);
    rx.template load<kPlain>(x + t * p.x_t, p.x_t, next, th.vn, A.wide);
    rd.template load<kPlain>(dt + t * p.dt_t, p.dt_t, next, th.vn, A.wide);
    rg.template load<kPlain>(g + t * row_stride, row_stride, next, th.vn, A.wide);
    rb.template load<kPlain>(bp, p.b_t, t0, sh.T, sh.N, mask);
    rc.template load<kPlain>(cp, p.c_t, t0, sh.T, sh.N, mask);
    th.load_kept(A.ckpt + ((size_t)th.b * sh.tiles + tile) * sh.D * sh.kn, first);
  };
  const auto ask_tile = [&](int tile) { tile < plain ? ask(tile, Plain()) : ask(tile, Ragged()); };
  const auto put = [&]() {
    here = next;
#pragma unroll
    for (int i = 0; i < Tile::kPasses; ++i) {
      float2 sig = make_float2(1.f, 1.f);
      const float2 v = make_float2(rd.v[i].get(0) + bias[0], rd.v[i].get(1) + bias[1]);
      const f32x2 delta = p.softplus ? softplus2<true>(v, sig) : pack2(v.x, v.y);
      const f32x2 dx = mul2(delta, pack2(rx.v[i].get(0), rx.v[i].get(1)));
      const bool on = here >> i & 1;
      *reinterpret_cast<ulonglong2*>(&sm.in[th.row + i * Tile::kRows][th.vpair]) = make_ulonglong2(on ? delta : 0, on ? dx : 0);
      sm.up[th.row + i * Tile::kRows][th.vpair] = make_float4(rg.v[i].get(0), rg.v[i].get(1), sig.x, sig.y);
      kept.v[i] = rx.v[i];
    }
    rb.store(sm.b);
    rc.store(sm.c);
  };

  ask_tile(tile1 - 1);
  for (int tile = tile1 - 1; tile >= tile0; --tile) {
    f32x2 s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = first[j];
    put();
    __syncthreads();
    if (tile > tile0) ask_tile(tile - 1);
    const int64_t t0 = (int64_t)tile * kScanTile;

    // The states in front of each part of the tile, then part by part from the last: forward with what the way back needs, and back.
#pragma unroll 1
    for (int part = 0; part < kScanTile / kRun; ++part) {
      f32x2 delta[kRun], dx[kRun], e[kRun][4];
      sm.start[part][0][threadIdx.x] = make_ulonglong2(s[0], s[1]);
      sm.start[part][1][threadIdx.x] = make_ulonglong2(s[2], s[3]);
      if (part == kScanTile / kRun - 1) break;
#pragma unroll
      for (int r = 0; r < kRun; ++r) {
        const ulonglong2 in = *reinterpret_cast<const ulonglong2*>(&sm.in[part * kRun + r][th.pair]);
        delta[r] = in.x;
        dx[r] = in.y;
      }
      decays<kRun>(delta, a2, e);
#pragma unroll
      for (int r = 0; r < kRun; ++r) {
        float bt[4];
        lane_states(sm.b[part * kRun + r], th.ln, bt);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = fma2(e[r][j], s[j], scale(split2(dx[r]), bt[j]));
      }
    }
#pragma unroll 1
    for (int part = kScanTile / kRun - 1; part >= 0; --part) {
      const int base = part * kRun;
      f32x2 delta[kRun], dx[kRun], e[kRun][4], st[kRun + 1][4];      // decays; the states in front of each token
      const ulonglong2 lo = sm.start[part][0][threadIdx.x], hi = sm.start[part][1][threadIdx.x];
      st[0][0] = lo.x; st[0][1] = lo.y; st[0][2] = hi.x; st[0][3] = hi.y;
#pragma unroll
      for (int r = 0; r < kRun; ++r) {
        const ulonglong2 in = *reinterpret_cast<const ulonglong2*>(&sm.in[base + r][th.pair]);
        delta[r] = in.x;
        dx[r] = in.y;
      }
      decays<kRun>(delta, a2, e);
#pragma unroll
      for (int r = 0; r < kRun; ++r) {
        float bt[4];
        lane_states(sm.b[base + r], th.ln, bt);
#pragma unroll
        for (int j = 0; j < 4; ++j) st[r + 1][j] = fma2(e[r][j], st[r][j], scale(split2(dx[r]), bt[j]));
      }
#pragma unroll
      for (int t = kRun - 1; t >= 0; --t) {
        const float2 gt = *reinterpret_cast<const float2*>(&sm.up[base + t][th.pair]), dxt = split2(dx[t]);
        float bt[4], ct[4], gb[4], gc[4];              // gb, gc: of the four states, over both channels
        f32x2 over_b = both(0.f), over_p = both(0.f);  // sum_n G b, sum_n a2 p of both channels
        lane_states(sm.b[base + t], th.ln, bt);
        lane_states(sm.c[base + t], th.ln, ct);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x2 Gt = scale_add(gt, ct[j], G[j]), pt = mul2(Gt, mul2(e[t][j], st[t][j]));
          const float2 Gs = split2(Gt), ss = split2(st[t + 1][j]);
          gb[j] = fmaf(Gs.x, dxt.x, Gs.y * dxt.y);
          gc[j] = fmaf(ss.x, gt.x, ss.y * gt.y);
          over_b = scale_add(Gs, bt[j], over_b);
          over_p = fma2(pt, a2[j], over_p);
          da[j] = fma2(pt, delta[t], da[j]);
          G[j] = mul2(Gt, e[t][j]);
        }
        sm.part[base + t][0][th.pair][th.ln] = make_float4(gb[0], gb[1], gb[2], gb[3]);
        sm.part[base + t][1][th.pair][th.ln] = make_float4(gc[0], gc[1], gc[2], gc[3]);
        const float2 ob = split2(over_b), op = split2(over_p);
        float over_n[4] = {ob.x, ob.y, op.x, op.y};
        lanes_sum<4, LN>(over_n, th.ln);
        float* res = reinterpret_cast<float*>(&sm.res[base + t][th.pair]);
        if constexpr (LN <= 4) {
#pragma unroll
          for (int i = 0; i < 4 / LN; ++i) res[th.ln * (4 / LN) + i] = over_n[i];
        } else {
          if (th.ln % (LN / 4) == 0) res[th.ln / (LN / 4)] = over_n[0];
        }
      }
    }
    __syncthreads();
    // gb and gc of the CTA's channels: kEach neighbouring threads share the sum of one token's four states
    constexpr int kOut = kScanTile * 2 * LN, kEach = kOut < kScanThreads ? kScanThreads / kOut : 1;
#pragma unroll
    for (int o = threadIdx.x / kEach; o < kOut; o += kScanThreads / kEach) {
      const int l = o % LN, which = o / LN % 2, t = o / (2 * LN);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int r = 0; r < Smem::kParts / kEach; ++r) {
        const float4 w = sm.part[t][which][r * kEach + threadIdx.x % kEach][l];
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
      }
      float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int w = kEach / 2; w > 0; w >>= 1)
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] += __shfl_xor_sync(0xffffffffu, f[j], w);
      const int64_t token = t0 + t;
      if (token >= sh.T || threadIdx.x % kEach) continue;
      const bool gone = mask && mask[token];
      const int64_t to = ((token * sh.B + th.b) * sh.G + th.group) * sh.N;
      const int64_t part = (int64_t)(blockIdx.x % sh.per_group) * sh.T * sh.B * sh.G * sh.N + to;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = j * LN + l;
        if (n >= sh.N) continue;
        const float out = gone ? 0.f : f[j];
        if (sh.per_group == 1) static_cast<T*>(which ? A.gc : A.gb)[to + n] = from_f<T>(out);
        else (which ? A.part_c : A.part_b)[part + n] = out;
      }
    }
#pragma unroll
    for (int i = 0; i < Tile::kPasses; ++i) {
      const int t = th.row + i * Tile::kRows;
      if (t0 + t >= sh.T) continue;
      Raw<T, 2> ox, od;
      ox.zero(); od.zero();
      if (here >> i & 1) {
        const float4 in = sm.in[t][th.vpair], up = sm.up[t][th.vpair], res = sm.res[t][th.vpair];
        const float delta[2] = {in.x, in.y}, gt[2] = {up.x, up.y}, sig[2] = {up.z, up.w}, gu[2] = {res.x, res.y}, gp[2] = {res.z, res.w};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float xv = kept.v[i].get(k), v = fmaf(xv, gu[k], kLn2 * gp[k]) * sig[k];
          ox.set(k, from_f<T>(fmaf(delta[k], gu[k], skip[k] * gt[k])));
          od.set(k, from_f<T>(v));
          gd[k] = fmaf(xv, gt[k], gd[k]);
          gbias[k] += v;
        }
      }
      ox.store(static_cast<T*>(A.gx) + (t0 + t) * row_stride + out0, th.vn, A.wide);
      od.store(static_cast<T*>(A.gdt) + (t0 + t) * row_stride + out0, th.vn, A.wide);
    }
    __syncthreads();
  }

  const size_t row = (size_t)th.b * sh.segs + seg;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    th.put(A.part_a + row * sh.D * sh.N, j, sh.N, da[j]);
    if (seg == 0 && A.gs_in) th.put(A.gs_in + (size_t)th.b * sh.D * sh.N, j, sh.N, G[j]);
  }
  float4* over_rows = &sm.in[0][0];                    // gd and gbias over the rows of loading threads
  over_rows[threadIdx.x] = make_float4(gd[0], gd[1], gbias[0], gbias[1]);
  __syncthreads();
  if (th.row == 0) {
    float4 v = over_rows[threadIdx.x];
    for (int r = 1; r < Tile::kRows; ++r) {
      const float4 w = over_rows[r * Tile::kPairs + threadIdx.x];
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

template <typename T, int LN> int launch_bwd(const BwdArgs& a, cudaStream_t stream) {
  constexpr int bytes = (int)sizeof(BwdSmem<LN>);
  const dim3 grid(a.sh.per_group * a.sh.G, a.sh.B, a.sh.segs);
  const cudaError_t err = cudaFuncSetAttribute(scan_bwd_kernel<T, LN>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  RFA_REQUIRE(err == cudaSuccess, (int)err, "selective_scan_bwd: %s", cudaGetErrorString(err));
  if (a.sh.segs > 1) {
    scan_bwd_summary_kernel<T, LN><<<dim3(grid.x, grid.y, a.sh.segs - 1), kScanThreads, 0, stream>>>(a);
    if (int r = check_launch("selective_scan_bwd (segments)")) return r;
  }
  scan_bwd_kernel<T, LN><<<grid, kScanThreads, bytes, stream>>>(a);
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
