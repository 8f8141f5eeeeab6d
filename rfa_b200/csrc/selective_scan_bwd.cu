// Selective scan, backward.  With G_t = c_t g_t + exp(delta_(t+1) a) G_(t+1) (the gradient of s_t) and p_t = G_t exp(delta_t a) s_(t-1):
//   gc_t = sum over the group's channels of s_t g_t        gb_t = sum over them of G_t delta_t x_t
//   gx_t = delta_t sum_n G_t b_t + d g_t                   ga = sum_t delta_t p_t,  gd = sum_t x_t g_t
//   gdt_t = softplus'(dt_t + bias) (x_t sum_n G_t b_t + sum_n a p_t),  gbias = sum_t gdt_t.
//
// Layout in scan.cuh; tiles from the last to the first.  The states come back from the forward's checkpoints, one in front of every
// 16 tokens (as many bytes as two 16-bit activations at 16 states, instead of all states): a half of 8 tokens is walked forward with
// its decays and decayed states left in registers (128 of them), then backward; the first half's walk is made twice.
// Sums over states go over the LN lanes of a channel, sums over channels over the rest of the warp, then over the CTA's
// warps through shared memory, then over CTAs in sum_parts: a fixed order, no atomics.
//
// Few rows: segments as in the forward, whose summaries run backward here (the gradient a segment hands to the one before it).
#include "scan.cuh"

namespace rfa {
namespace {

constexpr int kHalf = kScanTile / 2;

template <int LN> struct __align__(16) BwdSmem {
  using Tile = ScanTile<LN>;
  float4 in[kScanTile][Tile::kPairs];       // delta, delta', x, x' of two adjacent channels
  float4 up[kScanTile][Tile::kPairs];       // g, g', and softplus' of both
  float4 res[kScanTile][Tile::kPairs];      // sum_n G b of both channels, sum_n a log2(e) p of both
  float b[kScanTile][Tile::kN], c[kScanTile][Tile::kN];
  float part[4][kScanTile][2][Tile::kN];    // gb and gc of each warp's channels
  float acc[16][kScanThreads];              // gd and gbias of each loading thread's eight channels
  float bias[Tile::kChannels], skip[Tile::kChannels];
};

struct BwdArgs {
  ScanShape sh;
  rfa_scan_t p;
  const void* g;
  const float *g_s, *ckpt;
  void *gx, *gdt, *gb, *gc;
  float *gs_in, *part_b, *part_c;           // part_b, part_c [per_group][T][B][G][N], used where per_group > 1
  float *part_a, *part_d, *part_bias;       // [B * segs][D][N], [B * segs][D]
  float *seg_grad, *seg_sum;                // of segments 1 ...: [segs - 1][B][D][n4], [segs - 1][B][D]
  bool wide;
};

// The gradient that the tokens of a segment alone hand to the state in front of it, and the segment's sum of deltas.
template <typename T, int LN>
__global__ void __launch_bounds__(kScanThreads) scan_bwd_summary_kernel(const __grid_constant__ BwdArgs A) {
  using Tile = ScanTile<LN>;
  extern __shared__ char smem_raw[];
  BwdSmem<LN>& sm = *reinterpret_cast<BwdSmem<LN>*>(smem_raw);
  const ScanShape& sh = A.sh;
  const rfa_scan_t& p = A.p;
  const ScanThread<LN> th(sh);
  const int seg = blockIdx.z + 1, tile0 = seg * sh.seg_tiles, tile1 = min(tile0 + sh.seg_tiles, sh.tiles);
  const int n0 = 4 * th.ln, ns = max(0, min(4, sh.N - n0));
  float a2[2][4], G[2][4] = {}, sum[2] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int ch = th.first_channel() + k;
    load4u(p.a + (size_t)(th.c0 + ch) * sh.N + n0, ch < th.nch ? ns : 0, a2[k]);
#pragma unroll
    for (int j = 0; j < 4; ++j) a2[k][j] *= kLog2e;
  }
  const int vch = 8 * th.vec, vn = min(8, th.nch - vch);
  const bool loads = th.row < kScanTile && vn > 0;
  const T* dt = static_cast<const T*>(p.dt) + (int64_t)th.b * p.dt_b + th.c0 + vch;
  const T* g = static_cast<const T*>(A.g) + (int64_t)th.b * sh.D + th.c0 + vch;
  const T* cp = static_cast<const T*>(p.c) + (int64_t)th.b * p.c_b + (int64_t)th.group * p.c_g;
  const uint8_t* mask = p.mask ? p.mask + (int64_t)th.b * sh.T : nullptr;
  for (int i = threadIdx.x; i < Tile::kChannels; i += kScanThreads) sm.bias[i] = p.dt_bias && i < th.nch ? p.dt_bias[th.c0 + i] : 0.f;

  Raw<T, 8> rd[Tile::kPasses], rg[Tile::kPasses];
  RawStates<T, LN> rc;
  uint32_t next = 0;
  const auto ask = [&](int tile) {
    const int64_t t0 = (int64_t)tile * kScanTile;
    const int tokens = (int)min((int64_t)kScanTile, sh.T - t0);
    next = 0;
#pragma unroll
    for (int i = 0; i < Tile::kPasses; ++i) {
      const int t = th.row + i * Tile::kRows;
      rd[i].zero(); rg[i].zero();
      if (loads && t < tokens && !(mask && mask[t0 + t])) {
        next |= 1u << i;
        rd[i].load(dt + (t0 + t) * p.dt_t, vn, A.wide);
        rg[i].load(g + (t0 + t) * (int64_t)sh.B * sh.D, vn, A.wide);
      }
    }
    rc.load(cp + t0 * p.c_t, p.c_t, tokens, sh.N, mask ? mask + t0 : nullptr);
  };
  const auto put = [&]() {
    if (th.row < kScanTile) {
#pragma unroll
      for (int i = 0; i < Tile::kPasses; ++i)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (next >> i & 1) {
            float sig;
            const float u0 = rd[i].get(j) + sm.bias[vch + j], u1 = rd[i].get(j + 1) + sm.bias[vch + j + 1];
            v = make_float4(p.softplus ? softplus(u0, sig) : u0, p.softplus ? softplus(u1, sig) : u1, rg[i].get(j), rg[i].get(j + 1));
          }
          sm.in[th.row + i * Tile::kRows][th.vec * 4 + j / 2] = v;
        }
    }
    rc.store(&sm.c[0][0]);
  };
  ask(tile1 - 1);
  __syncthreads();
  for (int tile = tile1 - 1; tile >= tile0; --tile) {
    put();
    __syncthreads();
    if (tile > tile0) ask(tile - 1);
#pragma unroll 4
    for (int t = kScanTile - 1; t >= 0; --t) {
      const float4 in = sm.in[t][th.pair];
      const float4 cv = *reinterpret_cast<const float4*>(&sm.c[t][n0]);
      const float ct[4] = {cv.x, cv.y, cv.z, cv.w}, delta[2] = {in.x, in.y}, gt[2] = {in.z, in.w};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        sum[k] += delta[k];
#pragma unroll
        for (int j = 0; j < 4; ++j) G[k][j] = fmaf(ct[j], gt[k], G[k][j]) * ex2(delta[k] * a2[k][j]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int ch = th.first_channel() + k;
    if (ch >= th.nch) continue;
    const size_t at = ((size_t)(seg - 1) * sh.B + th.b) * sh.D + th.c0 + ch;
    if (n0 < sh.n4) store4u(A.seg_grad + at * sh.n4 + n0, 4, G[k], true);
    if (th.ln == 0) A.seg_sum[at] = sum[k];
  }
}

template <typename T, int LN>
__global__ void __launch_bounds__(kScanThreads, 2) scan_bwd_kernel(const __grid_constant__ BwdArgs A) {
  using Tile = ScanTile<LN>;
  constexpr int kSlots = 32 / LN;                      // pairs of channels of a warp
  extern __shared__ char smem_raw[];
  BwdSmem<LN>& sm = *reinterpret_cast<BwdSmem<LN>*>(smem_raw);
  const ScanShape& sh = A.sh;
  const rfa_scan_t& p = A.p;
  const ScanThread<LN> th(sh);
  const int seg = blockIdx.z, tile0 = seg * sh.seg_tiles, tile1 = min(tile0 + sh.seg_tiles, sh.tiles);
  const int n0 = 4 * th.ln, ns = max(0, min(4, sh.N - n0));

  float a2[2][4], G[2][4], da[2][4] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int ch = th.first_channel() + k, nk = ch < th.nch ? ns : 0;
    load4u(p.a + (size_t)(th.c0 + ch) * sh.N + n0, nk, a2[k]);
#pragma unroll
    for (int j = 0; j < 4; ++j) a2[k][j] *= kLog2e;
    if (A.g_s) load4u(A.g_s + ((size_t)th.b * sh.D + th.c0 + ch) * sh.N + n0, nk, G[k]);
    else load4u(nullptr, 0, G[k]);
    for (int i = sh.segs - 2; i >= seg; --i) {         // the segments behind this one
      if (ch >= th.nch) continue;
      const size_t at = ((size_t)i * sh.B + th.b) * sh.D + th.c0 + ch;
      float v[4];
      load4f(A.seg_grad + at * sh.n4 + n0, n0 < sh.n4 ? 4 : 0, v);
      const float total = A.seg_sum[at];
#pragma unroll
      for (int j = 0; j < 4; ++j) G[k][j] = fmaf(ex2(total * a2[k][j]), G[k][j], v[j]);
    }
  }

  const int vch = 8 * th.vec, vn = min(8, th.nch - vch);
  const bool loads = th.row < kScanTile && vn > 0;
  const T* x = static_cast<const T*>(p.x) + (int64_t)th.b * p.x_b + th.c0 + vch;
  const T* dt = static_cast<const T*>(p.dt) + (int64_t)th.b * p.dt_b + th.c0 + vch;
  const T* g = static_cast<const T*>(A.g) + (int64_t)th.b * sh.D + th.c0 + vch;
  const T* bp = static_cast<const T*>(p.b) + (int64_t)th.b * p.b_b + (int64_t)th.group * p.b_g;
  const T* cp = static_cast<const T*>(p.c) + (int64_t)th.b * p.c_b + (int64_t)th.group * p.c_g;
  const uint8_t* mask = p.mask ? p.mask + (int64_t)th.b * sh.T : nullptr;
  const int64_t row_stride = (int64_t)sh.B * sh.D, out0 = (int64_t)th.b * sh.D + th.c0 + vch;
  for (int i = threadIdx.x; i < Tile::kChannels; i += kScanThreads) {
    sm.bias[i] = p.dt_bias && i < th.nch ? p.dt_bias[th.c0 + i] : 0.f;
    sm.skip[i] = p.d && i < th.nch ? p.d[th.c0 + i] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) sm.acc[i][threadIdx.x] = 0.f;

  Raw<T, 8> rx[Tile::kPasses], rd[Tile::kPasses], rg[Tile::kPasses];
  RawStates<T, LN> rb, rc;
  float first[2][4];                                   // the state in front of the tile
  uint32_t here = 0, next = 0;
  const auto ask = [&](int tile) {
    const int64_t t0 = (int64_t)tile * kScanTile;
    const int tokens = (int)min((int64_t)kScanTile, sh.T - t0);
    next = 0;
#pragma unroll
    for (int i = 0; i < Tile::kPasses; ++i) {
      const int t = th.row + i * Tile::kRows;
      rx[i].zero(); rd[i].zero(); rg[i].zero();
      if (loads && t < tokens && !(mask && mask[t0 + t])) {
        next |= 1u << i;
        rx[i].load(x + (t0 + t) * p.x_t, vn, A.wide);
        rd[i].load(dt + (t0 + t) * p.dt_t, vn, A.wide);
        rg[i].load(g + (t0 + t) * row_stride, vn, A.wide);
      }
    }
    rb.load(bp + t0 * p.b_t, p.b_t, tokens, sh.N, mask ? mask + t0 : nullptr);
    rc.load(cp + t0 * p.c_t, p.c_t, tokens, sh.N, mask ? mask + t0 : nullptr);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int ch = th.first_channel() + k;
      load4f(A.ckpt + (((size_t)th.b * sh.tiles + tile) * sh.D + th.c0 + ch) * sh.n4 + n0, ch < th.nch && n0 < sh.n4 ? 4 : 0, first[k]);
    }
  };
  const auto put = [&]() {
    here = next;
    if (th.row < kScanTile) {
#pragma unroll
      for (int i = 0; i < Tile::kPasses; ++i)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f), u = v;
          if (here >> i & 1) {
            const float u0 = rd[i].get(j) + sm.bias[vch + j], u1 = rd[i].get(j + 1) + sm.bias[vch + j + 1];
            float s0 = 1.f, s1 = 1.f;
            v = make_float4(p.softplus ? softplus(u0, s0) : u0, p.softplus ? softplus(u1, s1) : u1, rx[i].get(j), rx[i].get(j + 1));
            u = make_float4(rg[i].get(j), rg[i].get(j + 1), s0, s1);
          }
          sm.in[th.row + i * Tile::kRows][th.vec * 4 + j / 2] = v;
          sm.up[th.row + i * Tile::kRows][th.vec * 4 + j / 2] = u;
        }
    }
    rb.store(&sm.b[0][0]);
    rc.store(&sm.c[0][0]);
  };

  ask(tile1 - 1);
  __syncthreads();
  for (int tile = tile1 - 1; tile >= tile0; --tile) {
    float s0[2][4];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) s0[k][j] = first[k][j];
    put();
    __syncthreads();
    if (tile > tile0) ask(tile - 1);

    float e[kHalf][2][4], q[kHalf][2][4], s[2][4];     // decays, decayed states
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[k][j] = s0[k][j];
#pragma unroll
    for (int t = 0; t < kHalf; ++t) {                  // the first half, for the state behind it
      const float4 in = sm.in[t][th.pair];
      const float4 bv = *reinterpret_cast<const float4*>(&sm.b[t][n0]);
      const float bt[4] = {bv.x, bv.y, bv.z, bv.w}, delta[2] = {in.x, in.y}, dx[2] = {in.x * in.z, in.y * in.w};
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[k][j] = fmaf(ex2(delta[k] * a2[k][j]), s[k][j], dx[k] * bt[j]);
    }
#pragma unroll 1
    for (int half = 1; half >= 0; --half) {
      const int base = half * kHalf;
#pragma unroll
      for (int t = 0; t < kHalf; ++t) {
        const float4 in = sm.in[base + t][th.pair];
        const float4 bv = *reinterpret_cast<const float4*>(&sm.b[base + t][n0]);
        const float bt[4] = {bv.x, bv.y, bv.z, bv.w}, delta[2] = {in.x, in.y}, dx[2] = {in.x * in.z, in.y * in.w};
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            e[t][k][j] = ex2(delta[k] * a2[k][j]);
            q[t][k][j] = e[t][k][j] * s[k][j];
            s[k][j] = fmaf(dx[k], bt[j], q[t][k][j]);
          }
      }
#pragma unroll
      for (int t = kHalf - 1; t >= 0; --t) {
        const float4 in = sm.in[base + t][th.pair], up = sm.up[base + t][th.pair];
        const float4 bv = *reinterpret_cast<const float4*>(&sm.b[base + t][n0]), cv = *reinterpret_cast<const float4*>(&sm.c[base + t][n0]);
        const float bt[4] = {bv.x, bv.y, bv.z, bv.w}, ct[4] = {cv.x, cv.y, cv.z, cv.w};
        const float delta[2] = {in.x, in.y}, dx[2] = {in.x * in.z, in.y * in.w}, gt[2] = {up.x, up.y};
        float over_n[4] = {}, over_ch[8] = {};         // sum_n G b, sum_n a2 p of both channels; gb, gc of the four states
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float Gt = fmaf(ct[j], gt[k], G[k][j]), st = fmaf(dx[k], bt[j], q[t][k][j]), pt = Gt * q[t][k][j];
            over_ch[j] = fmaf(Gt, dx[k], over_ch[j]);
            over_ch[4 + j] = fmaf(st, gt[k], over_ch[4 + j]);
            over_n[k] = fmaf(Gt, bt[j], over_n[k]);
            over_n[2 + k] = fmaf(pt, a2[k][j], over_n[2 + k]);
            da[k][j] = fmaf(pt, delta[k], da[k][j]);
            G[k][j] = Gt * e[t][k][j];
          }
        lanes_sum<4, LN>(over_n, th.ln);
        float* res = reinterpret_cast<float*>(&sm.res[base + t][th.pair]);
        if constexpr (LN <= 4) {
#pragma unroll
          for (int i = 0; i < 4 / LN; ++i) res[th.ln * (4 / LN) + i] = over_n[i];
        } else {
          if (th.ln % (LN / 4) == 0) res[th.ln / (LN / 4)] = over_n[0];
        }
        const int slot = th.lane / LN;
        lanes_sum<8, kSlots>(over_ch, slot, LN);
        float* part = &sm.part[th.warp][base + t][0][0];
        if constexpr (kSlots <= 8) {
          constexpr int kEach = 8 / kSlots;
#pragma unroll
          for (int i = 0; i < kEach; ++i) {
            const int v = slot * kEach + i;
            part[(v / 4) * Tile::kN + n0 + v % 4] = over_ch[i];
          }
        } else {
          const int v = slot / (kSlots / 8);
          if (slot % (kSlots / 8) == 0) part[(v / 4) * Tile::kN + n0 + v % 4] = over_ch[0];
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[k][j] = s0[k][j];
    }
    __syncthreads();

    const int64_t t0 = (int64_t)tile * kScanTile;
#pragma unroll
    for (int i = 0; i < Tile::kPasses; ++i) {
      const int t = th.row + i * Tile::kRows;
      if (!loads || t0 + t >= sh.T) continue;
      Raw<T, 8> ox, od;
      ox.zero(); od.zero();
      if (here >> i & 1) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 in = sm.in[t][th.vec * 4 + j / 2], up = sm.up[t][th.vec * 4 + j / 2], res = sm.res[t][th.vec * 4 + j / 2];
          const float delta = j & 1 ? in.y : in.x, xv = j & 1 ? in.w : in.z, gv = j & 1 ? up.y : up.x, sig = j & 1 ? up.w : up.z;
          const float gu = j & 1 ? res.y : res.x, gp = j & 1 ? res.w : res.z;
          const float gd = fmaf(xv, gu, kLn2 * gp) * sig;
          ox.set(j, from_f<T>(fmaf(delta, gu, sm.skip[vch + j] * gv)));
          od.set(j, from_f<T>(gd));
          sm.acc[j][threadIdx.x] += xv * gv;
          sm.acc[8 + j][threadIdx.x] += gd;
        }
      }
      ox.store(static_cast<T*>(A.gx) + (t0 + t) * row_stride + out0, vn, A.wide);
      od.store(static_cast<T*>(A.gdt) + (t0 + t) * row_stride + out0, vn, A.wide);
    }
#pragma unroll
    for (int i = 0; i < Tile::kBc; ++i) {
      const int at = threadIdx.x + i * kScanThreads, t = at / Tile::kN, n = at % Tile::kN;
      if (t0 + t >= sh.T || n >= sh.N) continue;
      float vb = 0.f, vc = 0.f;
      if (!(mask && mask[t0 + t])) {
#pragma unroll
        for (int w = 0; w < 4; ++w) { vb += sm.part[w][t][0][n]; vc += sm.part[w][t][1][n]; }
      }
      const int64_t to = (((t0 + t) * sh.B + th.b) * sh.G + th.group) * sh.N + n;
      if (sh.per_group == 1) {
        static_cast<T*>(A.gb)[to] = from_f<T>(vb);
        static_cast<T*>(A.gc)[to] = from_f<T>(vc);
      } else {
        const int64_t part = (int64_t)(blockIdx.x % sh.per_group) * sh.T * sh.B * sh.G * sh.N + to;
        A.part_b[part] = vb;
        A.part_c[part] = vc;
      }
    }
    __syncthreads();
  }

  const size_t row = (size_t)th.b * sh.segs + seg;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int ch = th.first_channel() + k;
    if (ch >= th.nch) continue;
    store4u(A.part_a + (row * sh.D + th.c0 + ch) * sh.N + n0, ns, da[k], false);
    if (seg == 0 && A.gs_in) store4u(A.gs_in + ((size_t)th.b * sh.D + th.c0 + ch) * sh.N + n0, ns, G[k], false);
  }
  for (int i = threadIdx.x; i < th.nch; i += kScanThreads) {
    float vd = 0.f, vb = 0.f;
    const int rows = min(Tile::kRows, kScanTile);
    for (int r = 0; r < rows; ++r) {
      vd += sm.acc[i % 8][r * Tile::kVecs + i / 8];
      vb += sm.acc[8 + i % 8][r * Tile::kVecs + i / 8];
    }
    A.part_d[row * sh.D + th.c0 + i] = vd;
    A.part_bias[row * sh.D + th.c0 + i] = vb;
  }
}

template <typename T, int LN> int launch_bwd(const BwdArgs& a, cudaStream_t stream) {
  constexpr int bytes = (int)sizeof(BwdSmem<LN>);
  const dim3 grid(a.sh.per_group * a.sh.G, a.sh.B, a.sh.segs);
  cudaError_t err = cudaFuncSetAttribute(scan_bwd_kernel<T, LN>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess) err = cudaFuncSetAttribute(scan_bwd_summary_kernel<T, LN>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  RFA_REQUIRE(err == cudaSuccess, (int)err, "selective_scan_bwd: %s", cudaGetErrorString(err));
  if (a.sh.segs > 1) {
    scan_bwd_summary_kernel<T, LN><<<dim3(grid.x, grid.y, a.sh.segs - 1), kScanThreads, bytes, stream>>>(a);
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
    grad = (size_t)(s.segs - 1) * s.B * s.D * s.n4;
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
  return (size_t)(s.segs - 1) * B * D * (s.n4 + 1) * 4;
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
  a.wide = wide_ok(scan->x, scan->x_t, scan->x_b, size, 8) && wide_ok(scan->dt, scan->dt_t, scan->dt_b, size, 8) &&
           wide_ok(g, scan->D, a.sh.heads, size, 8) && wide_ok(gx, 0, 0, size, 8) && wide_ok(gdt, 0, 0, size, 8);
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
