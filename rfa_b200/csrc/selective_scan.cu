// Selective scan, forward and one token:
//   delta = softplus(dt + bias),  s_t = exp(delta_t a) s_(t-1) + delta_t b_t x_t,  y_t = c_t . s_t + d x_t.
//
// Bound by arithmetic: one exponential per token, channel and state, where a token and channel of 16 states moves 6 bytes in 16 bits
// (8 x 2048 tokens x 2048 channels: 537 M exponentials are 119 us of the special function units, 201 MB are 31 us of memory).  That size
// takes 230 to 232 us in bf16: of the 105 cycles of a token on an SM's scheduler the special function unit is busy for 56 (with softplus),
// the FMA units for 63, shared memory for 61 of the SM's, and 68 are issue slots; 256 CTAs on 148 SMs leave a seventh of the card idle.
// Tiles of 32 tokens: 226 us, for twice the shared memory and code.  Layout in scan.cuh.
//
// Few rows (a prompt of one sequence) leave SMs idle: the tokens are then cut into segments.  A first kernel leaves each segment's own state
// from zero and the sum of its deltas -- over which a whole segment's decay is exp(a sum delta), one exponential -- and the main kernel's
// CTAs begin with the states of the segments before theirs joined up, which costs the first kernel's pass over dt, x and b once more.
// 1 x 16384 tokens x 1024 channels, fp16, 37 segments: 87 us the first kernel (special function unit 65 % busy, FMA units 60 %), 118 the main one.
#include "scan.cuh"

namespace rfa {

int scan_lanes(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

// Two CTAs run side by side on an SM, 296 in all; one alone takes 0.63 of the time of two (forward, 0.66 backward).  A segment more costs the
// forward about half of its pass again, the backward an eighth.  us at T = 2048 (N = 16, bf16; a call with its host time of about 10 us), one segment /
// what the rule takes (other numbers):
//   forward   16 CTAs 148 / 44 in 19, 64 CTAs 150 / 110 in ten (four 119); above 120 one: 128 CTAs 158 (two 192), 160 CTAs 239 (two 277, four 244),
//             256 CTAs 241 (two 328)
//   backward  16 CTAs 527 / 87 in 19, 64 CTAs 579 / 286 in ten; above 120 whatever fills the last round: 128 CTAs 607 / 551 in two (four 548),
//             160 CTAs 903 / 655 in five (three 716, six 642), 320 CTAs (T = 1024) 726 / 603 in six (three 624), 256 CTAs 937 in one (four 955)
// Segments of less than 96 tokens lose to their own ends (16 CTAs, T = 2048: 19 segments 42 us, 32 segments 47, 64 segments 66).
ScanShape scan_shape(int64_t T, int B, int D, int N, int G, bool backward) {
  ScanShape s{};
  const int channels = 256 / scan_lanes(N);
  s.T = T; s.B = B; s.D = D; s.N = N; s.G = G;
  s.heads = D / G;
  s.per_group = (s.heads + channels - 1) / channels;
  const int tokens = backward ? kept_tokens(scan_lanes(N)) : kScanTile;
  s.tiles = (int)((T + tokens - 1) / tokens);
  s.kn = 4 * scan_lanes(N);
  const int64_t ctas = (int64_t)s.per_group * G * B;
  int64_t segs = 1;
  if (ctas < 120) {
    segs = (592 + ctas - 1) / ctas;
  } else if (backward) {
    double best = 1e30;
    for (int n = 1; n <= 6; ++n) {
      const int64_t last = ctas * n % 296;
      const double cost = (ctas * n / 296 + (last == 0 ? 0. : last <= 148 ? 0.66 : 1.) + 0.12 * (n - 1)) / n;
      if (cost < 0.97 * best) { best = cost; segs = n; }
    }
  }
  const int64_t most = T / 96;
  segs = segs < most ? segs : most;
  if (segs < 1) segs = 1;
  s.seg_tiles = (int)((s.tiles + segs - 1) / segs);
  s.segs = (s.tiles + s.seg_tiles - 1) / s.seg_tiles;
  return s;
}

int scan_check(const rfa_scan_t* s, const char* what) {
  RFA_REQUIRE(s, RFA_EINVAL, "%s: null argument", what);
  RFA_REQUIRE(s->x && s->dt && s->a && s->b && s->c, RFA_EINVAL, "%s: null pointer", what);
  RFA_REQUIRE(s->T > 0 && s->B > 0 && s->D > 0 && s->N > 0 && s->G > 0, RFA_EINVAL, "%s: empty or negative size", what);
  RFA_REQUIRE(s->dtype == RFA_F16 || s->dtype == RFA_F32 || s->dtype == RFA_BF16, RFA_EUNSUPPORTED, "%s: dtype %d", what, s->dtype);
  RFA_REQUIRE(s->D % s->G == 0, RFA_EUNSUPPORTED, "%s: %d channels in %d groups", what, s->D, s->G);
  RFA_REQUIRE(s->N <= 64, RFA_EUNSUPPORTED, "%s: %d states (at most 64)", what, s->N);
  RFA_REQUIRE(s->T < ((int64_t)1 << 31) - 64 && s->B <= 65535 && s->D <= kMaxChannels, RFA_EUNSUPPORTED, "%s: T %lld, B %d, D %d", what, (long long)s->T,
              s->B, s->D);
  RFA_REQUIRE(aligned16(s->s_in), RFA_EALIGN, "%s: s_in is not 16-byte aligned", what);
  return 0;
}

namespace {

template <int LN> struct __align__(16) FwdSmem {
  using Tile = ScanTile<LN>;
  static constexpr int kRow = Tile::kPairs * 2 + 8;    // the 8: neighbouring rows in other banks
  float4 in[2][kScanTile][Tile::kPairs];               // delta, delta', delta x, delta' x' of two adjacent channels
  float b[2][kScanTile][Tile::kN], c[2][kScanTile][Tile::kN];
  f32x2 y[2][kScanTile][LN / 2][kRow];                 // c . s, each lane's share; two lanes' side by side
};

constexpr int kFwdScan = 128, kFwdBring = 128, kFwdThreads = kFwdScan + kFwdBring;
template <int LN> using FwdThread = ScanThread<LN, kFwdScan, kFwdBring, kScanTile>;

struct FwdArgs {
  ScanShape sh;
  rfa_scan_t p;
  void* y;
  float *s_out, *ckpt, *seg_state, *seg_sum;      // seg_state [segs - 1][B][D][kn], seg_sum [segs - 1][B][D]
  int ckpts;                                      // of a batch row
  bool wide;                                      // pairs of x, dt and y as one word
};

// Brings the tiles of a segment and takes their outputs away.  kSummary: no c, no y.
template <typename T, int LN, bool kSummary>
__device__ __forceinline__ void fwd_bring(const FwdArgs& A, FwdSmem<LN>& sm, const FwdThread<LN>& th, int tile0, int tile1) {
  using Tile = ScanTile<LN>;
  const ScanShape& sh = A.sh;
  const rfa_scan_t& p = A.p;
  const int ch = th.c0 + 2 * th.vpair;
  const T* x = static_cast<const T*>(p.x) + (int64_t)th.b * p.x_b + ch;
  const T* dt = static_cast<const T*>(p.dt) + (int64_t)th.b * p.dt_b + ch;
  const T* bp = static_cast<const T*>(p.b) + (int64_t)th.b * p.b_b + (int64_t)th.group * p.b_g;
  const T* cp = static_cast<const T*>(p.c) + (int64_t)th.b * p.c_b + (int64_t)th.group * p.c_g;
  T* y = static_cast<T*>(A.y) + (int64_t)th.b * sh.D + ch;
  const int64_t y_t = (int64_t)sh.B * sh.D;
  const uint8_t* mask = p.mask ? p.mask + (int64_t)th.b * sh.T : nullptr;
  float bias[2], skip[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    bias[k] = p.dt_bias && k < th.vn ? p.dt_bias[ch + k] : 0.f;
    skip[k] = !kSummary && p.d && k < th.vn ? p.d[ch + k] : 0.f;
  }
  using Thread = FwdThread<LN>;
  RawPairs<T, Thread> rx, rd, kept;
  RawStates<T, LN, Thread> rb, rc;
  uint32_t here = 0, next = 0;                         // which of this thread's tokens are there: in the tile that is scanned, in the next one
  const int plain = A.wide && !mask && th.nch == Tile::kChannels ? (int)(sh.T / kScanTile) : 0;      // tiles in front of it are
  const auto ask = [&](int tile, auto kind) {
    constexpr bool kPlain = decltype(kind)::value;
    const int64_t t0 = (int64_t)tile * kScanTile, t = t0 + th.row;
    next = kPlain ? ~0u : th.tokens_here(mask, t0, sh.T);
    rx.template load<kPlain>(x + t * p.x_t, p.x_t, next, th.vn, A.wide);
    rd.template load<kPlain>(dt + t * p.dt_t, p.dt_t, next, th.vn, A.wide);
    rb.template load<kPlain>(th, bp, p.b_t, t0, sh.T, sh.N, mask);
    if (!kSummary) rc.template load<kPlain>(th, cp, p.c_t, t0, sh.T, sh.N, mask);
  };
  const auto ask_tile = [&](int tile) { tile < plain ? ask(tile, Plain()) : ask(tile, Ragged()); };
  const auto put = [&](int buf) {
#pragma unroll
    for (int i = 0; i < Thread::kPasses; ++i) {
      float2 sig;
      const float2 v = make_float2(rd.v[i].get(0) + bias[0], rd.v[i].get(1) + bias[1]);
      const f32x2 delta = p.softplus ? softplus2<false>(v, sig) : pack2(v.x, v.y);
      const f32x2 dx = mul2(delta, pack2(rx.v[i].get(0), rx.v[i].get(1)));
      const bool on = next >> i & 1;
      *reinterpret_cast<ulonglong2*>(&sm.in[buf][th.row + i * Thread::kRows][th.vpair]) = make_ulonglong2(on ? delta : 0, on ? dx : 0);
    }
    rb.store(th, sm.b[buf]);
    if (!kSummary) rc.store(th, sm.c[buf]);
  };
  const auto take = [&](int tile, int buf) {
    const int64_t t0 = (int64_t)tile * kScanTile;
#pragma unroll
    for (int i = 0; i < Thread::kPasses; ++i) {
      const int t = th.row + i * Thread::kRows;
      if (t0 + t >= sh.T) continue;
      f32x2 v[LN];
#pragma unroll
      for (int l = 0; l < LN; l += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&sm.y[buf][t][l / 2][2 * th.vpair]);
        v[l] = two.x; v[l + 1] = two.y;
      }
#pragma unroll
      for (int w = LN / 2; w > 0; w /= 2)
#pragma unroll
        for (int l = 0; l < w; ++l) v[l] = add2(v[l], v[l + w]);
      const float2 f = split2(v[0]);
      const bool on = here >> i & 1;
      Raw<T, 2> out;
      out.zero();
      out.set2(0, on ? fmaf(skip[0], kept.v[i].get(0), f.x) : 0.f, on ? fmaf(skip[1], kept.v[i].get(1), f.y) : 0.f);
      out.store(y + (t0 + t) * y_t, th.vn, A.wide);
    }
  };

  ask_tile(tile0);
  for (int tile = tile0; tile < tile1; ++tile) {
    const int buf = (tile - tile0) & 1;
    put(buf);
    meet_go<kFwdThreads>(kFull + buf);
    RawPairs<T, Thread> x_now = rx;
    const uint32_t here_now = next;
    if (tile + 1 < tile1) ask_tile(tile + 1);
    if (tile > tile0) {                                // the other buffer's tile
      meet_wait<kFwdThreads>(kDone + (buf ^ 1));
      if (!kSummary) take(tile - 1, buf ^ 1);
    }
    kept = x_now;
    here = here_now;
  }
  const int last = (tile1 - 1 - tile0) & 1;
  meet_wait<kFwdThreads>(kDone + last);
  if (!kSummary) take(tile1 - 1, last);
}

// kSummary: the state a segment reaches from zero, and its sum of deltas.
template <typename T, int LN, bool kSummary>
__global__ void __launch_bounds__(kFwdThreads, 2) scan_fwd_kernel(const __grid_constant__ FwdArgs A) {
  using Tile = ScanTile<LN>;
  extern __shared__ char smem_raw[];
  FwdSmem<LN>& sm = *reinterpret_cast<FwdSmem<LN>*>(smem_raw);
  const ScanShape& sh = A.sh;
  const rfa_scan_t& p = A.p;
  const FwdThread<LN> th(sh);
  const int seg = blockIdx.z, tile0 = seg * sh.seg_tiles, tile1 = min(tile0 + sh.seg_tiles, sh.tiles);
  if (!th.scans) {
    fwd_bring<T, LN, kSummary>(A, sm, th, tile0, tile1);
    return;
  }

  f32x2 a2[4], s[4], sum = both(0.f);                  // a in units of log 2
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    a2[j] = mul2(th.get(p.a, j, sh.N), both(kLog2e));
    s[j] = !kSummary && p.s_in ? th.get(p.s_in + (size_t)th.b * sh.D * sh.N, j, sh.N) : both(0.f);
  }
  if (!kSummary) join_segments(th, sh, A.seg_state, A.seg_sum, 0, seg, 1, a2, s);      // the segments before this one
  for (int tile = tile0; tile < tile1; ++tile) {
    const int buf = (tile - tile0) & 1;
    meet_wait<kFwdThreads>(kFull + buf);
    constexpr int kRun = 4;                            // tokens whose decays are formed side by side
#pragma unroll
    for (int t0 = 0; t0 < kScanTile; t0 += kRun) {
      if (!kSummary && A.ckpt && t0 % kept_tokens(LN) == 0) {
        const int at = tile * (kScanTile / kept_tokens(LN)) + t0 / kept_tokens(LN);
        if (at < A.ckpts) th.store_kept(A.ckpt + ((size_t)th.b * A.ckpts + at) * sh.D * sh.kn, s);
      }
      f32x2 delta[kRun], dx[kRun], e[kRun][4];
#pragma unroll
      for (int r = 0; r < kRun; ++r) {
        const ulonglong2 in = *reinterpret_cast<const ulonglong2*>(&sm.in[buf][t0 + r][th.pair]);
        delta[r] = in.x;
        dx[r] = in.y;
      }
      decays<kRun, true>(delta, a2, e);
#pragma unroll
      for (int r = 0; r < kRun; ++r) {
        float bt[4];
        lane_states(sm.b[buf][t0 + r], th.ln, bt);
#pragma unroll
        for (int j = 0; j < 4; ++j) e[r][j] = s[j] = fma2(e[r][j], s[j], mul2(dx[r], both(bt[j])));
      }
      if constexpr (kSummary) {
        sum = add2(sum, add2(add2(delta[0], delta[1]), add2(delta[2], delta[3])));
      } else {
        f32x2 out[kRun];
#pragma unroll
        for (int r = 0; r < kRun; ++r) {
          float ct[4];
          lane_states(sm.c[buf][t0 + r], th.ln, ct);
          out[r] = mul2(e[r][0], both(ct[0]));
#pragma unroll
          for (int j = 1; j < 4; ++j) out[r] = fma2(e[r][j], both(ct[j]), out[r]);
        }
#pragma unroll
        for (int r = 0; r < kRun; ++r) sm.y[buf][t0 + r][th.ln / 2][2 * th.pair + th.ln % 2] = out[r];
      }
    }
    meet_go<kFwdThreads>(kDone + buf);
  }

  if (kSummary) {
    const size_t at = ((size_t)seg * sh.B + th.b) * sh.D;
    th.store_kept(A.seg_state + at * sh.kn, s);
    th.put1(A.seg_sum + at, sum);
  } else if (A.s_out && seg == sh.segs - 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) th.put(A.s_out + (size_t)th.b * sh.D * sh.N, j, sh.N, s[j]);
  }
}

template <typename T, int LN> int launch_fwd(const FwdArgs& a, cudaStream_t stream) {
  constexpr int bytes = (int)sizeof(FwdSmem<LN>);
  cudaError_t err = cudaFuncSetAttribute(scan_fwd_kernel<T, LN, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess) err = cudaFuncSetAttribute(scan_fwd_kernel<T, LN, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  RFA_REQUIRE(err == cudaSuccess, (int)err, "selective_scan_fwd: %s", cudaGetErrorString(err));
  const dim3 grid(a.sh.per_group * a.sh.G, a.sh.B, a.sh.segs);
  if (a.sh.segs > 1) {
    scan_fwd_kernel<T, LN, true><<<dim3(grid.x, grid.y, a.sh.segs - 1), kFwdThreads, bytes, stream>>>(a);
    if (int r = check_launch("selective_scan_fwd (segments)")) return r;
  }
  scan_fwd_kernel<T, LN, false><<<grid, kFwdThreads, bytes, stream>>>(a);
  return check_launch("selective_scan_fwd");
}

// n of 4 floats, the rest 0; `wide`: as one 16-byte word
__device__ __forceinline__ void load4(const float* p, int n, bool wide, float* v) {
  if (wide && n >= 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.f;
  }
}
__device__ __forceinline__ void store4(float* p, int n, bool wide, const float* v) {
  if (wide && n >= 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = v[i];
  }
}

// ---- one token ---------------------------------------------------------------------------------------------------------------
// Bound by the state's way from memory and back, 8 bytes per element, where it is large enough.  A thread has eight adjacent states (two
// 16-byte words) of one channel, LN / 2 lanes a channel, in kRows batch rows, all of whose loads are on the way at once: the step size, a, the
// group and the addresses, which are most of the instructions, are found once for them.  256 x 2048 x 16 in bf16: 13.8 us in a graph, 16.4 by itself,
// 10.8 of memory.  Registers are limited to what leaves an SM four CTAs (three in fp32): 68 of them took 16.9 us.
template <typename T, int LN, int kRows>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 3 : 4) scan_step_kernel(const __grid_constant__ rfa_scan_t p, T* y, float* state, bool wide, bool wide_bc) {
  constexpr int kLanes = LN / 2, kPoly = LN < 8 ? LN / 2 : 4;      // pairs of a thread's states
  const int at_ch = (blockIdx.x * 256 + threadIdx.x) / kLanes, n0 = 8 * (threadIdx.x % kLanes), b0 = blockIdx.y * kRows;
  const bool there = at_ch < p.D;
  const int ch = there ? at_ch : 0, rows = min(kRows, p.B - b0);
  const int n[2] = {there ? p.N - n0 : 0, there ? p.N - n0 - 4 : 0};
  const int g = p.G == 1 ? 0 : ch / (p.D / p.G);
  const T* bp = static_cast<const T*>(p.b) + (int64_t)g * p.b_g + n0;
  const T* cp = static_cast<const T*>(p.c) + (int64_t)g * p.c_g + n0;
  float* at = state + ((int64_t)b0 * p.D + ch) * p.N + n0;
  const int64_t row = (int64_t)p.D * p.N;
  float s[kRows][8], a[8];
  Raw<T, 4> rb[kRows][2], rc[kRows][2];
  T x[kRows], dt[kRows];
  const float bias = p.dt_bias ? p.dt_bias[ch] : 0.f, skip = p.d ? p.d[ch] : 0.f;
  // What the decays want is asked for in front of the states or behind: 256 x 2048 x 16 in front 14.9 us in bf16
  // and 15.4 in fp32, behind 13.9 and 16.6
  constexpr bool kSmallFirst = sizeof(T) == 4;
  if constexpr (kSmallFirst) {
#pragma unroll
    for (int h = 0; h < 2; ++h) load4(p.a + (size_t)ch * p.N + n0 + 4 * h, n[h], wide, a + 4 * h);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int b = b0 + (r < rows ? r : 0);             // a row that is not there: another's loads, nothing stored
    if constexpr (kSmallFirst) {
      dt[r] = static_cast<const T*>(p.dt)[(int64_t)b * p.dt_b + ch];
      x[r] = static_cast<const T*>(p.x)[(int64_t)b * p.x_b + ch];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      load4(at + (b - b0) * row + 4 * h, n[h], wide, s[r] + 4 * h);
      rb[r][h].load(bp + (int64_t)b * p.b_b + 4 * h, n[h], wide_bc);
      rc[r][h].load(cp + (int64_t)b * p.c_b + 4 * h, n[h], wide_bc);
    }
    if constexpr (!kSmallFirst) {
      dt[r] = static_cast<const T*>(p.dt)[(int64_t)b * p.dt_b + ch];
      x[r] = static_cast<const T*>(p.x)[(int64_t)b * p.x_b + ch];
    }
  }
  if constexpr (!kSmallFirst) {
#pragma unroll
    for (int h = 0; h < 2; ++h) load4(p.a + (size_t)ch * p.N + n0 + 4 * h, n[h], wide, a + 4 * h);
  }
  f32x2 a2[4];                                         // in units of log 2; adjacent states in pairs
#pragma unroll
  for (int i = 0; i < 4; ++i) a2[i] = mul2(pack2(a[2 * i], a[2 * i + 1]), both(kLog2e));
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const float xv = to_f(x[r]);
    float delta = to_f(dt[r]) + bias, sig;
    if (p.softplus) delta = softplus(delta, sig);
    const f32x2 dx = both(delta * xv), step = both(delta);
    f32x2 e[4], out2 = both(0.f);
    Poly<kPoly> poly;                                  // the slow states' decays: an error of one sign would add up from call to call
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < kPoly) poly.template begin<true>(i, mul2(step, a2[i]));
      else e[i] = exp2_unit(mul2(step, a2[i]));
    }
    poly.run();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 bt = rb[r][i / 2].get2(i % 2), ct = rc[r][i / 2].get2(i % 2);
      const f32x2 now = fma2(i < kPoly ? poly.end(i) : e[i], pack2(s[r][2 * i], s[r][2 * i + 1]), mul2(dx, pack2(bt.x, bt.y)));
      out2 = fma2(now, pack2(ct.x, ct.y), out2);
      const float2 f = split2(now);
      s[r][2 * i] = f.x;
      s[r][2 * i + 1] = f.y;
    }
    const float2 halves = split2(out2);
    float out = halves.x + halves.y;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) out += __shfl_xor_sync(0xffffffffu, out, o);
    if (r >= rows || !there) continue;
    const bool gone = p.mask && p.mask[b0 + r];
    if (!gone) {
#pragma unroll
      for (int h = 0; h < 2; ++h) store4(at + r * row + 4 * h, n[h], wide, s[r] + 4 * h);
    }
    if (n0 == 0) y[(int64_t)(b0 + r) * p.D + ch] = from_f<T>(gone ? 0.f : p.d ? fmaf(skip, xv, out) : out);
  }
}

}  // namespace
}  // namespace rfa

extern "C" size_t rfa_selective_scan_checkpoint_bytes(int64_t T, int B, int D, int N) {
  if (T <= 0 || B <= 0 || D <= 0 || N <= 0) return 0;
  const int lanes = rfa::scan_lanes(N), tokens = rfa::kept_tokens(lanes);
  return (size_t)((T + tokens - 1) / tokens) * B * D * (4 * lanes) * 4;
}

extern "C" int rfa_selective_scan_fwd(const rfa_scan_t* scan, void* y, float* s_out, float* checkpoints, void* workspace, size_t workspace_bytes,
                                      rfa_stream_t stream) {
  using namespace rfa;
  if (int r = scan_check(scan, "selective_scan_fwd")) return r;
  RFA_REQUIRE(y, RFA_EINVAL, "selective_scan_fwd: null pointer");
  // a segment's CTA may read s_in after the last segment's has written s_out
  RFA_REQUIRE(!s_out || s_out != scan->s_in, RFA_EINVAL, "selective_scan_fwd: s_out is s_in");
  RFA_REQUIRE(aligned16(s_out) && aligned16(checkpoints) && aligned16(workspace), RFA_EALIGN, "selective_scan_fwd: s_out, checkpoints or workspace is not 16-byte aligned");
  const size_t need = rfa_selective_scan_workspace_bytes(scan->T, scan->B, scan->D, scan->N, scan->G, 0);
  RFA_REQUIRE(!need || (workspace && workspace_bytes >= need), RFA_EWORKSPACE, "selective_scan_fwd: workspace %zu bytes, %zu needed", workspace_bytes, need);
  FwdArgs a{};
  a.sh = scan_shape(scan->T, scan->B, scan->D, scan->N, scan->G, false);
  a.p = *scan;
  a.y = y; a.s_out = s_out; a.ckpt = checkpoints;
  a.ckpts = (int)((scan->T + kept_tokens(scan_lanes(scan->N)) - 1) / kept_tokens(scan_lanes(scan->N)));
  a.seg_state = static_cast<float*>(workspace);
  a.seg_sum = a.seg_state + (size_t)(a.sh.segs - 1) * scan->B * scan->D * a.sh.kn;
  const int size = scan->dtype == RFA_F32 ? 4 : 2;
  a.wide = wide_ok(scan->x, scan->x_t, scan->x_b, size, 2) && wide_ok(scan->dt, scan->dt_t, scan->dt_b, size, 2) && wide_ok(y, scan->D, a.sh.heads, size, 2);
#define CALL(T, LN) return launch_fwd<T, LN>(a, as_stream(stream))
  RFA_SCAN_DISPATCH(scan->dtype, scan_lanes(scan->N), CALL);
#undef CALL
  return 0;
}

extern "C" int rfa_selective_scan_step(const rfa_scan_t* scan, void* y, float* s, rfa_stream_t stream) {
  using namespace rfa;
  if (int r = scan_check(scan, "selective_scan_step")) return r;
  RFA_REQUIRE(y && s, RFA_EINVAL, "selective_scan_step: null pointer");
  RFA_REQUIRE(scan->T == 1, RFA_EINVAL, "selective_scan_step: %lld tokens", (long long)scan->T);
  RFA_REQUIRE(aligned16(s), RFA_EALIGN, "selective_scan_step: s is not 16-byte aligned");
  const int size = scan->dtype == RFA_F32 ? 4 : 2;
  const bool wide = scan->N % 4 == 0 && aligned16(scan->a);
  const bool wide_bc = wide_ok(scan->b, scan->b_b, scan->b_g, size, 4) && wide_ok(scan->c, scan->c_b, scan->c_g, size, 4);
  // Two rows a thread from eight CTAs of one row per SM on; below, all SMs are wanted.  us of B x 2048 x 16 in bf16, one row / two: B = 16 2.45 / 2.55,
  // 32 3.15 / 3.36, 64 (7 a SM) 4.84 / 4.74, 74 (8) 5.23 / 4.91, 128 7.48 / 7.20, 256 14.9 / 14.4
#define CALL(T, LN)                                                                                                          \
  do {                                                                                                                       \
    const unsigned x = (unsigned)(((int64_t)scan->D * (LN / 2) + 255) / 256);                                                \
    if ((int64_t)x * scan->B >= 8 * 148)                                                                                     \
      scan_step_kernel<T, LN, 2><<<dim3(x, (scan->B + 1) / 2), 256, 0, as_stream(stream)>>>(*scan, static_cast<T*>(y), s, wide, wide_bc); \
    else                                                                                                                     \
      scan_step_kernel<T, LN, 1><<<dim3(x, scan->B), 256, 0, as_stream(stream)>>>(*scan, static_cast<T*>(y), s, wide, wide_bc);           \
  } while (0)
  RFA_SCAN_DISPATCH(scan->dtype, scan_lanes(scan->N), CALL);
#undef CALL
  return check_launch("selective_scan_step");
}
