// Selective scan, forward and one token:
//   delta = softplus(dt + bias),  s_t = exp(delta_t a) s_(t-1) + delta_t b_t x_t,  y_t = c_t . s_t + d x_t.
//
// Bound by the exponentials: one per token, channel and state, 16 a clock and SM, where a token and channel of 16 states moves 6 bytes in
// 16 bits (8 x 2048 tokens x 2048 channels: 537 M exponentials are 119 us of that unit, 201 MB are 31 us of memory).  Layout in scan.cuh.
//
// Few rows (a prompt of one sequence) leave SMs idle: the tokens are then cut into segments.  A first kernel leaves each segment's own state
// from zero and the sum of its deltas -- over which a whole segment's decay is exp(a sum delta), one exponential -- and the main kernel's
// CTAs begin with the states of the segments before theirs joined up, which costs the first kernel's pass over dt, x and b once more.
#include "scan.cuh"

namespace rfa {

int scan_lanes(int N) { return N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

ScanShape scan_shape(int64_t T, int B, int D, int N, int G, bool backward) {
  ScanShape s{};
  const int channels = 256 / scan_lanes(N);
  s.T = T; s.B = B; s.D = D; s.N = N; s.G = G;
  s.heads = D / G;
  s.per_group = (s.heads + channels - 1) / channels;
  s.tiles = (int)((T + kScanTile - 1) / kScanTile);
  s.n4 = (N + 3) / 4 * 4;
  const int64_t ctas = (int64_t)s.per_group * G * B, want = 148 * (backward ? 2 : 4);
  int64_t segs = ctas >= want ? 1 : (want + ctas - 1) / ctas;
  segs = segs < s.tiles / 4 ? segs : s.tiles / 4;
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
  RFA_REQUIRE(s->T < ((int64_t)1 << 31) - 64 && s->B <= 65535, RFA_EUNSUPPORTED, "%s: T %lld, B %d", what, (long long)s->T, s->B);
  RFA_REQUIRE(aligned16(s->s_in), RFA_EALIGN, "%s: s_in is not 16-byte aligned", what);
  return 0;
}

namespace {

template <int LN> struct __align__(16) FwdSmem {
  float4 in[2][kScanTile][ScanTile<LN>::kPairs];      // delta, delta', x, x' of two adjacent channels; then y, y' in place of the deltas
  float b[2][kScanTile][ScanTile<LN>::kN], c[2][kScanTile][ScanTile<LN>::kN];
};

struct FwdArgs {
  ScanShape sh;
  rfa_scan_t p;
  void* y;
  float *s_out, *ckpt, *seg_state, *seg_sum;      // seg_state [segs - 1][B][D][n4], seg_sum [segs - 1][B][D]
  bool wide, states16;                            // x and dt in 16-byte words; states in 16-byte words
};

// kSummary: the state a segment reaches from zero, and its sum of deltas; no c, no y.
template <typename T, int LN, bool kSummary>
__global__ void __launch_bounds__(kScanThreads) scan_fwd_kernel(const __grid_constant__ FwdArgs A) {
  using Tile = ScanTile<LN>;
  extern __shared__ char smem_raw[];
  FwdSmem<LN>& sm = *reinterpret_cast<FwdSmem<LN>*>(smem_raw);
  const ScanShape& sh = A.sh;
  const rfa_scan_t& p = A.p;
  const ScanThread<LN> th(sh);
  const int seg = blockIdx.z, tile0 = seg * sh.seg_tiles, tile1 = min(tile0 + sh.seg_tiles, sh.tiles);
  const int n0 = 4 * th.ln, ns = max(0, min(4, sh.N - n0));

  // this thread's states: a in units of log 2, and s
  float a2[2][4], s[2][4], sum[2] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int ch = th.first_channel() + k;
    const int nk = ch < th.nch ? ns : 0;
    load4u(p.a + (size_t)(th.c0 + ch) * sh.N + n0, nk, a2[k]);
#pragma unroll
    for (int j = 0; j < 4; ++j) a2[k][j] *= kLog2e;
    if (kSummary || !p.s_in) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[k][j] = 0.f;
    } else {
      load4u(p.s_in + ((size_t)th.b * sh.D + th.c0 + ch) * sh.N + n0, nk, s[k]);
    }
    if (!kSummary)
      for (int i = 0; i < seg; ++i) {                  // the segments before this one
        if (ch >= th.nch) continue;
        const size_t at = ((size_t)i * sh.B + th.b) * sh.D + th.c0 + ch;
        float v[4];
        load4f(A.seg_state + at * sh.n4 + n0, n0 < sh.n4 ? 4 : 0, v);
        const float total = A.seg_sum[at];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[k][j] = fmaf(ex2(total * a2[k][j]), s[k][j], v[j]);
      }
  }

  // what this thread loads and writes: eight channels, kPasses tokens of a tile
  const T *x = static_cast<const T*>(p.x), *dt = static_cast<const T*>(p.dt);
  const T* bp = static_cast<const T*>(p.b) + (int64_t)th.b * p.b_b + (int64_t)th.group * p.b_g;
  const T* cp = static_cast<const T*>(p.c) + (int64_t)th.b * p.c_b + (int64_t)th.group * p.c_g;
  const int vch = 8 * th.vec, vn = min(8, th.nch - vch);
  const bool loads = th.row < kScanTile && vn > 0;
  x += (int64_t)th.b * p.x_b + th.c0 + vch;
  dt += (int64_t)th.b * p.dt_b + th.c0 + vch;
  T* y = static_cast<T*>(A.y) + (int64_t)th.b * sh.D + th.c0 + vch;
  const uint8_t* mask = p.mask ? p.mask + (int64_t)th.b * sh.T : nullptr;
  float bias[8], skip[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bias[i] = p.dt_bias && i < vn ? p.dt_bias[th.c0 + vch + i] : 0.f;
    skip[i] = !kSummary && p.d && i < vn ? p.d[th.c0 + vch + i] : 0.f;
  }

  Raw<T, 8> rx[Tile::kPasses], rd[Tile::kPasses];
  RawStates<T, LN> rb, rc;
  uint32_t here = 0, next = 0;                         // which of this thread's tokens are there: bit i of pass i
  const auto ask = [&](int tile) {
    const int64_t t0 = (int64_t)tile * kScanTile;
    const int tokens = (int)min((int64_t)kScanTile, sh.T - t0);
    next = 0;
#pragma unroll
    for (int i = 0; i < Tile::kPasses; ++i) {
      const int t = th.row + i * Tile::kRows;
      rx[i].zero(); rd[i].zero();
      if (loads && t < tokens && !(mask && mask[t0 + t])) {
        next |= 1u << i;
        rx[i].load(x + (t0 + t) * p.x_t, vn, A.wide);
        rd[i].load(dt + (t0 + t) * p.dt_t, vn, A.wide);
      }
    }
    rb.load(bp + t0 * p.b_t, p.b_t, tokens, sh.N, mask ? mask + t0 : nullptr);
    if (!kSummary) rc.load(cp + t0 * p.c_t, p.c_t, tokens, sh.N, mask ? mask + t0 : nullptr);
  };
  const auto put = [&](int buf) {
    here = next;
    if (th.row < kScanTile) {
#pragma unroll
      for (int i = 0; i < Tile::kPasses; ++i) {
        const bool on = here >> i & 1;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (on) {
            float sig;
            const float u0 = rd[i].get(j) + bias[j], u1 = rd[i].get(j + 1) + bias[j + 1];
            v = make_float4(p.softplus ? softplus(u0, sig) : u0, p.softplus ? softplus(u1, sig) : u1, rx[i].get(j), rx[i].get(j + 1));
          }
          sm.in[buf][th.row + i * Tile::kRows][th.vec * 4 + j / 2] = v;
        }
      }
    }
    rb.store(&sm.b[buf][0][0]);
    if (!kSummary) rc.store(&sm.c[buf][0][0]);
  };

  ask(tile0);
  put(0);
  for (int tile = tile0; tile < tile1; ++tile) {
    const int buf = (tile - tile0) & 1;
    __syncthreads();
    const uint32_t mine = here;
    if (tile + 1 < tile1) ask(tile + 1);
    if (!kSummary && A.ckpt && n0 < sh.n4) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (th.first_channel() + k < th.nch)
          store4u(A.ckpt + (((size_t)th.b * sh.tiles + tile) * sh.D + th.c0 + th.first_channel() + k) * sh.n4 + n0, 4, s[k], true);
    }
    constexpr int kRun = kSummary ? 4 : (LN / 2 < 1 ? 1 : LN / 2);      // tokens whose outputs are summed over the lanes together
#pragma unroll
    for (int t0 = 0; t0 < kScanTile; t0 += kRun) {
      float out[2 * kRun];
#pragma unroll
      for (int r = 0; r < kRun; ++r) {
        const float4 in = sm.in[buf][t0 + r][th.pair];
        const float4 bv = *reinterpret_cast<const float4*>(&sm.b[buf][t0 + r][n0]);
        const float bt[4] = {bv.x, bv.y, bv.z, bv.w};
        const float delta[2] = {in.x, in.y}, dx[2] = {in.x * in.z, in.y * in.w};
        float ct[4];
        if (!kSummary) {
          const float4 cv = *reinterpret_cast<const float4*>(&sm.c[buf][t0 + r][n0]);
          ct[0] = cv.x; ct[1] = cv.y; ct[2] = cv.z; ct[3] = cv.w;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float acc = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[k][j] = fmaf(ex2(delta[k] * a2[k][j]), s[k][j], dx[k] * bt[j]);
            if (!kSummary) acc = fmaf(s[k][j], ct[j], acc);
          }
          if (kSummary) sum[k] += delta[k];
          else out[2 * r + k] = acc;
        }
      }
      if constexpr (!kSummary) {
        lanes_sum<2 * kRun, LN>(out, th.ln);           // lane l has value l: token l / 2, channel l % 2
        __syncwarp();                                  // every lane of the pair has read the deltas
        float* at = reinterpret_cast<float*>(&sm.in[buf][t0 + th.ln / 2][th.pair]);
        at[th.ln % 2] = out[0];
      }
    }
    if constexpr (!kSummary) {
      __syncthreads();
      const int64_t t0 = (int64_t)tile * kScanTile;
#pragma unroll
      for (int i = 0; i < Tile::kPasses; ++i) {
        const int t = th.row + i * Tile::kRows;
        if (loads && t0 + t < sh.T) {
          Raw<T, 8> out;
          out.zero();
          if (mine >> i & 1) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
              const float4 v = sm.in[buf][t][th.vec * 4 + j / 2];
              out.set(j, from_f<T>(fmaf(skip[j], v.z, v.x)));
              out.set(j + 1, from_f<T>(fmaf(skip[j + 1], v.w, v.y)));
            }
          }
          out.store(y + (t0 + t) * (int64_t)sh.B * sh.D, vn, A.wide);
        }
      }
    }
    if (tile + 1 < tile1) put(buf ^ 1);
  }

#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int ch = th.first_channel() + k;
    if (ch >= th.nch) continue;
    const size_t row = (size_t)th.b * sh.D + th.c0 + ch;
    if (kSummary) {
      const size_t at = (size_t)seg * sh.B * sh.D + row;
      if (n0 < sh.n4) store4u(A.seg_state + at * sh.n4 + n0, 4, s[k], true);
      if (th.ln == 0) A.seg_sum[at] = sum[k];
    } else if (A.s_out && seg == sh.segs - 1) {
      store4u(A.s_out + row * sh.N + n0, ns, s[k], A.states16);
    }
  }
}

template <typename T, int LN> int launch_fwd(const FwdArgs& a, cudaStream_t stream) {
  constexpr size_t bytes = sizeof(FwdSmem<LN>);
  static_assert(bytes <= 48 * 1024, "no opt-in is made for more");
  const dim3 grid(a.sh.per_group * a.sh.G, a.sh.B, a.sh.segs);
  if (a.sh.segs > 1) {
    scan_fwd_kernel<T, LN, true><<<dim3(grid.x, grid.y, a.sh.segs - 1), kScanThreads, bytes, stream>>>(a);
    if (int r = check_launch("selective_scan_fwd (segments)")) return r;
  }
  scan_fwd_kernel<T, LN, false><<<grid, kScanThreads, bytes, stream>>>(a);
  return check_launch("selective_scan_fwd");
}

// ---- one token ---------------------------------------------------------------------------------------------------------------
// Bound by the state's way from memory and back, 8 bytes per element.  LN lanes a channel, four states (one 16-byte word) each.
template <typename T, int LN, bool kWide>
__global__ void __launch_bounds__(256) scan_step_kernel(const __grid_constant__ rfa_scan_t p, T* y, float* state) {
  const int at_ch = (blockIdx.x * 256 + threadIdx.x) / LN, n0 = 4 * (threadIdx.x % LN), b = blockIdx.y;
  const bool there = at_ch < p.D;
  const int ch = there ? at_ch : 0, n = there ? max(0, min(4, p.N - n0)) : 0;
  const int64_t item = (int64_t)b * p.D + ch;
  const bool gone = p.mask && p.mask[b];
  float s[4], a[4];
  float* at = state + item * p.N + n0;
  if (kWide) {
    load4f(at, n, s);
    load4f(p.a + (size_t)ch * p.N + n0, n, a);
  } else {
    load4u(at, n, s);
    load4u(p.a + (size_t)ch * p.N + n0, n, a);
  }
  const int g = ch / (p.D / p.G);
  const T* bp = static_cast<const T*>(p.b) + (int64_t)b * p.b_b + (int64_t)g * p.b_g + n0;
  const T* cp = static_cast<const T*>(p.c) + (int64_t)b * p.c_b + (int64_t)g * p.c_g + n0;
  float bt[4], ct[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    bt[j] = j < n ? to_f(bp[j]) : 0.f;
    ct[j] = j < n ? to_f(cp[j]) : 0.f;
  }
  const float x = to_f(static_cast<const T*>(p.x)[(int64_t)b * p.x_b + ch]);
  float delta = to_f(static_cast<const T*>(p.dt)[(int64_t)b * p.dt_b + ch]) + (p.dt_bias ? p.dt_bias[ch] : 0.f), sig;
  if (p.softplus) delta = softplus(delta, sig);
  const float dx = delta * x;
  float out = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    s[j] = fmaf(ex2(delta * (a[j] * kLog2e)), s[j], dx * bt[j]);
    out = fmaf(s[j], ct[j], out);
  }
#pragma unroll
  for (int o = LN / 2; o > 0; o >>= 1) out += __shfl_xor_sync(0xffffffffu, out, o);
  if (!there) return;
  if (!gone) store4u(at, n, s, kWide);
  if (n0 == 0) y[item] = from_f<T>(gone ? 0.f : p.d ? fmaf(p.d[ch], x, out) : out);
}

}  // namespace
}  // namespace rfa

extern "C" size_t rfa_selective_scan_checkpoint_bytes(int64_t T, int B, int D, int N) {
  if (T <= 0 || B <= 0 || D <= 0 || N <= 0) return 0;
  return (size_t)((T + rfa::kScanTile - 1) / rfa::kScanTile) * B * D * ((N + 3) / 4 * 4) * 4;
}

extern "C" int rfa_selective_scan_fwd(const rfa_scan_t* scan, void* y, float* s_out, float* checkpoints, void* workspace, size_t workspace_bytes,
                                      rfa_stream_t stream) {
  using namespace rfa;
  if (int r = scan_check(scan, "selective_scan_fwd")) return r;
  RFA_REQUIRE(y, RFA_EINVAL, "selective_scan_fwd: null pointer");
  RFA_REQUIRE(aligned16(s_out) && aligned16(checkpoints) && aligned16(workspace), RFA_EALIGN, "selective_scan_fwd: s_out, checkpoints or workspace is not 16-byte aligned");
  const size_t need = rfa_selective_scan_workspace_bytes(scan->T, scan->B, scan->D, scan->N, scan->G, 0);
  RFA_REQUIRE(!need || (workspace && workspace_bytes >= need), RFA_EWORKSPACE, "selective_scan_fwd: workspace %zu bytes, %zu needed", workspace_bytes, need);
  FwdArgs a{};
  a.sh = scan_shape(scan->T, scan->B, scan->D, scan->N, scan->G, false);
  a.p = *scan;
  a.y = y; a.s_out = s_out; a.ckpt = checkpoints;
  a.seg_state = static_cast<float*>(workspace);
  a.seg_sum = a.seg_state + (size_t)(a.sh.segs - 1) * scan->B * scan->D * a.sh.n4;
  const int size = scan->dtype == RFA_F32 ? 4 : 2;
  a.wide = wide_ok(scan->x, scan->x_t, scan->x_b, size, 8) && wide_ok(scan->dt, scan->dt_t, scan->dt_b, size, 8) && wide_ok(y, scan->D, a.sh.heads, size, 8);
  a.states16 = scan->N % 4 == 0;
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
  const bool wide = scan->N % 4 == 0 && aligned16(scan->a);
#define CALL(T, LN)                                                                                                       \
  do {                                                                                                                    \
    const dim3 grid((unsigned)(((int64_t)scan->D * LN + 255) / 256), scan->B);                                            \
    if (wide) scan_step_kernel<T, LN, true><<<grid, 256, 0, as_stream(stream)>>>(*scan, static_cast<T*>(y), s);           \
    else scan_step_kernel<T, LN, false><<<grid, 256, 0, as_stream(stream)>>>(*scan, static_cast<T*>(y), s);               \
  } while (0)
  RFA_SCAN_DISPATCH(scan->dtype, scan_lanes(scan->N), CALL);
#undef CALL
  return check_launch("selective_scan_step");
}
