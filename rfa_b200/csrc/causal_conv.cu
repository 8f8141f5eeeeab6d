// Causal depthwise convolution over the last W tokens, with SiLU: pre_t = bias + sum_j w_j x_(t-W+1+j), y_t = silu(pre_t); and its gradients.
// Padded tokens are left out of the sequence: a window holds the last W tokens that are there.
//
// Bound by memory: x once, y once (backward: x, g, gx).  A warp takes 32 vectors of adjacent channels and a run of tokens, and keeps the
// window in registers, so that x is read once but for the W - 1 tokens in front of a run; four tokens are on the way at a
// time.  The backward walks a run and the W - 1 tokens behind it with the gradients of the last W tokens pending in registers: a
// token's gradient is written when the last window that holds it has passed.  Weight gradients stay in registers over the run,
// are summed over the CTA's warps in shared memory and over CTAs in sum_parts, in a fixed order.
#include "state_space.cuh"

namespace rfa {
namespace {

constexpr int kConvWarps = 4, kConvRun = 16, kConvBwdRun = 32, kConvFlight = 4, kConvMax = 8;

struct ConvArgs {
  rfa_causal_conv_t p;
  void *y, *state_out;
  const void *g, *g_state;
  int64_t g_t, g_b;
  void *gx, *g_state_in;
  float *part_w, *part_b;      // [gridDim.x * B][D][W], [gridDim.x * B][D]; null: not wanted
  bool wide;
};

// The last token before t that is not masked, -1 for none; all lanes of a warp together.
__device__ __forceinline__ int64_t token_before(const uint8_t* mask, int64_t t) {
  const int lane = threadIdx.x & 31;
  for (; t > 0; t -= 32) {
    const int64_t at = t - 1 - lane;
    const uint32_t there = __ballot_sync(0xffffffffu, at >= 0 && !mask[at]);
    if (there) return t - __ffs(there);
  }
  return -1;
}

__device__ __forceinline__ float silu_or(float v, bool silu) { return silu ? v * sigmoid(v) : v; }

template <typename T, int NV> __device__ __forceinline__ void load_row(const T* p, int n, bool wide, float* v) {
  Raw<T, NV> r;
  r.load(p, n, wide);
#pragma unroll
  for (int c = 0; c < NV; ++c) v[c] = r.get(c);
}

// What a thread of either kernel is; the window in front of its run.
template <typename T, int NV, int W, bool kMask> struct ConvThread {
  const rfa_causal_conv_t& p;
  int c0, n, b;
  int64_t t0, t1;
  bool wide;
  const T* x;
  const uint8_t* mask;
  float w[W][NV], bias[NV];
  __device__ ConvThread(const ConvArgs& a, int run) : p(a.p), wide(a.wide) {
    c0 = (blockIdx.y * 32 + (threadIdx.x & 31)) * NV;
    n = min(NV, p.D - c0);                             // may be negative: such a thread only takes part in its warp's ballots
    b = blockIdx.z;
    t0 = ((int64_t)blockIdx.x * kConvWarps + (threadIdx.x >> 5)) * run;
    t1 = min(t0 + run, p.T);
    x = static_cast<const T*>(p.x) + (int64_t)b * p.x_b + c0;
    mask = kMask ? p.mask + (int64_t)b * p.T : nullptr;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
#pragma unroll
      for (int j = 0; j < W; ++j) w[j][c] = c < n ? to_f(static_cast<const T*>(p.weight)[(size_t)(c0 + c) * W + j]) : 0.f;
      bias[c] = p.bias && c < n ? to_f(static_cast<const T*>(p.bias)[c0 + c]) : 0.f;
    }
  }
  __device__ __forceinline__ bool gone(int64_t t) const { return kMask && mask[t]; }
  // win[0 .. W - 2]: the tokens in front of t0, oldest first; at[]: where they stand (-1 ... -(W - 1): in the incoming state)
  __device__ __forceinline__ void before(float (*win)[NV], int64_t* at) const {
    int64_t t = t0;
    int slot = W - 2;                                  // of the incoming state
#pragma unroll
    for (int j = W - 2; j >= 0; --j) {
      if (t > 0) t = kMask ? token_before(mask, t) : t - 1;
      else t = -1;
      if (t >= 0) {
        load_row<T, NV>(x + t * p.x_t, n, wide, win[j]);
        at[j] = t;
      } else {
        if (p.state_in) load_row<T, NV>(static_cast<const T*>(p.state_in) + ((size_t)b * (W - 1) + slot) * p.D + c0, n, wide, win[j]);
        else
#pragma unroll
          for (int c = 0; c < NV; ++c) win[j][c] = 0.f;
        at[j] = slot - (W - 1);
        --slot;
        t = 0;                                         // nothing further in front
      }
    }
  }
};

template <typename T, int NV, int W, bool kMask>
__global__ void __launch_bounds__(32 * kConvWarps) conv_fwd_kernel(const __grid_constant__ ConvArgs a) {
  const ConvThread<T, NV, W, kMask> th(a, kConvRun);
  const rfa_causal_conv_t& p = a.p;
  if (th.t0 >= p.T) return;
  const bool last = th.t1 == p.T && a.state_out;
  const int64_t out_t = (int64_t)p.B * p.D;
  T* y = static_cast<T*>(a.y) + (int64_t)th.b * p.D + th.c0;
  Raw<T, NV> none;
  none.zero();
  if (kMask && !last) {                                // a run of padding has no window to look for
    const int64_t t = th.t0 + (threadIdx.x & 31);
    if (!__ballot_sync(0xffffffffu, t < th.t1 && !th.mask[t])) {
      for (int64_t u = th.t0; u < th.t1; ++u) none.store(y + u * out_t, th.n, th.wide);
      return;
    }
  }
  float win[W - 1 + kConvFlight][NV];
  int64_t at[W];
  th.before(win, at);
  for (int64_t t = th.t0; t < th.t1; t += kConvFlight) {
    Raw<T, NV> raw[kConvFlight];
#pragma unroll
    for (int i = 0; i < kConvFlight; ++i) {
      raw[i].zero();
      if (t + i < th.t1 && !th.gone(t + i)) raw[i].load(th.x + (t + i) * p.x_t, th.n, th.wide);
    }
    int len = 0;                                       // tokens of these that are there
#pragma unroll
    for (int i = 0; i < kConvFlight; ++i) {
      if (t + i >= th.t1) break;
      if (th.gone(t + i)) {
        none.store(y + (t + i) * out_t, th.n, th.wide);
        continue;
      }
      const int at_i = kMask ? 0 : i;                  // with a mask the window is moved on token by token, else after four
#pragma unroll
      for (int c = 0; c < NV; ++c) win[W - 1 + at_i][c] = raw[i].get(c);
      Raw<T, NV> out;
      out.zero();
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        float pre = th.bias[c];
#pragma unroll
        for (int j = 0; j < W; ++j) pre = fmaf(th.w[j][c], win[at_i + j][c], pre);
        out.set(c, from_f<T>(silu_or(pre, p.silu)));
      }
      out.store(y + (t + i) * out_t, th.n, th.wide);
      if (kMask) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
          for (int c = 0; c < NV; ++c) win[j][c] = win[j + 1][c];
      }
      ++len;
    }
    if (!kMask) {
#pragma unroll
      for (int k = 1; k <= kConvFlight; ++k)           // len is at most four, and less only at the end
        if (len == k) {
#pragma unroll
          for (int j = 0; j < W - 1; ++j)
#pragma unroll
            for (int c = 0; c < NV; ++c) win[j][c] = win[j + k][c];
        }
    }
  }
  if (last) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      Raw<T, NV> out;
      out.zero();
#pragma unroll
      for (int c = 0; c < NV; ++c) out.set(c, from_f<T>(win[j][c]));
      out.store(static_cast<T*>(a.state_out) + ((size_t)th.b * (W - 1) + j) * p.D + th.c0, th.n, th.wide);
    }
  }
}

template <typename T, int NV, int W, bool kMask>
__global__ void __launch_bounds__(32 * kConvWarps) conv_bwd_kernel(const __grid_constant__ ConvArgs a) {
  __shared__ float red[kConvWarps][32 * NV + 1];
  const ConvThread<T, NV, W, kMask> th(a, kConvBwdRun);
  const rfa_causal_conv_t& p = a.p;
  const int64_t out_t = (int64_t)p.B * p.D;
  const T* g = static_cast<const T*>(a.g) + (int64_t)th.b * a.g_b + th.c0;
  T* gx = static_cast<T*>(a.gx) + (int64_t)th.b * p.D + th.c0;
  float dw[W][NV] = {}, db[NV] = {};
  bool walk = th.t0 < p.T;
  if (kMask && walk) {                                 // padded tokens' gradients; a run without others has nothing to do but the state's
    Raw<T, NV> none;
    none.zero();
    for (int64_t u = th.t0; u < th.t1; ++u)
      if (th.mask[u]) none.store(gx + u * out_t, th.n, th.wide);
    const int64_t t = th.t0 + (threadIdx.x & 31);
    const bool any = __ballot_sync(0xffffffffu, t < th.t1 && !th.mask[t]);
    walk = any || (th.t0 == 0 && a.g_state_in);
  }
  if (walk) {
    float win[W][NV], pend[W][NV];                     // the last W tokens, oldest first, and their gradients as far as they have come
    int64_t at[W];
    th.before(win, at);
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int c = 0; c < NV; ++c) pend[j][c] = 0.f;
    const auto give = [&](int64_t where, const float* v) {
      const bool mine = where >= th.t0 && where < th.t1, state = where < 0 && th.t0 == 0 && a.g_state_in;
      if (!mine && !state) return;
      Raw<T, NV> out;
      out.zero();
#pragma unroll
      for (int c = 0; c < NV; ++c) out.set(c, from_f<T>(v[c]));
      T* to = mine ? gx + where * out_t : static_cast<T*>(a.g_state_in) + ((size_t)th.b * (W - 1) + (W - 1 + where)) * p.D + th.c0;
      out.store(to, th.n, th.wide);
    };
    int more = W - 1;                                  // tokens behind the run that its own still take part in
    for (int64_t t = th.t0; t < p.T && (t < th.t1 || more > 0); t += kConvFlight) {
      Raw<T, NV> rx[kConvFlight], rg[kConvFlight];
#pragma unroll
      for (int i = 0; i < kConvFlight; ++i) {
        rx[i].zero(); rg[i].zero();
        if (t + i < p.T && !th.gone(t + i)) {
          rx[i].load(th.x + (t + i) * p.x_t, th.n, th.wide);
          rg[i].load(g + (t + i) * a.g_t, th.n, th.wide);
        }
      }
#pragma unroll
      for (int i = 0; i < kConvFlight; ++i) {
        const bool own = t + i < th.t1;
        if (t + i >= p.T || (!own && more == 0)) break;
        if (th.gone(t + i)) continue;
        if (!own) --more;
        at[W - 1] = t + i;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
          win[W - 1][c] = rx[i].get(c);
          float gp = rg[i].get(c);
          if (p.silu) {
            float pre = th.bias[c];
#pragma unroll
            for (int j = 0; j < W; ++j) pre = fmaf(th.w[j][c], win[j][c], pre);
            const float sig = sigmoid(pre);
            gp *= fmaf(pre * sig, 1.f - sig, sig);
          }
#pragma unroll
          for (int j = 0; j < W; ++j) {
            pend[j][c] = fmaf(th.w[j][c], gp, pend[j][c]);
            if (own) dw[j][c] = fmaf(gp, win[j][c], dw[j][c]);
          }
          if (own) db[c] += gp;
        }
        give(at[0], pend[0]);
#pragma unroll
        for (int j = 0; j + 1 < W; ++j) {
          at[j] = at[j + 1];
#pragma unroll
          for (int c = 0; c < NV; ++c) { win[j][c] = win[j + 1][c]; pend[j][c] = pend[j + 1][c]; }
        }
#pragma unroll
        for (int c = 0; c < NV; ++c) pend[W - 1][c] = 0.f;
      }
    }
    if (more > 0) {                                    // the sequence ended: the last W - 1 tokens are the outgoing state
#pragma unroll
      for (int j = 0; j < W - 1; ++j) {
        if (a.g_state) {
          float v[NV];
          load_row<T, NV>(static_cast<const T*>(a.g_state) + ((size_t)th.b * (W - 1) + j) * p.D + th.c0, th.n, th.wide, v);
#pragma unroll
          for (int c = 0; c < NV; ++c) pend[j][c] += v[c];
        }
        give(at[j], pend[j]);
      }
    }
  }
  if (!a.part_w) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t part = (size_t)blockIdx.z * gridDim.x + blockIdx.x;
  for (int j = 0; j <= W; ++j) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      float v = db[c];
#pragma unroll
      for (int k = 0; k < W; ++k)
        if (k == j) v = dw[k][c];
      red[warp][lane * NV + c] = v;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * NV; i += 32 * kConvWarps) {
      const int ch = blockIdx.y * 32 * NV + i;
      if (ch >= p.D) continue;
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < kConvWarps; ++k) v += red[k][i];
      if (j < W) a.part_w[(part * p.D + ch) * W + j] = v;
      else a.part_b[part * p.D + ch] = v;
    }
  }
}

constexpr int conv_vec(int size) { return size == 2 ? 8 : 4; }
constexpr int conv_bwd_vec(int) { return 4; }
int conv_row_blocks(int64_t T, int run) { return (int)((T + kConvWarps * run - 1) / (kConvWarps * run)); }

int conv_check(const rfa_causal_conv_t* p, const char* what) {
  RFA_REQUIRE(p, RFA_EINVAL, "%s: null argument", what);
  RFA_REQUIRE(p->x && p->weight, RFA_EINVAL, "%s: null pointer", what);
  RFA_REQUIRE(p->T > 0 && p->B > 0 && p->D > 0, RFA_EINVAL, "%s: empty or negative size", what);
  RFA_REQUIRE(p->dtype == RFA_F16 || p->dtype == RFA_F32 || p->dtype == RFA_BF16, RFA_EUNSUPPORTED, "%s: dtype %d", what, p->dtype);
  RFA_REQUIRE(p->W >= 1 && p->W <= kConvMax, RFA_EUNSUPPORTED, "%s: a window of %d tokens (1 to %d)", what, p->W, kConvMax);
  RFA_REQUIRE(p->T < ((int64_t)1 << 31) - 64 && p->B <= 65535 && p->D <= 65535 * 128, RFA_EUNSUPPORTED, "%s: T %lld, B %d, D %d", what,
              (long long)p->T, p->B, p->D);
  return 0;
}

template <typename T, int W, bool kMask> int conv_launch(const ConvArgs& a, bool backward, cudaStream_t stream) {
  if (backward) {
    constexpr int NV = conv_bwd_vec(sizeof(T));
    const dim3 grid(conv_row_blocks(a.p.T, kConvBwdRun), (a.p.D + 32 * NV - 1) / (32 * NV), a.p.B);
    conv_bwd_kernel<T, NV, W, kMask><<<grid, 32 * kConvWarps, 0, stream>>>(a);
    return check_launch("causal_conv_bwd");
  }
  constexpr int NV = conv_vec(sizeof(T));
  const dim3 grid(conv_row_blocks(a.p.T, kConvRun), (a.p.D + 32 * NV - 1) / (32 * NV), a.p.B);
  conv_fwd_kernel<T, NV, W, kMask><<<grid, 32 * kConvWarps, 0, stream>>>(a);
  return check_launch("causal_conv_fwd");
}
template <typename T> int conv_width(const ConvArgs& a, bool backward, cudaStream_t stream) {
  switch (a.p.W * 2 + (a.p.mask != nullptr)) {
#define CASE(W) \
  case 2 * W: return conv_launch<T, W, false>(a, backward, stream); \
  case 2 * W + 1: return conv_launch<T, W, true>(a, backward, stream);
    CASE(1) CASE(2) CASE(3) CASE(4) CASE(5) CASE(6) CASE(7) CASE(8)
#undef CASE
  }
  return 0;
}
int conv_dtype(const ConvArgs& a, bool backward, cudaStream_t stream) {
  return a.p.dtype == RFA_F16    ? conv_width<__half>(a, backward, stream)
         : a.p.dtype == RFA_BF16 ? conv_width<__nv_bfloat16>(a, backward, stream)
                                 : conv_width<float>(a, backward, stream);
}

}  // namespace
}  // namespace rfa

extern "C" int rfa_causal_conv_fwd(const rfa_causal_conv_t* conv, void* y, void* state_out, rfa_stream_t stream) {
  using namespace rfa;
  if (int r = conv_check(conv, "causal_conv_fwd")) return r;
  RFA_REQUIRE(y, RFA_EINVAL, "causal_conv_fwd: null pointer");
  RFA_REQUIRE(!state_out || state_out != conv->state_in || conv->T == 1, RFA_EINVAL, "causal_conv_fwd: the state in place of %lld tokens", (long long)conv->T);
  ConvArgs a{};
  a.p = *conv;
  a.y = y; a.state_out = conv->W > 1 ? state_out : nullptr;
  const int size = conv->dtype == RFA_F32 ? 4 : 2, nv = conv_vec(size);
  a.wide = wide_ok(conv->x, conv->x_t, conv->x_b, size, nv) && wide_ok(y, conv->D, 0, size, nv) && wide_ok(state_out, 0, 0, size, nv) &&
           wide_ok(conv->state_in, 0, 0, size, nv);
  return conv_dtype(a, false, as_stream(stream));
}

extern "C" size_t rfa_causal_conv_workspace_bytes(int64_t T, int B, int D, int W) {
  using namespace rfa;
  if (T <= 0 || B <= 0 || D <= 0 || W < 1 || W > kConvMax) return 0;
  return (size_t)conv_row_blocks(T, kConvBwdRun) * B * D * (W + 1) * 4;
}

extern "C" int rfa_causal_conv_bwd(const rfa_causal_conv_t* conv, const void* g, int64_t g_t, int64_t g_b, const void* g_state, void* gx, void* g_weight,
                                   void* g_bias, void* g_state_in, void* workspace, size_t workspace_bytes, rfa_stream_t stream) {
  using namespace rfa;
  if (int r = conv_check(conv, "causal_conv_bwd")) return r;
  RFA_REQUIRE(g && gx, RFA_EINVAL, "causal_conv_bwd: null pointer");
  const bool weights = g_weight || g_bias;
  const size_t need = weights ? rfa_causal_conv_workspace_bytes(conv->T, conv->B, conv->D, conv->W) : 0;
  RFA_REQUIRE(!need || (workspace && workspace_bytes >= need), RFA_EWORKSPACE, "causal_conv_bwd: workspace %zu bytes, %zu needed", workspace_bytes, need);
  RFA_REQUIRE(aligned16(workspace), RFA_EALIGN, "causal_conv_bwd: the workspace is not 16-byte aligned");
  ConvArgs a{};
  a.p = *conv;
  a.g = g; a.g_t = g_t; a.g_b = g_b;
  a.gx = gx;
  if (conv->W > 1) { a.g_state = g_state; a.g_state_in = g_state_in; }
  const int parts = conv_row_blocks(conv->T, kConvBwdRun) * conv->B;
  if (weights) {
    a.part_w = static_cast<float*>(workspace);
    a.part_b = a.part_w + (size_t)parts * conv->D * conv->W;
  }
  const int size = conv->dtype == RFA_F32 ? 4 : 2, nv = conv_bwd_vec(size);
  a.wide = wide_ok(conv->x, conv->x_t, conv->x_b, size, nv) && wide_ok(g, g_t, g_b, size, nv) && wide_ok(gx, conv->D, 0, size, nv) &&
           wide_ok(conv->state_in, 0, 0, size, nv) && wide_ok(a.g_state, 0, 0, size, nv) && wide_ok(a.g_state_in, 0, 0, size, nv);
  if (int r = conv_dtype(a, true, as_stream(stream))) return r;
  const SumJob jobs[2] = {{a.part_w, g_weight, (int64_t)conv->D * conv->W, parts, conv->dtype}, {a.part_b, g_bias, conv->D, parts, conv->dtype}};
  return weights ? sum_parts(jobs, 2, as_stream(stream)) : 0;
}
