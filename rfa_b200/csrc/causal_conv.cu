// Causal depthwise convolution over the last W tokens, with SiLU: pre_t = bias + sum_j w_j x_(t-W+1+j), y_t = silu(pre_t); and its gradients.
// Padded tokens are left out of the sequence: a window holds the last W tokens that are there.
//
// Bound by memory and the sigmoid's two special functions: x once, y once (backward: x, g, gx); 8 x 2048 tokens x 2048 channels of a
// wider array, W = 4, bf16, forward: 20.5 us of memory, 24 us of that unit, 39 us measured (3.5 TB/s; latency and issue slots, 56 %
// busy; fp32 51 us, 5.3 TB/s).  A warp takes 32 vectors of four adjacent channels and a run of 32 tokens, and keeps the window in
// registers, so that x is read once but for the W - 1 tokens in front of a run; four tokens that are there are worked on together
// while the next four are on the way (token by token, a padded batch took 57 us instead of 39).  Vectors of eight: 43 us, runs of
// 16: 43.  The backward walks a run and the W - 1 tokens behind it with the gradients of the last W tokens pending in registers: a
// token's gradient is written when the last window that holds it has passed.  Weight gradients stay in registers over the run,
// are summed over the CTA's warps in shared memory and over CTAs in sum_parts, in a fixed order.
// Backward, 64 x 1024 x 1024 in fp16, padded: 184 us, 62 of memory.  Bound by latency: 130 registers leave three CTAs an SM (18 % of the warps), a
// CTA's four runs are of one row, and issue slots are 46 % busy.
#include "state_space.cuh"

namespace rfa {
namespace {

constexpr int kConvWarps = 4, kConvRun = 32, kConvFlight = 4, kConvMax = 8;
constexpr int kConvVec = 4;      // adjacent channels of a thread

struct ConvArgs {
  rfa_causal_conv_t p;
  void *y, *state_out;
  const void *g, *g_state;
  int64_t g_t, g_b;
  void *gx, *g_state_in;
  float *part_w, *part_b;      // [row_blocks * B][D][W], [row_blocks * B][D]; null: not wanted
  int row_blocks, ch_blocks;   // a CTA's place: channels fastest, so that what runs side by side reads whole rows
  bool wide, wide_w;           // vectors of activations and states, a vector's weights in wide accesses
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

// The first token from t on that is not masked, T for none.
__device__ __forceinline__ int64_t token_after(const uint8_t* mask, int64_t t, int64_t T) {
  const int lane = threadIdx.x & 31;
  for (; t < T; t += 32) {
    const uint32_t there = __ballot_sync(0xffffffffu, t + lane < T && !mask[t + lane]);
    if (there) return t + __ffs(there) - 1;
  }
  return T;
}

template <typename T, int NV, bool kConst = true> __device__ __forceinline__ void load_row(const T* p, int n, bool wide, float* v) {
  Raw<T, NV> r;
  r.template load<kConst>(p, n, wide);
#pragma unroll
  for (int c = 0; c < NV; ++c) v[c] = r.get(c);
}

// Whether the four tokens from the run's i-th on are there.
__device__ __forceinline__ bool four_there(uint32_t there, int i) {
  static_assert(kConvFlight == 4 && kConvRun == 32, "bits of a run, four at a time");
  return i < kConvRun && (there >> i & 15u) == 15u;
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
  int ch_block, row_block;
  __device__ ConvThread(const ConvArgs& a) : p(a.p), wide(a.wide) {
    ch_block = blockIdx.x % a.ch_blocks;
    row_block = blockIdx.x / a.ch_blocks;
    c0 = (ch_block * 32 + (threadIdx.x & 31)) * NV;
    n = min(NV, p.D - c0);                             // may be negative: such a thread only takes part in its warp's ballots
    b = blockIdx.y;
    t0 = ((int64_t)row_block * kConvWarps + (threadIdx.x >> 5)) * kConvRun;
    t1 = min(t0 + kConvRun, p.T);
    x = static_cast<const T*>(p.x) + (int64_t)b * p.x_b + c0;
    mask = kMask ? p.mask + (int64_t)b * p.T : nullptr;
    Raw<T, NV * W> rw;
    rw.load(static_cast<const T*>(p.weight) + (size_t)c0 * W, n * W, a.wide_w);
    Raw<T, NV> rb;
    rb.zero();
    if (p.bias) rb.load(static_cast<const T*>(p.bias) + c0, n, wide);
#pragma unroll
    for (int c = 0; c < NV; ++c) {
#pragma unroll
      for (int j = 0; j < W; ++j) w[j][c] = rw.get(c * W + j);
      bias[c] = rb.get(c);
    }
  }
  // The run's tokens that are there: bit t - t0.
  __device__ __forceinline__ uint32_t tokens() const {
    const int64_t t = t0 + (threadIdx.x & 31);
    return __ballot_sync(0xffffffffu, t < t1 && !(kMask && mask[t]));
  }
  // win[0 .. W - 2]: the tokens in front of t0, oldest first; at[]: where they stand (-1 ... -(W - 1): in the incoming state,
  // which may be the outgoing one of a single token: not a constant of the launch)
  __device__ __forceinline__ void before(float (*win)[NV], int* at) const {
    int64_t t = t0;
    int slot = W - 2;                                  // of the incoming state
#pragma unroll
    for (int j = W - 2; j >= 0; --j) {
      if (t > 0) t = kMask ? token_before(mask, t) : t - 1;
      else t = -1;
      if (t >= 0) {
        load_row<T, NV>(x + t * p.x_t, n, wide, win[j]);
        at[j] = (int)t;
      } else {
        if (p.state_in) load_row<T, NV, false>(static_cast<const T*>(p.state_in) + ((size_t)b * (W - 1) + slot) * p.D + c0, n, wide, win[j]);
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
  const ConvThread<T, NV, W, kMask> th(a);
  const rfa_causal_conv_t& p = a.p;
  if (th.t0 >= p.T) return;
  const bool last = th.t1 == p.T && a.state_out;
  const int64_t out_t = (int64_t)p.B * p.D;
  const int count = (int)(th.t1 - th.t0);
  const uint32_t there = th.tokens();
  const T* from = th.x + th.t0 * p.x_t;
  T* to = static_cast<T*>(a.y) + (int64_t)th.b * p.D + th.c0 + th.t0 * out_t;
  float win[W - 1 + kConvFlight][NV];
  if (there || last) {                                 // (a run of padding has no window to look for)
    int at[W];
    th.before(win, at);
  }
  const auto put = [&](int first, T* out_at) {         // one output, from the window that begins at `first`
    float v[NV];
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      v[c] = th.bias[c];
#pragma unroll
      for (int j = 0; j < W; ++j) v[c] = fmaf(th.w[j][c], win[first + j][c], v[c]);
    }
    if (p.silu) {
#pragma unroll
      for (int c = 0; c < NV; ++c) v[c] *= sigmoid(v[c]);
    }
    Raw<T, NV> out;
#pragma unroll
    for (int c = 0; c < NV; c += 2) out.set2(c / 2, v[c], v[c + 1]);
    out.store(out_at, th.n, th.wide);
  };
  const auto move = [&](int by) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
#pragma unroll
      for (int c = 0; c < NV; ++c) win[j][c] = win[j + by][c];
  };
  Raw<T, NV> raw[kConvFlight];
  const auto ask = [&](const T* at) {
#pragma unroll
    for (int k = 0; k < kConvFlight; ++k, at += p.x_t) raw[k].load(at, th.n, th.wide);
  };
  const auto four = [&](int i) { return kMask ? four_there(there, i) : i + kConvFlight <= count; };
  bool on_way = false;
  for (int i = 0; i < count;) {
    if (four(i)) {                                     // four tokens together, the next four on the way
      if (!on_way) ask(from);
      from += kConvFlight * p.x_t;
#pragma unroll
      for (int k = 0; k < kConvFlight; ++k)
#pragma unroll
        for (int c = 0; c < NV; ++c) win[W - 1 + k][c] = raw[k].get(c);
      i += kConvFlight;
      on_way = four(i);
      if (on_way) ask(from);
#pragma unroll
      for (int k = 0; k < kConvFlight; ++k, to += out_t) put(k, to);
      move(kConvFlight);
    } else {
      if (!kMask || (there >> i & 1)) {
        load_row<T, NV>(from, th.n, th.wide, win[W - 1]);
        put(0, to);
        move(1);
      } else {
        Raw<T, NV> none;
        none.zero();
        none.store(to, th.n, th.wide);
      }
      ++i;
      from += p.x_t;
      to += out_t;
    }
  }
  if (last) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      Raw<T, NV> out;
      out.zero();
#pragma unroll
      for (int c = 0; c < NV; c += 2) out.set2(c / 2, win[j][c], win[j][c + 1]);
      out.store(static_cast<T*>(a.state_out) + ((size_t)th.b * (W - 1) + j) * p.D + th.c0, th.n, th.wide);
    }
  }
}

template <typename T, int NV, int W, bool kMask>
__global__ void __launch_bounds__(32 * kConvWarps) conv_bwd_kernel(const __grid_constant__ ConvArgs a) {
  __shared__ float red[kConvWarps][32 * NV + 1];
  const ConvThread<T, NV, W, kMask> th(a);
  const rfa_causal_conv_t& p = a.p;
  const int64_t out_t = (int64_t)p.B * p.D;
  const T* g = static_cast<const T*>(a.g) + (int64_t)th.b * a.g_b + th.c0;
  T* gx = static_cast<T*>(a.gx) + (int64_t)th.b * p.D + th.c0;
  float dw[W][NV] = {}, db[NV] = {};
  const int count = th.t0 < p.T ? (int)(th.t1 - th.t0) : 0;
  const uint32_t there = th.tokens();
  if (kMask)                                           // padded tokens' gradients
    for (int i = 0; i < count; ++i)
      if (!(there >> i & 1)) {
        Raw<T, NV> none;
        none.zero();
        none.store(gx + (th.t0 + i) * out_t, th.n, th.wide);
      }
  if (there || (count && th.t0 == 0 && a.g_state_in)) {      // a run of padding has nothing to do but the state's
    // The last W - 1 tokens and their gradients as far as they have come, oldest first; then those that are worked on.
    float win[W - 1 + kConvFlight][NV], pend[W - 1 + kConvFlight][NV];
    int at[W - 1 + kConvFlight];
    th.before(win, at);
#pragma unroll
    for (int j = 0; j < W - 1 + kConvFlight; ++j)
#pragma unroll
      for (int c = 0; c < NV; ++c) pend[j][c] = 0.f;
    const auto give = [&](int where, const float* v) {
      const bool mine = where >= th.t0 && where < th.t1, state = where < 0 && th.t0 == 0 && a.g_state_in;
      if (!mine && !state) return;
      Raw<T, NV> out;
#pragma unroll
      for (int c = 0; c < NV; c += 2) out.set2(c / 2, v[c], v[c + 1]);
      T* to = mine ? gx + (int64_t)where * out_t : static_cast<T*>(a.g_state_in) + ((size_t)th.b * (W - 1) + (W - 1 + where)) * p.D + th.c0;
      out.store(to, th.n, th.wide);
    };
    // the token whose window begins at `first`
    const auto work = [&](int first, const Raw<T, NV>& rx, const Raw<T, NV>& rg, bool own) {
      float gp[NV];
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        win[first + W - 1][c] = rx.get(c);
        gp[c] = rg.get(c);
      }
      if (p.silu) {
#pragma unroll
        for (int c = 0; c < NV; ++c) {
          float pre = th.bias[c];
#pragma unroll
          for (int j = 0; j < W; ++j) pre = fmaf(th.w[j][c], win[first + j][c], pre);
          const float sig = sigmoid(pre);
          gp[c] *= fmaf(pre * sig, 1.f - sig, sig);
        }
      }
#pragma unroll
      for (int c = 0; c < NV; ++c) {
#pragma unroll
        for (int j = 0; j < W; ++j) pend[first + j][c] = fmaf(th.w[j][c], gp[c], pend[first + j][c]);
        if (own) {
#pragma unroll
          for (int j = 0; j < W; ++j) dw[j][c] = fmaf(gp[c], win[first + j][c], dw[j][c]);
          db[c] += gp[c];
        }
      }
    };
    const auto move = [&](int by) {
#pragma unroll
      for (int j = 0; j < W - 1 + kConvFlight; ++j)
#pragma unroll
        for (int c = 0; c < NV; ++c) {
          if (j < W - 1) win[j][c] = win[j + by][c];
          pend[j][c] = j < W - 1 ? pend[j + by][c] : 0.f;
        }
    };
    // the oldest `by` tokens have passed
    const auto pass = [&](int by) {
#pragma unroll
      for (int k = 0; k < kConvFlight; ++k)
        if (k < by) give(at[k], pend[k]);
      move(by);
#pragma unroll
      for (int j = 0; j < W - 1; ++j) at[j] = at[j + by];
    };
    const T *from_x = th.x + th.t0 * p.x_t, *from_g = g + th.t0 * a.g_t;
    Raw<T, NV> rx[kConvFlight], rg[kConvFlight];
    const auto ask = [&](const T* at_x, const T* at_g) {
#pragma unroll
      for (int k = 0; k < kConvFlight; ++k, at_x += p.x_t, at_g += a.g_t) {
        rx[k].load(at_x, th.n, th.wide);
        rg[k].load(at_g, th.n, th.wide);
      }
    };
    const auto four = [&](int i) { return kMask ? four_there(there, i) : i + kConvFlight <= count; };
    bool on_way = false;
    for (int i = 0; i < count;) {
      if (four(i)) {                                   // four tokens together, the next four on the way
        if (!on_way) ask(from_x, from_g);
        Raw<T, NV> ux[kConvFlight], ug[kConvFlight];
#pragma unroll
        for (int k = 0; k < kConvFlight; ++k) { ux[k] = rx[k]; ug[k] = rg[k]; }
        from_x += kConvFlight * p.x_t;
        from_g += kConvFlight * a.g_t;
        on_way = four(i + kConvFlight);
        if (on_way) ask(from_x, from_g);
#pragma unroll
        for (int k = 0; k < kConvFlight; ++k) {
          at[W - 1 + k] = (int)th.t0 + i + k;
          work(k, ux[k], ug[k], true);
        }
        if (!kMask && i >= W - 1) {                    // four of the run's own, side by side
          T* to = gx + (th.t0 + i - (W - 1)) * out_t;
#pragma unroll
          for (int k = 0; k < kConvFlight; ++k, to += out_t) {
            Raw<T, NV> out;
#pragma unroll
            for (int c = 0; c < NV; c += 2) out.set2(c / 2, pend[k][c], pend[k][c + 1]);
            out.store(to, th.n, th.wide);
          }
          move(kConvFlight);
#pragma unroll
          for (int j = 0; j < W - 1; ++j) at[j] = at[j + kConvFlight];
        } else {
          pass(kConvFlight);
        }
        i += kConvFlight;
      } else {
        if (!kMask || (there >> i & 1)) {
          rx[0].load(from_x, th.n, th.wide);
          rg[0].load(from_g, th.n, th.wide);
          at[W - 1] = (int)th.t0 + i;
          work(0, rx[0], rg[0], true);
          pass(1);
        }
        ++i;
        from_x += p.x_t;
        from_g += a.g_t;
      }
    }
    // the tokens behind the run that its own still take part in
    int64_t behind[W];
    Raw<T, NV> bx[W], bg[W];
    int more = W - 1;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      const int64_t t = j ? behind[j - 1] + 1 : th.t1;
      behind[j] = kMask ? token_after(th.mask, t, p.T) : t;
      if (behind[j] < p.T) {
        bx[j].load(th.x + behind[j] * p.x_t, th.n, th.wide);
        bg[j].load(g + behind[j] * a.g_t, th.n, th.wide);
      }
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      if (behind[j] >= p.T) continue;
      --more;
      at[W - 1] = (int)behind[j];
      work(0, bx[j], bg[j], false);
      pass(1);
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
  const size_t part = (size_t)th.b * a.row_blocks + th.row_block;
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
      const int ch = th.ch_block * 32 * NV + i;
      if (ch >= p.D) continue;
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < kConvWarps; ++k) v += red[k][i];
      if (j < W) a.part_w[(part * p.D + ch) * W + j] = v;
      else a.part_b[part * p.D + ch] = v;
    }
  }
}

int conv_row_blocks(int64_t T) { return (int)((T + kConvWarps * kConvRun - 1) / (kConvWarps * kConvRun)); }

int conv_check(const rfa_causal_conv_t* p, const char* what) {
  RFA_REQUIRE(p, RFA_EINVAL, "%s: null argument", what);
  RFA_REQUIRE(p->x && p->weight, RFA_EINVAL, "%s: null pointer", what);
  RFA_REQUIRE(p->T > 0 && p->B > 0 && p->D > 0, RFA_EINVAL, "%s: empty or negative size", what);
  RFA_REQUIRE(p->dtype == RFA_F16 || p->dtype == RFA_F32 || p->dtype == RFA_BF16, RFA_EUNSUPPORTED, "%s: dtype %d", what, p->dtype);
  RFA_REQUIRE(p->W >= 1 && p->W <= kConvMax, RFA_EUNSUPPORTED, "%s: a window of %d tokens (1 to %d)", what, p->W, kConvMax);
  RFA_REQUIRE(p->T < ((int64_t)1 << 31) - 64 && p->B <= 65535 && p->D <= kMaxChannels && p->T / 128 * p->D < (int64_t)1 << 37, RFA_EUNSUPPORTED, "%s: T %lld, B %d, D %d", what,
              (long long)p->T, p->B, p->D);
  return 0;
}

template <typename T, int W, bool kMask> int conv_launch(const ConvArgs& a, bool backward, cudaStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.row_blocks * a.ch_blocks), a.p.B);
  if (backward) conv_bwd_kernel<T, kConvVec, W, kMask><<<grid, 32 * kConvWarps, 0, stream>>>(a);
  else conv_fwd_kernel<T, kConvVec, W, kMask><<<grid, 32 * kConvWarps, 0, stream>>>(a);
  return check_launch(backward ? "causal_conv_bwd" : "causal_conv_fwd");
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
  RFA_REQUIRE(y != conv->x, RFA_EINVAL, "causal_conv_fwd: y is x");      // other runs' warps read it
  ConvArgs a{};
  a.p = *conv;
  a.y = y; a.state_out = conv->W > 1 ? state_out : nullptr;
  const int size = conv->dtype == RFA_F32 ? 4 : 2, nv = kConvVec;
  a.row_blocks = conv_row_blocks(conv->T);
  a.ch_blocks = (conv->D + 32 * nv - 1) / (32 * nv);
  a.wide = wide_ok(conv->x, conv->x_t, conv->x_b, size, nv) && wide_ok(y, conv->D, 0, size, nv) && wide_ok(state_out, 0, 0, size, nv) &&
           wide_ok(conv->state_in, 0, 0, size, nv) && wide_ok(conv->bias, 0, 0, size, nv);
  a.wide_w = wide_ok(conv->weight, 0, 0, size, nv * conv->W);
  return conv_dtype(a, false, as_stream(stream));
}

extern "C" size_t rfa_causal_conv_workspace_bytes(int64_t T, int B, int D, int W) {
  using namespace rfa;
  if (T <= 0 || B <= 0 || D <= 0 || W < 1 || W > kConvMax) return 0;
  return (size_t)conv_row_blocks(T) * B * D * (W + 1) * 4;
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
  // other runs' warps read what these would overwrite
  RFA_REQUIRE(gx != g && gx != conv->x, RFA_EINVAL, "causal_conv_bwd: gx is g or x");
  RFA_REQUIRE(!g_state_in || (g_state_in != g_state && g_state_in != conv->state_in), RFA_EINVAL, "causal_conv_bwd: g_state_in is g_state or state_in");
  ConvArgs a{};
  a.p = *conv;
  a.g = g; a.g_t = g_t; a.g_b = g_b;
  a.gx = gx;
  if (conv->W > 1) { a.g_state = g_state; a.g_state_in = g_state_in; }
  const int parts = conv_row_blocks(conv->T) * conv->B;
  if (weights) {
    a.part_w = static_cast<float*>(workspace);
    a.part_b = a.part_w + (size_t)parts * conv->D * conv->W;
  }
  const int size = conv->dtype == RFA_F32 ? 4 : 2, nv = kConvVec;
  a.row_blocks = conv_row_blocks(conv->T);
  a.ch_blocks = (conv->D + 32 * nv - 1) / (32 * nv);
  a.wide = wide_ok(conv->x, conv->x_t, conv->x_b, size, nv) && wide_ok(g, g_t, g_b, size, nv) && wide_ok(gx, conv->D, 0, size, nv) &&
           wide_ok(conv->state_in, 0, 0, size, nv) && wide_ok(a.g_state, 0, 0, size, nv) && wide_ok(a.g_state_in, 0, 0, size, nv) &&
           wide_ok(conv->bias, 0, 0, size, nv);
  a.wide_w = wide_ok(conv->weight, 0, 0, size, nv * conv->W);
  if (int r = conv_dtype(a, true, as_stream(stream))) return r;
  const SumJob jobs[2] = {{a.part_w, g_weight, (int64_t)conv->D * conv->W, parts, conv->dtype}, {a.part_b, g_bias, conv->D, parts, conv->dtype}};
  return weights ? sum_parts(jobs, 2, as_stream(stream)) : 0;
}
