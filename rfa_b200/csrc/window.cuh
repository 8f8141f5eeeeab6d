// Shared by the kernels of sliding-window attention (window.cu, window_tiles.cu, window_step.cu).
//
// Tokens are numbered within their sequence, padded ones not counted; token number n sees number m <= n where n - m < window or m < sinks.  Without
// padding and without a cache in front a token's number is its place.  Otherwise `order` holds it, or ~(the number of real tokens before) for a place that holds
// none, and `pos` the place of each number (S behind the last): both grow along the places, so that a tile's span of keys is two look-ups.
#pragma once

#include "state_space.cuh"

namespace rfa {

constexpr int kWindowMaxWidth = 256;

struct WindowRows {      // [T][B][heads] of D adjacent elements, strides in elements
  const void* p;
  int64_t t, b, h;
};
struct WindowArgs {
  WindowRows q, k, v, g, o;
  const int32_t *order, *pos;      // [B][S], [B][S + 1]; null: places are numbers
  void *out, *gq, *gk, *gv;        // contiguous
  float *lse, *delta;              // [B][H][T], in units of the exponential's base e; the backward's sum of g . out
  int64_t T, S;                    // queries, keys: query t stands at place S - T + t
  int B, H, G, D, window, sinks, dtype;
  float scale;
  float* parts;                    // [B][G][splits][min(sinks, T)][2][D]: what each part of the queries adds to gk and gv of the first tokens
  int splits;                      // 1: no parts
};

#ifdef __CUDACC__
// The reference of weights before a key has been seen: the lowest number, so that any finite score moves it, and not -inf, which taken from itself is no number.
constexpr float kLowest = -3.402823466e38f;
struct WindowNumbers {
  const int32_t *order, *pos;
  int64_t S;
  int window, sinks;
  __device__ __forceinline__ WindowNumbers(const WindowArgs& a, int b)
      : order(a.order ? a.order + b * a.S : nullptr), pos(a.pos ? a.pos + b * (a.S + 1) : nullptr), S(a.S), window(a.window), sinks(a.sinks) {}
  // the number at a place, negative where there is none
  __device__ __forceinline__ int at(int64_t s) const { return s < 0 || s >= S ? -1 : order ? order[s] : (int)s; }
  // of a key in a tile in front of all windows (`front`): there only first tokens count, and the rows beside them are cleared like those of padding -- a weight of nothing
  // times what is not finite is not nothing
  __device__ __forceinline__ int key_of_tile(int64_t s, bool front) const {
    const int n = at(s);
    return front && n >= sinks ? -1 : n;
  }
  __device__ __forceinline__ int64_t real_before(int64_t s) const { const int n = at(s); return n < 0 ? ~n : n; }      // 0 <= s < S
  __device__ __forceinline__ int64_t place(int64_t n) const { return n < 0 ? 0 : n >= S ? S : pos ? pos[n] : n; }
  __device__ __forceinline__ int64_t real_to(int64_t s) const { const int n = at(s); return n < 0 ? ~n : n + 1; }           // up to s, 0 <= s < S
  // queries at places [p0, p1) see keys from front() to first_end() and keys from first_key(p0) to last_key(p0, p1), 0 where no query is real
  __device__ __forceinline__ int64_t front() const { return place(0); }
  __device__ __forceinline__ int64_t first_key(int64_t p0) const { return place(max((int64_t)0, real_before(p0) - window + 1)); }
  __device__ __forceinline__ int64_t first_end() const { return sinks > 0 ? min(S, place(sinks - 1) + 1) : 0; }
  __device__ __forceinline__ int64_t last_key(int64_t p0, int64_t p1) const {
    if (!order) return p1;
    const int64_t n = real_to(p1 - 1);
    return n > real_before(p0) ? place(n - 1) + 1 : 0;
  }
  // A query that sees one key gives it the weight 1 whatever both are: its gradient is exactly 0, not the rounding of g . v - g . out; so is the gradient of a
  // key that only such queries see.  Factors for query number n and for any key of the sequence.
  __device__ __forceinline__ bool single() const { return window == 1 && sinks <= 0; }
  __device__ __forceinline__ float query_factor(int n) const { return n == 0 || single() ? 0.f : 1.f; }
  __device__ __forceinline__ float key_factor() const { return place(1) >= S || single() ? 0.f : 1.f; }
  // The first tokens' keys are seen by all queries behind, many times a window's.  Where `splits` > 1, what a tile of `rows` keys that holds some of them takes is
  // split: the queries up to near_query(), which is all for its other keys, and the rest of them in splits - 1 parts.  Of tiles from front() on this many are
  // split: all that hold first tokens, unless padding is among these; the ones behind then go through all their queries.
  __device__ __forceinline__ int first_tiles(int rows) const { return (int)((min((int64_t)sinks, S) + rows - 1) / rows) + (order ? 1 : 0); }
  __device__ __forceinline__ bool is_split(int64_t p0, int rows, int splits) const {
    const int64_t tile = p0 / rows - front() / rows;
    return splits > 1 && p0 < first_end() && tile >= 0 && tile < first_tiles(rows);
  }
  __device__ __forceinline__ int64_t near_query(int64_t p0, int64_t p1) const {
    if (!order) return min(S, p1 - 1 + window);
    if (real_to(p1 - 1) == real_before(p0)) return p0;
    return min(place(real_to(S - 1) - 1) + 1, place(real_before(p1 - 1) + window));
  }
  // keys at places [p0, p1) are seen by no query at or behind this place, p0 where no key is real
  __device__ __forceinline__ int64_t last_query(int64_t p0, int64_t p1) const {
    if (!order) return p0 < first_end() ? S : min(S, p1 - 1 + window);
    if (real_to(p1 - 1) == real_before(p0)) return p0;
    const int64_t end = place(real_to(S - 1) - 1) + 1;
    return p0 < first_end() ? end : min(end, place(real_before(p1 - 1) + window));
  }
};
__device__ __forceinline__ bool window_sees(int n, int m, int window, int sinks) { return m >= 0 && m <= n && (n - m < window || m < sinks); }
#endif

int launch_window_order(const uint8_t* mask, const int64_t* length, int cap, int32_t* order, int32_t* pos, int64_t T, int B, cudaStream_t stream);
int launch_window_fwd_tiles(const WindowArgs& a, cudaStream_t stream);        // window_tiles.cu: any sizes and types
int launch_window_bwd_tiles(const WindowArgs& a, cudaStream_t stream);
int launch_window_parts(const WindowArgs& a, int rows, float scale, cudaStream_t stream);      // the parts' sums, those of gk times scale, for tiles of `rows` keys
bool window_tc_ok(const WindowArgs& a);                                       // window_tc.cu: fp16 and bf16, heads of up to 128 in rows that a tensor map can describe
int launch_window_fwd_tc(const WindowArgs& a, cudaStream_t stream);
int launch_window_bwd_tc(const WindowArgs& a, const uint8_t* mask, cudaStream_t stream);      // window_bwd_tc.cu
int launch_window_step(const rfa_window_t& c, void* cache_k, void* cache_v, int64_t* length, void* out, cudaStream_t stream);      // window_step.cu
// the cache in front of the new tokens, in the order of their numbers and then themselves: [cap + T][B][G][D]; and back
int launch_window_gather(const rfa_window_t& c, const void* cache_k, const void* cache_v, const int64_t* length, void* keys, void* values, cudaStream_t stream);
int launch_window_keep(const rfa_window_t& c, void* cache_k, void* cache_v, int64_t* length, const int32_t* order, bool empty, cudaStream_t stream);

}  // namespace rfa
