// Shared by the tensor-core kernels of sliding-window attention (window_tc.cu, window_bwd_tc.cu).
#pragma once

#include "tc_rows.cuh"
#include "window.cuh"

namespace rfa {

// Of keys or values as tiles of 64: the map that ends behind the first tokens, where tiles may lie in front of all windows and places are numbers; else the map of all.
inline int make_tmap_first(CUtensorMap* m, const CUtensorMap& all, const WindowArgs& a, const WindowRows& x) {
  *m = all;
  if (a.order || a.sinks <= 0 || a.sinks >= a.S || a.S <= a.window) return 0;
  return make_tmap_heads(m, x.p, a.dtype == RFA_BF16, a.sinks, a.B, a.G, a.D, x.t, x.b, x.h, 64);
}

#ifdef __CUDACC__
// The tiles of kTile keys that queries see: those of the first tokens, then from `first` on.
struct WindowSpan {
  int front, firsts, first, end;      // tiles [front, firsts) hold first tokens
  __device__ __forceinline__ int begin() const { return firsts > 0 ? front : first; }
  __device__ __forceinline__ int next(int kt) const { return kt + 1 < firsts ? kt + 1 : max(kt + 1, first); }
  __device__ __forceinline__ bool has(int kt) const { return kt < end && ((kt >= front && kt < firsts) || kt >= first); }
};
// of the 128 queries from row0 on, which stand at places at + row
template <int kTile = 128>
__device__ __forceinline__ WindowSpan window_span(const WindowNumbers& num, int64_t at, int64_t row0, int64_t T) {
  if (row0 >= T) return {0, 0, 0, 0};
  const int64_t end = num.last_key(at + row0, at + min(T, row0 + 128));
  if (end == 0) {      // no query is real: one tile, of which they see nothing
    const int own = (int)((at + row0) / kTile);
    return {own, 0, own, own + 1};
  }
  return {(int)(num.front() / kTile), (int)((num.first_end() + kTile - 1) / kTile), (int)(num.first_key(at + row0) / kTile), (int)((end + kTile - 1) / kTile)};
}
// scale (a - top), scale (b - top)
__device__ __forceinline__ float2 scaled_rest(float a, float b, float top, float scale) {
  float2 r;
  asm("{\n\t.reg .b64 v, f, t;\n\t"
      "mov.b64 v, {%2, %3};\n\tmov.b64 t, {%4, %4};\n\tmov.b64 f, {%5, %5};\n\t"
      "add.rn.f32x2 v, v, t;\n\tmul.rn.f32x2 v, v, f;\n\t"
      "mov.b64 {%0, %1}, v;\n\t}" : "=f"(r.x), "=f"(r.y) : "f"(a), "f"(b), "f"(-top), "f"(scale));
  return r;
}
// the lowest n bits
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
#endif

}  // namespace rfa
