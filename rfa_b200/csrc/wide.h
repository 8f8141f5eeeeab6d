// Which runs of elements may be taken in wide accesses: the host's decision and the kernels' accesses (state_space.cuh) from one rule.
#pragma once

#include <cstdint>

namespace rfa {

// Bytes of the accesses that a run of `bytes` adjacent bytes is taken in: the largest power of two that divides it, at most 16.
constexpr int access_bytes(int bytes) {
  const int low = bytes & -bytes;
  return low < 16 ? low : 16;
}

// Whether runs of nv elements at p, p + stride ... may be taken so.
inline bool wide_ok(const void* p, int64_t stride, int64_t stride2, int size, int nv) {
  const int64_t bytes = access_bytes(nv * size);
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * size % bytes == 0 && stride2 * size % bytes == 0;
}

}  // namespace rfa
