// What the tensor-core kernels of decaying and windowed attention share beyond tc_common.cuh: tiles of rows with any strides, fp16 and bf16.
#pragma once

#include "state_space.cuh"
#include "tc_common.cuh"

namespace rfa {

// Rows [T][B][heads] of `width` adjacent 16-bit elements, strides in elements, as boxes of 64 columns by `box_rows` tokens of one (batch row, head) with the 128-byte
// swizzle; out of range reads as zero.
inline int make_tmap_heads(CUtensorMap* m, const void* base, bool bf16, int64_t T, int B, int heads, int width, int64_t s_t, int64_t s_b, int64_t s_h, uint32_t box_rows) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (!enc) return -1;
  static thread_local bool ctx_bound = false;      // see make_tmap_rows
  if (!ctx_bound) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return -2;
    ctx_bound = true;
  }
  const auto bytes = [&](int64_t n, int64_t stride) { return n > 1 ? (cuuint64_t)stride * 2 : (cuuint64_t)((width + 7) / 8) * 16; };      // one row: never stepped over
  cuuint64_t dims[4] = {(cuuint64_t)width, (cuuint64_t)heads, (cuuint64_t)B, (cuuint64_t)T};
  cuuint64_t strides[3] = {bytes(heads, s_h), bytes(B, s_b), bytes(T, s_t)};
  cuuint32_t box[4] = {64, 1, 1, box_rows}, estr[4] = {1, 1, 1, 1};
  CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)r;
}
// Whether a tensor map can describe them: 16-byte rows and steps, none of them backwards or zero.
inline bool tmap_rows_ok(const void* p, int64_t T, int B, int heads, int width, int64_t s_t, int64_t s_b, int64_t s_h) {
  const auto ok = [](int64_t n, int64_t s) { return n <= 1 || (s > 0 && s % 8 == 0 && s < ((int64_t)1 << 38)); };
  return aligned16(p) && width % 8 == 0 && ok(T, s_t) && ok(B, s_b) && ok(heads, s_h);
}

#ifdef __CUDACC__
// box of 64 columns from c0 on, of head h, batch row b, tokens from t on
__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int c0, int h, int b, int t) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(smem_dst)),
               "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(h), "r"(b), "r"(t)
               : "memory");
}
// untiled copies between 16-byte aligned places
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// the same towards L2 alone
__device__ __forceinline__ void tma_prefetch_4d(const CUtensorMap* m, int c0, int h, int b, int t) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global [%0, {%1, %2, %3, %4}];" ::"l"(reinterpret_cast<uint64_t>(m)), "r"(c0), "r"(h), "r"(b), "r"(t) : "memory");
}
__device__ __forceinline__ void bulk_prefetch(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, const void* smem_src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(smem_src)), "r"(bytes) : "memory");
}

// the instruction descriptor for fp16 or bf16 operands, fp32 accumulator
template <typename T>
__host__ __device__ constexpr uint32_t umma_idesc(int M, int N, bool a_mn_major, bool b_mn_major) {
  return umma_idesc_f16(M, N, a_mn_major, b_mn_major) | (std::is_same_v<T, __nv_bfloat16> ? (1u << 7) | (1u << 10) : 0u);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2h(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    return pack_half2(a, b);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack2h(uint32_t u) {
  if constexpr (std::is_same_v<T, __half>) return unpack_half2(u);
  else return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), RFA_TMEM_ST_REGS8(r, 0) : "memory");
}
// 16 fp32 numbers -> 32 bytes of a row of a global array that has `left` elements from here on (a multiple of 8)
template <typename T>
__device__ __forceinline__ void store_row16(T* p, const float* v, int left, bool wide) {
  uint32_t w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = pack2h<T>(v[2 * e], v[2 * e + 1]);
  if (wide && left >= 16) {      // a whole sector
    st_global_v8(p, w);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    if (left > 8) *reinterpret_cast<uint4*>(p + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
#endif

}  // namespace rfa
