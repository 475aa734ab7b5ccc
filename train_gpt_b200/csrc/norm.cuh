// What the norm kernels share: a row's sums, its pieces in shared memory, and the launches' shared-memory limit.
#pragma once

#include <atomic>

#include "common.cuh"

namespace tg {

// Sum of squares of the 8 bf16 values in w, as a balanced tree (keeps the rounding error of
// a row's variance at a few 2^-24 regardless of outliers).
__device__ __forceinline__ float sumsq8(const uint4& w) {
  const float2 v0 = bf16x2_unpack(w.x), v1 = bf16x2_unpack(w.y), v2 = bf16x2_unpack(w.z), v3 = bf16x2_unpack(w.w);
  const float2 t = __fadd2_rn(__ffma2_rn(v2, v2, __fmul2_rn(v0, v0)), __ffma2_rn(v3, v3, __fmul2_rn(v1, v1)));
  return t.x + t.y;
}

template <int N>
__device__ __forceinline__ float tree_sum(float (&v)[N]) {
#pragma unroll
  for (int stride = 1; stride < N; stride *= 2)
#pragma unroll
    for (int i = 0; i + stride < N; i += 2 * stride) v[i] += v[i + stride];
  return v[0];
}

// Sum over the lanes of a warp and, where a row has several, over its WPR warps in order.  `red` holds one float per warp of
// the block and alternates between two buffers from row to row: a warp writes one only after its group's barrier of the row
// before, which every warp of the group reaches after reading the other.
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* red, int warp, int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (WPR > 1) {
    if (lane == 0) red[warp] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / WPR), "n"(WPR * 32) : "memory");   // this row's warps only
    const int g0 = (warp / WPR) * WPR;
    v = red[g0];
#pragma unroll
    for (int i = 1; i < WPR; ++i) v += red[g0 + i];
  }
  return v;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

constexpr int pow2_at_least(int n) { return n <= 1 ? 1 : 2 * pow2_at_least((n + 1) / 2); }

// Dynamic shared memory of `bytes` for `kern`, once per device.
template <typename K>
static int allow_smem(K kern, int bytes, std::atomic<bool> (&done)[64]) {
  int dev = 0;
  TG_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return TG_ERR_SHAPE;
  if (!done[dev].load(std::memory_order_acquire)) {
    TG_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done[dev].store(true, std::memory_order_release);
  }
  return TG_OK;
}

}  // namespace tg
