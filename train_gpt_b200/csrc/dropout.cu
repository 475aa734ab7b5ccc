// Dropout from a counter-based generator, with the residual add behind it:
//
//     y = bf16(residual + keep x 65536 / (65536 - t)),   keep = (16 random bits >= t),   t = round(65536 p)
//
// The random bits of the eight elements 8 i .. 8 i + 7 are the four words of Philox4x32 with ten rounds (J. Salmon, M. Moraes, R. Dror,
// D. Shaw, Parallel random numbers: as easy as 1, 2, 3, 2011), of the counter (low word of i, high word of i, site, 0) and the seed as the
// key, the low half of each word before the high one.  So the mask is a function of seed, site and place: none is stored, and the backward
// pass makes it again (the same call on the gradient, without a residual).  Sixteen bits an element resolve p to 2^-17; the factor is that
// of the rounded p, so the expectation is the input's.  A dropped element is 0 whatever it was, infinities and NaN included.
//
// Bound by memory: 4 bytes an element, 6 with a residual.  A counter's ten rounds are 20 wide products and 20 three-way exclusive ors for
// eight elements, some 100 warp instructions with everything else, a third of what the SMs can issue meanwhile.
#include <math.h>

#include <algorithm>

#include "common.cuh"

namespace tg {

struct DropoutArgs {
  const __nv_bfloat16 *x, *residual;
  __nv_bfloat16* y;
  const int64_t* seed;
  uint32_t site, threshold;      // threshold <= 65535, in the high half of the word
  float scale;
  int64_t n;
};

__device__ __forceinline__ void philox(uint64_t piece, uint32_t site, uint32_t k0, uint32_t k1, uint32_t (&c)[4]) {
  c[0] = uint32_t(piece);
  c[1] = uint32_t(piece >> 32);
  c[2] = site;
  c[3] = 0u;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = uint64_t(c[0]) * 0xD2511F53u, b = uint64_t(c[2]) * 0xCD9E8D57u;
    c[0] = uint32_t(b >> 32) ^ c[1] ^ (k0 + uint32_t(i) * 0x9E3779B9u);
    c[1] = uint32_t(b);
    c[2] = uint32_t(a >> 32) ^ c[3] ^ (k1 + uint32_t(i) * 0xBB67AE85u);
    c[3] = uint32_t(a);
  }
}

// two elements of word w of the counter
template <bool RES>
__device__ __forceinline__ uint32_t drop2(uint32_t x, uint32_t res, uint32_t word, uint32_t threshold, float scale) {
  const float lo = (word << 16) >= threshold ? bf16lo(x) * scale : 0.f, hi = word >= threshold ? bf16hi(x) * scale : 0.f;
  return RES ? pack_bf16x2(lo + bf16lo(res), hi + bf16hi(res)) : pack_bf16x2(lo, hi);
}

constexpr int kDropThreads = 128;

// A thread has PIECES pieces of a block's contiguous part, all of them on their way before the first is worked on.
template <bool RES, int PIECES>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const DropoutArgs p) {
  grid_trigger();
  grid_wait();
  const uint64_t seed = uint64_t(*p.seed);
  const uint32_t k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
  const int64_t pieces = p.n / 8;
  constexpr int kChunk = kDropThreads * PIECES;
  const int64_t first = int64_t(blockIdx.x) * kChunk + threadIdx.x;
  for (int64_t at = first; at < pieces; at += int64_t(gridDim.x) * kChunk) {
    uint4 x[PIECES], r[PIECES];
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const int64_t i = at + u * kDropThreads;
      x[u] = r[u] = make_uint4(0u, 0u, 0u, 0u);
      if (i < pieces) {
        x[u] = ld_stream_v4(p.x + 8 * i);
        if (RES) r[u] = ld_stream_v4(p.residual + 8 * i);
      }
    }
#pragma unroll
    for (int u = 0; u < PIECES; ++u) {
      const int64_t i = at + u * kDropThreads;
      if (i >= pieces) break;
      uint32_t c[4];
      philox(uint64_t(i), p.site, k0, k1, c);
      uint4 o;
      o.x = drop2<RES>(x[u].x, r[u].x, c[0], p.threshold, p.scale);
      o.y = drop2<RES>(x[u].y, r[u].y, c[1], p.threshold, p.scale);
      o.z = drop2<RES>(x[u].z, r[u].z, c[2], p.threshold, p.scale);
      o.w = drop2<RES>(x[u].w, r[u].w, c[3], p.threshold, p.scale);
      *reinterpret_cast<uint4*>(p.y + 8 * i) = o;
    }
  }
  if (first == 0 && pieces * 8 < p.n) {      // the last, incomplete piece
    uint32_t c[4];
    philox(uint64_t(pieces), p.site, k0, k1, c);
    for (int64_t e = pieces * 8; e < p.n; ++e) {
      const int j = int(e & 7);
      const uint32_t word = j < 2 ? c[0] : j < 4 ? c[1] : j < 6 ? c[2] : c[3];
      const float v = ((j & 1) != 0 ? word : word << 16) >= p.threshold ? __bfloat162float(p.x[e]) * p.scale : 0.f;
      p.y[e] = __float2bfloat16_rn(RES ? v + __bfloat162float(p.residual[e]) : v);
    }
  }
}

}  // namespace tg

using namespace tg;

extern "C" int tg_dropout(const void* x, const void* residual, double p, const int64_t* seed, uint32_t site, void* y, int64_t n, void* stream) {
  if (n < 0 || !(p >= 0.0 && p <= 1.0)) return TG_ERR_SHAPE;
  if (n == 0) return TG_OK;
  if (x == nullptr || y == nullptr || seed == nullptr) return TG_ERR_SHAPE;
  if (!aligned16(x) || !aligned16(residual) || !aligned16(y) || (reinterpret_cast<uintptr_t>(seed) & 7u) != 0) return TG_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int threshold = int(nearbyint(p * 65536.0));
  if (threshold == 65536) {                  // nothing is kept
    if (residual == nullptr) TG_CUDA_CHECK(cudaMemsetAsync(y, 0, size_t(n) * 2, st));
    else if (residual != y) TG_CUDA_CHECK(cudaMemcpyAsync(y, residual, size_t(n) * 2, cudaMemcpyDeviceToDevice, st));
    return TG_OK;
  }
  using B = const __nv_bfloat16*;
  const DropoutArgs a = {B(x), B(residual), static_cast<__nv_bfloat16*>(y), seed, site, uint32_t(threshold) << 16,
                         float(65536.0 / double(65536 - threshold)), n};
  // Eight pieces a thread where every SM has some blocks of those, else one: 32768 x 1024 with a residual 34.1 us (two 37, sixteen 41),
  // 128 x 128 1.9 us (eight 2.7).
  const int64_t pieces = (n + 7) / 8, most = int64_t(1) << 30;
  const bool many = pieces >= int64_t(sm_count()) * 4 * kDropThreads * 8;
  const int64_t per_block = int64_t(kDropThreads) * (many ? 8 : 1);
  auto kern = residual != nullptr ? (many ? dropout_kernel<true, 8> : dropout_kernel<true, 1>) : (many ? dropout_kernel<false, 8> : dropout_kernel<false, 1>);
  TG_CUDA_CHECK(launch_early(kern, int(std::min(most, (pieces + per_block - 1) / per_block)), kDropThreads, 0, st, a));
  return TG_OK;
}
