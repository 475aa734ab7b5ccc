// The gated feed-forward's first half in bf16,
//
//     h = act(x Wg) * (x Wu)            x [M, D], Wg and Wu [D, F]; act silu, gelu (by erf) or relu
//
// as one kernel: both projections, the activation and the product.  Backward, for the gradient g of h, with G = x Wg and U = x Wu:
//
//     dG = g U act'(G),  dU = g act(G),    dx = dG Wg^T + dU Wu^T,    dWg = x^T dG,  dWu = x^T dU
//
// one pass for dG and dU, in bf16 (of small problems as the sum of two), and one launch for the three products.  Products are bf16 tcgen05.mma on pairs of SMs (cta_group::2) with float32
// accumulators in tensor memory; no operand is transposed in memory, the descriptors carry the major-ness.  A cluster of two CTAs has a
// tile of 256 rows and 256 accumulator columns: CTA r owns rows 128 r.. of it and loads them of A, and half of the 256 rows of B.
//   forward   A = x, B: the first CTA loads 128 columns of Wg, the second the same of Wu.  Accumulator columns 0-127 are then G and 128-255
//             are U of the same 128 columns of h, and a thread of the epilogue finds both of an element in its own tensor-memory lane.
//   dx        A = dG and then dU, B = Wg and then Wu: one contraction of 2 F, so the sum of the two products is made in the accumulator.
//   dW        A = x^T, B = dG for the first half of the column tiles and dU for the second.
// dx and dW do not depend on one another: one launch, the problem with the longer items first, pairs that its last round leaves idle
// begin with the other one.
//
// What the forward pass keeps for the backward one is G and U in 16 bits.  bf16 there would cost dx and dW half as much precision again as
// the rounding of dG and dU (which the tensor cores need) does: fp16 has three more bits, and a power of two per 64 columns of a row
// (a byte each) that puts the largest of them below 2^15 makes up for its range: half a step is 2^-11 of a value, but 2^-39 of the largest (finite)
// of its 64 at least, so that values below 2^-28 of that one have fewer bits than 11, and what is below 2^-40 of it is kept as 0.
//
// Warp roles of a CTA (320 threads): 0-7 epilogue (warp w reads TMEM lanes 32 (w % 4).., half w / 4 of the columns), 8 TMA producer,
// 9 MMA issuer (in the first CTA).  Two accumulators take turns, so a tile's epilogue runs beside the next tile's products; results leave
// through swizzled staging rows and bulk tensor stores, which also clip ragged edges.  Ragged operands arrive as zeros.
//
// Every wait on an mbarrier is bounded, as in gemm_fp8.cu (the same codes).
#include <cuda.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "cluster.cuh"
#include "common.cuh"
#include "gemm_tiles.cuh"
#include "host_api.h"
#include "mbarrier.cuh"
#include "norm.cuh"
#include "umma.cuh"

namespace tg {

// ---- activations ---------------------------------------------------------------------------------------------------

// Phi(-a) = exp(-a^2 / 2) t R(t) with t = 1 / (1 + 0.3 a): erfc scaled by its exponential is smooth in t, and R is a polynomial fitted to it for
// a in [0, 14.5] by least squares of the relative error at Chebyshev points, reweighted towards the largest (1.6e-7; 4e-7 in float32).
// Relative, unlike the quantiser's: a product with U may have any size.
__device__ __forceinline__ float gated_phi(float g, float e) {      // e = exp(-g^2 / 2)
  const float t = __fdividef(1.f, fmaf(0.3f, fabsf(g), 1.f));
  float r = 0.03542373329401016f;
  r = fmaf(r, t, -0.156158447265625f);
  r = fmaf(r, t, 0.20455677807331085f);
  r = fmaf(r, t, -0.05203401297330856f);
  r = fmaf(r, t, 0.12769177556037903f);
  r = fmaf(r, t, 0.10017594695091248f);
  r = fmaf(r, t, 0.12071213871240616f);
  r = fmaf(r, t, 0.11963200569152832f);
  const float tail = e * t * r;
  return g > 0.f ? 1.f - tail : tail;
}
template <int ACT>
__device__ __forceinline__ float gated_act(float g) {
  if constexpr (ACT == TG_GATED_SILU) return __fdividef(g, 1.f + __expf(-g));
  if constexpr (ACT == TG_GATED_GELU) return g * gated_phi(g, __expf(-0.5f * g * g));
  return g > 0.f || g != g ? g : 0.f;
}
// act(g) and its derivative
template <int ACT>
__device__ __forceinline__ float2 gated_act_slope(float g) {
  if constexpr (ACT == TG_GATED_SILU) {
    const float s = __fdividef(1.f, 1.f + __expf(-g)), a = g * s;
    return make_float2(a, s * (1.f + g * (1.f - s)));
  }
  if constexpr (ACT == TG_GATED_GELU) {
    const float e = __expf(-0.5f * g * g), phi = gated_phi(g, e);
    return make_float2(g * phi, fmaf(0.3989422804014327f * g, e, phi));
  }
  return make_float2(g > 0.f || g != g ? g : 0.f, g > 0.f ? 1.f : 0.f);
}

// ---- the products --------------------------------------------------------------------------------------------------

constexpr int kGbK = 64;                        // contraction of a stage: 128 bytes of bf16
constexpr int kGbBox = 64 * 128;                // bytes of an operand box: 64 rows of 128 bytes
constexpr int kGbStage = 4 * kGbBox;            // a CTA's: two boxes of A, two of B
constexpr int kGbWarps = 8, kGbThreads = 32 * (kGbWarps + 2);
constexpr int kGbOutBox = 32 * 128;             // bytes of an output box: 32 rows of 64 columns
constexpr int kGbBand = 8;                      // 256-row tiles per band of the tile numbering
enum { kGbForward = 0, kGbData = 1, kGbWeights = 2 };

// A problem of either kernel.  Operand maps have boxes of 64 x 64, output maps of 64 columns x 32 rows.
struct GatedProblem {
  CUtensorMap a[2], b[2], d[2];
  int kind, tiles_m, tiles_n, blocks;           // blocks: stages of the contraction of a tile
  int half;                                     // kGbData: its first stage that reads the second operands; kGbWeights: column tiles of dWg
  // dG and dU may have a second piece (see gated_slopes_kernel), `low` rows behind the first: stages from `piece` on read that one.
  int piece, low;
  // The contraction may be cut into ranges: item i is tile i % tiles of range i / tiles, and its float32 sums go to `partial`, 256 KB an item,
  // in the order in which the epilogue's threads hold them (see gated_join_kernel).
  int ranges;
  float4* partial;
};
struct GatedSaved {
  CUtensorMap gate, up;
  uint8_t* exponents;
  int64_t rows;
  int chunks;                                   // of 64 columns
};

__device__ __forceinline__ void gated_place(int tiles_m, int tiles_n, int tile, int& tm, int& tn) {
  const int per_band = kGbBand * tiles_n, b = tile / per_band, w = tile - b * per_band, rows = min(kGbBand, tiles_m - b * kGbBand);
  tn = w / rows;
  tm = b * kGbBand + (w - tn * rows);
}
// item -> tile, and the stages of its range
__device__ __forceinline__ void gated_tile(const GatedProblem& p, int item, int& tm, int& tn, int& first, int& last) {
  first = 0;
  last = p.blocks;
  if (p.ranges > 1) {
    const int tiles = p.tiles_m * p.tiles_n, range = item / tiles;
    item -= range * tiles;
    first = int(int64_t(p.blocks) * range / p.ranges);
    last = int(int64_t(p.blocks) * (range + 1) / p.ranges);
  }
  gated_place(p.tiles_m, p.tiles_n, item, tm, tn);
}

__device__ __forceinline__ void umma_bf16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(x), "r"(y)
               : "memory");
}
// As make_smem_desc: 128-byte swizzle, 8-row groups 1024 bytes apart.  MN-major operands lie in chunks of 64 rows or columns, a box each.
__device__ __forceinline__ uint64_t gated_desc(uint32_t saddr) {
  return uint64_t((saddr >> 4) & 0x3FFFu) | uint64_t(kGbBox >> 4) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// The running maximum of magnitudes by a float's bits: without the sign, and a step of the exponent up, which takes infinities and NaN past 2^32,
// below every finite value.
__device__ __forceinline__ uint32_t max_magnitude(uint32_t m, uint32_t bits) { return max(m, 2u * bits + 0x01000000u); }

// Sixteen bytes of this lane's staging row: chunk c of its 128 bytes, swizzled
__device__ __forceinline__ void stage16(uint32_t row, int lane, int c, uint4 v) { sts128(row + (uint32_t(c ^ (lane & 7)) << 4), v); }

template <int BUFS>
struct GatedCfg {
  static constexpr int bufs = BUFS;             // output boxes of a warp
  static constexpr int out_bytes = kGbWarps * BUFS * kGbOutBox;
  static constexpr int stages_fit = (kSmemLimit - 1024 - out_bytes) / kGbStage;
  static constexpr int stages = stages_fit > 6 ? 6 : stages_fit;
  static constexpr int smem_bytes = stages * kGbStage + out_bytes;
  static_assert(stages >= 4 && smem_bytes + 1024 <= kSmemLimit, "shared-memory plan");
};

// What a row's 64 values are scaled by to be kept, from max_magnitude over them: the power of two that puts the largest finite one into [2^14, 2^15), up or
// down (2^126 at most, for values below 2^-112 and a row of zeros).  Returns the exponent field of the float that undoes it.
__device__ __forceinline__ uint32_t save_exponent(uint32_t m, float& scale) {
  const uint32_t e = max(m >> 24, 16u);          // the largest's exponent field, and one
  scale = __uint_as_float((269u - e) << 23);
  return e - 15u;
}
__device__ __forceinline__ float saved_scale(uint32_t field) { return __uint_as_float(field << 23); }
// relu's gate (POSITIVE): what is above 0 stays so, since the slope goes by that
template <bool POSITIVE>
__device__ __forceinline__ float save_scaled(float v, float scale) {
  return POSITIVE && v > 0.f ? fmaxf(v * scale, 0x1p-24f) : v * scale;
}
// f16 of 64 accumulator values, scaled; returns the exponent field
template <bool POSITIVE>
__device__ __forceinline__ uint32_t save_row(const uint32_t (&v0)[32], const uint32_t (&v1)[32], uint32_t row, int lane) {
  uint32_t m = 0u;
#pragma unroll
  for (int j = 0; j < 32; ++j) m = max_magnitude(max_magnitude(m, v0[j]), v1[j]);
  float scale;
  const uint32_t e = save_exponent(m, scale);
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = 8 * c + 2 * j;
      const float lo = __uint_as_float(at < 32 ? v0[at & 31] : v1[at & 31]), hi = __uint_as_float(at < 32 ? v0[(at + 1) & 31] : v1[(at + 1) & 31]);
      o[j] = pack_f16x2(save_scaled<POSITIVE>(lo, scale), save_scaled<POSITIVE>(hi, scale));
    }
    stage16(row, lane, c, make_uint4(o[0], o[1], o[2], o[3]));
  }
  return e;
}

// `one` and, where two is set, `two` with the walk that walk_second gives.
template <int KIND, int ACT, bool SAVE, typename C>
__device__ __forceinline__ void gated_body(const GatedProblem& one, const GatedProblem& two, bool both, int rounds, const GatedSaved& saved, unsigned* status) {
  constexpr int kStages = C::stages;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(16) uint64_t ctl_bars[2 * kStages + 5];
  __shared__ uint32_t ctl_tmem_ptr;
  __shared__ int ctl_abort;
  const uint32_t sbase = smem_u32(smem);
  const uint32_t full0 = smem_u32(ctl_bars), empty0 = full0 + 8u * kStages, tfull0 = empty0 + 8u * kStages, tempty0 = tfull0 + 16u, drain_bar = tempty0 + 16u;
  volatile uint32_t* tmem_ptr_smem = &ctl_tmem_ptr;
  volatile int* abort_flag = &ctl_abort;
  if ((sbase & 1023u) != 0) {   // the swizzled layouts need this alignment (both CTAs have the same layout)
    if (threadIdx.x == 0 && status != nullptr) atomicCAS(status, 0u, 6u);
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int unit = int(blockIdx.x) / 2, units = int(gridDim.x) / 2;
  const int n1 = one.tiles_m * one.tiles_n * one.ranges;
  const Walk walk1 = walk_alone(unit, units, n1);
  const Walk walk2 = both ? walk_second(unit, units, n1, two.tiles_m * two.tiles_n * two.ranges, rounds) : Walk{0, 0, 0, 1, 0};

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full0 + 8u * s, 1);             // (the first CTA's counts the bytes of both)
      mbar_init(empty0 + 8u * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull0 + 8u * b, 1);
      mbar_init(tempty0 + 8u * b, 2 * kGbWarps);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kGbWarps + 1) tmem_take_pair(smem_u32(&ctl_tmem_ptr));
  tc_fence_before();
  cluster_sync();                               // both CTAs' barriers exist before either signals across, both have their tensor memory
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr_smem;
  grid_trigger();
  grid_wait();

  if (warp == kGbWarps) {
    // ------------------------------ TMA producer -------------------------------------
    uint32_t s = 0, ph = 1;
    bool ok = true;
    const uint32_t full_leader = map_rank(full0, 0u);
    auto produce = [&](const GatedProblem& p, const Walk& w) {
      for (int item = w.first; ok && item < w.n; item = w.next(item)) {
        int tm, tn, first, last;
        gated_tile(p, item, tm, tn, first, last);
        const int m0 = (2 * tm + int(rank)) * 128;
        for (int kb = first; kb < last; ++kb) {
          ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8u * s, ph, abort_flag, status, 1u));
          if (!ok) break;
          if (elect_one()) {
            const uint32_t dst = sbase + s * kGbStage, fb = full_leader + 8u * s;
            // The first CTA announces the bytes of both.  The second's may land before that: its barrier phase is the same one,
            // since the stage was free in both CTAs only after the phase before had completed.
            if (rank == 0) mbar_expect_tx(full0 + 8u * s, 2 * kGbStage);
            if constexpr (KIND == kGbForward) {
              const int k0 = kb * kGbK, n0 = tn * 128;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                tma_load_2d_pair(dst + i * kGbBox, &p.a[0], fb, k0, m0 + 64 * i);
                tma_load_2d_pair(dst + (2 + i) * kGbBox, &p.b[rank], fb, n0 + 64 * i, k0);
              }
            } else if (p.kind == kGbData) {
              const bool second = kb >= p.piece;
              const int stage = kb - (second ? p.piece : 0), sel = stage >= p.half, k0 = (stage - (sel ? p.half : 0)) * kGbK, n0 = tn * 256 + int(rank) * 128;
              const int a0 = m0 + (second ? p.low : 0);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                tma_load_2d_pair(dst + i * kGbBox, &p.a[sel], fb, k0, a0 + 64 * i);
                tma_load_2d_pair(dst + (2 + i) * kGbBox, &p.b[sel], fb, k0, n0 + 64 * i);
              }
            } else {
              const bool second = kb >= p.piece;
              const int sel = tn >= p.half, k0 = (kb - (second ? p.piece : 0)) * kGbK, n0 = (tn - (sel ? p.half : 0)) * 256 + int(rank) * 128;
              const int b0 = k0 + (second ? p.low : 0);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                tma_load_2d_pair(dst + i * kGbBox, &p.a[0], fb, m0 + 64 * i, k0);
                tma_load_2d_pair(dst + (2 + i) * kGbBox, &p.b[sel], fb, n0 + 64 * i, b0);
              }
            }
          }
          __syncwarp();
          if (++s == kStages) { s = 0; ph ^= 1u; }
        }
      }
    };
    produce(one, walk1);
    if (KIND != kGbForward && both) produce(two, walk2);
  } else if (warp == kGbWarps + 1) {
    // ------------------------------ MMA issuer (first CTA) ----------------------------
    if (rank == 0) {
      const uint64_t desc_a0 = gated_desc(sbase), desc_b0 = gated_desc(sbase + 2 * kGbBox);
      const uint32_t desc_hi = uint32_t(desc_a0 >> 32), a_lo0 = uint32_t(desc_a0), b_lo0 = uint32_t(desc_b0);
      bool ok = true;
      uint32_t s = 0, sph = 0, buf = 0, bph = 1;
      auto issue = [&](const GatedProblem& p, const Walk& w) {
        const int kind = KIND == kGbForward ? kGbForward : p.kind;
        const uint32_t a_mn = kind == kGbWeights, b_mn = kind != kGbData;
        // D f32 (bit 4), A and B bf16 (7, 10), major bits 15/16, N>>3 at 17, M>>4 at 24
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (a_mn << 15) | (b_mn << 16) | (uint32_t(256 >> 3) << 17) | (uint32_t(256 >> 4) << 24);
        // descriptor step per 16 of the contraction: 32 bytes along a K-major row, 16 rows of 128 bytes otherwise
        const uint32_t a_step = a_mn ? 128u : 2u, b_step = b_mn ? 128u : 2u;
        for (int item = w.first; ok && item < w.n; item = w.next(item)) {
          int tm, tn, first, last;
          gated_tile(p, item, tm, tn, first, last);
          for (int kb = first; kb < last; ++kb) {
            ok = __all_sync(0xffffffffu, (kb > first || mbar_wait(tempty0 + 8u * buf, bph, abort_flag, status, 2u)) &&
                                             mbar_wait(full0 + 8u * s, sph, abort_flag, status, 3u));
            if (!ok) break;
            __syncwarp();
            tc_fence_after();
            if (elect_one()) {
              const uint32_t soff = s * uint32_t(kGbStage >> 4);
#pragma unroll
              for (int k = 0; k < kGbK / 16; ++k)
                umma_bf16_pair(tmem_base + buf * 256u, (uint64_t(desc_hi) << 32) | (a_lo0 + soff + k * a_step),
                               (uint64_t(desc_hi) << 32) | (b_lo0 + soff + k * b_step), idesc, kb > first || k > 0 ? 1u : 0u);
              umma_commit_both(empty0 + 8u * s);
              if (kb + 1 == last) umma_commit_both(tfull0 + 8u * buf);
            }
            __syncwarp();
            if (++s == kStages) { s = 0; sph ^= 1u; }
          }
          if ((buf ^= 1u) == 0u) bph ^= 1u;
        }
      };
      issue(one, walk1);
      if (KIND != kGbForward && both) issue(two, walk2);
      // nothing issued here may still be running when tensor memory is freed
      if (elect_one()) {
        umma_commit_here(drain_bar);
        mbar_wait(drain_bar, 0u, abort_flag, status, 4u);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------ epilogue ------------------------------------------
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t lanes = tmem_base + (uint32_t(quarter * 32) << 16);
    const uint32_t out = sbase + kStages * kGbStage + uint32_t(warp) * (C::bufs * kGbOutBox), row = out + uint32_t(lane) * 128u;
    const uint32_t tempty_leader = map_rank(tempty0, 0u), is_lane0 = lane == 0;
    uint32_t buf = 0, bph = 0;
    bool ok = true;
    auto release = [&]() {
      tc_fence_before();
      __syncwarp();
      mbar_arrive_cluster_if(tempty_leader + 8u * buf, is_lane0);
    };
    auto rows_free = [&]() {            // the stores before have read their staging rows
      if (is_lane0) tma_store_wait_read();
      __syncwarp();
    };
    auto staged = [&]() {               // generic writes -> visible to the copy engine
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    };
    auto finish = [&](const GatedProblem& p, const Walk& w) {
      for (int item = w.first; item < w.n; item = w.next(item)) {
        int tm, tn, first, last;
        gated_tile(p, item, tm, tn, first, last);
        const int m0 = (2 * tm + int(rank)) * 128 + quarter * 32;
        ok = __all_sync(0xffffffffu, mbar_wait(tfull0 + 8u * buf, bph, abort_flag, status, 5u));
        if (!ok) break;
        __syncwarp();
        tc_fence_after();
        if constexpr (KIND == kGbForward) {
          const uint32_t at = lanes + buf * 256u + uint32_t(half) * 64u;
          uint32_t g0[32], g1[32], u0[32], u1[32];
          tmem_ld32(at, g0);
          tmem_ld32(at + 32u, g1);
          tmem_ld32(at + 128u, u0);
          tmem_ld32(at + 160u, u1);
          tmem_wait_ld(g0);
          tmem_wait_ld(g1);
          tmem_wait_ld(u0);
          tmem_wait_ld(u1);
          release();
          rows_free();
          const int n0 = tn * 128 + half * 64;
          if constexpr (SAVE) {
            // one staging box for the gate's, the up-projection's and the result's rows in turn: with three, four stages were left for the operands
            // (32768 x 1024 -> 4096 with its backward pass 1352 us, 1332 so)
            auto send = [&](const CUtensorMap* map) {
              staged();
              if (is_lane0) {
                tma_store_2d(map, out, n0, m0);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
              }
              rows_free();
            };
            const uint32_t eg = save_row<ACT == TG_GATED_RELU>(g0, g1, row, lane);
            send(&saved.gate);
            const uint32_t eu = save_row<false>(u0, u1, row, lane);
            send(&saved.up);
            if (m0 + lane < saved.rows && n0 / 64 < saved.chunks)
              reinterpret_cast<uint16_t*>(saved.exponents)[int64_t(n0 / 64) * saved.rows + m0 + lane] = uint16_t(eg | eu << 8);
          }
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int i = 8 * (c & 3) + 2 * j;
              const uint32_t(&g)[32] = c < 4 ? g0 : g1;
              const uint32_t(&u)[32] = c < 4 ? u0 : u1;
              o[j] = pack_bf16x2(gated_act<ACT>(__uint_as_float(g[i])) * __uint_as_float(u[i]),
                                 gated_act<ACT>(__uint_as_float(g[i + 1])) * __uint_as_float(u[i + 1]));
            }
            stage16(row, lane, c, make_uint4(o[0], o[1], o[2], o[3]));
          }
          staged();
          if (is_lane0) {
            tma_store_2d(&p.d[0], out, n0, m0);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          __syncwarp();
        } else {
          const int sel = p.kind == kGbWeights && tn >= p.half, n0 = (tn - (sel ? p.half : 0)) * 256 + half * 128;
          const uint32_t at = lanes + buf * 256u + uint32_t(half) * 128u;
          if (p.ranges > 1) {           // four columns a lane, a warp's rows side by side
            float4* to = p.partial + ((int64_t(item) * 2 + rank) * kGbWarps + warp) * 1024 + lane;
#pragma unroll
            for (int piece = 0; piece < 4; ++piece) {
              uint32_t v[32];
              tmem_ld32(at + 32u * piece, v);
              tmem_wait_ld(v);
              if (piece == 3) release();
#pragma unroll
              for (int j = 0; j < 8; ++j)
                to[(8 * piece + j) * 32] = make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]), __uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3]));
            }
            if ((buf ^= 1u) == 0u) bph ^= 1u;
            continue;
          }
          rows_free();
#pragma unroll
          for (int box = 0; box < 2; ++box) {
            uint32_t v0[32], v1[32];
            tmem_ld32(at + 64u * box, v0);
            tmem_ld32(at + 64u * box + 32u, v1);
            tmem_wait_ld(v0);
            tmem_wait_ld(v1);
            if (box == 1) release();
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              uint32_t o[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int i = 8 * (c & 3) + 2 * j;
                const uint32_t(&v)[32] = c < 4 ? v0 : v1;
                o[j] = pack_bf16x2(__uint_as_float(v[i]), __uint_as_float(v[i + 1]));
              }
              stage16(row + box * kGbOutBox, lane, c, make_uint4(o[0], o[1], o[2], o[3]));
            }
          }
          staged();
          if (is_lane0) {
#pragma unroll
            for (int box = 0; box < 2; ++box) tma_store_2d(&p.d[sel], out + box * kGbOutBox, n0 + 64 * box, m0);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          __syncwarp();
        }
        if ((buf ^= 1u) == 0u) bph ^= 1u;
      }
    };
    finish(one, walk1);
    if (KIND != kGbForward && both && ok) finish(two, walk2);
    // the last bulk stores must have read their staging rows before the CTA's shared memory goes away
    if (is_lane0) tma_store_wait_read();
    __syncwarp();
  }

  // ------------------------------ teardown ----------------------------------------------
  __syncwarp();
  tc_fence_before();
  cluster_sync();              // the partner no longer reads this CTA's shared memory or signals its barriers
  if (warp == kGbWarps + 1) {
    __syncwarp();
    tc_fence_after();
    tmem_give_pair(tmem_base);
  }
}

template <int ACT, bool SAVE>
__global__ void __launch_bounds__(kGbThreads, 1) gated_fwd_kernel(const __grid_constant__ GatedProblem p, const __grid_constant__ GatedSaved saved, unsigned* status) {
  gated_body<kGbForward, ACT, SAVE, GatedCfg<1>>(p, p, false, 0, saved, status);
}
__global__ void __launch_bounds__(kGbThreads, 1)
gated_bwd_kernel(const __grid_constant__ GatedProblem one, const __grid_constant__ GatedProblem two, int both, int rounds, unsigned* status) {
  gated_body<kGbData, 0, false, GatedCfg<2>>(one, two, both != 0, rounds, GatedSaved{}, status);
}

// The ranges of a problem that was cut, added up in order.  A warp has eight columns of the 32 rows of an epilogue's warp at a time.
struct GatedJoin {
  const float4* partial;
  __nv_bfloat16* d[2];
  int kind, tiles_m, tiles_n, half, ranges;
  int64_t rows, cols;                           // of a result; its pitch is cols
};
__global__ void __launch_bounds__(256) gated_join_kernel(const __grid_constant__ GatedJoin a, const __grid_constant__ GatedJoin b, int blocks_a) {
  grid_trigger();
  grid_wait();
  const bool second = int(blockIdx.x) >= blocks_a;
  const GatedJoin& p = second ? b : a;
  const int lane = threadIdx.x & 31;
  const int64_t unit = int64_t(int(blockIdx.x) - (second ? blocks_a : 0)) * 8 + (threadIdx.x >> 5);      // (tile, CTA, warp, eight columns)
  const int tiles = p.tiles_m * p.tiles_n, piece = int(unit & 15), slab = int(unit >> 4), tile = slab >> 4, rank = (slab >> 3) & 1, warp = slab & 7;
  if (tile >= tiles) return;
  int tm, tn;
  gated_place(p.tiles_m, p.tiles_n, tile, tm, tn);
  const float4* at = p.partial + int64_t(slab) * 1024 + piece * 64 + lane;
  const int64_t step = int64_t(tiles) * 16 * 1024;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
#pragma unroll 4
  for (int r = 0; r < p.ranges; ++r) {
    const float4 v = __ldcg(at + r * step), w = __ldcg(at + r * step + 32);
    x = make_float4(x.x + v.x, x.y + v.y, x.z + v.z, x.w + v.w);
    y = make_float4(y.x + w.x, y.y + w.y, y.z + w.z, y.w + w.w);
  }
  const int sel = p.kind == kGbWeights && tn >= p.half;
  const int64_t row = (2 * tm + rank) * 128 + (warp & 3) * 32 + lane, col = int64_t(tn - (sel ? p.half : 0)) * 256 + (warp >> 2) * 128 + piece * 8;
  if (row < p.rows && col < p.cols)
    *reinterpret_cast<uint4*>(p.d[sel] + row * p.cols + col) = make_uint4(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w), pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
}

// ---- few tokens ----------------------------------------------------------------------------------------------------

// Few tokens are bound by the pass over the weights, so the tiles are made for that (and small problems, which are launches and ramps, have more of
// them to share out; few_plan).  A block has 128 rows and 64 columns of h (128 of the accumulator: the gate's, then the up-projection's), two blocks run on an SM, and where there are fewer tiles than
// places for them the contraction is cut into up to eight ranges, a cluster's blocks one each: their partial sums meet in shared memory,
// in the order of the ranges, and the blocks share the rows out.  (All places busy at once is what counts: 1 x 4096 -> 11008 has 86 tiles of 128 columns for 74 pairs, 55 us there.)
// A stage holds no more rows of x than there are, in boxes of eight at least: rows of a box that lie outside the tensor are not free
// (1 x 4096 -> 11008 29.4 us, in boxes of 64 44.8), and more than four stages measured slower (16 x 8192 -> 8192 41.8, six 45.1).
// 1, 16 and 128 x 8192 -> 8192 41.5, 41.8 and 46.8 us (6.5, 6.4 and 5.7 TB/s of weights).
// Warps 0-3 epilogue, 4 TMA producer, 5 MMA issuer.
constexpr int kGfRows = 128, kGfThreads = 192, kGfCols = 64, kGfPitch = 2 * kGfCols + 4;      // pitch of a row of partial sums, floats
constexpr int kGfStages = 4, kGfMost = 110 * 1024;      // at most; shared memory of a block, two of which an SM has room for
static_assert(2 * (kGfMost + 2048) <= 228 * 1024, "two blocks on an SM");

struct GatedFew {
  CUtensorMap x, gate, up;                      // boxes of x_rows x 64, 64 x 64
  __nv_bfloat16* h;
  __half *saved_gate, *saved_up;
  uint8_t* exponents;
  int rows, inner, blocks;                      // blocks: stages of the whole contraction
  int tiles_m;                                  // row tiles, the blocks of a column tile's side by side
  int stages;                                   // of the ring
  int x_rows, x_boxes;                          // rows of x in a stage: boxes of a multiple of eight rows
};

__device__ __forceinline__ void umma_bf16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float4 lds_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// This block's share of the rows, sixteen lanes each: the ranges' partial sums, all on their way at once and added up in order, then h and
// what the backward pass needs.
template <int ACT, bool SAVE, int RANGES>
__device__ __forceinline__ void few_join(const GatedFew& p, uint32_t sums, uint32_t rank, int m0, int n0) {
  const int lane = threadIdx.x & 31, col = 4 * (lane & 15);
  const int rows = min(kGfRows, p.rows - m0);
  for (int i = 2 * int(threadIdx.x >> 5); i * RANGES < rows; i += 2 * kGfThreads / 32) {
    const int row = (i + (lane >> 4)) * RANGES + int(rank);
    const bool there = row < rows;
    float4 g = make_float4(0.f, 0.f, 0.f, 0.f), u = g;
    if (there) {
      const uint32_t from = sums + uint32_t(row * kGfPitch + col) * 4u;
      float4 a[RANGES], b[RANGES];
#pragma unroll
      for (uint32_t r = 0; r < RANGES; ++r) {
        const uint32_t peer = map_rank(from, r);
        a[r] = lds_cluster(peer);
        b[r] = lds_cluster(peer + 4u * kGfCols);
      }
      g = a[0];
      u = b[0];
#pragma unroll
      for (int r = 1; r < RANGES; ++r) {
        g = make_float4(g.x + a[r].x, g.y + a[r].y, g.z + a[r].z, g.w + a[r].w);
        u = make_float4(u.x + b[r].x, u.y + b[r].y, u.z + b[r].z, u.w + b[r].w);
      }
    }
    const bool stores = there && n0 + col < p.inner;
    const int64_t at = int64_t(m0 + row) * p.inner + n0 + col;
    if constexpr (SAVE) {
      uint32_t e[2];
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const float4 v = which ? u : g;
        uint32_t m = max_magnitude(max_magnitude(max_magnitude(max_magnitude(0u, __float_as_uint(v.x)), __float_as_uint(v.y)), __float_as_uint(v.z)), __float_as_uint(v.w));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        float scale;
        e[which] = save_exponent(m, scale);
        auto kept = [&](float w) { return ACT == TG_GATED_RELU && which == 0 ? save_scaled<true>(w, scale) : save_scaled<false>(w, scale); };
        if (stores) *reinterpret_cast<uint2*>((which ? p.saved_up : p.saved_gate) + at) = make_uint2(pack_f16x2(kept(v.x), kept(v.y)), pack_f16x2(kept(v.z), kept(v.w)));
      }
      if (there && col == 0) reinterpret_cast<uint16_t*>(p.exponents)[int64_t(n0 / kGfCols) * p.rows + m0 + row] = uint16_t(e[0] | e[1] << 8);
    }
    if (stores)
      *reinterpret_cast<uint2*>(p.h + at) =
          make_uint2(pack_bf16x2(gated_act<ACT>(g.x) * u.x, gated_act<ACT>(g.y) * u.y), pack_bf16x2(gated_act<ACT>(g.z) * u.z, gated_act<ACT>(g.w) * u.w));
  }
}

template <int ACT, bool SAVE>
__global__ void __launch_bounds__(kGfThreads, 2) gated_few_kernel(const __grid_constant__ GatedFew p, unsigned* status) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(16) uint64_t ctl_bars[2 * kGfStages + 1];
  __shared__ uint32_t ctl_tmem_ptr;
  __shared__ int ctl_abort;
  const uint32_t sbase = smem_u32(smem);
  const uint32_t full0 = smem_u32(ctl_bars), empty0 = full0 + 8u * kGfStages, done_bar = empty0 + 8u * kGfStages;
  const uint32_t x_bytes = uint32_t(p.x_rows * p.x_boxes) * 128u, stage_bytes = x_bytes + 2 * kGbBox;
  volatile uint32_t* tmem_ptr_smem = &ctl_tmem_ptr;
  volatile int* abort_flag = &ctl_abort;
  if ((sbase & 1023u) != 0) {   // the swizzled layouts need this alignment (all blocks have the same layout)
    if (threadIdx.x == 0 && status != nullptr) atomicCAS(status, 0u, 6u);
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  uint32_t ranges;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ranges));
  const uint32_t rank = cluster_rank();
  const int tile = int(blockIdx.x / ranges), n0 = tile / p.tiles_m * kGfCols, m0 = (tile - tile / p.tiles_m * p.tiles_m) * kGfRows;
  const int first = int(uint64_t(p.blocks) * rank / ranges), last = int(uint64_t(p.blocks) * (rank + 1) / ranges);
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full0 + 8u * s, 1);
      mbar_init(empty0 + 8u * s, 1);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) {
    tmem_take(smem_u32(&ctl_tmem_ptr), 2 * kGfCols);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr_smem;
  grid_trigger();
  grid_wait();

  if (warp == 4) {
    uint32_t s = 0, ph = 1;
    for (int kb = first; kb < last; ++kb) {
      if (!__all_sync(0xffffffffu, mbar_wait(empty0 + 8u * s, ph, abort_flag, status, 1u))) break;
      if (elect_one()) {
        const uint32_t dst = sbase + s * stage_bytes, fb = full0 + 8u * s;
        mbar_expect_tx(fb, stage_bytes);
        tma_load_2d(dst + x_bytes, &p.gate, fb, n0, kb * kGbK);
        tma_load_2d(dst + x_bytes + kGbBox, &p.up, fb, n0, kb * kGbK);
        for (int i = 0; i < p.x_boxes; ++i) tma_load_2d(dst + i * kGbBox, &p.x, fb, kb * kGbK, m0 + 64 * i);
      }
      __syncwarp();
      if (++s == uint32_t(p.stages)) { s = 0; ph ^= 1u; }
    }
  } else if (warp == 5) {
    // A K-major (rows of the tile beyond those of x are whatever lies behind them in the stage: rows of the result that nobody reads), B MN-major
    const uint64_t desc_a0 = gated_desc(sbase), desc_b0 = gated_desc(sbase + x_bytes);
    const uint32_t desc_hi = uint32_t(desc_a0 >> 32), a_lo0 = uint32_t(desc_a0), b_lo0 = uint32_t(desc_b0);
    const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (uint32_t(2 * kGfCols >> 3) << 17) | (uint32_t(kGfRows >> 4) << 24);
    uint32_t s = 0, ph = 0;
    for (int kb = first; kb < last; ++kb) {
      if (!__all_sync(0xffffffffu, mbar_wait(full0 + 8u * s, ph, abort_flag, status, 3u))) break;
      __syncwarp();
      tc_fence_after();
      if (elect_one()) {
        const uint32_t soff = s * (stage_bytes >> 4);
#pragma unroll
        for (int k = 0; k < kGbK / 16; ++k)
          umma_bf16(tmem_base, (uint64_t(desc_hi) << 32) | (a_lo0 + soff + k * 2u), (uint64_t(desc_hi) << 32) | (b_lo0 + soff + k * 128u), idesc,
                    kb > first || k > 0 ? 1u : 0u);
        umma_commit(empty0 + 8u * s);
      }
      __syncwarp();
      if (++s == uint32_t(p.stages)) { s = 0; ph ^= 1u; }
    }
    // (after a wait that gave up too: nothing issued here may still be running when tensor memory is freed)
    if (elect_one()) umma_commit(done_bar);
    __syncwarp();
  }
  // every warp: the products are done, and with them the last look at the operands' shared memory
  const bool ok = __all_sync(0xffffffffu, mbar_wait(done_bar, 0u, abort_flag, status, 5u)) && !*abort_flag;
  __syncwarp();
  tc_fence_after();
  if (warp < 4 && ok && m0 + warp * 32 < p.rows) {
    const uint32_t at = tmem_base + (uint32_t(warp * 32) << 16);
    const int row = warp * 32 + lane;
    uint32_t g0[32], g1[32], u0[32], u1[32];
    tmem_ld32(at, g0);
    tmem_ld32(at + 32u, g1);
    tmem_ld32(at + 64u, u0);
    tmem_ld32(at + 96u, u1);
    tmem_wait_ld(g0);
    tmem_wait_ld(g1);
    tmem_wait_ld(u0);
    tmem_wait_ld(u1);
    if (m0 + row < p.rows) {
      const uint32_t to = sbase + uint32_t(row) * (kGfPitch * 4);
#pragma unroll
      for (int c = 0; c < 32; ++c) {
        const uint32_t(&v)[32] = c < 8 ? g0 : c < 16 ? g1 : c < 24 ? u0 : u1;
        sts128(to + 16u * c, make_uint4(v[4 * (c & 7)], v[4 * (c & 7) + 1], v[4 * (c & 7) + 2], v[4 * (c & 7) + 3]));
      }
    }
  }
  __syncwarp();
  cluster_sync();                              // the partial sums are there
  if (ok) {
    if (ranges == 1) few_join<ACT, SAVE, 1>(p, sbase, rank, m0, n0);
    else if (ranges == 2) few_join<ACT, SAVE, 2>(p, sbase, rank, m0, n0);
    else if (ranges == 4) few_join<ACT, SAVE, 4>(p, sbase, rank, m0, n0);
    else few_join<ACT, SAVE, 8>(p, sbase, rank, m0, n0);
  }
  __syncwarp();
  cluster_sync();                              // the partners have read this block's sums
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * kGfCols);
  }
}

// ---- dG and dU -----------------------------------------------------------------------------------------------------

struct GatedSlopes {
  const __nv_bfloat16* g;
  const __half *gate, *up;
  const uint16_t* exponents;
  __nv_bfloat16 *dgate, *dup;
  int64_t rows, low;                            // low: rows from the first pieces to the second ones, 0 for none
  int inner, chunks;
};
constexpr int kGsThreads = 128, kGsRows = kGsThreads / 8, kGsUnroll = 4;

// what is left of two values beside their bf16 (of an infinity or not-a-number nothing)
__device__ __forceinline__ uint32_t second_piece(float2 v, uint32_t first) {
  const float2 f = bf16x2_unpack(first);
  return pack_bf16x2(fabsf(f.x) < INFINITY ? v.x - f.x : 0.f, fabsf(f.y) < INFINITY ? v.y - f.y : 0.f);
}
// A block takes 64 columns of 64 rows, eight lanes a row: a row's 128 bytes of each tensor are one request, and its
// exponents one of a few in the same sector.
// TWO: dG and dU as the sum of two bf16, what the first leaves of them rounded in the second, for small problems (gated_low); rows up to the
// second pieces are zeros, since stages of dW run on into them.
template <int ACT, bool TWO>
__global__ void __launch_bounds__(kGsThreads) gated_slopes_kernel(const GatedSlopes p) {
  grid_trigger();
  grid_wait();
  const int lane8 = threadIdx.x & 7, r0 = threadIdx.x >> 3;
  {
    const uint32_t group = blockIdx.x / uint32_t(p.chunks);
    const int chunk = int(blockIdx.x - group * uint32_t(p.chunks)), col = chunk * 64 + lane8 * 8;
    uint4 g[kGsUnroll], a[kGsUnroll], u[kGsUnroll];
    uint32_t e[kGsUnroll];
    int64_t row[kGsUnroll];
#pragma unroll
    for (int k = 0; k < kGsUnroll; ++k) {
      row[k] = (int64_t(group) * kGsUnroll + k) * kGsRows + r0;
      if (col >= p.inner || row[k] >= (TWO ? p.low : p.rows)) row[k] = -1;
      if (row[k] < 0) continue;
      if constexpr (TWO) {
        if (row[k] >= p.rows) {
          g[k] = a[k] = u[k] = make_uint4(0u, 0u, 0u, 0u);
          e[k] = 0u;
          continue;
        }
      }
      const int64_t at = row[k] * p.inner + col;
      g[k] = ld_stream_v4(p.g + at);
      a[k] = ld_stream_v4(p.gate + at);
      u[k] = ld_stream_v4(p.up + at);
      e[k] = p.exponents[int64_t(chunk) * p.rows + row[k]];
    }
#pragma unroll
    for (int k = 0; k < kGsUnroll; ++k) {
      if (row[k] < 0) continue;
      const float sa = saved_scale(e[k] & 255u), su = saved_scale(e[k] >> 8);
      uint32_t og[4], ou[4], lg[4], lu[4];
      const uint32_t *gw = &g[k].x, *aw = &a[k].x, *uw = &u[k].x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 gv = bf16x2_unpack(gw[j]);
        const float2 av = __half22float2(*reinterpret_cast<const __half2*>(&aw[j])), uv = __half22float2(*reinterpret_cast<const __half2*>(&uw[j]));
        const float2 s0 = gated_act_slope<ACT>(av.x * sa), s1 = gated_act_slope<ACT>(av.y * sa);
        const float2 dg = make_float2(gv.x * (uv.x * su) * s0.y, gv.y * (uv.y * su) * s1.y), du = make_float2(gv.x * s0.x, gv.y * s1.x);
        og[j] = pack_bf16x2(dg.x, dg.y);
        ou[j] = pack_bf16x2(du.x, du.y);
        if constexpr (TWO) {
          lg[j] = second_piece(dg, og[j]);
          lu[j] = second_piece(du, ou[j]);
        }
      }
      const int64_t at = row[k] * p.inner + col;
      *reinterpret_cast<uint4*>(p.dgate + at) = make_uint4(og[0], og[1], og[2], og[3]);
      *reinterpret_cast<uint4*>(p.dup + at) = make_uint4(ou[0], ou[1], ou[2], ou[3]);
      if constexpr (TWO) {
        const int64_t behind = at + p.low * p.inner;
        *reinterpret_cast<uint4*>(p.dgate + behind) = make_uint4(lg[0], lg[1], lg[2], lg[3]);
        *reinterpret_cast<uint4*>(p.dup + behind) = make_uint4(lu[0], lu[1], lu[2], lu[3]);
      }
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------

// [rows][cols] of 16-bit elements, row pitch ld: boxes of 64 columns (128 bytes, swizzled) and box_rows rows
static int gated_map(CUtensorMap* m, const void* base, bool f16, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  return make_tmap(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, cols, rows, ld * 2, 128, box_rows);
}

// A launch on pairs: the kernel's shared memory is set, and the pairs that fit at a time are counted, once per device.
template <typename K, typename... A>
static int launch_gated(K kern, int smem, std::atomic<int>* units_of, int64_t items, bool early, cudaStream_t st, int& units, A... args) {
  int dev = 0;
  TG_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return TG_ERR_SHAPE;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = 2;
  attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kGbThreads);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.attrs = attrs;
  cfg.numAttrs = 1;
  cfg.stream = st;
  int fit = units_of[dev].load(std::memory_order_acquire);
  if (fit == 0) {
    TG_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cfg.gridDim = dim3(unsigned(sm_count() & ~1));
    TG_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&fit, kern, &cfg));
    if (fit < 1) return record_cuda_error(cudaErrorLaunchOutOfResources, "no CTA pair fits on this device");
    units_of[dev].store(fit, std::memory_order_release);
  }
  units = int(std::min<int64_t>(std::max(1, std::min(fit, gemm_pairs())), items));
  if constexpr (sizeof...(A) > 0) {
    cfg.gridDim = dim3(unsigned(2 * units));
    cfg.numAttrs = early ? 2 : 1;
    TG_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, args...));
  }
  return TG_OK;
}

static int gated_check(const tg_gated_args* a) {
  if (a == nullptr || a->rows < 0 || a->cols < 8 || a->inner < 8 || a->cols % 8 != 0 || a->inner % 8 != 0) return TG_ERR_SHAPE;
  if (a->act != TG_GATED_SILU && a->act != TG_GATED_GELU && a->act != TG_GATED_RELU) return TG_ERR_SHAPE;
  if (a->ldx < a->cols || a->ld_gate < a->inner || a->ld_up < a->inner) return TG_ERR_SHAPE;
  // (a tile's contraction stays far below what its barriers' waits are bounded by)
  if (a->rows > int64_t(1) << 30 || a->cols > int64_t(1) << 26 || a->inner > int64_t(1) << 26) return TG_ERR_TOO_LARGE;
  auto tiles = [](int64_t n, int64_t t) { return (n + t - 1) / t; };      // (every grid and every item number fits an int)
  if (tiles(a->rows, 256) * tiles(a->inner, 128) > INT32_MAX / 2 || tiles(a->rows, 256) * tiles(a->cols, 256) > INT32_MAX / 2 ||
      2 * tiles(a->cols, 256) * tiles(a->inner, 256) > INT32_MAX / 2 || tiles(a->rows, 64) * tiles(a->inner, 64) > INT32_MAX)
    return TG_ERR_TOO_LARGE;
  return TG_OK;
}
static bool gated_aligned(const tg_gated_args* a) {
  return aligned16(a->x) && aligned16(a->w_gate) && aligned16(a->w_up) && a->ldx % 8 == 0 && a->ld_gate % 8 == 0 && a->ld_up % 8 == 0;
}
static int64_t gated_chunks(int64_t inner) { return (inner + 63) / 64; }

// Whether that kernel takes a problem, and how.
struct FewPlan {
  int tiles_m = 1, tiles = 0, ranges = 1;
  bool takes = false;
};
static FewPlan few_plan(const tg_gated_args* a) {
  FewPlan f;
  const int64_t tiles_m = (a->rows + kGfRows - 1) / kGfRows, tiles = tiles_m * ((a->inner + kGfCols - 1) / kGfCols), blocks = (a->cols + kGbK - 1) / kGbK;
  const int64_t places = 2 * sm_count(), rows = std::min<int64_t>(a->rows, kGfRows);
  if (a->rows > 64 && tiles > places) return f;
  // As many ranges as find a place at once, of four stages at least and of one per eight tokens, whose sums take their time to meet: 128 x 1024 -> 4096
  // 10.5 us in one range, 12.5 in four; 128 x 4096 -> 4096 28.7 and 19.9; 16 x 1024 -> 4096 6.9 in four.
  while (f.ranges < 8 && tiles * f.ranges * 2 <= places && blocks >= 8 * f.ranges && 8 * (blocks / (2 * f.ranges)) >= rows) f.ranges *= 2;
  f.tiles_m = int(tiles_m);
  f.tiles = int(tiles);
  // Beyond 64 tokens by what the two take, in microseconds (a stage costs a block 0.2 with few of them and 0.45 with 128 and more, a pair's tile
  // 0.3): 1024 x 8192 -> 1024 32.8 here, 43 on pairs; 256 x 4096 -> 4096 21.5 and 25; 512 x 2048 -> 2048 13.5 and 14.8, 768 18.6 and 15.8; 300 x
  // 1024 -> 1024 7.9 and 9.2; 129 x 1024 -> 4096 11.2 and 10.1.
  const int64_t pair_tiles = (a->rows + 255) / 256 * ((a->inner + 127) / 128), pairs = sm_count() / 2;
  const double stage = 0.14 + 0.31 * std::min(1.0, double(tiles * f.ranges) / 128.0);
  const double here = 4.0 + (f.ranges > 1 ? 1.5 : 0.0) + stage * double(blocks) / f.ranges;
  const double on_pairs = 4.3 + 0.3 * double((pair_tiles + pairs - 1) / pairs * (blocks + 3));
  f.takes = a->rows <= 64 || here < on_pairs;
  return f;
}
template <int ACT, bool SAVE>
static int launch_few(const GatedFew& p, int tiles, int ranges, int smem, unsigned* status, cudaStream_t st) {
  static std::atomic<bool> done[64];
  if (int rc = allow_smem(gated_few_kernel<ACT, SAVE>, kGfMost, done)) return rc;
  TG_CUDA_CHECK(launch_early_clusters(gated_few_kernel<ACT, SAVE>, ranges, tiles * ranges, kGfThreads, smem, st, p, status));
  return TG_OK;
}
template <bool SAVE>
static int run_gated_few(const tg_gated_args* a, cudaStream_t st) {
  GatedFew p = {};
  p.x_rows = std::min(64, pow2_at_least(int(std::max<int64_t>(a->rows, 8))));
  p.x_boxes = a->rows > 64 ? 2 : 1;
  if (int rc = gated_map(&p.x, a->x, false, a->rows, a->cols, a->ldx, p.x_rows)) return rc;
  if (int rc = gated_map(&p.gate, a->w_gate, false, a->cols, a->inner, a->ld_gate, 64)) return rc;
  if (int rc = gated_map(&p.up, a->w_up, false, a->cols, a->inner, a->ld_up, 64)) return rc;
  p.h = static_cast<__nv_bfloat16*>(a->h);
  p.saved_gate = static_cast<__half*>(a->saved_gate);
  p.saved_up = static_cast<__half*>(a->saved_up);
  p.exponents = a->saved_exponents;
  p.rows = int(a->rows);
  p.inner = int(a->inner);
  p.blocks = int((a->cols + kGbK - 1) / kGbK);
  const FewPlan plan = few_plan(a);
  p.tiles_m = plan.tiles_m;
  const int tiles = plan.tiles, ranges = plan.ranges, rows = int(std::min<int64_t>(a->rows, kGfRows));
  const int stage = p.x_rows * p.x_boxes * 128 + 2 * kGbBox;
  p.stages = std::min(kGfStages, kGfMost / stage);
  const int smem = std::max(p.stages * stage, rows * kGfPitch * 4);
  static_assert(kGfRows * kGfPitch * 4 <= kGfMost, "partial sums fit where the operands were");
  if (a->act == TG_GATED_SILU) return launch_few<TG_GATED_SILU, SAVE>(p, tiles, ranges, smem, a->status, st);
  if (a->act == TG_GATED_GELU) return launch_few<TG_GATED_GELU, SAVE>(p, tiles, ranges, smem, a->status, st);
  return launch_few<TG_GATED_RELU, SAVE>(p, tiles, ranges, smem, a->status, st);
}

template <int ACT, bool SAVE>
static int run_gated_fwd(const GatedProblem& p, const GatedSaved& s, unsigned* status, cudaStream_t st) {
  static std::atomic<int> units_of[64];
  const int64_t items = int64_t(p.tiles_m) * p.tiles_n;
  int units = 0;
  return launch_gated(gated_fwd_kernel<ACT, SAVE>, GatedCfg<1>::smem_bytes, units_of, items, items <= 4 * gemm_pairs() && p.blocks <= 64, st,
                      units, p, s, status);
}
template <bool SAVE>
static int run_gated_fwd(int act, const GatedProblem& p, const GatedSaved& s, unsigned* status, cudaStream_t st) {
  if (act == TG_GATED_SILU) return run_gated_fwd<TG_GATED_SILU, SAVE>(p, s, status, st);
  if (act == TG_GATED_GELU) return run_gated_fwd<TG_GATED_GELU, SAVE>(p, s, status, st);
  return run_gated_fwd<TG_GATED_RELU, SAVE>(p, s, status, st);
}

}  // namespace tg

using namespace tg;

extern "C" int64_t tg_gated_linear_exponent_bytes(int64_t rows, int64_t inner) {
  return rows <= 0 || inner <= 0 ? 0 : 2 * rows * gated_chunks(inner);
}

extern "C" int tg_gated_linear_fwd(const tg_gated_args* a, void* stream) {
  if (int rc = gated_check(a)) return rc;
  const bool save = a->saved_gate != nullptr;
  if (save != (a->saved_up != nullptr) || save != (a->saved_exponents != nullptr)) return TG_ERR_SHAPE;
  if (a->rows == 0) return TG_OK;
  if (a->x == nullptr || a->w_gate == nullptr || a->w_up == nullptr || a->h == nullptr) return TG_ERR_SHAPE;
  if (!gated_aligned(a) || !aligned16(a->h) || !aligned16(a->saved_gate) || !aligned16(a->saved_up) || !aligned16(a->saved_exponents)) return TG_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  const int64_t M = a->rows, D = a->cols, F = a->inner;
  if (few_plan(a).takes) return save ? run_gated_few<true>(a, static_cast<cudaStream_t>(stream)) : run_gated_few<false>(a, static_cast<cudaStream_t>(stream));
  GatedProblem p = {};
  GatedSaved s = {};
  if (int rc = gated_map(&p.a[0], a->x, false, M, D, a->ldx, 64)) return rc;
  if (int rc = gated_map(&p.b[0], a->w_gate, false, D, F, a->ld_gate, 64)) return rc;
  if (int rc = gated_map(&p.b[1], a->w_up, false, D, F, a->ld_up, 64)) return rc;
  if (int rc = gated_map(&p.d[0], a->h, false, M, F, F, 32)) return rc;
  if (save) {
    if (int rc = gated_map(&s.gate, a->saved_gate, true, M, F, F, 32)) return rc;
    if (int rc = gated_map(&s.up, a->saved_up, true, M, F, F, 32)) return rc;
    s.exponents = a->saved_exponents;
    s.rows = M;
    s.chunks = int(gated_chunks(F));
  }
  p.kind = kGbForward;
  p.ranges = 1;
  p.tiles_m = int((M + 255) / 256);
  p.tiles_n = int((F + 127) / 128);
  p.blocks = int((D + kGbK - 1) / kGbK);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return save ? run_gated_fwd<true>(a->act, p, s, a->status, st) : run_gated_fwd<false>(a->act, p, s, a->status, st);
}

// Where dG and dU have two pieces: up to so many stages of the products with one, per pair of SMs.  With one, dx and dW have that rounding's error beside their
// own, as large in 2-norm where many terms average it (so the root of two of what a float32 form is off); where a few terms decide a result, as in small
// problems, up to 2.5 times.  With two they have their own rounding alone, so two are taken where the products are short next to the launches (forward and
// backward, us): 34 x 80 x 136 10.5 -> 13.3, 128 x 128 x 512 17.4 -> 20.7, 128 x 1024 x 1024 26.6 -> 30.6.  Past that it costs too much for a factor that
// averages: at 16 stages 8 x 1024 x 4096 26.5 -> 35.8, 1024 x 1024 x 1024 30.5 -> 41.  (A pair has the stages that a B200's 74 leave it.)
constexpr int64_t kGatedTwoStages = 4;

// Sizes of a problem as the launch sees them
struct GatedTiles {
  int64_t tiles = 0, blocks = 0, ranges = 1;
};
static double gated_makespan(const GatedTiles& x, const GatedTiles& y, int64_t units, int& rounds) {
  const GatedTiles &a = x.blocks * y.ranges >= y.blocks * x.ranges ? x : y, &b = &a == &x ? y : x;
  auto item = [](const GatedTiles& t) { return double(t.blocks) / double(t.ranges) + 3.0; };
  rounds = 0;
  if (a.tiles == 0 || b.tiles == 0) {
    const GatedTiles& t = a.tiles == 0 ? b : a;
    return double((t.tiles * t.ranges + units - 1) / units) * item(t);
  }
  return two_problems_us(a.tiles * a.ranges, item(a), b.tiles * b.ranges, item(b), units, rounds);
}
// How many ranges the contractions of dx and dW are cut into, in units of a stage (0.3 us): where whole items leave a fifth of the pairs' time
// unused or more, into items of a third of what each pair has to do, if that gains more than the sums' way through memory and a launch cost.
// 65536 x 512 -> 64 has four tiles of dW, of 1024 stages.
static void gated_ranges(GatedTiles& data, GatedTiles& weights) {
  const int64_t units = sm_count() / 2;
  int rounds;
  const double load = double(data.tiles * data.blocks + weights.tiles * weights.blocks) / double(units);
  const double whole = gated_makespan(data, weights, units, rounds);
  if (whole < 1.2 * load + 10.0) return;
  const int64_t length = std::max<int64_t>(16, int64_t(load / 3.0));
  double best = whole;
  const GatedTiles x = data, y = weights;
  for (int which = 1; which < 4; ++which) {
    GatedTiles u = x, v = y;
    if (which & 1) u.ranges = std::max<int64_t>(1, std::min<int64_t>(u.blocks / 8, (u.blocks + length - 1) / length));
    if (which & 2) v.ranges = std::max<int64_t>(1, std::min<int64_t>(v.blocks / 8, (v.blocks + length - 1) / length));
    const int64_t moved = (u.ranges > 1 ? u.tiles * u.ranges : 0) + (v.ranges > 1 ? v.tiles * v.ranges : 0);
    if (moved == 0 || moved > 1024) continue;
    const double time = gated_makespan(u, v, units, rounds) + 10.0 + 0.5 * double(moved);
    if (time < best) {
      best = time;
      data = u;
      weights = v;
    }
  }
}
// Rows from the first pieces of dG and dU to the second ones, 0 where one piece does: by the sizes alone, not by which gradients are asked for.
static int64_t gated_low(const tg_gated_args* a) {
  auto over = [](int64_t n, int64_t t) { return (n + t - 1) / t; };
  const int64_t data = over(a->rows, 256) * over(a->cols, 256) * 2 * over(a->inner, kGbK), weights = over(a->cols, 256) * 2 * over(a->inner, 256) * over(a->rows, kGbK);
  return data + weights <= kGatedTwoStages * (sm_count() / 2) ? over(a->rows, kGbK) * kGbK : 0;
}
static void gated_tiles(const tg_gated_args* a, bool two, GatedTiles& data, GatedTiles& weights) {
  auto over = [](int64_t n, int64_t t) { return (n + t - 1) / t; };
  if (a->dx != nullptr) {
    data.tiles = over(a->rows, 256) * over(a->cols, 256);
    data.blocks = (two ? 4 : 2) * over(a->inner, kGbK);
  }
  if (a->dw_gate != nullptr) {
    weights.tiles = over(a->cols, 256) * 2 * over(a->inner, 256);
    weights.blocks = (two ? 2 : 1) * over(a->rows, kGbK);
  }
  gated_ranges(data, weights);
}
// of dG, and of dU
static int64_t gated_half_bytes(const tg_gated_args* a, int64_t low) { return ((low > 0 ? 2 * low : a->rows) * a->inner * 2 + 255) / 256 * 256; }
static int64_t gated_partial_items(const GatedTiles& t) { return t.ranges > 1 ? t.tiles * t.ranges : 0; }

extern "C" int64_t tg_gated_linear_bwd_scratch_bytes(const tg_gated_args* a) {
  if (gated_check(a) != TG_OK || a->rows == 0) return 0;
  GatedTiles data, weights;
  const int64_t low = gated_low(a);
  gated_tiles(a, low > 0, data, weights);
  return 2 * gated_half_bytes(a, low) + (gated_partial_items(data) + gated_partial_items(weights)) * 262144;
}

extern "C" int tg_gated_linear_bwd(const tg_gated_args* a, void* stream) {
  if (int rc = gated_check(a)) return rc;
  if ((a->dw_gate == nullptr) != (a->dw_up == nullptr)) return TG_ERR_SHAPE;
  const int64_t M = a->rows, D = a->cols, F = a->inner;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (M == 0) {
    if (int rc = check_arch()) return rc;
    for (void* v : {a->dw_gate, a->dw_up})
      if (v != nullptr) TG_CUDA_CHECK(cudaMemsetAsync(v, 0, size_t(D) * F * 2, st));
    return TG_OK;
  }
  const bool dx = a->dx != nullptr, dw = a->dw_gate != nullptr;
  if (a->g == nullptr || a->saved_gate == nullptr || a->saved_up == nullptr || a->saved_exponents == nullptr || a->scratch == nullptr || a->scratch_bytes < 2 * gated_half_bytes(a, 0) ||
      (dx && (a->w_gate == nullptr || a->w_up == nullptr)) || (dw && a->x == nullptr))
    return TG_ERR_SHAPE;
  if (!gated_aligned(a) || !aligned16(a->g) || !aligned16(a->saved_gate) || !aligned16(a->saved_up) || !aligned16(a->saved_exponents) || !aligned16(a->dx) ||
      !aligned16(a->dw_gate) || !aligned16(a->dw_up) || !aligned16(a->scratch))
    return TG_ERR_ALIGN;
  GatedTiles data_tiles, weights_tiles;
  const bool all = a->scratch_bytes >= tg_gated_linear_bwd_scratch_bytes(a);
  const int64_t low = all ? gated_low(a) : 0, half_bytes = gated_half_bytes(a, low);
  gated_tiles(a, low > 0, data_tiles, weights_tiles);
  if (!all) data_tiles.ranges = weights_tiles.ranges = 1;
  // (an item's stages stay far below what its barriers' waits are bounded by: 0.6 s here; the ranges see to that, without them rows do up to 2^27)
  if (weights_tiles.blocks / weights_tiles.ranges > 1 << 21) return TG_ERR_TOO_LARGE;
  if (int rc = check_arch()) return rc;
  if (!dx && !dw) return TG_OK;
  GatedSlopes s = {};
  s.g = static_cast<const __nv_bfloat16*>(a->g);
  s.gate = static_cast<const __half*>(a->saved_gate);
  s.up = static_cast<const __half*>(a->saved_up);
  s.exponents = reinterpret_cast<const uint16_t*>(a->saved_exponents);
  s.dgate = static_cast<__nv_bfloat16*>(a->scratch);
  s.dup = reinterpret_cast<__nv_bfloat16*>(static_cast<uint8_t*>(a->scratch) + half_bytes);
  s.rows = M;
  s.low = low;
  s.inner = int(F);
  s.chunks = int(gated_chunks(F));
  const int64_t items = (M + kGsRows * kGsUnroll - 1) / (kGsRows * kGsUnroll) * s.chunks;
  static_assert(kGsRows * kGsUnroll == kGbK, "a block's rows end where the second pieces begin");
  auto slopes = [&](auto act) { return low > 0 ? gated_slopes_kernel<act.value, true> : gated_slopes_kernel<act.value, false>; };
  auto kern = a->act == TG_GATED_SILU   ? slopes(std::integral_constant<int, TG_GATED_SILU>())
              : a->act == TG_GATED_GELU ? slopes(std::integral_constant<int, TG_GATED_GELU>())
                                        : slopes(std::integral_constant<int, TG_GATED_RELU>());
  TG_CUDA_CHECK(launch_if_short(items <= 8 * sm_count(), kern, dim3(unsigned(items)), kGsThreads, 0, st, s));

  GatedProblem data = {}, weights = {};
  GatedJoin joins[2] = {};
  int n_joins = 0;
  uint8_t* partial = static_cast<uint8_t*>(a->scratch) + 2 * half_bytes;
  auto cut = [&](GatedProblem& p, const GatedTiles& t, void* d0, void* d1, int64_t rows, int64_t cols) {
    p.ranges = int(t.ranges);
    if (t.ranges == 1) return;
    p.partial = reinterpret_cast<float4*>(partial);
    partial += gated_partial_items(t) * 262144;
    joins[n_joins++] = {p.partial, {static_cast<__nv_bfloat16*>(d0), static_cast<__nv_bfloat16*>(d1)}, p.kind, p.tiles_m, p.tiles_n, p.half, p.ranges, rows, cols};
  };
  if (dx) {
    for (int i = 0; i < 2; ++i) {
      if (int rc = gated_map(&data.a[i], i ? s.dup : s.dgate, false, low > 0 ? 2 * low : M, F, F, 64)) return rc;
      if (int rc = gated_map(&data.b[i], i ? a->w_up : a->w_gate, false, D, F, i ? a->ld_up : a->ld_gate, 64)) return rc;
    }
    if (int rc = gated_map(&data.d[0], a->dx, false, M, D, D, 32)) return rc;
    data.kind = kGbData;
    data.tiles_m = int((M + 255) / 256);
    data.tiles_n = int((D + 255) / 256);
    data.half = int((F + kGbK - 1) / kGbK);
    data.piece = 2 * data.half;
    data.low = int(low);
    data.blocks = int(data_tiles.blocks);
    cut(data, data_tiles, a->dx, nullptr, M, D);
  }
  if (dw) {
    if (int rc = gated_map(&weights.a[0], a->x, false, M, D, a->ldx, 64)) return rc;
    for (int i = 0; i < 2; ++i) {
      if (int rc = gated_map(&weights.b[i], i ? s.dup : s.dgate, false, low > 0 ? 2 * low : M, F, F, 64)) return rc;
      if (int rc = gated_map(&weights.d[i], i ? a->dw_up : a->dw_gate, false, D, F, F, 32)) return rc;
    }
    weights.kind = kGbWeights;
    weights.tiles_m = int((D + 255) / 256);
    weights.half = int((F + 255) / 256);
    weights.tiles_n = 2 * weights.half;
    weights.piece = int((M + kGbK - 1) / kGbK);
    weights.low = int(low);
    weights.blocks = int(weights_tiles.blocks);
    cut(weights, weights_tiles, a->dw_gate, a->dw_up, D, F);
  }
  // the longer items first
  const bool both = dx && dw, data_first = dx && (!dw || data_tiles.blocks * weights_tiles.ranges >= weights_tiles.blocks * data_tiles.ranges);
  const GatedProblem &one = data_first ? data : weights, &two = data_first ? weights : data;
  const int64_t n1 = int64_t(one.tiles_m) * one.tiles_n * one.ranges, n2 = both ? int64_t(two.tiles_m) * two.tiles_n * two.ranges : 0;
  static std::atomic<int> units_of[64];
  using C = GatedCfg<2>;
  int units = 0, rounds = 0;
  if (int rc = launch_gated(gated_bwd_kernel, C::smem_bytes, units_of, n1 + n2, false, st, units)) return rc;
  gated_makespan(data_tiles, weights_tiles, units, rounds);
  const bool early = n1 + n2 <= 4 * units && one.blocks / one.ranges <= 64;
  if (int rc = launch_gated(gated_bwd_kernel, C::smem_bytes, units_of, n1 + n2, early, st, units, one, two, int(both), rounds, reinterpret_cast<unsigned*>(a->status)))
    return rc;
  if (n_joins > 0) {
    auto blocks_of = [](const GatedJoin& j) { return j.ranges > 1 ? j.tiles_m * j.tiles_n * 32 : 0; };
    const int first = blocks_of(joins[0]);
    TG_CUDA_CHECK(launch_if_short(true, gated_join_kernel, dim3(unsigned(first + blocks_of(joins[1]))), 256, 0, st, joins[0], joins[1], first));
  }
  return TG_OK;
}
