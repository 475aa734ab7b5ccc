// The junction between two blocks of a network whose blocks have a norm on both sides, as one kernel each way:
//
//     x' = bf16(alpha x + G (y * rsqrt(mean y^2 + eps) * post)),   h = bf16(x' * rsqrt(mean x'^2 + eps) * pre)
//
// y is the block's output, x the residual stream, G a gate per channel or per token (or 1), h what the next block reads -- in bf16 and,
// where an FP8 linear reads it, in 1 x 128 e4m3 tiles (fp8.py:39-47 on the bf16 h).  x' is rounded before it is normalised: it is what the
// stream keeps, and what the backward pass computes from.  All else is float32, rounded once.
//
// Backward, for the gradients g of x' and gh of h, with r and s the two norms' factors (r of x', s of y):
//     a = gh pre,  d = g + r (a - x' r^2 mean(a x')),  dx = alpha d,  dpre = sum_rows r gh x'
//     t = d post (gate per channel: times the gate),  dy = G s (t - y s^2 mean(t y)),  C = sum_rows G s d y
//     dpost = C (times the gate per channel),  dgate per channel = C post,  per token = s sum_columns t y
//
// A pass of either is bound by memory (8 bytes an element forward, 12 backward), so each is one read of its inputs: rows are staged
// through shared memory by cp.async, the next ones on their way while one is worked on.  Every lane reads only the 16-byte pieces that
// it fetched itself, so the warps of a row meet only at its sums, of which there are two rounds.
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "host_api.h"
#include "norm.cuh"

namespace tg {

constexpr int kSwWarps = 16;                   // of a block
constexpr int kSwMaxCols = 8192;

// N sums over a row of wpr warps; `red` holds N floats per warp of the block.  Two rounds a row with a buffer of their own each: a warp
// that writes one of the next row has passed the other's barrier, which every warp of the row reaches after reading the first.
template <int N>
__device__ __forceinline__ void group_sums(float (&v)[N], float (*red)[kSwWarps], int warp, int lane, int wpr, int first, int barrier) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  if (wpr > 1) {
    if (lane == 0) {
#pragma unroll
      for (int n = 0; n < N; ++n) red[n][warp] = v[n];
    }
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(wpr * 32) : "memory");   // this row's warps only
    const int at = lane & (kSwWarps - 1);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = at < wpr ? red[n][first + at] : 0.f;
#pragma unroll
      for (int o = kSwWarps / 2; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    }
  }
}

struct SandwichVectors {
  const __nv_bfloat16 *post, *pre, *gate;
  int gate_kind;
};

// post (times the gate per channel) and pre, widened to float, in two planes each (columns 8i..8i+3 of every piece, then 8i+4..8i+7): a
// warp's 16-byte reads of either plane are contiguous
__device__ __forceinline__ void fill_planes(const SandwichVectors& v, float4* s_w, float4* s_pre, int pieces) {
  for (int i = threadIdx.x; i < pieces; i += blockDim.x) {
    const uint4 a = reinterpret_cast<const uint4*>(v.post)[i], b = reinterpret_cast<const uint4*>(v.pre)[i];
    float4 lo = make_float4(bf16lo(a.x), bf16hi(a.x), bf16lo(a.y), bf16hi(a.y));
    float4 hi = make_float4(bf16lo(a.z), bf16hi(a.z), bf16lo(a.w), bf16hi(a.w));
    if (v.gate_kind == TG_GATE_CHANNEL) {      // (a product of two bf16 values is exact)
      const uint4 g = reinterpret_cast<const uint4*>(v.gate)[i];
      lo = make_float4(lo.x * bf16lo(g.x), lo.y * bf16hi(g.x), lo.z * bf16lo(g.y), lo.w * bf16hi(g.y));
      hi = make_float4(hi.x * bf16lo(g.z), hi.y * bf16hi(g.z), hi.z * bf16lo(g.w), hi.w * bf16hi(g.w));
    }
    s_w[i] = lo;
    s_w[pieces + i] = hi;
    s_pre[i] = make_float4(bf16lo(b.x), bf16hi(b.x), bf16lo(b.y), bf16hi(b.y));
    s_pre[pieces + i] = make_float4(bf16lo(b.z), bf16hi(b.z), bf16lo(b.w), bf16hi(b.w));
  }
}
__device__ __forceinline__ void plane8(const float4* s, int pieces, int piece, float2 (&v)[4]) {
  const float4 a = s[piece], b = s[pieces + piece];
  v[0] = make_float2(a.x, a.y);
  v[1] = make_float2(a.z, a.w);
  v[2] = make_float2(b.x, b.y);
  v[3] = make_float2(b.z, b.w);
}
__device__ __forceinline__ void unpack8(const uint4& w, float2 (&v)[4]) {
  v[0] = bf16x2_unpack(w.x);
  v[1] = bf16x2_unpack(w.y);
  v[2] = bf16x2_unpack(w.z);
  v[3] = bf16x2_unpack(w.w);
}
__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }

// ---- forward -----------------------------------------------------------------------------------------------------

struct SandwichFwd {
  const __nv_bfloat16 *x, *y;
  SandwichVectors v;
  float alpha, eps;
  __nv_bfloat16 *x_new, *h;
  uint8_t* q;
  float* scales;
  int64_t rows;
  int cols;
};

// x' of a piece
__device__ __forceinline__ uint4 junction8(const uint4& xw, const uint4& yw, const float2 (&w)[4], float alpha, float rg) {
  float2 x[4], y[4];
  unpack8(xw, x);
  unpack8(yw, y);
  uint4 o;
  uint32_t* op = &o.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 n = __fmul2_rn(__fmul2_rn(y[j], splat(rg)), w[j]);
    const float2 t = __ffma2_rn(splat(alpha), x[j], n);
    op[j] = pack_bf16x2(t.x, t.y);
  }
  return o;
}
__device__ __forceinline__ uint4 normed8(const uint4& xw, const float2 (&g)[4], float r) {
  float2 x[4];
  unpack8(xw, x);
  uint4 o;
  uint32_t* op = &o.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 t = __fmul2_rn(__fmul2_rn(x[j], splat(r)), g[j]);
    op[j] = pack_bf16x2(t.x, t.y);
  }
  return o;
}

// Sixteen warps a block.  A row of up to 512 columns has a warp, two slots and two blocks per SM (65536 x 256 21.3 us, 32768 x 512 20.6,
// with one 26.9 and 26.7); up to 1024 a warp, with one block (16384 x 1024 20.0; two: 22.7); up to 2048 four warps with two pieces of 256
// columns each and three slots (32768 x 2048 83.7 us, 6.4 TB/s; two warps of four pieces 99.5, with two slots 97.4); above, as many warps
// as have three or four pieces each and two slots (8191 x 8184 90.5 us, 8000 x 3400 39.1; with two pieces 115 and 49, as a block then has half the rows).
constexpr int sw_fwd_per_sm(int nchunk, int slots) { return nchunk <= 2 && slots == 2 ? 2 : 1; }

template <int NCHUNK, int SLOTS, bool FULL>
__global__ void __launch_bounds__(kSwWarps * 32, sw_fwd_per_sm(NCHUNK, SLOTS)) sandwich_fwd_kernel(const SandwichFwd p, int wpr) {
  constexpr int WARPS = kSwWarps, kRowBytes = NCHUNK * 512, kSlotBytes = 2 * kRowBytes;
  __shared__ float s_red[2][1][WARPS];
  extern __shared__ float4 s_w[];              // planes of w and pre, then [warps][slots][x row | y row]
  const int cols = p.cols, pieces = cols / 8, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rpb = WARPS / wpr, row_of_block = warp / wpr, first = row_of_block * wpr, barrier = 1 + row_of_block;
  const bool works = row_of_block < rpb;       // (sixteen is not a multiple of every row's warps)
  const int col_base = (warp - first) * (NCHUNK * 256) + lane * 8;
  const bool token = p.v.gate_kind == TG_GATE_TOKEN;
  float4* s_pre = s_w + 2 * pieces;
  const uint32_t slot0 = uint32_t(__cvta_generic_to_shared(s_w)) + uint32_t(cols) * 8u + uint32_t(warp) * SLOTS * kSlotBytes + uint32_t(lane) * 16u;
  grid_trigger();
  grid_wait();
  fill_planes(p.v, s_w, s_pre, pieces);
  __syncthreads();

  const int64_t stride = int64_t(gridDim.x) * rpb;
  int64_t row = works ? int64_t(blockIdx.x) * rpb + row_of_block : p.rows;
  auto prefetch = [&](int64_t r, int slot) {
    if (r < p.rows) {
#pragma unroll
      for (int c = 0; c < NCHUNK; ++c) {
        const int col = col_base + c * 256;
        if (FULL || col < cols) {
          cp_async16(slot0 + slot * kSlotBytes + c * 512, p.x + r * cols + col);
          cp_async16(slot0 + slot * kSlotBytes + kRowBytes + c * 512, p.y + r * cols + col);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");   // an empty group keeps the wait count uniform
  };
#pragma unroll
  for (int s = 0; s < SLOTS - 1; ++s) prefetch(row + s * stride, s);
  int slot = 0, slot_in = SLOTS - 1;
  const uint16_t* gates = reinterpret_cast<const uint16_t*>(p.v.gate);
  uint32_t next_gate = token && row < p.rows ? gates[row] : 0x3f80u;     // its bits, a row ahead (16000 x 1280 33.4 us, loaded in its turn 41.1)
  for (; row < p.rows; row += stride) {
    const uint32_t base = slot0 + uint32_t(slot) * kSlotBytes;
    prefetch(row + (SLOTS - 1) * stride, slot_in);    // into the slot that the previous row has left
    const float gate = __uint_as_float(next_gate << 16);
    if (token && row + stride < p.rows) next_gate = gates[row + stride];
    asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 1) : "memory");
    slot_in = slot;
    if (++slot == SLOTS) slot = 0;
    float part[NCHUNK];
#pragma unroll
    for (int c = 0; c < NCHUNK; ++c) part[c] = (FULL || col_base + c * 256 < cols) ? sumsq8(lds128(base + kRowBytes + c * 512)) : 0.f;
    float ss[1] = {tree_sum(part)};
    group_sums<1>(ss, s_red[0], warp, lane, wpr, first, barrier);
    const float rg = __frsqrt_rn(__fdiv_rn(ss[0], float(cols)) + p.eps) * gate;

    uint4 xo[NCHUNK];
#pragma unroll
    for (int c = 0; c < NCHUNK; ++c) {
      const int col = col_base + c * 256;
      xo[c] = make_uint4(0u, 0u, 0u, 0u);
      if (FULL || col < cols) {
        float2 w[4];
        plane8(s_w, pieces, col >> 3, w);
        xo[c] = junction8(lds128(base + c * 512), lds128(base + kRowBytes + c * 512), w, p.alpha, rg);
        *reinterpret_cast<uint4*>(p.x_new + row * cols + col) = xo[c];
      }
      part[c] = sumsq8(xo[c]);
    }
    ss[0] = tree_sum(part);
    group_sums<1>(ss, s_red[1], warp, lane, wpr, first, barrier);
    const float r = __frsqrt_rn(__fdiv_rn(ss[0], float(cols)) + p.eps);

    constexpr int G = pow2_at_least(NCHUNK);
    uint32_t amax_bits[G];
#pragma unroll
    for (int u = NCHUNK; u < G; ++u) amax_bits[u] = 0u;
#pragma unroll
    for (int c = 0; c < NCHUNK; ++c) {
      const int col = col_base + c * 256;
      amax_bits[c] = 0u;
      if (FULL || col < cols) {
        float2 g[4];
        plane8(s_pre, pieces, col >> 3, g);
        xo[c] = normed8(xo[c], g, r);
        if (p.h != nullptr) *reinterpret_cast<uint4*>(p.h + row * cols + col) = xo[c];
        amax_bits[c] = absmax8_h(xo[c]);
      }
    }
    if (p.q == nullptr) continue;
    float s[G], inv[G], s_mine;
    bool fin;
    tile_scales_own<G>(exchange_tile_amax<G>(amax_bits), s, inv, s_mine, fin);
    {
      const int j = lane & 15;
      const int col = col_base - lane * 8 + j * 256 + (lane & 16) * 8;     // first column of the tile this lane computed
      if (j < NCHUNK && (FULL || col < cols)) p.scales[row * (cols / kTile) + col / kTile] = s_mine;
    }
    uint8_t* qp = p.q + row * cols + col_base;
#pragma unroll
    for (int c = 0; c < NCHUNK; ++c)
      if (FULL || col_base + c * 256 < cols) *reinterpret_cast<uint2*>(qp + c * 256) = fin ? quantize8_sr(xo[c], s[c], inv[c]) : quantize8(xo[c], s[c]);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---- backward ----------------------------------------------------------------------------------------------------

struct SandwichBwd {
  const __nv_bfloat16 *x_new, *y;
  SandwichVectors v;
  float alpha, eps;
  const __nv_bfloat16 *g_new, *g_h;            // either may be NULL: zero
  __nv_bfloat16 *dx, *dy, *dgate_token;
  float* partial;                              // [blocks][2][cols]: sums of r gh x', and C
  int64_t rows;
  int cols;
};

// Sixteen warps a block, one block per SM.  A warp has two pieces of 256 columns of a row (their column sums are 32 registers), a row as many
// warps as it needs: `wpr`, the rest of the sixteen their own rows.  Three pieces where a block then has five thirds of the rows or more
// (32768 x 768 56.5 us instead of 64.2, 4096 x 2304 27.2 instead of 30.5; 20000 x 1536, eight rows instead of five, 67.5 instead of 63.0).  With the reduction behind it: 32768 x 2048 128 us (6.3 TB/s), 16384 x
// 1024 37.4, 3001 x 4096 38.9, 8191 x 8184 188, 65536 x 256 39.7, 128 x 128 5.0; with four pieces a warp and eight warps 127, 37.8, 39.4,
// 204, 50.7 and 4.7.
template <int NCHUNK, int SLOTS, bool FULL>
__global__ void __launch_bounds__(kSwWarps * 32) sandwich_bwd_kernel(const SandwichBwd p, int wpr) {
  constexpr int WARPS = kSwWarps, kRowBytes = NCHUNK * 512, kSlotBytes = 4 * kRowBytes;
  __shared__ float s_red3[3][WARPS], s_red1[1][WARPS];
  extern __shared__ float4 s_w[];              // planes of w and pre, then [warps][slots][x' | y | g | gh]
  const int cols = p.cols, pieces = cols / 8, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rpb = WARPS / wpr, row_of_block = warp / wpr, first = row_of_block * wpr, barrier = 1 + row_of_block;
  const bool works = row_of_block < rpb;       // (sixteen is not a multiple of every row's warps)
  const int col_base = (warp - first) * (NCHUNK * 256) + lane * 8;
  float4* s_pre = s_w + 2 * pieces;
  const uint32_t slot0 = uint32_t(__cvta_generic_to_shared(s_w)) + uint32_t(cols) * 8u + uint32_t(warp) * SLOTS * kSlotBytes + uint32_t(lane) * 16u;
  const float inv_d = __fdiv_rn(1.0f, float(cols));
  const bool has_g = p.g_new != nullptr, has_h = p.g_h != nullptr, token = p.v.gate_kind == TG_GATE_TOKEN;
  grid_wait();
  fill_planes(p.v, s_w, s_pre, pieces);
  __syncthreads();

  float2 acc_p[NCHUNK][4], acc_c[NCHUNK][4];
#pragma unroll
  for (int c = 0; c < NCHUNK; ++c)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc_p[c][j] = acc_c[c][j] = splat(0.f);

  const int64_t stride = int64_t(gridDim.x) * rpb;
  int64_t row = works ? int64_t(blockIdx.x) * rpb + row_of_block : p.rows;
  auto prefetch = [&](int64_t r, int slot) {
    if (r < p.rows) {
      const uint32_t dst = slot0 + uint32_t(slot) * kSlotBytes;
#pragma unroll
      for (int c = 0; c < NCHUNK; ++c) {
        const int col = col_base + c * 256;
        if (FULL || col < cols) {
          const int64_t at = r * cols + col;
          cp_async16(dst + c * 512, p.x_new + at);
          cp_async16(dst + kRowBytes + c * 512, p.y + at);
          if (has_g) cp_async16(dst + 2 * kRowBytes + c * 512, p.g_new + at);
          if (has_h) cp_async16(dst + 3 * kRowBytes + c * 512, p.g_h + at);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int s = 0; s < SLOTS - 1; ++s) prefetch(row + s * stride, s);
  int slot = 0, slot_in = SLOTS - 1;
  for (; row < p.rows; row += stride) {
    const uint32_t xs = slot0 + uint32_t(slot) * kSlotBytes, ys = xs + kRowBytes, gs = ys + kRowBytes, hs = gs + kRowBytes;
    prefetch(row + (SLOTS - 1) * stride, slot_in);    // into the slot that the previous row has left
    const float gate = token ? __bfloat162float(p.v.gate[row]) : 1.0f;
    asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 1) : "memory");
    slot_in = slot;
    if (++slot == SLOTS) slot = 0;

    // ---- sums of x'^2, a x' and y^2
    float sums[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NCHUNK; ++c) {
      const int col = col_base + c * 256;
      if (!(FULL || col < cols)) continue;
      const uint4 xw = lds128(xs + c * 512);
      sums[0] += sumsq8(xw);
      sums[2] += sumsq8(lds128(ys + c * 512));
      if (has_h) {
        float2 x[4], g[4], m[4];
        unpack8(xw, x);
        unpack8(lds128(hs + c * 512), g);
        plane8(s_pre, pieces, col >> 3, m);
        float2 t = splat(0.f);
#pragma unroll
        for (int j = 0; j < 4; ++j) t = __ffma2_rn(__fmul2_rn(g[j], m[j]), x[j], t);
        sums[1] += t.x + t.y;
      }
    }
    group_sums<3>(sums, s_red3, warp, lane, wpr, first, barrier);
    const float r = __frsqrt_rn(__fmaf_rn(sums[0], inv_d, p.eps)), s = __frsqrt_rn(__fmaf_rn(sums[2], inv_d, p.eps));
    const float nm = -(r * r) * (sums[1] * inv_d);    // d = g + r (a + x' nm)

    // ---- d, dx, the sum of t y
    float2 d[NCHUNK][4];
    float sum4[1] = {0.f};
#pragma unroll
    for (int c = 0; c < NCHUNK; ++c) {
      const int col = col_base + c * 256;
      if (!(FULL || col < cols)) continue;
      float2 x[4], y[4], g[4], gh[4], m[4];
      unpack8(lds128(xs + c * 512), x);
      unpack8(has_g ? lds128(gs + c * 512) : zero, g);
      unpack8(has_h ? lds128(hs + c * 512) : zero, gh);
      plane8(s_pre, pieces, col >> 3, m);
      uint4 o;
      uint32_t* op = &o.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = __fmul2_rn(gh[j], m[j]);
        d[c][j] = __ffma2_rn(splat(r), __ffma2_rn(x[j], splat(nm), a), g[j]);
        acc_p[c][j] = __ffma2_rn(__fmul2_rn(x[j], splat(r)), gh[j], acc_p[c][j]);
        const float2 t = __fmul2_rn(d[c][j], splat(p.alpha));
        op[j] = pack_bf16x2(t.x, t.y);
      }
      *reinterpret_cast<uint4*>(p.dx + row * cols + col) = o;
      unpack8(lds128(ys + c * 512), y);
      plane8(s_w, pieces, col >> 3, m);
      float2 t = splat(0.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) t = __ffma2_rn(__fmul2_rn(d[c][j], m[j]), y[j], t);
      sum4[0] += t.x + t.y;
    }
    group_sums<1>(sum4, s_red1, warp, lane, wpr, first, barrier);
    if (token && p.dgate_token != nullptr && lane == 0 && warp == first) p.dgate_token[row] = __float2bfloat16_rn(s * sum4[0]);
    const float gsr = gate * s, nm2 = -(s * s) * (sum4[0] * inv_d);

    // ---- dy and C
#pragma unroll
    for (int c = 0; c < NCHUNK; ++c) {
      const int col = col_base + c * 256;
      if (!(FULL || col < cols)) continue;
      float2 y[4], m[4];
      unpack8(lds128(ys + c * 512), y);
      plane8(s_w, pieces, col >> 3, m);
      uint4 o;
      uint32_t* op = &o.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc_c[c][j] = __ffma2_rn(__fmul2_rn(y[j], splat(gsr)), d[c][j], acc_c[c][j]);
        const float2 t = __fmul2_rn(splat(gsr), __ffma2_rn(y[j], splat(nm2), __fmul2_rn(d[c][j], m[j])));
        op[j] = pack_bf16x2(t.x, t.y);
      }
      *reinterpret_cast<uint4*>(p.dy + row * cols + col) = o;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  grid_trigger();          // the reduction's blocks may take the places of this kernel's as they leave
  // every warp's column sums over the (now idle) slots, then the block's rows added up in order and published
  __syncthreads();
  float* s_sum = reinterpret_cast<float*>(s_w) + 2 * cols;
  constexpr int kWarpCols = NCHUNK * 256;
#pragma unroll
  for (int c = 0; c < NCHUNK; ++c) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const float2(&v)[4] = which ? acc_c[c] : acc_p[c];
      float4* dst = reinterpret_cast<float4*>(s_sum + (warp * 2 + which) * kWarpCols + c * 256 + lane * 8);
      dst[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
      dst[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    }
  }
  __syncthreads();
  float* out = p.partial + int64_t(blockIdx.x) * 2 * cols;
  for (int i = threadIdx.x; i < 2 * cols; i += blockDim.x) {
    const int which = i >= cols, col = which ? i - cols : i, w = col / kWarpCols;
    const float* from = s_sum + (w * 2 + which) * kWarpCols + (col - w * kWarpCols);
    float t = 0.f;
    for (int r = 0; r < rpb; ++r) t += from[r * wpr * 2 * kWarpCols];
    out[i] = t;
  }
}

// Column sums of the blocks' partial ones, 32 columns a block, warp w those of blocks w, w + 32, ...: an order that the number of blocks
// alone fixes.  dpre is the first sum; dpost and the gate's gradient come from the second.
struct SandwichReduce {
  const float* partial;
  SandwichVectors v;
  __nv_bfloat16 *dpost, *dpre, *dgate;
  int blocks, cols;
};
__global__ void __launch_bounds__(1024) sandwich_reduce_kernel(const SandwichReduce p) {
  __shared__ float s_part[2][32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  grid_wait();
  float a = 0.f, b = 0.f;
  if (col < p.cols) {
#pragma unroll 4
    for (int i = warp; i < p.blocks; i += 32) {
      const float* at = p.partial + int64_t(i) * 2 * p.cols + col;
      a += __ldcg(at);
      b += __ldcg(at + p.cols);
    }
  }
  s_part[0][warp][lane] = a;
  s_part[1][warp][lane] = b;
  __syncthreads();
  if (warp < 2 && col < p.cols) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) t += s_part[warp][w][lane];
    if (warp == 0) {
      p.dpre[col] = __float2bfloat16_rn(t);
    } else {
      const bool channel = p.v.gate_kind == TG_GATE_CHANNEL;
      p.dpost[col] = __float2bfloat16_rn(channel ? t * __bfloat162float(p.v.gate[col]) : t);
      if (channel && p.dgate != nullptr) p.dgate[col] = __float2bfloat16_rn(t * __bfloat162float(p.v.post[col]));
    }
  }
}

// ---- launches ----------------------------------------------------------------------------------------------------

template <int NC, int SLOTS, bool FULL>
static int launch_sandwich_fwd(const SandwichFwd& a, int wpr, cudaStream_t st) {
  static std::atomic<bool> done[64];
  auto kern = sandwich_fwd_kernel<NC, SLOTS, FULL>;
  constexpr int stage = kSwWarps * SLOTS * NC * 1024, most = kSwMaxCols * 8 + stage;
  static_assert(most + 512 <= 227 * 1024, "row slots exceed shared memory");
  if (int rc = allow_smem(kern, most, done)) return rc;
  const int rpb = kSwWarps / wpr;
  const int blocks = int(std::min<int64_t>((a.rows + rpb - 1) / rpb, int64_t(sm_count()) * sw_fwd_per_sm(NC, SLOTS)));
  TG_CUDA_CHECK(launch_early(kern, blocks, kSwWarps * 32, a.cols * 8 + stage, st, a, wpr));
  return TG_OK;
}
template <int NC, int SLOTS>
static int launch_fwd_case(const SandwichFwd& a, int chunks, cudaStream_t st) {
  const int wpr = (chunks + NC - 1) / NC;
  return a.cols == wpr * NC * 256 ? launch_sandwich_fwd<NC, SLOTS, true>(a, wpr, st) : launch_sandwich_fwd<NC, SLOTS, false>(a, wpr, st);
}
static int launch_fwd_case(const SandwichFwd& a, cudaStream_t st) {
  const int chunks = (a.cols + 255) / 256;
  if (chunks == 1) return launch_fwd_case<1, 2>(a, chunks, st);
  if (chunks == 2) return launch_fwd_case<2, 2>(a, chunks, st);
  if (chunks > 4 && chunks <= 8) return launch_fwd_case<2, 3>(a, chunks, st);
  // three pieces a warp where a block then has four fifths of the rows that it has with four (8000 x 2816 30.8 us with three, 32.6 with
  // four; 8000 x 4600, two rows instead of three, 57.0 and 52.3)
  if (kSwWarps / ((chunks + 2) / 3) * 5 >= kSwWarps / ((chunks + 3) / 4) * 4) return launch_fwd_case<3, 2>(a, chunks, st);
  return launch_fwd_case<4, 2>(a, chunks, st);
}

constexpr int kSwThreeMax = 15 * 256;          // (columns whose vectors fit beside the rows of three pieces a warp)
struct SandwichBwdGeom {
  int nchunk, wpr;
};
static SandwichBwdGeom sandwich_bwd_geom(int64_t cols) {
  const int chunks = int((cols + 255) / 256);
  const bool three = kSwWarps / ((chunks + 2) / 3) * 3 >= kSwWarps / ((chunks + 1) / 2) * 5 && chunks <= kSwThreeMax / 256;
  const int nchunk = chunks == 1 ? 1 : three ? 3 : 2;
  return {nchunk, (chunks + nchunk - 1) / nchunk};
}
static int sandwich_bwd_blocks(int64_t rows, int64_t cols) {
  const int rpb = kSwWarps / sandwich_bwd_geom(cols).wpr;
  return int(std::min<int64_t>((rows + rpb - 1) / rpb, sm_count()));
}
template <int NC, int SLOTS, bool FULL>
static int launch_sandwich_bwd(const SandwichBwd& a, int wpr, int blocks, cudaStream_t st) {
  static std::atomic<bool> done[64];
  auto kern = sandwich_bwd_kernel<NC, SLOTS, FULL>;
  constexpr int stage = kSwWarps * SLOTS * NC * 2048, most = (NC == 3 ? kSwThreeMax : SLOTS == 2 ? kSwMaxCols : kSwMaxCols / 2) * 8 + stage;
  static_assert(most + 512 <= 227 * 1024, "row slots exceed shared memory");
  if (int rc = allow_smem(kern, most, done)) return rc;
  TG_CUDA_CHECK(launch_early(kern, blocks, kSwWarps * 32, a.cols * 8 + stage, st, a, wpr));
  return TG_OK;
}


// Rows on their way while one is worked on: two, but one where the vectors or the pieces leave no room.
static int launch_bwd_case(const SandwichBwd& a, int blocks, cudaStream_t st) {
  const SandwichBwdGeom g = sandwich_bwd_geom(a.cols);
  const bool full = a.cols == g.wpr * g.nchunk * 256;
  if (g.nchunk == 1) return full ? launch_sandwich_bwd<1, 3, true>(a, g.wpr, blocks, st) : launch_sandwich_bwd<1, 3, false>(a, g.wpr, blocks, st);
  if (g.nchunk == 3) return full ? launch_sandwich_bwd<3, 2, true>(a, g.wpr, blocks, st) : launch_sandwich_bwd<3, 2, false>(a, g.wpr, blocks, st);
  if (a.cols <= 4096) return full ? launch_sandwich_bwd<2, 3, true>(a, g.wpr, blocks, st) : launch_sandwich_bwd<2, 3, false>(a, g.wpr, blocks, st);
  return full ? launch_sandwich_bwd<2, 2, true>(a, g.wpr, blocks, st) : launch_sandwich_bwd<2, 2, false>(a, g.wpr, blocks, st);
}

static bool gate_ok(const void* gate, int kind) {
  return kind == TG_GATE_NONE || ((kind == TG_GATE_CHANNEL || kind == TG_GATE_TOKEN) && gate != nullptr);
}
static bool gate_aligned(const void* gate, int kind) { return kind != TG_GATE_CHANNEL || aligned16(gate); }

}  // namespace tg

using namespace tg;

extern "C" int tg_sandwich_norm_fwd(const void* x, const void* branch, const void* post, const void* pre, const void* gate, int gate_kind,
                                    float residual_scale, float eps, void* x_new, void* h, void* q, float* scales, int64_t rows,
                                    int64_t cols, void* stream) {
  if (rows < 0 || cols <= 0 || cols % 8 != 0 || !gate_ok(gate, gate_kind) || post == nullptr || pre == nullptr || x_new == nullptr) return TG_ERR_SHAPE;
  if ((q == nullptr) != (scales == nullptr) || (q == nullptr && h == nullptr) || (q != nullptr && cols % kTile != 0)) return TG_ERR_SHAPE;
  if (cols > kSwMaxCols) return TG_ERR_TOO_LARGE;
  if (rows == 0) return TG_OK;
  if (x == nullptr || branch == nullptr) return TG_ERR_SHAPE;
  if (!aligned16(x) || !aligned16(branch) || !aligned16(post) || !aligned16(pre) || !gate_aligned(gate, gate_kind) || !aligned16(x_new) ||
      !aligned16(h) || !aligned16(q))
    return TG_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  using B = const __nv_bfloat16*;
  const SandwichFwd a = {B(x), B(branch), {B(post), B(pre), B(gate), gate_kind}, residual_scale, eps, static_cast<__nv_bfloat16*>(x_new),
                         static_cast<__nv_bfloat16*>(h), static_cast<uint8_t*>(q), scales, rows, int(cols)};
  return launch_fwd_case(a, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t tg_sandwich_norm_bwd_scratch_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > kSwMaxCols) return 0;
  return int64_t(sandwich_bwd_blocks(rows, cols)) * 2 * cols * int64_t(sizeof(float));
}

extern "C" int tg_sandwich_norm_bwd(const void* x_new, const void* branch, const void* post, const void* pre, const void* gate, int gate_kind,
                                    float residual_scale, float eps, const void* g_new, const void* g_h, void* dx, void* dbranch, void* dpost,
                                    void* dpre, void* dgate, void* scratch, int64_t rows, int64_t cols, void* stream) {
  if (rows < 0 || cols <= 0 || cols % 8 != 0 || !gate_ok(gate, gate_kind) || post == nullptr || pre == nullptr || dpost == nullptr || dpre == nullptr)
    return TG_ERR_SHAPE;
  if (cols > kSwMaxCols) return TG_ERR_TOO_LARGE;
  if (rows > 0 && (x_new == nullptr || branch == nullptr || dx == nullptr || dbranch == nullptr || scratch == nullptr)) return TG_ERR_SHAPE;
  if (!aligned16(x_new) || !aligned16(branch) || !aligned16(post) || !aligned16(pre) || !gate_aligned(gate, gate_kind) || !aligned16(g_new) ||
      !aligned16(g_h) || !aligned16(dx) || !aligned16(dbranch) || !aligned16(scratch))
    return TG_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    for (void* v : {dpost, dpre, gate_kind == TG_GATE_CHANNEL ? dgate : nullptr})
      if (v != nullptr) TG_CUDA_CHECK(cudaMemsetAsync(v, 0, size_t(cols) * 2, st));
    return TG_OK;
  }
  using B = const __nv_bfloat16*;
  using M = __nv_bfloat16*;
  const int blocks = sandwich_bwd_blocks(rows, cols);
  const SandwichVectors v = {B(post), B(pre), B(gate), gate_kind};
  const SandwichBwd a = {B(x_new), B(branch), v, residual_scale, eps, B(g_new), B(g_h), M(dx), M(dbranch), gate_kind == TG_GATE_TOKEN ? M(dgate) : nullptr,
                         static_cast<float*>(scratch), rows, int(cols)};
  if (int rc = launch_bwd_case(a, blocks, st)) return rc;
  const SandwichReduce red = {static_cast<const float*>(scratch), v, M(dpost), M(dpre), gate_kind == TG_GATE_CHANNEL ? M(dgate) : nullptr, blocks, int(cols)};
  TG_CUDA_CHECK(launch_if_short(true, sandwich_reduce_kernel, dim3(unsigned((cols + 31) / 32)), 1024, 0, st, red));
  return TG_OK;
}
