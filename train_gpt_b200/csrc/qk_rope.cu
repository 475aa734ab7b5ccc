// The norm of every head of queries and keys and the rotation by position, as one pass:
//
//     y = R(t) (w x r),   r = rsqrt(mean x^2 + eps)        backward, for the gradient g of y:  g' = R(-t) g,  a = w g',
//                                                           dx = r (a - x r^2 mean(a x)),  dw = sum over tokens and heads of g' x r
//
// x is a head of `dim` elements, w (dim) the scale of the queries or of the keys, R(t) the rotation of the pair (i, i + rotary / 2) -- or
// (2 i, 2 i + 1), interleaved -- by the angle t theta^(-2 i / rotary), i < rotary / 2; elements beyond `rotary` are not rotated.  Without
// scales there is no norm: y = R(t) x, and its backward pass is R(-t) g.  Float32 between the loads and the one rounding.  Angles are counted
// in turns, in 64 bits until whole turns are off: float32 would lose the place of a token far into a context (position 10^6 has an error of
// 0.06 rad in it).
//
// A pass is bound by memory (4 bytes an element forward, 6 backward), so the rest is kept small: a warp takes a token, its lanes work out
// the rotary / 2 sines and cosines once, and every head of queries and keys uses them from registers.  A head is a group of lanes, a power of
// two, with two 16-byte pieces each: piece c and the one rotary / 2 elements on, so that both elements of a pair are in one lane.  Heads
// go to several warps where there are few tokens.
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "norm.cuh"

namespace tg {

constexpr int kQkWarps = 4, kQkMaxDim = 512;

struct QkHeads {
  const __nv_bfloat16* at;
  int64_t batch, token, head;          // strides, elements
};
struct QkParams {
  QkHeads q, k, gq, gk;
  __nv_bfloat16 *q_out, *k_out;        // [token][head][dim]
  const __nv_bfloat16 *wq, *wk;
  const void* positions;
  int64_t pos_batch, pos_token;
  int pos_64;
  uint32_t tokens, n_tokens;           // of a sequence, of all
  int heads, kv_heads, dim, rotary;
  int splits, rounds;                  // warps that share a token, rounds of heads of each
  float eps, sign;                     // sign -1: the other way round
  float* partial;                      // [block][queries, keys][dim]
  double turns[kQkMaxDim / 2];         // theta^(-2 i / rotary) / 2 pi
};

__device__ __forceinline__ void qk_unpack(const uint4& w, float2 (&v)[4]) {
  v[0] = bf16x2_unpack(w.x);
  v[1] = bf16x2_unpack(w.y);
  v[2] = bf16x2_unpack(w.z);
  v[3] = bf16x2_unpack(w.w);
}
__device__ __forceinline__ uint4 qk_pack(const float2 (&v)[4]) {
  return make_uint4(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[1].x, v[1].y), pack_bf16x2(v[2].x, v[2].y), pack_bf16x2(v[3].x, v[3].y));
}
__device__ __forceinline__ float2 qk_splat(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 qk_neg(float2 v) { return make_float2(-v.x, -v.y); }

template <int G>
__device__ __forceinline__ float qk_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The two pieces of a lane, turned: cs holds four cosines of the first angles, then of the second, sn the sines.
template <bool INTER>
__device__ __forceinline__ void qk_rotate(float2 (&lo)[4], float2 (&hi)[4], const float2 (&cs)[4], const float2 (&sn)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (INTER) {     // pair j of a piece: its angle is half of cs[j / 2] (low piece) and cs[2 + j / 2]
      const float c0 = j & 1 ? cs[j / 2].y : cs[j / 2].x, s0 = j & 1 ? sn[j / 2].y : sn[j / 2].x;
      const float c1 = j & 1 ? cs[2 + j / 2].y : cs[2 + j / 2].x, s1 = j & 1 ? sn[2 + j / 2].y : sn[2 + j / 2].x;
      lo[j] = make_float2(fmaf(lo[j].x, c0, -lo[j].y * s0), fmaf(lo[j].x, s0, lo[j].y * c0));
      hi[j] = make_float2(fmaf(hi[j].x, c1, -hi[j].y * s1), fmaf(hi[j].x, s1, hi[j].y * c1));
    } else {
      const float2 a = lo[j], b = hi[j];
      lo[j] = __ffma2_rn(a, cs[j], qk_neg(__fmul2_rn(b, sn[j])));
      hi[j] = __ffma2_rn(a, sn[j], __fmul2_rn(b, cs[j]));
    }
  }
}

// What a lane does: its place in a head, and where its pieces are.
template <int G, bool INTER>
struct QkLane {
  int lane, warp, row, c, lo, hi, angle, angle2;
  bool on, rot;
  __device__ __forceinline__ explicit QkLane(const QkParams& p) {
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    row = lane / G;
    c = lane % G;
    on = c < p.dim / 16;
    const int n = p.rotary / 16;
    rot = c < n;
    lo = rot ? 8 * c : 16 * c;
    hi = rot ? p.rotary / 2 + 8 * c : lo + 8;
    angle = rot ? (INTER ? 4 * c : 8 * c) : 0;
    angle2 = rot ? (INTER ? p.rotary / 4 + 4 * c : 8 * c + 4) : 0;
  }
};

// A token's sines and cosines: worked out by the warp's lanes in turn, handed over in shared memory.
struct QkAngles {
  float2 cs[4], sn[4];
};
template <int G, bool INTER>
__device__ __forceinline__ void qk_angles(const QkParams& p, const QkLane<G, INTER>& l, const double* turns, float2* s_cs, uint32_t b, uint32_t t, QkAngles& a) {
  double at = double(t);
  if (p.positions != nullptr) {
    const int64_t i = int64_t(b) * p.pos_batch + int64_t(t) * p.pos_token;
    at = p.pos_64 ? double(static_cast<const int64_t*>(p.positions)[i]) : double(static_cast<const int32_t*>(p.positions)[i]);
  }
  __syncwarp();                        // the token before has been read
  for (int i = l.lane; i < p.rotary / 2; i += 32) {
    const double turn = at * turns[i];
    float s, c;
    sincospif(2.f * float(turn - rint(turn)), &s, &c);
    s_cs[i] = make_float2(c, p.sign * s);
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = (j < 2 ? l.angle : l.angle2) + 2 * (j & 1);
    const float2 u = l.rot ? s_cs[i] : make_float2(1.f, 0.f), v = l.rot ? s_cs[i + 1] : make_float2(1.f, 0.f);
    a.cs[j] = make_float2(u.x, v.x);
    a.sn[j] = make_float2(u.y, v.y);
  }
}

__device__ __forceinline__ const __nv_bfloat16* qk_at(const QkHeads& h, uint32_t b, uint32_t t, int head) {
  return h.at + int64_t(b) * h.batch + int64_t(t) * h.token + int64_t(head) * h.head;
}

template <int G, bool NORM, bool INTER>
__global__ void __launch_bounds__(kQkWarps * 32) qk_fwd_kernel(const __grid_constant__ QkParams p) {
  __shared__ double s_turns[kQkMaxDim / 2];
  __shared__ float2 s_cs[kQkWarps][kQkMaxDim / 2];
  constexpr int RW = 32 / G, U = 2;
  const QkLane<G, INTER> l(p);
  for (int i = threadIdx.x; i < p.rotary / 2; i += kQkWarps * 32) s_turns[i] = p.turns[i];
  __syncthreads();
  grid_trigger();
  grid_wait();
  const int rows = p.heads + p.kv_heads;
  const float inv_dim = 1.f / float(p.dim);
  uint4 wq[2], wk[2];
  wq[0] = wq[1] = wk[0] = wk[1] = make_uint4(0u, 0u, 0u, 0u);      // (of lanes beyond the head: they add nothing to its sums)
  if (NORM && l.on) {
    wq[0] = *reinterpret_cast<const uint4*>(p.wq + l.lo);
    wq[1] = *reinterpret_cast<const uint4*>(p.wq + l.hi);
    wk[0] = *reinterpret_cast<const uint4*>(p.wk + l.lo);
    wk[1] = *reinterpret_cast<const uint4*>(p.wk + l.hi);
  }
  const uint64_t items = uint64_t(p.n_tokens) * uint32_t(p.splits);
  for (uint64_t item = uint64_t(blockIdx.x) * kQkWarps + l.warp; item < items; item += uint64_t(gridDim.x) * kQkWarps) {
    const uint32_t n = p.splits == 1 ? uint32_t(item) : uint32_t(item / uint32_t(p.splits));
    const int split = int(item - uint64_t(n) * uint32_t(p.splits));
    const uint32_t b = n / p.tokens, t = n - b * p.tokens;
    QkAngles a;
    bool turned = false;
    for (int round = 0; round < p.rounds; round += U) {
      uint4 x[U][2];
      int r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        r[u] = ((round + u) * p.splits + split) * RW + l.row;
        if (!l.on || round + u >= p.rounds) r[u] = rows;
        if (r[u] < rows) {
          const __nv_bfloat16* at = r[u] < p.heads ? qk_at(p.q, b, t, r[u]) : qk_at(p.k, b, t, r[u] - p.heads);
          x[u][0] = ld_stream_v4(at + l.lo);
          x[u][1] = ld_stream_v4(at + l.hi);
        } else {
          x[u][0] = x[u][1] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      if (!turned) {
        qk_angles(p, l, s_turns, s_cs[l.warp], b, t, a);
        turned = true;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float2 lo[4], hi[4];
        qk_unpack(x[u][0], lo);
        qk_unpack(x[u][1], hi);
        const bool is_q = r[u] < p.heads;
        if constexpr (NORM) {
          const float s = qk_sum<G>(sumsq8(x[u][0]) + sumsq8(x[u][1]));
          const float2 rn = qk_splat(__frsqrt_rn(fmaf(s, inv_dim, p.eps)));
          float2 w[4];
          qk_unpack(is_q ? wq[0] : wk[0], w);
#pragma unroll
          for (int j = 0; j < 4; ++j) lo[j] = __fmul2_rn(__fmul2_rn(lo[j], rn), w[j]);
          qk_unpack(is_q ? wq[1] : wk[1], w);
#pragma unroll
          for (int j = 0; j < 4; ++j) hi[j] = __fmul2_rn(__fmul2_rn(hi[j], rn), w[j]);
        }
        if (l.rot) qk_rotate<INTER>(lo, hi, a.cs, a.sn);
        if (r[u] < rows) {
          __nv_bfloat16* out = is_q ? p.q_out + (int64_t(n) * p.heads + r[u]) * p.dim : p.k_out + (int64_t(n) * p.kv_heads + (r[u] - p.heads)) * p.dim;
          *reinterpret_cast<uint4*>(out + l.lo) = qk_pack(lo);
          *reinterpret_cast<uint4*>(out + l.hi) = qk_pack(hi);
        }
      }
    }
  }
}

template <int G, bool INTER>
__global__ void __launch_bounds__(kQkWarps * 32) qk_bwd_kernel(const __grid_constant__ QkParams p) {
  __shared__ double s_turns[kQkMaxDim / 2];
  __shared__ float2 s_cs[kQkWarps][kQkMaxDim / 2];
  __shared__ float s_sum[kQkWarps][2][kQkMaxDim];
  constexpr int RW = 32 / G, U = 2;
  const QkLane<G, INTER> l(p);
  for (int i = threadIdx.x; i < p.rotary / 2; i += kQkWarps * 32) s_turns[i] = p.turns[i];
  __syncthreads();
  grid_trigger();
  grid_wait();
  const int rows = p.heads + p.kv_heads;
  const float inv_dim = 1.f / float(p.dim);
  uint4 wq[2], wk[2];
  wq[0] = wq[1] = wk[0] = wk[1] = make_uint4(0u, 0u, 0u, 0u);      // (of lanes beyond the head: they add nothing to its sums)
  if (l.on) {
    wq[0] = *reinterpret_cast<const uint4*>(p.wq + l.lo);
    wq[1] = *reinterpret_cast<const uint4*>(p.wq + l.hi);
    wk[0] = *reinterpret_cast<const uint4*>(p.wk + l.lo);
    wk[1] = *reinterpret_cast<const uint4*>(p.wk + l.hi);
  }
  float2 acc[2][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[0][j] = acc[1][j] = make_float2(0.f, 0.f);
  const uint64_t items = uint64_t(p.n_tokens) * uint32_t(p.splits);
  for (uint64_t item = uint64_t(blockIdx.x) * kQkWarps + l.warp; item < items; item += uint64_t(gridDim.x) * kQkWarps) {
    const uint32_t n = p.splits == 1 ? uint32_t(item) : uint32_t(item / uint32_t(p.splits));
    const int split = int(item - uint64_t(n) * uint32_t(p.splits));
    const uint32_t b = n / p.tokens, t = n - b * p.tokens;
    QkAngles a;
    bool turned = false;
    for (int round = 0; round < p.rounds; round += U) {
      uint4 x[U][2], g[U][2];
      int r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        r[u] = ((round + u) * p.splits + split) * RW + l.row;
        if (!l.on || round + u >= p.rounds) r[u] = rows;
        if (r[u] < rows) {
          const bool is_q = r[u] < p.heads;
          const __nv_bfloat16* at = is_q ? qk_at(p.q, b, t, r[u]) : qk_at(p.k, b, t, r[u] - p.heads);
          const __nv_bfloat16* from = is_q ? qk_at(p.gq, b, t, r[u]) : qk_at(p.gk, b, t, r[u] - p.heads);
          x[u][0] = ld_stream_v4(at + l.lo);
          x[u][1] = ld_stream_v4(at + l.hi);
          g[u][0] = ld_stream_v4(from + l.lo);
          g[u][1] = ld_stream_v4(from + l.hi);
        } else {
          x[u][0] = x[u][1] = g[u][0] = g[u][1] = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      if (!turned) {
        qk_angles(p, l, s_turns, s_cs[l.warp], b, t, a);
        turned = true;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float2 lo[4], hi[4], v[8];
        qk_unpack(g[u][0], lo);
        qk_unpack(g[u][1], hi);
        if (l.rot) qk_rotate<INTER>(lo, hi, a.cs, a.sn);
        const bool is_q = r[u] < p.heads;
        {
          float2 x0[4], x1[4];
          qk_unpack(x[u][0], x0);
          qk_unpack(x[u][1], x1);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[j] = x0[j];
            v[4 + j] = x1[j];
          }
        }
        float2 w[8];
        {
          float2 w0[4], w1[4];
          qk_unpack(is_q ? wq[0] : wk[0], w0);
          qk_unpack(is_q ? wq[1] : wk[1], w1);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            w[j] = __fmul2_rn(w0[j], lo[j]);
            w[4 + j] = __fmul2_rn(w1[j], hi[j]);
          }
        }
        float2 d2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 8; ++j) d2 = __ffma2_rn(w[j], v[j], d2);
        const float s = qk_sum<G>(sumsq8(x[u][0]) + sumsq8(x[u][1])), d = qk_sum<G>(d2.x + d2.y);
        const float rn = __frsqrt_rn(fmaf(s, inv_dim, p.eps));
        const float2 r2 = qk_splat(rn), m2 = qk_splat(-rn * rn * d * inv_dim);
        if (r[u] < rows) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 gx = __fmul2_rn(__fmul2_rn(j < 4 ? lo[j] : hi[j - 4], v[j]), r2);
            if (is_q) acc[0][j] = __fadd2_rn(acc[0][j], gx);
            else acc[1][j] = __fadd2_rn(acc[1][j], gx);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            lo[j] = __fmul2_rn(r2, __ffma2_rn(v[j], m2, w[j]));
            hi[j] = __fmul2_rn(r2, __ffma2_rn(v[4 + j], m2, w[4 + j]));
          }
          __nv_bfloat16* out = is_q ? p.q_out + (int64_t(n) * p.heads + r[u]) * p.dim : p.k_out + (int64_t(n) * p.kv_heads + (r[u] - p.heads)) * p.dim;
          *reinterpret_cast<uint4*>(out + l.lo) = qk_pack(lo);
          *reinterpret_cast<uint4*>(out + l.hi) = qk_pack(hi);
        }
      }
    }
  }
  // the scales' gradients: the warp's rows, then the block's warps in order
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float2 v = acc[which][j];
#pragma unroll
      for (int o = 16; o >= G; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
      }
      if (l.row == 0 && l.on) *reinterpret_cast<float2*>(&s_sum[l.warp][which][(j < 4 ? l.lo : l.hi) + 2 * (j & 3)]) = v;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.dim; i += kQkWarps * 32) {
    const int which = i >= p.dim, e = which ? i - p.dim : i;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kQkWarps; ++w) v += s_sum[w][which][e];
    p.partial[int64_t(blockIdx.x) * 2 * p.dim + i] = v;
  }
}

// Sums of the blocks' partial ones, 32 elements of either scale a block, warp w those of blocks w, w + 32, ...: an order that the number of
// blocks alone fixes.
__global__ void __launch_bounds__(1024) qk_scale_reduce_kernel(const float* partial, __nv_bfloat16* dq, __nv_bfloat16* dk, int blocks, int dim) {
  __shared__ float s_part[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  grid_wait();
  float v = 0.f;
  if (e < 2 * dim) {
#pragma unroll 4
    for (int i = warp; i < blocks; i += 32) v += __ldcg(partial + int64_t(i) * 2 * dim + e);
  }
  s_part[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && e < 2 * dim) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) t += s_part[w][lane];
    (e < dim ? dq : dk)[e < dim ? e : e - dim] = __float2bfloat16_rn(t);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------

static int qk_group(int dim) { return pow2_at_least(dim / 16) < 2 ? 2 : pow2_at_least(dim / 16); }

// How many warps share a token, so that few tokens still give every SM some, and the blocks of a launch.
struct QkGeom {
  int splits, rounds, blocks;
};
static QkGeom qk_geom(const tg_qk_args* a, int blocks_per_sm) {
  const int rw = 32 / qk_group(a->dim), rounds = (a->heads + a->kv_heads + rw - 1) / rw;
  const int64_t n = a->batch * a->tokens, want = int64_t(sm_count()) * kQkWarps * blocks_per_sm;
  QkGeom g;
  g.splits = int(std::max<int64_t>(1, std::min<int64_t>(rounds, want / std::max<int64_t>(n, 1))));
  g.rounds = (rounds + g.splits - 1) / g.splits;
  g.blocks = int(std::min<int64_t>((n * g.splits + kQkWarps - 1) / kQkWarps, int64_t(sm_count()) * blocks_per_sm));
  return g;
}
constexpr int kQkFwdPerSm = 8, kQkBwdPerSm = 4;

static bool qk_sizes_ok(const tg_qk_args* a) {
  return a->batch >= 0 && a->tokens >= 0 && a->heads >= 1 && a->kv_heads >= 1 && a->dim >= 16 && a->dim % 16 == 0 && a->rotary_dim >= 0 &&
         a->rotary_dim % 16 == 0 && a->rotary_dim <= a->dim && a->theta > 0.0 && isfinite(a->theta) && (a->q_scale == nullptr) == (a->k_scale == nullptr);
}
static bool qk_too_large(const tg_qk_args* a) {
  return a->dim > kQkMaxDim || a->heads > 65536 || a->kv_heads > 65536 || (a->tokens > 0 && a->batch >= (int64_t(1) << 31) / a->tokens);
}
static bool qk_strides_ok(const int64_t* s) { return s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0; }

static QkParams qk_params(const tg_qk_args* a, const QkGeom& g, float sign) {
  using B = const __nv_bfloat16*;
  QkParams p = {};
  p.q = {B(a->q), a->q_stride[0], a->q_stride[1], a->q_stride[2]};
  p.k = {B(a->k), a->k_stride[0], a->k_stride[1], a->k_stride[2]};
  p.gq = {B(a->g_q), a->g_q_stride[0], a->g_q_stride[1], a->g_q_stride[2]};
  p.gk = {B(a->g_k), a->g_k_stride[0], a->g_k_stride[1], a->g_k_stride[2]};
  p.q_out = static_cast<__nv_bfloat16*>(a->q_out);
  p.k_out = static_cast<__nv_bfloat16*>(a->k_out);
  p.wq = B(a->q_scale);
  p.wk = B(a->k_scale);
  p.positions = a->positions;
  p.pos_64 = a->positions_64;
  p.pos_batch = a->positions_stride[0];
  p.pos_token = a->positions_stride[1];
  p.tokens = uint32_t(a->tokens);
  p.n_tokens = uint32_t(a->batch * a->tokens);
  p.heads = a->heads;
  p.kv_heads = a->kv_heads;
  p.dim = a->dim;
  p.rotary = a->rotary_dim;
  p.splits = g.splits;
  p.rounds = g.rounds;
  p.eps = a->eps;
  p.sign = sign;
  p.partial = static_cast<float*>(a->scratch);
  // every eighth angle's step by a power, the ones between by products: an error of 8 2^-53 at most
  const double step = p.rotary > 0 ? pow(a->theta, -2.0 / p.rotary) : 1.0;
  for (int i = 0; i < p.rotary / 2; ++i)
    p.turns[i] = i % 8 == 0 ? pow(a->theta, -2.0 * i / p.rotary) / 6.283185307179586476925 : p.turns[i - 1] * step;
  return p;
}

template <int G>
static cudaError_t launch_qk_fwd(const QkParams& p, bool norm, bool inter, int blocks, cudaStream_t st) {
  auto kern = norm ? (inter ? qk_fwd_kernel<G, true, true> : qk_fwd_kernel<G, true, false>)
                   : (inter ? qk_fwd_kernel<G, false, true> : qk_fwd_kernel<G, false, false>);
  return launch_early(kern, blocks, kQkWarps * 32, 0, st, p);
}
template <int G>
static cudaError_t launch_qk_bwd(const QkParams& p, bool, bool inter, int blocks, cudaStream_t st) {
  return launch_early(inter ? qk_bwd_kernel<G, true> : qk_bwd_kernel<G, false>, blocks, kQkWarps * 32, 0, st, p);
}

}  // namespace tg

using namespace tg;

static int qk_check(const tg_qk_args* a) {
  if (a == nullptr || !qk_sizes_ok(a)) return TG_ERR_SHAPE;
  return qk_too_large(a) ? TG_ERR_TOO_LARGE : TG_OK;
}

extern "C" int tg_qk_norm_rope_fwd(const tg_qk_args* a, void* stream) {
  if (int rc = qk_check(a)) return rc;
  if (a->batch == 0 || a->tokens == 0) return TG_OK;
  if (a->q == nullptr || a->k == nullptr || a->q_out == nullptr || a->k_out == nullptr) return TG_ERR_SHAPE;
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->q_out) || !aligned16(a->k_out) || !aligned16(a->q_scale) || !aligned16(a->k_scale) ||
      !qk_strides_ok(a->q_stride) || !qk_strides_ok(a->k_stride))
    return TG_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  const QkGeom g = qk_geom(a, kQkFwdPerSm);
  const QkParams p = qk_params(a, g, 1.f);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool norm = a->q_scale != nullptr, inter = a->interleaved != 0;
  switch (qk_group(a->dim)) {
    case 2: TG_CUDA_CHECK(launch_qk_fwd<2>(p, norm, inter, g.blocks, st)); break;
    case 4: TG_CUDA_CHECK(launch_qk_fwd<4>(p, norm, inter, g.blocks, st)); break;
    case 8: TG_CUDA_CHECK(launch_qk_fwd<8>(p, norm, inter, g.blocks, st)); break;
    case 16: TG_CUDA_CHECK(launch_qk_fwd<16>(p, norm, inter, g.blocks, st)); break;
    default: TG_CUDA_CHECK(launch_qk_fwd<32>(p, norm, inter, g.blocks, st)); break;
  }
  return TG_OK;
}

extern "C" int64_t tg_qk_norm_rope_bwd_scratch_bytes(const tg_qk_args* a) {
  if (qk_check(a) != TG_OK || a->batch == 0 || a->tokens == 0 || a->q_scale == nullptr) return 0;
  return int64_t(qk_geom(a, kQkBwdPerSm).blocks) * 2 * a->dim * int64_t(sizeof(float));
}

extern "C" int tg_qk_norm_rope_bwd(const tg_qk_args* a, void* stream) {
  if (int rc = qk_check(a)) return rc;
  const bool norm = a->q_scale != nullptr, inter = a->interleaved != 0;
  if (norm && (a->dq_scale == nullptr || a->dk_scale == nullptr)) return TG_ERR_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->batch == 0 || a->tokens == 0) {
    if (int rc = check_arch()) return rc;
    for (void* v : {a->dq_scale, a->dk_scale})
      if (norm) TG_CUDA_CHECK(cudaMemsetAsync(v, 0, size_t(a->dim) * 2, st));
    return TG_OK;
  }
  if (a->g_q == nullptr || a->g_k == nullptr || a->q_out == nullptr || a->k_out == nullptr) return TG_ERR_SHAPE;
  if (norm && (a->q == nullptr || a->k == nullptr || a->scratch == nullptr)) return TG_ERR_SHAPE;
  if (!aligned16(a->g_q) || !aligned16(a->g_k) || !aligned16(a->q_out) || !aligned16(a->k_out) || !qk_strides_ok(a->g_q_stride) || !qk_strides_ok(a->g_k_stride))
    return TG_ERR_ALIGN;
  if (norm && (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->q_scale) || !aligned16(a->k_scale) || !aligned16(a->scratch) ||
               !qk_strides_ok(a->q_stride) || !qk_strides_ok(a->k_stride)))
    return TG_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  const QkGeom g = qk_geom(a, norm ? kQkBwdPerSm : kQkFwdPerSm);
  QkParams p = qk_params(a, g, -1.f);
  if (!norm) {
    p.q = p.gq;
    p.k = p.gk;
  }
  switch (qk_group(a->dim)) {
#define TG_QK_BWD(G) TG_CUDA_CHECK(norm ? launch_qk_bwd<G>(p, true, inter, g.blocks, st) : launch_qk_fwd<G>(p, false, inter, g.blocks, st))
    case 2: TG_QK_BWD(2); break;
    case 4: TG_QK_BWD(4); break;
    case 8: TG_QK_BWD(8); break;
    case 16: TG_QK_BWD(16); break;
    default: TG_QK_BWD(32); break;
#undef TG_QK_BWD
  }
  if (norm)
    TG_CUDA_CHECK(launch_if_short(true, qk_scale_reduce_kernel, dim3(unsigned((2 * a->dim + 31) / 32)), 1024, 0, st,
                                  static_cast<const float*>(a->scratch), static_cast<__nv_bfloat16*>(a->dq_scale),
                                  static_cast<__nv_bfloat16*>(a->dk_scale), g.blocks, a->dim));
  return TG_OK;
}
