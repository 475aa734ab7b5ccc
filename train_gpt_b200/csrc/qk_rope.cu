// The norm of every head of queries and keys and the rotation by position, as one pass:
//
//     y = R(t) (w x r),   r = rsqrt(mean x^2 + eps)        backward, for the gradient g of y:  g' = R(-t) g,  a = w g',
//                                                           dx = r (a - x r^2 mean(a x)),  dw = sum over tokens and heads of g' x r
//
// x is a head of `dim` elements, w (dim) the scale of the queries or of the keys, R(t) the rotation of the pair (i, i + rotary / 2) -- or
// (2 i, 2 i + 1), interleaved -- by the angle t theta^(-2 i / rotary), i < rotary / 2; elements beyond `rotary` are not rotated.  Without
// scales there is no norm: y = R(t) x, and its backward pass is R(-t) g.  Float32 between the loads and the one rounding.  Angles are counted
// in turns, in 64 bits until whole turns are off: float32 would lose the place of a token far into a context (position 10^6 has an error of
// 0.06 rad in it).  Two roundings of 2^-53 on the way to the turn and float32 behind it: an angle a is off by |a| 2^-52 + 2^-23 rad at most.
//
// A pass is bound by memory (4 bytes an element forward, 6 backward), so the rest is kept small: a warp takes a token; its lanes
// work out the rotary / 2 sines and cosines once, and every head of queries and of keys uses them from registers.  A head is a group of lanes, a power of two,
// with two 16-byte pieces each: piece c and the one rotary / 2 elements on, so that both elements of a pair are in one lane.  Heads go to several
// warps where there are few tokens.
//
// Pieces come through slots in shared memory by cp.async, rounds of heads ahead and across tokens, so that a warp never waits for a whole
// round trip; a lane reads only what it fetched itself.  32768 tokens (of 32 + 8 heads of 128 / 16 + 16 heads of 64): forward 107 / 48.5 us (6.3 / 5.5
// TB/s), backward 164 / 76 (6.1 / 5.3 TB/s); loads straight into registers 118 / 52 and 206 / 92.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "norm.cuh"

namespace tg {

constexpr int kQkMaxDim = 512;

struct QkHeads {
  const __nv_bfloat16* at;
  int64_t batch, token, head;          // strides, elements
};
// The queries, or the keys
struct QkPart {
  QkHeads x, g;
  __nv_bfloat16* out;                  // [token][head][dim]
  const __nv_bfloat16* w;
  int heads, rounds;                   // rounds of heads of each warp
};
struct QkParams {
  QkPart part[2];
  const void* positions;
  int64_t pos_batch, pos_token;
  int pos_64;
  uint32_t tokens, n_tokens;           // of a sequence, of all
  int dim, rotary, splits;             // splits: warps that share a token
  float eps, sign;                     // sign -1: the other way round
  float* partial;                      // [block][queries, keys][dim]
  double turns[kQkMaxDim / 2];         // theta^(-2 i / rotary) / 2 pi
};

__device__ __forceinline__ float2 qk_splat(float v) { return make_float2(v, v); }

template <int G>
__device__ __forceinline__ float qk_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
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

// A token's sines and cosines, worked out by the warp's lanes in turn and handed over in shared memory, as the coefficients of
//     turned[j] = own[j] from[j] + other[j] across[j]
// for the eight pairs of floats of a lane, the low piece first: `other` is the other piece's or, interleaved, the pair itself, swapped.
struct QkTurn {
  float2 from[8], across[8];
};
__device__ __forceinline__ void qk_angles(const QkParams& p, int lane, const double* turns, float2* s_cs, uint32_t b, uint32_t t) {
  double at = double(t);
  if (p.positions != nullptr) {
    const int64_t i = int64_t(b) * p.pos_batch + int64_t(t) * p.pos_token;
    at = p.pos_64 ? double(static_cast<const int64_t*>(p.positions)[i]) : double(static_cast<const int32_t*>(p.positions)[i]);
  }
  __syncwarp();                        // the token before has been read
  for (int i = lane; i < p.rotary / 2; i += 32) {
    const double turn = at * turns[i];
    float s, c;
    sincospif(2.f * float(turn - rint(turn)), &s, &c);
    s_cs[i] = make_float2(c, p.sign * s);
  }
  __syncwarp();
}
template <int G, bool INTER>
__device__ __forceinline__ void qk_turn(const QkLane<G, INTER>& l, const float2* s_cs, QkTurn& a) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {        // (cosine, sine) of two angles
    const float4 v = l.rot ? reinterpret_cast<const float4*>(s_cs)[((j < 2 ? l.angle : l.angle2) >> 1) + (j & 1)] : make_float4(1.f, 0.f, 1.f, 0.f);
    if constexpr (INTER) {
      a.from[2 * j] = make_float2(v.x, v.x);
      a.across[2 * j] = make_float2(-v.y, v.y);
      a.from[2 * j + 1] = make_float2(v.z, v.z);
      a.across[2 * j + 1] = make_float2(-v.w, v.w);
    } else {
      a.from[j] = a.from[4 + j] = make_float2(v.x, v.z);
      a.across[j] = make_float2(-v.y, -v.w);
      a.across[4 + j] = make_float2(v.y, v.w);
    }
  }
}
template <bool INTER>
__device__ __forceinline__ float2 qk_other(const float2 (&v)[8], int j) {
  return INTER ? make_float2(v[j].y, v[j].x) : v[j ^ 4];
}
template <bool INTER>
__device__ __forceinline__ void qk_rotate(float2 (&v)[8], const QkTurn& a) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 lo = __ffma2_rn(v[j], a.from[j], __fmul2_rn(qk_other<INTER>(v, j), a.across[j]));
    v[4 + j] = __ffma2_rn(v[4 + j], a.from[4 + j], __fmul2_rn(qk_other<INTER>(v, 4 + j), a.across[4 + j]));
    v[j] = lo;
  }
}
__device__ __forceinline__ void qk_unpack(const uint4& lo, const uint4& hi, float2 (&v)[8]) {
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = bf16x2_unpack(w[j]);
}
__device__ __forceinline__ void qk_store(__nv_bfloat16* out, int delta, const float2 (&v)[8]) {
  *reinterpret_cast<uint4*>(out) = make_uint4(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[1].x, v[1].y), pack_bf16x2(v[2].x, v[2].y), pack_bf16x2(v[3].x, v[3].y));
  *reinterpret_cast<uint4*>(out + delta) = make_uint4(pack_bf16x2(v[4].x, v[4].y), pack_bf16x2(v[5].x, v[5].y), pack_bf16x2(v[6].x, v[6].y), pack_bf16x2(v[7].x, v[7].y));
}

// A lane's part of a scale: read again for every token, from the L1, rather than kept in registers (0 for lanes beyond the head, whose
// values are 0 too).
template <int G, bool INTER>
__device__ __forceinline__ void qk_scale(const QkPart& q, const QkLane<G, INTER>& l, float2 (&w)[8]) {
  uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
  if (l.on) {
    lo = *reinterpret_cast<const uint4*>(q.w + l.lo);
    hi = *reinterpret_cast<const uint4*>(q.w + l.hi);
  }
  qk_unpack(lo, hi, w);
}

// Warps of a block, of which an SM has one: a grid of small blocks that leaves room for more of them is spread unevenly where the launch before it
// ends, and the SM with most of them ends last (32768 tokens of 40 heads of 128, rotated alone through slots: 123 us in blocks of four warps, 117 so).  Twelve backward:
// with 164 registers that is what fits; at sixteen the sums spill (32 x 1024 tokens of 32 heads of 64: 76 us, 112 with spills).
constexpr int kQkFwdWarps = 16, kQkBwdWarps = 12, kQkFewWarps = 4;
// Slots of a warp: more measured slower (forward with eight 110 us for 108 at 32768 tokens of 40 heads of 128, backward with seven 170 for 166).
constexpr int kQkFwdSlots = 3, kQkBwdSlots = 3;

// Shared memory: the turns, every warp's sines and cosines, every warp's slots
struct QkShared {
  double* turns;
  float2* cs;
  uint8_t* slots;
  __device__ __forceinline__ QkShared(uint8_t* at, int rotary, int warp, int warps)
      : turns(reinterpret_cast<double*>(at)), cs(reinterpret_cast<float2*>(at) + rotary / 2 * (1 + warp)), slots(at + rotary * 4 * (1 + warps)) {}
};
static int qk_shared_bytes(int rotary, int warps, int slot_bytes) { return rotary * 4 * (1 + warps) + warps * slot_bytes; }

// Warp w of block b takes tokens w * blocks + b, and on by as many as there are warps: what is left at the end goes to all SMs alike (3 x 1021 tokens of
// 16 heads of 80 8.0 us, 9.4 where a block's warps have neighbours).  Its rounds on their way to it: queries, then keys, token after token.  TENSORS: 1 forward (x), 2 backward (x and the
// gradient); a slot is two 16-byte pieces a lane of each.
template <int G, bool INTER, int TENSORS, int SLOTS>
struct QkStream {
  static constexpr int RW = 32 / G, kSlot = TENSORS * 1024;
  uint64_t item, items, step;
  const __nv_bfloat16 *x, *g;
  int64_t x_step, g_step;
  uint32_t base, slot, slot_in, b, t;
  int round, head, heads, next;
  __device__ __forceinline__ QkStream(const QkParams& p, const QkLane<G, INTER>& l, uint32_t smem)
      : item(uint64_t(l.warp) * gridDim.x + blockIdx.x), items(uint64_t(p.n_tokens) * uint32_t(p.splits)), step(uint64_t(gridDim.x) * (blockDim.x >> 5)), x(nullptr), g(nullptr), x_step(0),
        g_step(0), base(smem + uint32_t(l.warp) * (SLOTS * kSlot) + uint32_t(l.lane) * 16u), slot(0), slot_in((SLOTS - 1) * kSlot), b(0), t(0), round(0), head(0), heads(0), next(p.splits * RW) {
    if (!l.on) {                         // of lanes beyond the head: they add nothing to its sums
#pragma unroll
      for (int i = 0; i < SLOTS * TENSORS * 2; ++i) sts128(base + 512u * i, make_uint4(0u, 0u, 0u, 0u));
    }
#pragma unroll
    for (int i = 0; i < SLOTS - 1; ++i) fetch(p, l, i * kSlot);
  }
  __device__ __forceinline__ void fetch(const QkParams& p, const QkLane<G, INTER>& l, uint32_t to) {
    if (item < items) {
      const int rounds = p.part[0].rounds;
      if (round == 0 || round == rounds) {
        const QkPart& q = p.part[round != 0];
        uint32_t n = uint32_t(item), split = 0;
        if (p.splits != 1) {
          n = uint32_t(item / uint32_t(p.splits));
          split = uint32_t(item - uint64_t(n) * uint32_t(p.splits));
        }
        b = n / p.tokens;
        t = n - b * p.tokens;
        head = int(split) * RW + l.row;
        heads = l.on ? q.heads : 0;
        x = q.x.at + (int64_t(b) * q.x.batch + int64_t(t) * q.x.token + int64_t(head) * q.x.head + l.lo);
        x_step = q.x.head * next;
        if (TENSORS == 2) {
          g = q.g.at + (int64_t(b) * q.g.batch + int64_t(t) * q.g.token + int64_t(head) * q.g.head + l.lo);
          g_step = q.g.head * next;
        }
      }
      if (head < heads) {
        const uint32_t dst = base + to;
        cp_async16(dst, x);
        cp_async16(dst + 512, x + (l.hi - l.lo));
        if (TENSORS == 2) {
          cp_async16(dst + 1024, g);
          cp_async16(dst + 1536, g + (l.hi - l.lo));
        }
      }
      head += next;
      x += x_step;
      if (TENSORS == 2) g += g_step;
      if (++round == rounds + p.part[1].rounds) {
        round = 0;
        item += step;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");   // an empty group keeps the wait count uniform
  }
  // The oldest slot, once its pieces have arrived; the one that the round before has left is filled again.
  __device__ __forceinline__ uint32_t take(const QkParams& p, const QkLane<G, INTER>& l) {
    fetch(p, l, slot_in);
    asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 1) : "memory");
    const uint32_t at = base + slot;
    slot_in = slot;
    slot = slot == (SLOTS - 1) * kSlot ? 0u : slot + kSlot;
    return at;
  }
};

template <int G, bool INTER>
__global__ void __launch_bounds__(kQkFwdWarps * 32, 1) qk_fwd_kernel(const __grid_constant__ QkParams p) {
  extern __shared__ __align__(16) uint8_t s_qk[];
  constexpr int RW = 32 / G;
  const QkLane<G, INTER> l(p);
  const int warps = blockDim.x >> 5;
  const QkShared s_at(s_qk, p.rotary, l.warp, warps);
  for (int i = threadIdx.x; i < p.rotary / 2; i += blockDim.x) s_at.turns[i] = p.turns[i];
  __syncthreads();
  grid_trigger();
  grid_wait();
  const float inv_dim = 1.f / float(p.dim);
  const int delta = l.hi - l.lo, next = p.splits * RW;       // heads from one round to the next
  QkStream<G, INTER, 1, kQkFwdSlots> stream(p, l, uint32_t(__cvta_generic_to_shared(s_at.slots)));
  for (uint64_t item = uint64_t(l.warp) * gridDim.x + blockIdx.x; item < stream.items; item += stream.step) {
    const uint32_t n = p.splits == 1 ? uint32_t(item) : uint32_t(item / uint32_t(p.splits));
    const uint32_t b = n / p.tokens, t = n - b * p.tokens;
    const int first = int(item - uint64_t(n) * uint32_t(p.splits)) * RW + l.row;
    qk_angles(p, l.lane, s_at.turns, s_at.cs, b, t);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const QkPart& q = p.part[i];
      int head = first;
      __nv_bfloat16* out = q.out + (int64_t(n) * q.heads + head) * p.dim + l.lo;
      const int64_t out_step = int64_t(p.dim) * next;
      QkTurn a;
      qk_turn(l, s_at.cs, a);
      float2 w[8];                             // the scale goes into the coefficients
      qk_scale(q, l, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a.from[j] = __fmul2_rn(a.from[j], w[j]);
        a.across[j] = __fmul2_rn(a.across[j], qk_other<INTER>(w, j));
      }
#pragma unroll 1
      for (int round = 0; round < q.rounds; ++round) {
        const uint32_t slot = stream.take(p, l);
        // (a lane of a head that does not exist works on what its slot held before: its sums stay in its group, and nothing is stored)
        float2 v[8];
        qk_unpack(lds128(slot), lds128(slot + 512), v);
        float2 s2 = __fmul2_rn(v[0], v[0]), t2 = __fmul2_rn(v[1], v[1]);
#pragma unroll
        for (int j = 2; j < 8; j += 2) {
          s2 = __ffma2_rn(v[j], v[j], s2);
          t2 = __ffma2_rn(v[j + 1], v[j + 1], t2);
        }
        const float s = qk_sum<G>((s2.x + t2.x) + (s2.y + t2.y));
        const float2 rn = qk_splat(__frsqrt_rn(fmaf(s, inv_dim, p.eps)));
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fmul2_rn(v[j], rn);
        if (l.rot) {
          qk_rotate<INTER>(v, a);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = __fmul2_rn(v[j], a.from[j]);
        }
        if (l.on && head < q.heads) qk_store(out, delta, v);
        out += out_step;
        head += next;
      }
    }
  }
}

// The rotation alone (without scales, and backward without them): nothing waits for a sum, and loads straight into registers, four rounds at a time in
// blocks of four warps, four of them at a time on an SM, are ahead of the slots: 32768 tokens of 40 heads of 128 105 us (6.4 TB/s), 117 through slots;
// two rounds at a time 107, one 116.
constexpr int kQkTurnWarps = 4, kQkTurnRounds = 4, kQkTurnPerSm = 8;
template <int G, bool INTER>
__global__ void __launch_bounds__(kQkTurnWarps * 32, kQkTurnPerSm / 2) qk_turn_kernel(const __grid_constant__ QkParams p) {
  extern __shared__ __align__(16) uint8_t s_qk[];
  constexpr int RW = 32 / G, U = kQkTurnRounds;
  const QkLane<G, INTER> l(p);
  const QkShared s_at(s_qk, p.rotary, l.warp, kQkTurnWarps);
  for (int i = threadIdx.x; i < p.rotary / 2; i += blockDim.x) s_at.turns[i] = p.turns[i];
  __syncthreads();
  grid_trigger();
  grid_wait();
  const int delta = l.hi - l.lo, next = p.splits * RW;
  const uint64_t items = uint64_t(p.n_tokens) * uint32_t(p.splits), step = uint64_t(gridDim.x) * kQkTurnWarps;
  for (uint64_t item = uint64_t(blockIdx.x) * kQkTurnWarps + l.warp; item < items; item += step) {
    const uint32_t n = p.splits == 1 ? uint32_t(item) : uint32_t(item / uint32_t(p.splits));
    const uint32_t b = n / p.tokens, t = n - b * p.tokens;
    const int first = int(item - uint64_t(n) * uint32_t(p.splits)) * RW + l.row;
    QkTurn a;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const QkPart& q = p.part[i];
      int head = first;
      const __nv_bfloat16* in = q.x.at + (int64_t(b) * q.x.batch + int64_t(t) * q.x.token + int64_t(head) * q.x.head + l.lo);
      __nv_bfloat16* out = q.out + (int64_t(n) * q.heads + head) * p.dim + l.lo;
      const int64_t in_step = q.x.head * next, out_step = int64_t(p.dim) * next;
      for (int round = 0; round < q.rounds; round += U) {
        uint4 x[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          x[u][0] = x[u][1] = make_uint4(0u, 0u, 0u, 0u);
          if (l.on && head + u * next < q.heads) {        // (a round beyond the last has no heads)
            x[u][0] = ld_stream_v4(in);
            x[u][1] = ld_stream_v4(in + delta);
          }
          in += in_step;
        }
        if (i == 0 && round == 0) {
          qk_angles(p, l.lane, s_at.turns, s_at.cs, b, t);
          qk_turn(l, s_at.cs, a);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float2 v[8];
          qk_unpack(x[u][0], x[u][1], v);
          if (l.rot) qk_rotate<INTER>(v, a);
          if (l.on && head < q.heads) qk_store(out, delta, v);
          out += out_step;
          head += next;
        }
      }
    }
  }
}

template <int G, bool INTER>
__global__ void __launch_bounds__(kQkBwdWarps * 32, 1) qk_bwd_kernel(const __grid_constant__ QkParams p) {
  extern __shared__ __align__(16) uint8_t s_qk[];
  constexpr int RW = 32 / G;
  const QkLane<G, INTER> l(p);
  const int warps = blockDim.x >> 5;
  const QkShared s_at(s_qk, p.rotary, l.warp, warps);
  for (int i = threadIdx.x; i < p.rotary / 2; i += blockDim.x) s_at.turns[i] = p.turns[i];
  __syncthreads();
  grid_trigger();
  grid_wait();
  const float inv_dim = 1.f / float(p.dim);
  const int delta = l.hi - l.lo, next = p.splits * RW;
  QkStream<G, INTER, 2, kQkBwdSlots> stream(p, l, uint32_t(__cvta_generic_to_shared(s_at.slots)));
  float2 acc[2][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[0][j] = acc[1][j] = make_float2(0.f, 0.f);
  for (uint64_t item = uint64_t(l.warp) * gridDim.x + blockIdx.x; item < stream.items; item += stream.step) {
    const uint32_t n = p.splits == 1 ? uint32_t(item) : uint32_t(item / uint32_t(p.splits));
    const uint32_t b = n / p.tokens, t = n - b * p.tokens;
    const int first = int(item - uint64_t(n) * uint32_t(p.splits)) * RW + l.row;
    qk_angles(p, l.lane, s_at.turns, s_at.cs, b, t);
    QkTurn a;
    qk_turn(l, s_at.cs, a);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const QkPart& q = p.part[i];
      int head = first;
      __nv_bfloat16* out = q.out + (int64_t(n) * q.heads + head) * p.dim + l.lo;
      const int64_t out_step = int64_t(p.dim) * next;
      float2 w[8];
      qk_scale(q, l, w);
#pragma unroll 1
      for (int round = 0; round < q.rounds; ++round) {
        const uint32_t slot = stream.take(p, l);
        float2 v[8], o[8], m[8];
        qk_unpack(lds128(slot + 1024), lds128(slot + 1536), o);
        if (l.rot) qk_rotate<INTER>(o, a);
        qk_unpack(lds128(slot), lds128(slot + 512), v);
        float2 d2[2], s2[2];
        d2[0] = d2[1] = s2[0] = s2[1] = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 8; ++j) {          // o: the gradient times x, of the scale; m: times the scale
          m[j] = __fmul2_rn(w[j], o[j]);
          o[j] = __fmul2_rn(v[j], o[j]);
          s2[j & 1] = __ffma2_rn(v[j], v[j], s2[j & 1]);
          d2[j & 1] = __ffma2_rn(v[j], m[j], d2[j & 1]);
        }
        const float s = qk_sum<G>((s2[0].x + s2[1].x) + (s2[0].y + s2[1].y)), d = qk_sum<G>((d2[0].x + d2[1].x) + (d2[0].y + d2[1].y));
        const float rn = __frsqrt_rn(fmaf(s, inv_dim, p.eps));
        const float2 r2 = qk_splat(rn), n2 = qk_splat(-rn * rn * d * inv_dim);
        if (l.on && head < q.heads) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            acc[i][j] = __ffma2_rn(o[j], r2, acc[i][j]);
            m[j] = __fmul2_rn(r2, __ffma2_rn(v[j], n2, m[j]));
          }
          qk_store(out, delta, m);
        }
        out += out_step;
        head += next;
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float(*s_sum)[2][kQkMaxDim] = reinterpret_cast<float(*)[2][kQkMaxDim]>(s_at.slots);      // (idle now)
  static_assert(kQkBwdSlots * 2048 >= sizeof(float) * 2 * kQkMaxDim, "the sums have room in the slots");
  // the scales' gradients: the warp's rows, then the block's warps in order
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float2 v = acc[i][j];
#pragma unroll
      for (int o = 16; o >= G; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
      }
      if (l.row == 0 && l.on) *reinterpret_cast<float2*>(&s_sum[l.warp][i][(j < 4 ? l.lo : l.hi) + 2 * (j & 3)]) = v;
    }
  }
  __syncthreads();
  for (int at = threadIdx.x; at < 2 * p.dim; at += blockDim.x) {
    const int i = at >= p.dim, e = i ? at - p.dim : at;
    float v = 0.f;
    for (int k = 0; k < warps; ++k) v += s_sum[k][i][e];
    p.partial[int64_t(blockIdx.x) * 2 * p.dim + at] = v;
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

static int qk_group(int dim) { return std::max(2, pow2_at_least(dim / 16)); }

// How many warps share a token, so that few tokens still give every SM some, and the launch: as many blocks as an SM has of them, or small ones
// where there is less.
struct QkGeom {
  int splits, rounds[2], warps, blocks;
};
static QkGeom qk_geom(const tg_qk_args* a, int warps, int blocks_per_sm) {
  const int rw = 32 / qk_group(a->dim), all[2] = {(a->heads + rw - 1) / rw, (a->kv_heads + rw - 1) / rw};
  const int64_t n = a->batch * a->tokens, most = int64_t(sm_count()) * blocks_per_sm * warps;
  QkGeom g;
  g.splits = int(std::max<int64_t>(1, std::min<int64_t>(std::max(all[0], all[1]), most / std::max<int64_t>(n, 1))));
  for (int i = 0; i < 2; ++i) g.rounds[i] = (all[i] + g.splits - 1) / g.splits;
  g.warps = n * g.splits < most ? std::min(warps, kQkFewWarps) : warps;
  g.blocks = int(std::min<int64_t>(n * g.splits, most) / g.warps + (std::min<int64_t>(n * g.splits, most) % g.warps != 0));
  return g;
}
static QkGeom qk_geom_fwd(const tg_qk_args* a) { return a->q_scale != nullptr ? qk_geom(a, kQkFwdWarps, 1) : qk_geom(a, kQkTurnWarps, kQkTurnPerSm); }
static QkGeom qk_geom_bwd(const tg_qk_args* a) { return a->q_scale != nullptr ? qk_geom(a, kQkBwdWarps, 1) : qk_geom(a, kQkTurnWarps, kQkTurnPerSm); }

static bool qk_sizes_ok(const tg_qk_args* a) {
  return a->batch >= 0 && a->tokens >= 0 && a->heads >= 1 && a->kv_heads >= 1 && a->dim >= 16 && a->dim % 16 == 0 && a->rotary_dim >= 0 &&
         a->rotary_dim % 16 == 0 && a->rotary_dim <= a->dim && a->theta >= 1e-30 && isfinite(a->theta) && (a->q_scale == nullptr) == (a->k_scale == nullptr);
}
static bool qk_too_large(const tg_qk_args* a) {
  return a->dim > kQkMaxDim || a->heads > 65536 || a->kv_heads > 65536 || (a->tokens > 0 && a->batch >= (int64_t(1) << 31) / a->tokens);
}
static bool qk_strides_ok(const int64_t* s) { return s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0; }

static QkParams qk_params(const tg_qk_args* a, const QkGeom& g, bool backward) {
  using B = const __nv_bfloat16*;
  QkParams p = {};
  auto heads = [](const void* at, const int64_t* s) { return QkHeads{B(at), s[0], s[1], s[2]}; };
  const QkHeads gq = heads(a->g_q, a->g_q_stride), gk = heads(a->g_k, a->g_k_stride);
  const bool turn_back = backward && a->q_scale == nullptr;      // (a rotation of the gradients alone)
  p.part[0] = {turn_back ? gq : heads(a->q, a->q_stride), gq, static_cast<__nv_bfloat16*>(a->q_out), B(a->q_scale), a->heads, g.rounds[0]};
  p.part[1] = {turn_back ? gk : heads(a->k, a->k_stride), gk, static_cast<__nv_bfloat16*>(a->k_out), B(a->k_scale), a->kv_heads, g.rounds[1]};
  p.splits = g.splits;
  p.positions = a->positions;
  p.pos_64 = a->positions_64;
  p.pos_batch = a->positions_stride[0];
  p.pos_token = a->positions_stride[1];
  p.tokens = uint32_t(a->tokens);
  p.n_tokens = uint32_t(a->batch * a->tokens);
  p.dim = a->dim;
  p.rotary = a->rotary_dim;
  p.eps = a->eps;
  p.sign = backward ? -1.f : 1.f;
  p.partial = static_cast<float*>(a->scratch);
  // A step by a power, corrected by one of Newton's for theta step^n = 1, and products, in 64-bit mantissas: of 255 of them less than 2^-55 is left beside
  // the one rounding to double (1.04 2^-53 in all, measured).  0.08 us for 64 turns; by powl 0.34, by powers of doubles for every eighth and products
  // between them 0.15 and off by up to 9 2^-53.
  const int n = p.rotary / 2;
  if (n > 0) {
    long double step = pow(a->theta, -1.0 / n), all = 1.0L, square = step, turns = 1.0L / 6.283185307179586476925286766559L;
    for (int bits = n;; square *= square) {
      if (bits & 1) all *= square;
      if ((bits >>= 1) == 0) break;
    }
    step += step * (1.0L - a->theta * all) / n;
    for (int i = 0; i < n; ++i, turns *= step) p.turns[i] = double(turns);
  }
  return p;
}

template <int G, bool INTER>
static int launch_qk_fwd(const QkParams& p, const QkGeom& g, cudaStream_t st) {
  static std::atomic<bool> done[64];
  constexpr int most = kQkMaxDim * 4 * (1 + kQkFwdWarps) + kQkFwdWarps * kQkFwdSlots * 1024;
  static_assert(most <= 227 * 1024, "slots exceed shared memory");
  if (int rc = allow_smem(qk_fwd_kernel<G, INTER>, most, done)) return rc;
  TG_CUDA_CHECK(launch_early(qk_fwd_kernel<G, INTER>, g.blocks, g.warps * 32, qk_shared_bytes(p.rotary, g.warps, kQkFwdSlots * 1024), st, p));
  return TG_OK;
}
template <int G>
static int launch_qk_fwd(const QkParams& p, const QkGeom& g, bool norm, bool inter, cudaStream_t st) {
  if (norm) return inter ? launch_qk_fwd<G, true>(p, g, st) : launch_qk_fwd<G, false>(p, g, st);
  TG_CUDA_CHECK(launch_early(inter ? qk_turn_kernel<G, true> : qk_turn_kernel<G, false>, g.blocks, g.warps * 32, qk_shared_bytes(p.rotary, g.warps, 0), st, p));
  return TG_OK;
}
template <int G, bool INTER>
static int launch_qk_bwd(const QkParams& p, const QkGeom& g, cudaStream_t st) {
  static std::atomic<bool> done[64];
  constexpr int most = kQkMaxDim * 4 * (1 + kQkBwdWarps) + kQkBwdWarps * kQkBwdSlots * 2048;
  static_assert(most <= 227 * 1024, "slots exceed shared memory");
  if (int rc = allow_smem(qk_bwd_kernel<G, INTER>, most, done)) return rc;
  TG_CUDA_CHECK(launch_early(qk_bwd_kernel<G, INTER>, g.blocks, g.warps * 32, qk_shared_bytes(p.rotary, g.warps, kQkBwdSlots * 2048), st, p));
  return TG_OK;
}
template <int G>
static int launch_qk_bwd(const QkParams& p, const QkGeom& g, bool norm, bool inter, cudaStream_t st) {
  if (!norm) return launch_qk_fwd<G>(p, g, false, inter, st);
  return inter ? launch_qk_bwd<G, true>(p, g, st) : launch_qk_bwd<G, false>(p, g, st);
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
  const QkGeom g = qk_geom_fwd(a);
  const QkParams p = qk_params(a, g, false);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool norm = a->q_scale != nullptr, inter = a->interleaved != 0;
  switch (qk_group(a->dim)) {
    case 2: return launch_qk_fwd<2>(p, g, norm, inter, st);
    case 4: return launch_qk_fwd<4>(p, g, norm, inter, st);
    case 8: return launch_qk_fwd<8>(p, g, norm, inter, st);
    case 16: return launch_qk_fwd<16>(p, g, norm, inter, st);
    default: return launch_qk_fwd<32>(p, g, norm, inter, st);
  }
}

extern "C" int64_t tg_qk_norm_rope_bwd_scratch_bytes(const tg_qk_args* a) {
  if (qk_check(a) != TG_OK || a->batch == 0 || a->tokens == 0 || a->q_scale == nullptr) return 0;
  return int64_t(qk_geom_bwd(a).blocks) * 2 * a->dim * int64_t(sizeof(float));
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
  const QkGeom g = qk_geom_bwd(a);
  const QkParams p = qk_params(a, g, true);
  int rc = TG_OK;
  switch (qk_group(a->dim)) {
    case 2: rc = launch_qk_bwd<2>(p, g, norm, inter, st); break;
    case 4: rc = launch_qk_bwd<4>(p, g, norm, inter, st); break;
    case 8: rc = launch_qk_bwd<8>(p, g, norm, inter, st); break;
    case 16: rc = launch_qk_bwd<16>(p, g, norm, inter, st); break;
    default: rc = launch_qk_bwd<32>(p, g, norm, inter, st); break;
  }
  if (rc != TG_OK) return rc;
  if (norm)
    TG_CUDA_CHECK(launch_if_short(true, qk_scale_reduce_kernel, dim3(unsigned((2 * a->dim + 31) / 32)), 1024, 0, st,
                                  static_cast<const float*>(a->scratch), static_cast<__nv_bfloat16*>(a->dq_scale),
                                  static_cast<__nv_bfloat16*>(a->dk_scale), g.blocks, a->dim));
  return TG_OK;
}
