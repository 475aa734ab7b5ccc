// Distillation from a teacher's top logits: the selection of those (forward only) and the student's loss with its gradient.
//
// Both work on capped logits z = c tanh(x / c) (train-gpt model.py:97) of bf16 logits x, in float32 and without the reference's bf16
// roundings in between.  No running maximum: |z / T| <= c / T <= 64, so that a sum of exp(z / T) neither overflows nor loses its terms.
//
// A row is cut into 16-byte pieces at the boundaries of MEMORY, so rows of any length and alignment are read with wide loads; the elements
// of its first and last piece that belong to other rows are read with them and take no part.
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "host_api.h"

namespace tg {

constexpr int kDsMaxThreads = 512;
constexpr int kDsMaxVocab = 1 << 20;
constexpr int64_t kDsDynamicMax = 208 * 1024;       // of shared memory; up to 17 KB more are static
constexpr int kTopMaxCandidates = 1024;
constexpr float kDsLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ds_ex2(float v) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v));
  return e;
}
__device__ __forceinline__ float ds_rcp(float v) {
  float e;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v));
  return e;
}

// The cap.  u = 1 - tanh |x / c| = 2 / (1 + exp(2 |x| / c)) keeps its relative precision where tanh saturates, so that
// sech^2(x / c) = u (2 - u) does too; z / T = sign(x) (c / T) (1 - u).
struct Cap {
  float k2;            // 2 log2(e) / c
  float zt;            // c log2(e) / T: z / T in powers of two is sign(x) zt (1 - u)
  float c, inv_c, inv_t;
  __device__ __forceinline__ Cap(float cap, float temperature) {
    c = cap;
    inv_c = __fdiv_rn(1.0f, cap);
    inv_t = __fdiv_rn(1.0f, temperature);
    k2 = 2.0f * kDsLog2e * inv_c;
    zt = cap * kDsLog2e * inv_t;
  }
  // u of the two logits of a word
  __device__ __forceinline__ float2 u2(uint32_t w) const {
    const float2 a = __fmul2_rn(bf16x2_unpack(w & 0x7fff7fffu), make_float2(k2, k2));
    const float2 d = __fadd2_rn(make_float2(ds_ex2(a.x), ds_ex2(a.y)), make_float2(1.f, 1.f));
    const float2 r = make_float2(ds_rcp(d.x), ds_rcp(d.y));
    return __fadd2_rn(r, r);
  }
  // s = sign(x) scale (1 - u), the capped logits in the units of `scale`
  static __device__ __forceinline__ float2 signed2(uint32_t w, float2 u, float scale) {
    const uint32_t b = __float_as_uint(scale);
    const float2 s = make_float2(__uint_as_float(b ^ ((w << 16) & 0x80000000u)), __uint_as_float(b ^ (w & 0x80000000u)));
    return __ffma2_rn(make_float2(-u.x, -u.y), s, s);
  }
  // the few logits of a row whose own value counts (kept ones, the target) by CUDA's accurate functions
  __device__ __forceinline__ float z_over_t(float x) const { return __fmul_rn(c * tanhf(x * inv_c), inv_t); }
  __device__ __forceinline__ float z(float x) const { return c * tanhf(x * inv_c); }
  __device__ __forceinline__ float sech2(float x) const {
    const float u = __fdiv_rn(2.0f, 1.0f + expf(2.0f * fabsf(x) * inv_c));
    return u * (2.0f - u);
  }
};

// A row's 16-byte pieces.
struct DsRow {
  const uint16_t* base;          // the 16-byte boundary at or below the row's start
  int off;                       // elements of the first piece that belong to what lies before the row
  int pieces, end;               // pieces that hold any element of the row; the row's end, counted from base
  __device__ __forceinline__ DsRow(const void* logits, int64_t row, int64_t ld, int vocab) {
    const uint16_t* s = static_cast<const uint16_t*>(logits) + row * ld;
    off = int((reinterpret_cast<uintptr_t>(s) & 15u) >> 1);
    base = s - off;
    end = off + vocab;
    pieces = (end + 7) >> 3;
  }
  // which elements of piece i are not the row's, a bit each
  __device__ __forceinline__ uint32_t outside(int i) const {
    uint32_t m = i == 0 ? (1u << off) - 1u : 0u;
    if (i == pieces - 1 && (end & 7)) m |= 0xffu & ~((1u << (end & 7)) - 1u);
    return m;
  }
};

__device__ __forceinline__ float ds_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sums over the block of N values a thread, the same bits in every thread.  `s` holds N floats a warp; a barrier has to lie between two
// uses of one `s`.
template <int N>
__device__ __forceinline__ void ds_block_sum(float (&v)[N], float* s, int warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = ds_warp_sum(v[n]);
  if (lane == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) s[n * (kDsMaxThreads / 32) + warp] = v[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float t = 0.f;
    for (int i = 0; i < warps; ++i) t += s[n * (kDsMaxThreads / 32) + i];
    v[n] = t;
  }
}

// log of part / (part + other), from the smaller of the two where the result is near 0
__device__ __forceinline__ float log_share(float part, float other) {
  const float total = part + other;
  return other < part ? log1pf(-__fdiv_rn(other, total)) : logf(__fdiv_rn(part, total));
}

// ---------------------------------------------------------------------------------------
// The student's loss and its gradient.  One thread block per row.  First pass: the sum of exp(z / T) (and of exp(z)) over all logits that the
// teacher does not name; those it does are marked in a bitmap, a byte per piece, and computed by one thread each.  Second pass: the gradient,
// from the row as it lies in shared memory (or, of a vocabulary that does not fit there, read again), after which the threads of the named
// logits and the target write theirs over it.
// ---------------------------------------------------------------------------------------
struct DistillArgs {
  const void* logits;
  const void* ids;
  const float* logp;
  const float* log_rest;
  const void* targets;
  int ids_64, targets_64;
  float cap, temperature, weight;
  void* d;
  const float* gscale;
  int only_if_scaled;
  float* row_loss;
  int rows, vocab, k;
  int64_t ld;
};

__device__ __forceinline__ int ds_index(const void* p, int is64, int64_t at, int vocab) {
  const int64_t v = is64 ? static_cast<const int64_t*>(p)[at] : static_cast<const int32_t*>(p)[at];
  return v >= 0 && v < vocab ? int(v) : -1;
}

template <bool TWO, bool GRAD, bool STAGED>
__global__ void __launch_bounds__(kDsMaxThreads) softcap_distill_kernel(const DistillArgs p) {
  grid_trigger();
  grid_wait();
  if (p.only_if_scaled && *p.gscale == 1.0f) return;
  extern __shared__ __align__(16) uint8_t s_ds[];
  __shared__ float s_red[6 * (kDsMaxThreads / 32)], s_loss[kDsMaxThreads / 32];
  __shared__ int s_ids[kDsMaxThreads];
  __shared__ float s_p[kDsMaxThreads];
  const int tid = int(threadIdx.x), nt = int(blockDim.x), warps = nt >> 5;
  const int map_words = (p.vocab + 14) / 8 / 4 + 1;
  uint32_t* s_map = reinterpret_cast<uint32_t*>(s_ds);
  const uint8_t* s_named = s_ds;
  uint4* s_row = reinterpret_cast<uint4*>(s_ds + (map_words * 4 + 15) / 16 * 16);
  for (int i = tid; i < map_words; i += nt) s_map[i] = 0u;
  const Cap cap(p.cap, p.temperature);
  const float z1 = p.cap * kDsLog2e;
  const float t = p.temperature, w_soft = p.weight, w_hard = 1.0f - p.weight;
  const float gs = GRAD ? (p.gscale != nullptr ? *p.gscale : 1.0f) * __fdiv_rn(1.0f, float(p.rows)) : 0.f;
  __syncthreads();

  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const DsRow q(p.logits, row, p.ld, p.vocab);
    const uint16_t* x_row = q.base + q.off;
    // ---- what the teacher names, a thread each
    int id = -1;
    float lp = 0.f, prob = 0.f, x = 0.f;
    if (tid < p.k) {
      id = ds_index(p.ids, p.ids_64, row * p.k + tid, p.vocab);
      if (id >= 0) {
        lp = p.logp[row * p.k + tid];
        prob = expf(lp);
        x = __uint_as_float(uint32_t(x_row[id]) << 16);
      }
    }
    const float rest = p.log_rest != nullptr ? p.log_rest[row] : -INFINITY;
    const int target = p.targets != nullptr ? ds_index(p.targets, p.targets_64, row, p.vocab) : -1;
    bool again = false;                        // another thread has the same logit
    if (id >= 0) {
      const int at = id + q.off;
      const uint32_t bit = 1u << (at & 31);
      again = atomicOr(s_map + (at >> 5), bit) & bit;
    }
    s_ids[tid] = id;
    s_p[tid] = prob;
    const bool repeats = __syncthreads_or(again);
    bool first = id >= 0;                      // it is this thread's to count the logit and to write its gradient
    float prob_here = prob;                    // the teacher's probability for the logit, entries that repeat it added up in order
    if (repeats && id >= 0) {
      prob_here = 0.f;
      for (int i = 0; i < p.k; ++i)
        if (s_ids[i] == id) {
          first &= i >= tid;
          prob_here += s_p[i];
        }
    }
    const float s_here = id >= 0 ? cap.z_over_t(x) : 0.f;
    const float e_here = id >= 0 ? expf(s_here) : 0.f;
    const float e1_here = TWO && id >= 0 ? expf(cap.z(x)) : 0.f;

    // ---- first pass
    float2 acc = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
    const uint4* src = reinterpret_cast<const uint4*>(q.base);
    uint4 w0 = tid < q.pieces ? ld_stream_v4(src + tid) : make_uint4(0u, 0u, 0u, 0u);
    uint4 w1 = tid + nt < q.pieces ? ld_stream_v4(src + tid + nt) : make_uint4(0u, 0u, 0u, 0u);
    for (int i = tid; i < q.pieces; i += nt) {
      const uint4 w = w0;
      w0 = w1;
      if (i + 2 * nt < q.pieces) w1 = ld_stream_v4(src + i + 2 * nt);
      if (GRAD && STAGED) s_row[i] = w;
      const uint32_t wi[4] = {w.x, w.y, w.z, w.w};
      const uint32_t skip = uint32_t(s_named[i]) | q.outside(i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 u = cap.u2(wi[j]);
        const float2 s = Cap::signed2(wi[j], u, cap.zt);
        float2 e = make_float2(ds_ex2(s.x), ds_ex2(s.y));
        if (skip) {
          if (skip >> (2 * j) & 1u) e.x = 0.f;
          if (skip >> (2 * j + 1) & 1u) e.y = 0.f;
        }
        acc = __fadd2_rn(acc, e);
        if (TWO) {
          const float2 sz = Cap::signed2(wi[j], u, z1);
          float2 e1 = make_float2(ds_ex2(sz.x), ds_ex2(sz.y));
          if (skip) {
            if (skip >> (2 * j) & 1u) e1.x = 0.f;
            if (skip >> (2 * j + 1) & 1u) e1.y = 0.f;
          }
          acc1 = __fadd2_rn(acc1, e1);
        }
      }
    }
    float sums[TWO ? 5 : 3] = {acc.x + acc.y, first ? e_here : 0.f, prob};
    if constexpr (TWO) {
      sums[3] = acc1.x + acc1.y;
      sums[4] = first ? e1_here : 0.f;
    }
    ds_block_sum(sums, s_red, warps);
    const float tail = sums[0], kept = sums[1], total = tail + kept, inv = __fdiv_rn(1.0f, total);
    const float total1 = TWO ? sums[3] + sums[TWO ? 4 : 0] : total;
    const float p_rest = expf(rest), mass = sums[2] + p_rest;

    // ---- the row's loss
    float term = 0.f;
    if (prob > 0.f) {
      const float share = e_here * inv;
      term = prob * (lp - (share > 1e-30f ? logf(share) : s_here - logf(total)));
    }
    float terms[1] = {term};
    ds_block_sum(terms, s_loss, warps);
    if (tid == 0 && p.row_loss != nullptr) {
      float loss = terms[0];
      if (p_rest > 0.f) loss += p_rest * (rest - log_share(tail, kept));
      loss *= w_soft * t * t;
      if (w_soft == 0.f) loss = 0.f;
      if (target >= 0 && w_hard != 0.f) {
        const float xt = __uint_as_float(uint32_t(x_row[target]) << 16);
        loss += w_hard * (logf(total1) - cap.z(xt));
      }
      p.row_loss[row] = loss;
    }

    // ---- second pass
    if constexpr (GRAD) {
      const float soft = w_soft * t;
      const float a = soft == 0.f ? 0.f : soft * (mass * inv - (p_rest > 0.f && tail > 0.f ? __fdiv_rn(p_rest, tail) : 0.f));
      const float b = target >= 0 && w_hard != 0.f ? w_hard * __fdiv_rn(1.0f, total1) : 0.f;
      uint16_t* d_base = static_cast<uint16_t*>(p.d) + (q.base - static_cast<const uint16_t*>(p.logits));
      const float ab = TWO ? a : a + b;
      const float2 a2 = make_float2(ab, ab), b2 = make_float2(b, b), gs2 = make_float2(gs, gs), two = make_float2(2.f, 2.f);
      for (int i = tid; i < q.pieces; i += nt) {
        const uint4 w = STAGED ? s_row[i] : ld_stream_v4(src + i);
        const uint32_t wi[4] = {w.x, w.y, w.z, w.w};
        uint4 o;
        uint32_t* op = &o.x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 u = cap.u2(wi[j]);
          const float2 s = Cap::signed2(wi[j], u, cap.zt);
          float2 g = __fmul2_rn(a2, make_float2(ds_ex2(s.x), ds_ex2(s.y)));
          if (TWO) {
            const float2 sz = Cap::signed2(wi[j], u, z1);
            g = __ffma2_rn(b2, make_float2(ds_ex2(sz.x), ds_ex2(sz.y)), g);
          }
          const float2 sech = __fmul2_rn(u, __fadd2_rn(two, make_float2(-u.x, -u.y)));
          g = __fmul2_rn(g, __fmul2_rn(sech, gs2));
          op[j] = pack_bf16x2(g.x, g.y);
        }
        const uint32_t skip = q.outside(i);
        if (skip == 0u) {
          *reinterpret_cast<uint4*>(d_base + i * 8) = o;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (!(skip >> j & 1u)) d_base[i * 8 + j] = uint16_t(j & 1 ? op[j >> 1] >> 16 : op[j >> 1] & 0xffffu);
        }
      }
      __syncthreads();
      auto write = [&](int at, float g, float x_at) {
        reinterpret_cast<__nv_bfloat16*>(d_base)[at + q.off] = __float2bfloat16_rn(g * (cap.sech2(x_at) * gs));
      };
      if (first) {
        float g = (soft == 0.f ? 0.f : soft * (mass * inv * e_here - prob_here)) + b * (TWO ? e1_here : e_here);
        if (id == target) g -= w_hard;
        write(id, g, x);
      }
      if (tid == 0 && target >= 0 && !(s_map[(target + q.off) >> 5] >> ((target + q.off) & 31) & 1u)) {
        const float xt = __uint_as_float(uint32_t(x_row[target]) << 16);
        const float e = expf(cap.z_over_t(xt));
        write(target, a * e + b * (TWO ? expf(cap.z(xt)) : e) - w_hard, xt);
      }
    }
    __syncthreads();                           // (the target's thread has read the bitmap)
    if (id >= 0) s_map[(id + q.off) >> 5] = 0u;
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------
// A teacher's top logits.  One thread block per row.  The first pass brings the row into shared memory and finds the largest logit of every
// group (the even and the odd elements of a thread's pieces are a group each).  The k-th largest of the groups' maxima is a lower bound of the
// k-th largest logit that few others reach: with 1024 groups about 1024 ln(1 / (1 - k / 1024)) logits.  The second pass collects those and sums
// exp(z / T) of all others; each candidate then counts the candidates before it, which is its place.
// Where the bound lets too many through (a row of equal logits, large ones side by side) the k-th largest logit is found by bisection on the
// row's 16-bit keys, and its equals are taken in the row's order.
// ---------------------------------------------------------------------------------------
struct TopArgs {
  const void* logits;
  float cap, temperature;
  int32_t* ids;
  float* logp;
  float* log_rest;
  int rows, vocab, k;
  int64_t ld;
};

// bf16 bits -> an unsigned key of the same order (-0 is 0; NaN above all)
__device__ __forceinline__ uint32_t top_key(uint32_t bits) {
  if ((bits & 0x7fffu) > 0x7f80u) return 0xffffu;
  return bits & 0x8000u ? 0x8000u - (bits & 0x7fffu) : 0x8000u + bits;
}
__device__ __forceinline__ uint32_t top_bits(uint32_t key) { return key >= 0x8000u ? key - 0x8000u : 0x8000u | (0x8000u - key); }

template <bool STAGED>
__global__ void __launch_bounds__(kDsMaxThreads) top_logits_kernel(const TopArgs p) {
  grid_trigger();
  grid_wait();
  extern __shared__ __align__(16) uint8_t s_ds[];
  __shared__ float s_red[2 * (kDsMaxThreads / 32)];
  __shared__ uint64_t s_cand[kTopMaxCandidates], s_sorted[kTopMaxCandidates];
  __shared__ int s_count[2][kDsMaxThreads / 32], s_n;
  uint4* s_row = reinterpret_cast<uint4*>(s_ds);
  const int tid = int(threadIdx.x), nt = int(blockDim.x), warps = nt >> 5, lane = tid & 31, warp = tid >> 5;
  const Cap cap(p.cap, p.temperature);
  const int k = p.k;

  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const DsRow q(p.logits, row, p.ld, p.vocab);
    const uint4* src = reinterpret_cast<const uint4*>(q.base);
    auto piece = [&](int i) { return STAGED ? s_row[i] : ld_stream_v4(src + i); };
    // ---- first pass: the groups' maxima
    uint32_t top[2] = {0u, 0u};
    {
      uint4 w0 = tid < q.pieces ? ld_stream_v4(src + tid) : make_uint4(0u, 0u, 0u, 0u);
      uint4 w1 = tid + nt < q.pieces ? ld_stream_v4(src + tid + nt) : make_uint4(0u, 0u, 0u, 0u);
      for (int i = tid; i < q.pieces; i += nt) {
        const uint4 w = w0;
        w0 = w1;
        if (i + 2 * nt < q.pieces) w1 = ld_stream_v4(src + i + 2 * nt);
        if (STAGED) s_row[i] = w;
        const uint32_t wi[4] = {w.x, w.y, w.z, w.w}, skip = q.outside(i);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(skip >> j & 1u)) top[j & 1] = max(top[j & 1], top_key(j & 1 ? wi[j >> 1] >> 16 : wi[j >> 1] & 0xffffu));
      }
    }
    // how many of the block's `n`s there are (the same value in every thread); two buffers, so that one barrier a call does
    int turn = 0;
    auto count = [&](int n) {
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) s_count[turn][warp] = n;
      __syncthreads();
      int c = 0;
      for (int i = 0; i < warps; ++i) c += s_count[turn][i];
      turn ^= 1;
      return c;
    };
    // the largest key that at least k of the groups reach (0: none)
    uint32_t lo = 0u;
    for (uint32_t bit = 0x8000u; bit != 0u; bit >>= 1)
      if (count(int(top[0] >= (lo | bit)) + int(top[1] >= (lo | bit))) >= k) lo |= bit;

    // ---- second pass: candidates, and the sum of the others.  `strict`: equals of the bound are counted, not collected
    float2 acc;
    int equal;
    auto collect = [&](uint32_t bound, bool strict) {
      if (tid == 0) s_n = 0;
      __syncthreads();
      acc = make_float2(0.f, 0.f);
      equal = 0;
      for (int i = tid; i < q.pieces; i += nt) {
        const uint4 w = piece(i);
        const uint32_t wi[4] = {w.x, w.y, w.z, w.w}, skip = q.outside(i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 u = cap.u2(wi[j]);
          const float2 s = Cap::signed2(wi[j], u, cap.zt);
          float2 e = make_float2(ds_ex2(s.x), ds_ex2(s.y));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = 2 * j + h;
            const uint32_t key = top_key(h ? wi[j] >> 16 : wi[j] & 0xffffu);
            if (skip >> at & 1u) {
              (h ? e.y : e.x) = 0.f;
            } else if (key >= bound) {
              (h ? e.y : e.x) = 0.f;
              if (strict && key == bound) {
                ++equal;
              } else {
                const int n = atomicAdd(&s_n, 1);
                if (n < kTopMaxCandidates) s_cand[n] = uint64_t(key) << 32 | uint32_t(~uint32_t(i * 8 + at - q.off));
              }
            }
          }
          acc = __fadd2_rn(acc, e);
        }
      }
      __syncthreads();
      return s_n;
    };
    int n = collect(lo, false);
    float extra = 0.f;                         // the sum of candidates that are not kept
    if (n > kTopMaxCandidates) {
      // the k-th largest key of the row
      uint32_t key = lo;
      for (uint32_t add = 0x8000u; add != 0u; add >>= 1) {
        const uint32_t probe = key + add;
        if (probe > 0xffffu) continue;
        int c = 0;
        for (int i = tid; i < q.pieces; i += nt) {
          const uint4 w = piece(i);
          const uint32_t wi[4] = {w.x, w.y, w.z, w.w}, skip = q.outside(i);
#pragma unroll
          for (int j = 0; j < 8; ++j) c += !(skip >> j & 1u) && top_key(j & 1 ? wi[j >> 1] >> 16 : wi[j >> 1] & 0xffffu) >= probe;
        }
        if (count(c) >= k) key = probe;
      }
      n = collect(key, true);                  // fewer than k
      const int equals = count(equal), want = k - n;
      // the first `want` of its equals: block after block of pieces, each thread's in its place by a prefix sum
      int have = 0;
      for (int i0 = 0; have < want; i0 += nt) {
        const int i = i0 + tid;
        uint32_t mine = 0u;
        if (i < q.pieces) {
          const uint4 w = piece(i);
          const uint32_t wi[4] = {w.x, w.y, w.z, w.w}, skip = q.outside(i);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (!(skip >> j & 1u) && top_key(j & 1 ? wi[j >> 1] >> 16 : wi[j >> 1] & 0xffffu) == key) mine |= 1u << j;
        }
        int before = __popc(mine);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += v;
        }
        if (lane == 31) s_count[turn][warp] = before;
        __syncthreads();
        int all = 0, at = have + before - __popc(mine);
        for (int v = 0; v < warps; ++v) {
          if (v < warp) at += s_count[turn][v];
          all += s_count[turn][v];
        }
        turn ^= 1;
        for (; mine != 0u && at < want; mine &= mine - 1u, ++at)
          s_cand[n + at] = uint64_t(key) << 32 | uint32_t(~uint32_t(i * 8 + __ffs(int(mine)) - 1 - q.off));
        have += all;
      }
      __syncthreads();
      if (tid == 0 && equals > want) extra = float(equals - want) * expf(cap.z_over_t(__uint_as_float(top_bits(key) << 16)));
      n = k;
    }
    // ---- each candidate's place; from there on all in the order of places, so that results do not depend on that of the atomics
    for (int i = tid; i < n; i += nt) {
      const uint64_t mine = s_cand[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += s_cand[j] > mine;
      s_sorted[r] = mine;
    }
    __syncthreads();
    float kept = 0.f, s = 0.f;
    for (int r = tid; r < n; r += nt) {
      const float v = cap.z_over_t(__uint_as_float(top_bits(uint32_t(s_sorted[r] >> 32)) << 16));
      if (r < k) {
        s = v;
        kept = expf(v);
      } else {
        extra += expf(v);
      }
    }
    float sums[2] = {acc.x + acc.y + extra, kept};
    ds_block_sum(sums, s_red, warps);
    if (tid < k) {
      p.ids[row * k + tid] = int32_t(~uint32_t(s_sorted[tid]));
      p.logp[row * k + tid] = s - logf(sums[0] + sums[1]);
    }
    if (tid == 0) p.log_rest[row] = log_share(sums[0], sums[1]);
    __syncthreads();
  }
}

// Threads for a row of `pieces` 16-byte pieces, two pieces each up to the most there are, and at least `least`.
static int ds_threads(int64_t pieces, int least) {
  const int64_t want = std::max<int64_t>((pieces + 63) / 64 * 32, (least + 31) / 32 * 32);
  return int(std::min<int64_t>(std::max<int64_t>(want, 32), kDsMaxThreads));
}
static int64_t ds_row_bytes(int64_t vocab) { return (vocab + 14) / 8 * 16; }
static int64_t ds_map_bytes(int64_t vocab) { return (((vocab + 14) / 8 / 4 + 1) * 4 + 15) / 16 * 16; }

// Dynamic shared memory for `kern`, once per device and kernel.
template <typename K>
static int ds_allow(K kern, std::atomic<bool> (&done)[64]) {
  int dev = 0;
  TG_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return TG_ERR_SHAPE;
  if (!done[dev].load(std::memory_order_acquire)) {
    TG_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kDsDynamicMax)));
    done[dev].store(true, std::memory_order_release);
  }
  return TG_OK;
}

template <bool TWO, bool GRAD, bool STAGED>
static int launch_distill(const DistillArgs& a, cudaStream_t st) {
  static std::atomic<bool> done[64];
  auto kern = softcap_distill_kernel<TWO, GRAD, STAGED>;
  if (int rc = ds_allow(kern, done)) return rc;
  const int64_t smem = ds_map_bytes(a.vocab) + (GRAD && STAGED ? ds_row_bytes(a.vocab) : 0);
  const int nt = ds_threads((a.vocab + 14) / 8, a.k);
  const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>({(227 * 1024) / (smem + 8 * 1024), 2048 / nt, 24}));
  const int blocks = int(std::min<int64_t>(a.rows, int64_t(sm_count()) * per_sm));
  TG_CUDA_CHECK(launch_if_short(int64_t(a.rows) * a.vocab <= 1 << 20, kern, dim3(unsigned(blocks)), nt, size_t(smem), st, a));
  return TG_OK;
}

template <bool STAGED>
static int launch_top(const TopArgs& a, cudaStream_t st) {
  static std::atomic<bool> done[64];
  auto kern = top_logits_kernel<STAGED>;
  if (int rc = ds_allow(kern, done)) return rc;
  const int64_t smem = STAGED ? ds_row_bytes(a.vocab) : 0;
  const int nt = ds_threads((a.vocab + 14) / 8, a.k);
  const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>({(227 * 1024) / (smem + 18 * 1024), 2048 / nt, 24}));
  const int blocks = int(std::min<int64_t>(a.rows, int64_t(sm_count()) * per_sm));
  TG_CUDA_CHECK(launch_if_short(int64_t(a.rows) * a.vocab <= 1 << 20, kern, dim3(unsigned(blocks)), nt, size_t(smem), st, a));
  return TG_OK;
}

static bool ds_cap_fits(float cap, float temperature) {
  return cap >= 0x1p-10f && cap <= 64.0f && temperature > 0.f && temperature <= 1024.0f && cap <= 64.0f * temperature;
}

}  // namespace tg

using namespace tg;

extern "C" int tg_top_logits(const void* logits, float cap, float temperature, int32_t* ids, float* logp, float* log_rest, int64_t rows,
                             int64_t vocab, int64_t ld, int k, void* stream) {
  if (rows < 0 || vocab <= 0 || ld < vocab || k <= 0 || k > vocab || ids == nullptr || logp == nullptr || log_rest == nullptr) return TG_ERR_SHAPE;
  if (!ds_cap_fits(cap, temperature)) return TG_ERR_SHAPE;
  if (rows > INT32_MAX || vocab > kDsMaxVocab || k > TG_TOP_LOGITS_MAX) return TG_ERR_TOO_LARGE;
  if (rows == 0) return TG_OK;
  if ((reinterpret_cast<uintptr_t>(logits) & 1u) != 0) return TG_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  const TopArgs a = {logits, cap, temperature, ids, logp, log_rest, int(rows), int(vocab), k, ld};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return ds_row_bytes(vocab) <= kDsDynamicMax ? launch_top<true>(a, st) : launch_top<false>(a, st);
}

extern "C" int tg_softcap_distill(const tg_distill_args* args, void* stream) {
  if (args == nullptr) return TG_ERR_SHAPE;
  const tg_distill_args& g = *args;
  if (g.rows < 0 || g.vocab <= 0 || g.ld < g.vocab || g.k < 0 || (g.k > 0 && (g.ids == nullptr || g.logp == nullptr))) return TG_ERR_SHAPE;
  if (!ds_cap_fits(g.cap, g.temperature) || !(g.weight >= 0.f && g.weight <= 1.f)) return TG_ERR_SHAPE;
  if (g.only_if_scaled && (g.gscale == nullptr || g.dlogits == nullptr)) return TG_ERR_SHAPE;
  if (g.dlogits == nullptr && g.row_loss == nullptr) return TG_ERR_SHAPE;
  if (g.rows > INT32_MAX || g.vocab > kDsMaxVocab || g.k > TG_TOP_LOGITS_MAX) return TG_ERR_TOO_LARGE;
  if (g.rows == 0) return TG_OK;
  if ((reinterpret_cast<uintptr_t>(g.logits) & 1u) != 0) return TG_ERR_ALIGN;
  if (g.dlogits != nullptr && ((reinterpret_cast<uintptr_t>(g.logits) ^ reinterpret_cast<uintptr_t>(g.dlogits)) & 15u) != 0) return TG_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  // one sum does where there is one temperature
  const bool soft = g.weight > 0.f, hard = g.weight < 1.f && g.targets != nullptr;
  const bool two = soft && hard && g.temperature != 1.0f;
  const DistillArgs a = {g.logits, g.ids, g.logp, g.log_rest, hard ? g.targets : nullptr, g.ids_64, g.targets_64, g.cap, soft ? g.temperature : 1.0f,
                         g.weight, g.dlogits, g.gscale, g.only_if_scaled, g.row_loss, int(g.rows), int(g.vocab), g.k, g.ld};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool staged = ds_map_bytes(g.vocab) + ds_row_bytes(g.vocab) <= kDsDynamicMax;
  if (g.dlogits == nullptr) return two ? launch_distill<true, false, false>(a, st) : launch_distill<false, false, false>(a, st);
  if (staged) return two ? launch_distill<true, true, true>(a, st) : launch_distill<false, true, true>(a, st);
  return two ? launch_distill<true, true, false>(a, st) : launch_distill<false, true, false>(a, st);
}
