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
#include "norm.cuh"

namespace tg {

constexpr int kDsMaxThreads = 512;
constexpr int kDsMaxVocab = 1 << 20;
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
__device__ __forceinline__ float ds_lds(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// The cap.  u = 1 - tanh |x / c| = 2 / (1 + exp(2 |x| / c)) keeps its relative precision where tanh saturates, so that
// sech^2(x / c) = u (2 - u) does too; z / T = sign(x) (c / T) (1 - u).  Handed out as -u.
//
// Two ways to it.  Two approximations of the special function unit, an exponential and a reciprocal (a third one is the exponential of
// z / T): 16 of them a clock and SM, so six clocks for 32 logits.  Or a table: x is a bf16 value, so between 2^-24 c, below
// which z is as good as +-2^-24 c, and 16 c, from where on tanh is 1, it has 29 binades of 128 values.  A look-up of 32 random entries
// takes 3.5 clocks of shared memory and leaves the special function unit two.
constexpr int kCapBinadesBelow = 24, kCapBinades = 29;
constexpr int kCapEntries = kCapBinades * 128 + 1;
constexpr int kCapTableBytes = (kCapEntries * 4 + 15) / 16 * 16;

template <bool TABLE>
struct Cap {
  float k2;            // 2 log2(e) / c
  float zt;            // c log2(e) / T: z / T in powers of two is sign(x) zt (1 - u)
  float c, inv_c, inv_t;
  uint32_t lo2, hi2;   // the table's first and last magnitude as bf16 bits, twice
  uint32_t tab2;       // (its address) - 4 lo, twice: plus a pair of magnitudes times 4, two 16-bit addresses
  __device__ __forceinline__ Cap(float cap, float temperature, void* table) {
    c = cap;
    inv_c = __fdiv_rn(1.0f, cap);
    inv_t = __fdiv_rn(1.0f, temperature);
    k2 = 2.0f * kDsLog2e * inv_c;
    zt = cap * kDsLog2e * inv_t;
    if constexpr (TABLE) {
      const uint32_t c_pow = (__float_as_uint(cap) >> 16) & 0x7f80u;     // 2^floor(log2 c)
      const uint32_t lo = c_pow - (kCapBinadesBelow << 7), hi = lo + (kCapBinades << 7);
      float* t = static_cast<float*>(table);
      for (int i = threadIdx.x; i < kCapEntries; i += blockDim.x)
        t[i] = __fdiv_rn(-2.0f, 1.0f + expf(2.0f * (__uint_as_float((lo + uint32_t(i)) << 16) * inv_c)));
      lo2 = lo * 0x10001u;
      hi2 = hi * 0x10001u;
      tab2 = (uint32_t(__cvta_generic_to_shared(table)) - 4u * lo) * 0x10001u;
    }
  }
  // -u of the two logits of a word.  `top` collects the largest magnitudes: the table has no NaN
  __device__ __forceinline__ float2 minus_u(uint32_t w, uint32_t& top) const {
    const uint32_t mag = w & 0x7fff7fffu;
    if constexpr (TABLE) {
      top = __vmaxu2(top, mag);
      const uint32_t at = __vminu2(__vmaxu2(mag, lo2), hi2) * 4u + tab2;
      return make_float2(ds_lds(at & 0xffffu), ds_lds(at >> 16));
    } else {
      const float2 a = __fmul2_rn(bf16x2_unpack(mag), make_float2(k2, k2));
      const float2 d = __fadd2_rn(make_float2(ds_ex2(a.x), ds_ex2(a.y)), make_float2(1.f, 1.f));
      return __fmul2_rn(make_float2(ds_rcp(d.x), ds_rcp(d.y)), make_float2(-2.f, -2.f));
    }
  }
  static __device__ __forceinline__ bool is_nan(uint32_t top) { return TABLE && ((top & 0xffffu) > 0x7f80u || (top >> 16) > 0x7f80u); }
  // sign(x) scale (1 - u), the capped logits in the units of `scale`
  static __device__ __forceinline__ float2 capped2(uint32_t w, float2 minus_u, float scale) {
    const uint32_t b = __float_as_uint(scale);
    const float2 s = make_float2(__uint_as_float(b ^ ((w << 16) & 0x80000000u)), __uint_as_float(b ^ (w & 0x80000000u)));
    return __ffma2_rn(minus_u, s, s);
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

// zeros in the place of a piece's elements that are not the row's
__device__ __forceinline__ void clear_outside(uint4& w, uint32_t out) {
  uint32_t* p = &w.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] &= (out >> (2 * j) & 1u ? 0u : 0xffffu) | (out >> (2 * j + 1) & 1u ? 0u : 0xffff0000u);
}

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
  for (int n = 0; n < N; ++n) v[n] = ds_warp_sum(lane < warps ? s[n * (kDsMaxThreads / 32) + lane] : 0.f);
}

// log of part / (part + other), from the smaller of the two where the result is near 0
__device__ __forceinline__ float log_share(float part, float other) {
  const float total = part + other;
  return other < part ? log1pf(-__fdiv_rn(other, total)) : logf(__fdiv_rn(part, total));
}

// ---------------------------------------------------------------------------------------
// The student's loss and its gradient.  One thread block per row.  First pass: the sum of exp(z / T) (and of exp(z)) over all logits that the
// teacher does not name; those it does are marked in a bitmap, a byte per piece, and computed by one thread each.  Second pass: the gradient,
// from the row read again -- 600 rows of 100 KB are in work at a time, which the L2 holds -- after which the threads of the named
// logits and the target write theirs over it.
// EXPS: 1 where one sum does (one temperature, or one of the two losses), 2 for two exponentials, 3 and 4 where the second is the first one
// squared once or twice (temperatures 2 and 4).
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

template <int EXPS, bool GRAD, bool TABLE>
__global__ void __launch_bounds__(kDsMaxThreads) softcap_distill_kernel(const DistillArgs p) {
  constexpr bool TWO = EXPS > 1;
  grid_trigger();
  grid_wait();
  if (p.only_if_scaled && *p.gscale == 1.0f) return;
  extern __shared__ __align__(16) uint8_t s_ds[];
  __shared__ float s_red[6 * (kDsMaxThreads / 32)], s_loss[kDsMaxThreads / 32];
  __shared__ int s_ids[kDsMaxThreads];
  __shared__ float s_p[kDsMaxThreads];
  const int tid = int(threadIdx.x), nt = int(blockDim.x), warps = nt >> 5;
  const int map_words = (p.vocab + 14) / 8 / 4 + 1;
  const uint8_t* s_named = s_ds + (TABLE ? kCapTableBytes : 0);
  uint32_t* s_map = reinterpret_cast<uint32_t*>(s_ds + (TABLE ? kCapTableBytes : 0));
  for (int i = tid; i < map_words; i += nt) s_map[i] = 0u;
  const Cap<TABLE> cap(p.cap, p.temperature, s_ds);
  const float z1 = p.cap * kDsLog2e;
  const float t = p.temperature, w_soft = p.weight, w_hard = 1.0f - p.weight;
  const float gs = GRAD ? (p.gscale != nullptr ? *p.gscale : 1.0f) * __fdiv_rn(1.0f, float(p.rows)) : 0.f;
  // exp(z) of a pair, from its exp(z / T) or anew
  auto second = [&](float2 e, uint32_t w, float2 nu) {
    if constexpr (EXPS > 2) {
#pragma unroll
      for (int i = 2; i < EXPS; ++i) e = __fmul2_rn(e, e);
      return e;
    } else {
      const float2 sz = Cap<TABLE>::capped2(w, nu, z1);
      return make_float2(ds_ex2(sz.x), ds_ex2(sz.y));
    }
  };
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
    uint32_t top = 0u;
    const uint4* src = reinterpret_cast<const uint4*>(q.base);
    uint4 w0 = tid < q.pieces ? ld_stream_v4(src + tid) : make_uint4(0u, 0u, 0u, 0u);
    uint4 w1 = tid + nt < q.pieces ? ld_stream_v4(src + tid + nt) : make_uint4(0u, 0u, 0u, 0u);
    for (int i = tid; i < q.pieces; i += nt) {
      uint4 w = w0;
      w0 = w1;
      if (i + 2 * nt < q.pieces) w1 = ld_stream_v4(src + i + 2 * nt);
      const uint32_t out = q.outside(i), skip = uint32_t(s_named[i]) | out;
      if (out) clear_outside(w, out);
      const uint32_t wi[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 nu = cap.minus_u(wi[j], top);
        const float2 s = Cap<TABLE>::capped2(wi[j], nu, cap.zt);
        float2 e = make_float2(ds_ex2(s.x), ds_ex2(s.y));
        if (skip) {
          if (skip >> (2 * j) & 1u) e.x = 0.f;
          if (skip >> (2 * j + 1) & 1u) e.y = 0.f;
        }
        acc = __fadd2_rn(acc, e);
        if constexpr (EXPS > 2) {
          acc1 = __fadd2_rn(acc1, second(e, wi[j], nu));
        } else if constexpr (EXPS == 2) {
          float2 e1 = second(e, wi[j], nu);
          if (skip) {
            if (skip >> (2 * j) & 1u) e1.x = 0.f;
            if (skip >> (2 * j + 1) & 1u) e1.y = 0.f;
          }
          acc1 = __fadd2_rn(acc1, e1);
        }
      }
    }
    if (Cap<TABLE>::is_nan(top)) acc.x = acc1.x = __int_as_float(0x7fffffff);
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
      const float2 a2 = make_float2(ab, ab), b2 = make_float2(b, b), gs2 = make_float2(-gs, -gs), two = make_float2(2.f, 2.f);
      w0 = tid < q.pieces ? ld_stream_v4(src + tid) : make_uint4(0u, 0u, 0u, 0u);
      w1 = tid + nt < q.pieces ? ld_stream_v4(src + tid + nt) : make_uint4(0u, 0u, 0u, 0u);
      for (int i = tid; i < q.pieces; i += nt) {
        const uint4 w = w0;
        w0 = w1;
        if (i + 2 * nt < q.pieces) w1 = ld_stream_v4(src + i + 2 * nt);
        const uint32_t wi[4] = {w.x, w.y, w.z, w.w};
        uint4 o;
        uint32_t* op = &o.x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 nu = cap.minus_u(wi[j], top);
          const float2 s = Cap<TABLE>::capped2(wi[j], nu, cap.zt);
          const float2 e = make_float2(ds_ex2(s.x), ds_ex2(s.y));
          float2 g = __fmul2_rn(a2, e);
          if (TWO) g = __ffma2_rn(b2, second(e, wi[j], nu), g);
          const float2 sech = __fmul2_rn(nu, __fadd2_rn(two, nu));       // (negative, as is gs2)
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
// A teacher's top logits.  One thread block per row.  The first pass finds the largest logit of every group (the even and the odd elements
// of a thread's pieces are a group each).  The k-th largest of the groups' maxima is a lower bound of the k-th largest logit
// that few others reach: with 1024 groups about 1024 ln(1 / (1 - k / 1024)) logits.  The second pass, over the row as the L2 holds it, collects
// those and sums exp(z / T) of all others.  Candidates are sorted by counting into bins of two keys, then within their bin.
// Where the bound lets too many through (a row of equal logits, large ones side by side), or a NaN is among them, the k-th largest logit is found by
// bisection on the row's 16-bit keys, and its equals are taken in the row's order.
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

constexpr int kTopBins = 256;

template <bool TABLE>
__global__ void __launch_bounds__(kDsMaxThreads) top_logits_kernel(const TopArgs p) {
  grid_trigger();
  grid_wait();
  extern __shared__ __align__(16) uint8_t s_ds[];
  __shared__ float s_red[2 * (kDsMaxThreads / 32)];
  __shared__ uint64_t s_cand[kTopMaxCandidates], s_sorted[kTopMaxCandidates];
  __shared__ __align__(16) int s_hist[kTopBins];
  __shared__ int s_begin[kTopBins], s_count[2][kDsMaxThreads / 32], s_n;
  __shared__ uint32_t s_bound;
  const int tid = int(threadIdx.x), nt = int(blockDim.x), warps = nt >> 5, lane = tid & 31, warp = tid >> 5;
  const Cap<TABLE> cap(p.cap, p.temperature, s_ds);
  const int k = p.k;
  __syncthreads();

  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const DsRow q(p.logits, row, p.ld, p.vocab);
    const uint4* src = reinterpret_cast<const uint4*>(q.base);
    // ---- first pass: the groups' maxima (NaN aside), as keys; 0 for a group of none
    uint32_t top[2];
    {
      uint4 w0 = tid < q.pieces ? ld_stream_v4(src + tid) : make_uint4(0u, 0u, 0u, 0u);
      uint4 w1 = tid + nt < q.pieces ? ld_stream_v4(src + tid + nt) : make_uint4(0u, 0u, 0u, 0u);
      __nv_bfloat162 m = __halves2bfloat162(__ushort_as_bfloat16(0x7fff), __ushort_as_bfloat16(0x7fff));
      for (int i = tid; i < q.pieces; i += nt) {
        uint4 w = w0;
        w0 = w1;
        if (i + 2 * nt < q.pieces) w1 = ld_stream_v4(src + i + 2 * nt);
        const uint32_t out = q.outside(i);
        uint32_t* wi = &w.x;
        if (out) {
#pragma unroll
          for (int j = 0; j < 4; ++j) wi[j] |= (out >> (2 * j) & 1u ? 0x7fffu : 0u) | (out >> (2 * j + 1) & 1u ? 0x7fff0000u : 0u);   // NaN
        }
        const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(wi);
        m = __hmax2(m, __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3])));
      }
      const uint32_t bits = *reinterpret_cast<const uint32_t*>(&m);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t b = h ? bits >> 16 : bits & 0xffffu;
        top[h] = (b & 0x7fffu) > 0x7f80u ? 0u : top_key(b);
      }
    }
    // how many of the block's `n`s there are (the same value in every thread); two buffers, so that one barrier a call does
    int turn = 0;
    auto count = [&](int n) {
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) s_count[turn][warp] = n;
      __syncthreads();
      const int c = __reduce_add_sync(0xffffffffu, lane < warps ? s_count[turn][lane] : 0);
      turn ^= 1;
      return c;
    };
    // ---- the bound: counts by distance from the largest, two keys a bin
    uint32_t largest = __reduce_max_sync(0xffffffffu, max(top[0], top[1]));
    if (lane == 0) s_count[turn][warp] = int(largest);
    for (int i = tid; i < kTopBins; i += nt) s_hist[i] = 0;
    __syncthreads();
    largest = __reduce_max_sync(0xffffffffu, lane < warps ? uint32_t(s_count[turn][lane]) : 0u);
    turn ^= 1;
    auto bin = [&](uint32_t key) { return key > largest ? 0u : min((largest - key) >> 1, uint32_t(kTopBins - 1)); };
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (top[h] != 0u) atomicAdd(s_hist + bin(top[h]), 1);
    __syncthreads();
    // warp 0: the first bin at which the running count reaches `want` (kTopBins: none), or all bins' beginnings
    auto scan = [&](int want, bool begins) {
      int v[kTopBins / 32], sum = 0;
#pragma unroll
      for (int j = 0; j < kTopBins / 32; j += 4) {
        const int4 b = reinterpret_cast<const int4*>(s_hist)[(lane * (kTopBins / 32) + j) / 4];
        v[j] = b.x; v[j + 1] = b.y; v[j + 2] = b.z; v[j + 3] = b.w;
      }
#pragma unroll
      for (int j = 0; j < kTopBins / 32; ++j) sum += v[j];
      int before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += x;
      }
      before -= sum;
      int found = kTopBins;
#pragma unroll
      for (int j = 0; j < kTopBins / 32; ++j) {
        if (begins) s_begin[lane * (kTopBins / 32) + j] = before;
        before += v[j];
        if (before >= want && found == kTopBins) found = lane * (kTopBins / 32) + j;
      }
      return int(__reduce_min_sync(0xffffffffu, unsigned(found)));
    };
    if (warp == 0) {
      const int b = scan(k, false);
      // (the last bin has everything further down: no bound)
      if (lane == 0) s_bound = b < kTopBins - 1 && largest > 2u * uint32_t(b) + 1u ? largest - 2u * uint32_t(b) - 1u : 0u;
      if (lane == 0) s_n = 0;
    }
    __syncthreads();
    uint32_t lo = s_bound;
    if (lo == 0u) {
      // the largest key that at least k of the groups reach (0: none)
      for (uint32_t bit = 0x8000u; bit != 0u; bit >>= 1)
        if (count(int(top[0] >= (lo | bit)) + int(top[1] >= (lo | bit))) >= k) lo |= bit;
    }

    // ---- second pass: candidates, and the sum of the others
    float2 acc = make_float2(0.f, 0.f);
    uint32_t nan = 0u;
    {
      const uint32_t bits = lo == 0u ? 0xff80u : top_bits(lo);           // (no bound: -inf)
      const __nv_bfloat162 bound = __halves2bfloat162(__ushort_as_bfloat16(uint16_t(bits)), __ushort_as_bfloat16(uint16_t(bits)));
      uint4 w0 = tid < q.pieces ? ld_stream_v4(src + tid) : make_uint4(0u, 0u, 0u, 0u);
      uint4 w1 = tid + nt < q.pieces ? ld_stream_v4(src + tid + nt) : make_uint4(0u, 0u, 0u, 0u);
      for (int i = tid; i < q.pieces; i += nt) {
        uint4 w = w0;
        w0 = w1;
        if (i + 2 * nt < q.pieces) w1 = ld_stream_v4(src + i + 2 * nt);
        const uint32_t out = q.outside(i);
        if (out) clear_outside(w, out);
        const uint32_t wi[4] = {w.x, w.y, w.z, w.w};
        uint32_t skip = out;
        uint32_t ge[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) ge[j] = __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&wi[j]), bound);
        if (ge[0] | ge[1] | ge[2] | ge[3]) {
          uint32_t hit = 0u;
#pragma unroll
          for (int j = 0; j < 4; ++j) hit |= (ge[j] & 1u) << (2 * j) | (ge[j] >> 31) << (2 * j + 1);
          hit &= ~out;
          skip |= hit;
          for (; hit != 0u; hit &= hit - 1u) {
            const int at = __ffs(int(hit)) - 1, n = atomicAdd(&s_n, 1);
            const uint32_t word = at < 4 ? (at < 2 ? wi[0] : wi[1]) : (at < 6 ? wi[2] : wi[3]);
            if (n < kTopMaxCandidates)
              s_cand[n] = uint64_t(top_key(at & 1 ? word >> 16 : word & 0xffffu)) << 32 | uint32_t(~uint32_t(i * 8 + at - q.off));
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 s = Cap<TABLE>::capped2(wi[j], cap.minus_u(wi[j], nan), cap.zt);
          float2 e = make_float2(ds_ex2(s.x), ds_ex2(s.y));
          if (skip) {
            if (skip >> (2 * j) & 1u) e.x = 0.f;
            if (skip >> (2 * j + 1) & 1u) e.y = 0.f;
          }
          acc = __fadd2_rn(acc, e);
        }
      }
    }
    if (Cap<TABLE>::is_nan(nan)) acc.x = __int_as_float(0x7fffffff);
    float others = acc.x + acc.y;
    const bool odd = __syncthreads_or(isnan(others));
    int n = s_n;
    float extra = 0.f;                         // the sum of candidates that are not kept
    if (n > kTopMaxCandidates || n < k || odd) {
      // the k-th largest key of the row
      auto keys_of = [&](int i, auto&& f) {
        const uint4 w = ld_stream_v4(src + i);
        const uint32_t wi[4] = {w.x, w.y, w.z, w.w}, skip = q.outside(i);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(skip >> j & 1u)) f(j, top_key(j & 1 ? wi[j >> 1] >> 16 : wi[j >> 1] & 0xffffu));
      };
      uint32_t key = 0u;
      for (uint32_t bit = 0x8000u; bit != 0u; bit >>= 1) {
        int c = 0;
        for (int i = tid; i < q.pieces; i += nt) keys_of(i, [&](int, uint32_t v) { c += v >= (key | bit); });
        if (count(c) >= k) key |= bit;
      }
      if (tid == 0) s_n = 0;
      __syncthreads();
      // those above it, fewer than k; how many equal it; the sum of those below
      int equal = 0;
      others = 0.f;
      for (int i = tid; i < q.pieces; i += nt)
        keys_of(i, [&](int j, uint32_t v) {
          if (v > key) s_cand[atomicAdd(&s_n, 1)] = uint64_t(v) << 32 | uint32_t(~uint32_t(i * 8 + j - q.off));
          else if (v == key) ++equal;
          else others += expf(cap.z_over_t(__uint_as_float(top_bits(v) << 16)));
        });
      const int equals = count(equal), above = s_n, want = k - above;
      // the first `want` of its equals: block after block of pieces, each thread's in its place by a prefix sum
      int have = 0;
      for (int i0 = 0; have < want; i0 += nt) {
        const int i = i0 + tid;
        uint32_t mine = 0u;
        if (i < q.pieces) keys_of(i, [&](int j, uint32_t v) { mine |= uint32_t(v == key) << j; });
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
          s_cand[above + at] = uint64_t(key) << 32 | uint32_t(~uint32_t(i * 8 + __ffs(int(mine)) - 1 - q.off));
        have += all;
      }
      __syncthreads();
      if (tid == 0 && equals > want) extra = float(equals - want) * expf(cap.z_over_t(__uint_as_float(top_bits(key) << 16)));
      n = k;
    }
    // ---- each candidate's place; from there on all in the order of places, so that results do not depend on that of the atomics
    for (int i = tid; i < kTopBins; i += nt) s_hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += nt) atomicAdd(s_hist + bin(uint32_t(s_cand[i] >> 32)), 1);
    __syncthreads();
    if (warp == 0) scan(0, true);
    __syncthreads();
    for (int i = tid; i < n; i += nt) {
      const uint64_t c = s_cand[i];
      s_sorted[atomicAdd(s_begin + bin(uint32_t(c >> 32)), 1)] = c;      // (a bin's beginning becomes its end)
    }
    __syncthreads();
    for (int i = tid; i < n; i += nt) {
      const uint64_t mine = s_sorted[i];
      const uint32_t b = bin(uint32_t(mine >> 32));
      const int end = s_begin[b], begin = end - s_hist[b];
      int r = begin;
      for (int j = begin; j < end; ++j) r += s_sorted[j] > mine;
      s_cand[r] = mine;
    }
    __syncthreads();
    float kept = 0.f, s = 0.f;
    for (int r = tid; r < n; r += nt) {
      const float v = cap.z_over_t(__uint_as_float(top_bits(uint32_t(s_cand[r] >> 32)) << 16));
      if (r < k) {
        s = v;
        kept = expf(v);
      } else {
        extra += expf(v);
      }
    }
    float sums[2] = {others + extra, kept};
    ds_block_sum(sums, s_red, warps);
    if (tid < k) {
      p.ids[row * k + tid] = int32_t(~uint32_t(s_cand[tid]));
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
static int64_t ds_map_bytes(int64_t vocab) { return (((vocab + 14) / 8 / 4 + 1) * 4 + 15) / 16 * 16; }

// Whether the logits that a block meets pay for its table.
static bool ds_table(int64_t rows, int64_t vocab) { return std::max<int64_t>(1, rows / (2 * sm_count())) * vocab >= 16384; }

// Blocks of nt threads that an SM holds of `kern`, whose registers and static shared memory are looked up once per device.
struct DsKernelInfo {
  std::atomic<int> registers[64];
  std::atomic<int> smem[64];
};
template <typename K>
static int ds_blocks(K kern, DsKernelInfo& info, int most_smem, int smem, int nt, int64_t rows, int* blocks) {
  int dev = 0;
  TG_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return TG_ERR_SHAPE;
  if (info.registers[dev].load(std::memory_order_acquire) == 0) {
    cudaFuncAttributes a;
    TG_CUDA_CHECK(cudaFuncGetAttributes(&a, kern));
    TG_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most_smem));
    info.smem[dev].store(int(a.sharedSizeBytes), std::memory_order_relaxed);
    info.registers[dev].store(a.numRegs, std::memory_order_release);
  }
  const int per_warp = (info.registers[dev].load(std::memory_order_acquire) * 32 + 255) / 256 * 256;
  const int64_t by_registers = 65536 / (int64_t(per_warp) * (nt / 32));
  const int64_t by_smem = (228 * 1024) / (smem + info.smem[dev].load(std::memory_order_relaxed) + 1024);
  const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>({by_registers, by_smem, 2048 / nt, 32}));
  *blocks = int(std::min<int64_t>(rows, sm_count() * per_sm));
  return TG_OK;
}

template <int EXPS, bool GRAD, bool TABLE>
static int launch_distill(const DistillArgs& a, int nt, cudaStream_t st) {
  static DsKernelInfo info;
  auto kern = softcap_distill_kernel<EXPS, GRAD, TABLE>;
  const int table = TABLE ? kCapTableBytes : 0, smem = int(ds_map_bytes(a.vocab)) + table;
  int blocks;
  if (int rc = ds_blocks(kern, info, int(ds_map_bytes(kDsMaxVocab)) + table, smem, nt, a.rows, &blocks)) return rc;
  TG_CUDA_CHECK(launch_if_short(int64_t(a.rows) * a.vocab <= 1 << 20, kern, dim3(unsigned(blocks)), nt, size_t(smem), st, a));
  return TG_OK;
}
template <int EXPS, bool GRAD>
static int launch_distill(const DistillArgs& a, cudaStream_t st) {
  const int nt = ds_threads((a.vocab + 14) / 8, a.k);
  return ds_table(a.rows, a.vocab) ? launch_distill<EXPS, GRAD, true>(a, nt, st) : launch_distill<EXPS, GRAD, false>(a, nt, st);
}

template <bool TABLE>
static int launch_top(const TopArgs& a, int nt, cudaStream_t st) {
  static DsKernelInfo info;
  const int smem = TABLE ? kCapTableBytes : 0;
  int blocks;
  if (int rc = ds_blocks(top_logits_kernel<TABLE>, info, smem, smem, nt, a.rows, &blocks)) return rc;
  TG_CUDA_CHECK(launch_if_short(int64_t(a.rows) * a.vocab <= 1 << 20, top_logits_kernel<TABLE>, dim3(unsigned(blocks)), nt, size_t(smem), st, a));
  return TG_OK;
}
static int launch_top(const TopArgs& a, cudaStream_t st) {
  const int nt = ds_threads((a.vocab + 14) / 8, a.k);
  return ds_table(a.rows, a.vocab) ? launch_top<true>(a, nt, st) : launch_top<false>(a, nt, st);
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
  return launch_top(a, st);
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
  const float t = soft ? g.temperature : 1.0f;
  const int exps = !(soft && hard) || t == 1.0f ? 1 : t == 2.0f ? 3 : t == 4.0f ? 4 : 2;
  const DistillArgs a = {g.logits, g.ids, g.logp, g.log_rest, hard ? g.targets : nullptr, g.ids_64, g.targets_64, g.cap, t,
                         g.weight, g.dlogits, g.gscale, g.only_if_scaled, g.row_loss, int(g.rows), int(g.vocab), g.k, g.ld};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool grad = g.dlogits != nullptr;
  if (exps == 1) return grad ? launch_distill<1, true>(a, st) : launch_distill<1, false>(a, st);
  if (exps == 2) return grad ? launch_distill<2, true>(a, st) : launch_distill<2, false>(a, st);
  if (exps == 3) return grad ? launch_distill<3, true>(a, st) : launch_distill<3, false>(a, st);
  return grad ? launch_distill<4, true>(a, st) : launch_distill<4, false>(a, st);
}
