// Distillation from a teacher's top logits: the selection of those (forward only) and the student's loss with its gradient.
//
// Both work on capped logits z = c tanh(x / c) (train-gpt model.py:97) of bf16 logits x, in float32 and without the reference's bf16
// roundings in between.  No running maximum: |z / T| <= c / T <= 64, so that a sum of exp(z / T) neither overflows nor loses its terms.
//
// A row is cut into 16-byte pieces at the boundaries of MEMORY, so rows of any length and alignment are read with wide loads; the elements
// of its first and last piece that belong to other rows are read with them and take no part.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "host_api.h"
#include "norm.cuh"

namespace tg {

constexpr int kDsMaxThreads = 512;                  // of a row
// Threads of a block.  Those that keep their rows have the registers of half as many: 8192 x 50304 with 64 logits takes 427 us with 256 threads a
// row and two pieces of a thread's at a time, 541 with 512 and two pieces, 551 with 512 and one (64 registers spill).  Rows that are not kept
// come from memory with every read, and need the threads: 4096 x 130000 735 us, with half of them 897.
constexpr int ds_block_threads(bool staged) { return staged ? kDsMaxThreads : 2 * kDsMaxThreads; }
constexpr int64_t kDsSmemMax = 227 * 1024;
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
  asm("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// The cap.  u = 1 - tanh |x / c| = 2 / (1 + exp(2 |x| / c)) keeps its relative precision where tanh saturates, so that
// sech^2(x / c) = u (2 - u) does too; z / T = sign(x) (c / T) (1 - u).  Handed out as -u.
//
// Three approximations of the special function unit a logit (two exponentials and a reciprocal), 16 of them a clock and SM, are six clocks for 32
// logits.  x is a bf16 value, though, and everything here a function of it: between 2^-22 c, below which z is as good as +-2^-22 c,
// and 16 c, from where on tanh is 1, it has 27 binades of 128 values.  A table over those (of -u by the magnitude, or of E = exp(z / T)
// by magnitude and sign, twice that) makes it a look-up, 3.5 clocks of shared memory for 32 random entries, and fewer instructions.
// u goes on falling where tanh is 1, and sech^2 with it: the table of -u has two binades more (14.5 KB), up to where exp(2 |x| / c) overflows and u is 0.
// A quarter of the logits (the last word of four) goes the other way, so that both units work.
enum { kTabU = 1, kTabE = 2 };
constexpr int kCapBinadesBelow = 22;
constexpr int cap_entries(int table) { return (table & kTabU ? 29 : 27) * 128 + 1; }
constexpr int kCapSign = 4096;                                             // entries from the positive logits' to the negative ones'
constexpr int cap_bytes(int table) { return table == 0 ? 0 : ((table == kTabE ? kCapSign : 0) * 4 + cap_entries(table) * 4 + 15) / 16 * 16; }

template <int TABLES>
struct Cap {
  float k2;            // 2 log2(e) / c
  float zt;            // c log2(e) / T: z / T in powers of two is sign(x) zt (1 - u)
  float c, inv_c, inv_t;
  uint32_t minus_lo2;  // minus the table's first magnitude as bf16 bits, twice
  uint32_t tab2;       // its address, twice: plus a pair of entries times 4, two 16-bit addresses (which a block of a cluster's would exceed)
  __device__ __forceinline__ Cap(float cap, float temperature, void* tables) {
    c = cap;
    inv_c = __fdiv_rn(1.0f, cap);
    inv_t = __fdiv_rn(1.0f, temperature);
    k2 = 2.0f * kDsLog2e * inv_c;
    zt = cap * kDsLog2e * inv_t;
    if constexpr (TABLES != 0) {
      const uint32_t c_pow = (__float_as_uint(cap) >> 16) & 0x7f80u;     // 2^floor(log2 c)
      const uint32_t lo = c_pow - (kCapBinadesBelow << 7);
      float* t = static_cast<float*>(tables);
      for (int i = threadIdx.x; i < cap_entries(TABLES); i += blockDim.x) {
        const float nu = __fdiv_rn(-2.0f, 1.0f + expf(2.0f * (__uint_as_float((lo + uint32_t(i)) << 16) * inv_c)));
        if (TABLES & kTabU) t[i] = nu;
        if (TABLES & kTabE) {
          const float s = __fmaf_rn(nu, zt, zt);
          t[i] = ds_ex2(s);
          t[kCapSign + i] = ds_ex2(-s);
        }
      }
      minus_lo2 = ((0x10000u - lo) & 0xffffu) * 0x10001u;
      tab2 = uint32_t(__cvta_generic_to_shared(tables)) * 0x10001u;
    }
  }
  // two entries by magnitude, or by magnitude and sign
  __device__ __forceinline__ float2 look_up(uint32_t w, bool by_sign) const {
    uint32_t at = __viaddmin_s16x2_relu(w & 0x7fff7fffu, minus_lo2, uint32_t(cap_entries(TABLES) - 1) * 0x10001u);   // max(min(mag - lo, last), 0)
    if (by_sign) at |= (w >> 3) & 0x10001000u;
    at = at * 4u + tab2;
    return make_float2(ds_lds(at & 0xffffu), ds_lds(at >> 16));
  }
  __device__ __forceinline__ float2 direct_minus_u(uint32_t w) const {
    const float2 a = __fmul2_rn(bf16x2_unpack(w & 0x7fff7fffu), make_float2(k2, k2));
    const float2 d = __fadd2_rn(make_float2(ds_ex2(a.x), ds_ex2(a.y)), make_float2(1.f, 1.f));
    return __fmul2_rn(make_float2(ds_rcp(d.x), ds_rcp(d.y)), make_float2(-2.f, -2.f));
  }
  // sign(x) scale (1 - u), the capped logits in the units of `scale`
  static __device__ __forceinline__ float2 capped2(uint32_t w, float2 minus_u, float scale) {
    const uint32_t b = __float_as_uint(scale);
    const float2 s = make_float2(__uint_as_float(b ^ ((w << 16) & 0x80000000u)), __uint_as_float(b ^ (w & 0x80000000u)));
    return __ffma2_rn(minus_u, s, s);
  }
  static __device__ __forceinline__ float2 ex2_2(float2 s) { return make_float2(ds_ex2(s.x), ds_ex2(s.y)); }
  // -sech^2
  static __device__ __forceinline__ float2 minus_sech2(float2 nu) { return __fmul2_rn(nu, __fadd2_rn(make_float2(2.f, 2.f), nu)); }

  // Of the two logits of word J of a piece: -u, and E
  template <int J>
  __device__ __forceinline__ float2 minus_u(uint32_t w) const {
    if constexpr ((TABLES & kTabU) && J != 3) return look_up(w, false);
    else return direct_minus_u(w);
  }
  template <int J>
  __device__ __forceinline__ float2 e(uint32_t w) const {
    if constexpr ((TABLES & kTabE) && J != 3) return look_up(w, true);
    else return ex2_2(capped2(w, minus_u<J>(w), zt));
  }
  // The table has no NaN: the largest magnitude of each half of the words that were looked up, and whether one was among them
  static __device__ __forceinline__ uint32_t largest(const uint4& w) {
    return TABLES == 0 ? 0u : __vimax3_u16x2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu, w.z & 0x7fff7fffu);
  }
  static __device__ __forceinline__ bool is_nan(uint32_t top) { return TABLES != 0 && ((top & 0xffffu) > 0x7f80u || (top >> 16) > 0x7f80u); }
  // the few logits of a row whose own value counts (kept ones, the target) by CUDA's accurate functions
  __device__ __forceinline__ float z_over_t(float x) const { return __fmul_rn(c * tanhf(x * inv_c), inv_t); }
  __device__ __forceinline__ float z(float x) const { return c * tanhf(x * inv_c); }
  __device__ __forceinline__ float sech2(float x) const {
    const float u = __fdiv_rn(2.0f, 1.0f + expf(2.0f * fabsf(x) * inv_c));
    return u * (2.0f - u);
  }
};
// f(0, w.x), ... with the word's number as a constant
template <typename F>
__device__ __forceinline__ void four_words(const uint4& w, F&& f) {
  f(std::integral_constant<int, 0>(), w.x);
  f(std::integral_constant<int, 1>(), w.y);
  f(std::integral_constant<int, 2>(), w.z);
  f(std::integral_constant<int, 3>(), w.w);
}

// A row's 16-byte pieces.
struct DsRow {
  const uint16_t* base;          // the 16-byte boundary at or below the row's start
  int off;                       // elements of the first piece that belong to what lies before the row
  int end;                       // the row's end, counted from base
  __device__ __forceinline__ DsRow(const void* logits, int64_t row, int64_t ld, int vocab) {
    const uint16_t* s = static_cast<const uint16_t*>(logits) + row * ld;
    off = int((reinterpret_cast<uintptr_t>(s) & 15u) >> 1);
    base = s - off;
    end = off + vocab;
  }
  // the pieces that are the row's as a whole: [first, last); one more may lie before them and one behind
  __device__ __forceinline__ int first() const { return off != 0; }
  __device__ __forceinline__ int last() const { return end >> 3; }
  __device__ __forceinline__ const uint4* pieces() const { return reinterpret_cast<const uint4*>(base); }
  // The elements of the other two, one for each of sixteen lanes: its place counted from base, or -1
  __device__ __forceinline__ int edge(int lane) const {
    if (lane < 8) return off != 0 && lane >= off && lane < end ? lane : -1;
    const int e = last() * 8 + lane - 8;
    return lane < 16 && last() >= first() && e >= off && e < end ? e : -1;
  }
  // which elements of piece i are not the row's, a bit each
  __device__ __forceinline__ uint32_t outside(int i) const {
    uint32_t m = i == 0 ? (1u << off) - 1u : 0u;
    if (i == last()) m |= 0xffu & ~((1u << (end & 7)) - 1u);
    return m;
  }
};

// A thread's whole pieces of a row, every nt-th from its first one on: two of them are fetched by themselves, long before they are needed, and
// two stay on their way.
struct Pieces {
  uint4 w0, w1;
  __device__ __forceinline__ void fetch(const DsRow& q, int tid, int nt) {
    const int i = q.first() + tid;
    w0 = i < q.last() ? ld_stream_v4(q.pieces() + i) : make_uint4(0u, 0u, 0u, 0u);
    w1 = i + nt < q.last() ? ld_stream_v4(q.pieces() + i + nt) : make_uint4(0u, 0u, 0u, 0u);
  }
  // f(w, i) for each i below `end` (what is beyond the row's last is not read)
  template <typename F>
  __device__ __forceinline__ void each(const DsRow& q, int end, int tid, int nt, F&& f) {
    const int last = q.last();
    int i = q.first() + tid;
    const uint4* p = q.pieces() + i + 2 * nt;
#pragma unroll 1
    for (; i < end; i += 2 * nt, p += 2 * nt) {
      f(w0, i);
      if (i + 2 * nt < last) w0 = ld_stream_v4(p);
      if (i + nt < end) {
        f(w1, i + nt);
        if (i + 3 * nt < last) w1 = ld_stream_v4(p + nt);
      }
    }
  }
};

__device__ __forceinline__ float ds_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The threads that work on one row: a thread block, or one of up to eight groups of a block that share its table.
constexpr int kDsMaxGroups = 8;
struct Group {
  int index, tid, nt;
  __device__ __forceinline__ void sync() const { asm volatile("bar.sync %0, %1;" ::"r"(1 + index), "r"(nt) : "memory"); }
  __device__ __forceinline__ bool sync_or(bool v) const {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"(uint32_t(v)), "r"(1 + index), "r"(nt) : "memory");
    return r != 0u;
  }
};

// Sums over a group of N values a thread, the same bits in every thread, in two halves with a barrier between them: each warp's into `s`
// (N floats a warp), and those of the first `warps`.
template <int N>
__device__ __forceinline__ void ds_warp_sums(float (&v)[N], float* s, int warp, bool wanted) {
  if (!wanted) return;
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = ds_warp_sum(v[n]);
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) s[n * (kDsMaxThreads / 32) + warp] = v[n];
  }
}
template <int N>
__device__ __forceinline__ void ds_add_warps(float (&v)[N], const float* s, int warps) {
  const int at = threadIdx.x & (kDsMaxThreads / 32 - 1);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float t = at < warps ? s[n * (kDsMaxThreads / 32) + at] : 0.f;
#pragma unroll
    for (int o = kDsMaxThreads / 64; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    v[n] = t;
  }
}

// log of part / (part + other), from the smaller of the two where the result is near 0
__device__ __forceinline__ float log_share(float part, float other) {
  const float total = part + other;
  return other < part ? log1pf(-__fdiv_rn(other, total)) : logf(__fdiv_rn(part, total));
}

// ---------------------------------------------------------------------------------------
// The student's loss and its gradient.  A group of threads per row.  First pass: the sum of exp(z / T) (and of exp(z)) over all logits that the
// teacher does not name.  Those it does are marked in a bitmap, a byte per piece, and computed by one thread each; what else is in a piece with a
// mark is added by the thread of its lowest one, which is the same whatever the order of the marks was.  Second pass: the gradient, from the
// row as the first has left it in shared memory, after which the threads of the named logits and the target write theirs over it.
// (A vocabulary that does not fit is read again, about a third of it from memory: 4096 x 130000 735 us, 1.3 times the time a logit.)  Two rows of
// 50304 logits fit on an SM only with one table for both, hence the groups.
// A row has three barriers, and a chain of loads (an id, its logit) at its beginning: the next row's ids and logits are fetched a phase ahead, and
// its pieces take the places of this one's as the second pass leaves them.
// 8192 x 50304 with 64 logits: 427 us (3.9 TB/s); with a target 448 at T = 1, 465 at 2 and 4 (below), 603 at any other.  A row's 28100 cycles are 11800 of the first pass, 14100
// of the second, 2300 around the barriers; with two rows at once look-ups (3.5 cycles of shared memory for 32) keep that pipe busy for 68 %,
// exponentials theirs for 59 %, and instructions are issued in 62 % of the cycles.
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
  int groups, group_bytes;                     // of a block; shared memory of each behind the table
};

// an id as it is given, and -1 for one outside the vocabulary
__device__ __forceinline__ int ds_index(const void* p, int is64, int64_t at, int vocab) {
  const int64_t v = is64 ? static_cast<const int64_t*>(p)[at] : static_cast<const int32_t*>(p)[at];
  return v >= 0 && v < vocab ? int(v) : -1;
}

constexpr int distill_table(int exps, bool grad) { return exps == 2 || grad ? kTabU : kTabE; }
constexpr int ds_map_bytes(int64_t vocab) { return int(((vocab + 14) / 8 + 15) / 16 * 16); }
constexpr int64_t ds_row_bytes(int64_t vocab) { return (vocab + 14) / 8 * 16; }

template <int EXPS, bool GRAD, bool TABLE, bool STAGED>
__global__ void __launch_bounds__(ds_block_threads(STAGED), 1) softcap_distill_kernel(const DistillArgs p) {
  constexpr bool TWO = EXPS > 1;
  constexpr int TABLES = TABLE ? distill_table(EXPS, GRAD) : 0;
  using C = Cap<TABLES>;
  grid_trigger();
  grid_wait();
  if (p.only_if_scaled && *p.gscale == 1.0f) return;
  extern __shared__ __align__(16) uint8_t s_ds[];
  static_assert(kDsMaxGroups * 6 * (kDsMaxThreads / 32) * sizeof(float) <= 3 * 1024, "static shared memory beyond kDsStatic");
  __shared__ float s_reds[kDsMaxGroups][5 * (kDsMaxThreads / 32)], s_losses[kDsMaxGroups][kDsMaxThreads / 32];
  const C cap(p.cap, p.temperature, s_ds);
  const int nt = int(blockDim.x) / p.groups, index = int(threadIdx.x) / nt;
  const Group group = {index, int(threadIdx.x) - index * nt, nt};
  const int tid = group.tid, warps = nt >> 5, lane = tid & 31, warp = tid >> 5;
  float *const s_red = s_reds[index], *const s_loss = s_losses[index];
  uint8_t* const s_mine = s_ds + cap_bytes(TABLES) + index * p.group_bytes;
  const int map_bytes = ds_map_bytes(p.vocab);
  uint32_t* const s_map = reinterpret_cast<uint32_t*>(s_mine);
  const uint8_t* const s_named = s_mine;
  uint4* const s_row = reinterpret_cast<uint4*>(s_mine + map_bytes);       // the row's whole pieces, each in a place of its thread's own
  for (int i = tid; i < map_bytes / 4; i += nt) s_map[i] = 0u;
  const float z1 = p.cap * kDsLog2e;
  const float t = p.temperature, w_soft = p.weight, w_hard = 1.0f - p.weight;
  const float gs = GRAD ? (p.gscale != nullptr ? *p.gscale : 1.0f) * __fdiv_rn(1.0f, float(p.rows)) : 0.f;
  // exp(z) of a pair from its exp(z / T)
  auto squared = [&](float2 e) {
#pragma unroll
    for (int i = 2; i < EXPS; ++i) e = __fmul2_rn(e, e);
    return e;
  };
  // exp(z / T) and exp(z) of word J of a piece
  auto both = [&](auto j, uint32_t w, float2& e1) {
    constexpr int J = decltype(j)::value;
    if constexpr (EXPS == 2) {
      const float2 nu = cap.template minus_u<J>(w);
      e1 = C::ex2_2(C::capped2(w, nu, z1));
      return C::ex2_2(C::capped2(w, nu, cap.zt));
    } else {
      const float2 e = cap.template e<J>(w);
      e1 = squared(e);
      return e;
    }
  };

  // what a row needs besides its pieces, fetched in two steps
  int id = -1, target = -1;
  float lp = 0.f, rest = 0.f;
  uint4 named = make_uint4(0u, 0u, 0u, 0u);    // the piece of logit `id`
  uint32_t x_target = 0u, x_end = 0u;          // the target's logit (thread 0), that of this lane at the row's ends (last warp)
  auto fetch_ids = [&](int64_t row) {
    id = tid < p.k ? ds_index(p.ids, p.ids_64, row * p.k + tid, p.vocab) : -1;
    lp = id >= 0 ? p.logp[row * p.k + tid] : 0.f;
    rest = p.log_rest != nullptr ? p.log_rest[row] : -INFINITY;
    target = p.targets != nullptr ? ds_index(p.targets, p.targets_64, row, p.vocab) : -1;
  };
  auto fetch_logits = [&](const DsRow& q) {
    if (id >= 0) named = ld_stream_v4(q.pieces() + ((id + q.off) >> 3));
    if (tid == 0 && target >= 0) x_target = q.base[q.off + target];
    if (warp == warps - 1 && q.edge(lane) >= 0) x_end = q.base[q.edge(lane)];
  };

  __syncthreads();                             // (the table; from here on the groups go their own ways)
  const int64_t step = int64_t(gridDim.x) * p.groups;
  int64_t row = int64_t(blockIdx.x) * p.groups + index;
  if (row >= p.rows) return;
  DsRow q(p.logits, row, p.ld, p.vocab);
  Pieces in;                                   // (not STAGED)
  const uint32_t slot0 = uint32_t(__cvta_generic_to_shared(s_row)) + uint32_t(tid) * 16u;
  if constexpr (STAGED) {
    uint32_t to = slot0;
    const uint4* from = q.pieces() + q.first() + tid;
    for (int i = q.first() + tid; i < q.last(); i += nt, to += uint32_t(nt) * 16u, from += nt) cp_async16(to, from);
    asm volatile("cp.async.commit_group;" ::: "memory");
  } else {
    in.fetch(q, tid, nt);
  }
  fetch_ids(row);
  fetch_logits(q);
  while (row < p.rows) {
    // ---- what the teacher names, a thread each
    const int at = id + q.off;
    const bool present = id >= 0;
    bool again = false;                        // another thread has the same logit
    if (present) again = atomicOr(s_map + (at >> 5), 1u << (at & 31)) >> (at & 31) & 1u;
    const float prob = present ? expf(lp) : 0.f;
    float x = 0.f, s_here = 0.f, e_here = 0.f, e1_here = 0.f;
    if (present) {
      const uint32_t word = at & 4 ? (at & 2 ? named.w : named.z) : (at & 2 ? named.y : named.x);
      x = __uint_as_float(at & 1 ? word & 0xffff0000u : word << 16);
      s_here = cap.z_over_t(x);
      e_here = expf(s_here);
      e1_here = TWO ? expf(cap.z(x)) : 0.f;
    }
    const float xt_here = __uint_as_float(x_target << 16);             // (thread 0's)
    const float rest_here = rest, lp_here = lp;
    const int target_here = target, id_here = id;
    const bool repeats = group.sync_or(again);
    bool first = present;                      // it is this thread's to count the logit and to write its gradient
    float prob_here = prob;                    // the teacher's probability for the logit, entries that repeat it added up in order
    if (repeats && present) {
      prob_here = 0.f;
      for (int i = 0; i < p.k; ++i)
        if (ds_index(p.ids, p.ids_64, row * p.k + i, p.vocab) == id) {
          first &= i >= tid;
          prob_here += expf(p.logp[row * p.k + i]);
        }
    }
    const bool target_named = tid == 0 && target >= 0 && (s_map[(target + q.off) >> 5] >> ((target + q.off) & 31) & 1u);

    // ---- first pass
    float2 acc = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
    uint32_t top = 0u;
    auto add_some = [&](const uint4& w, uint32_t skip) {               // a piece's elements without a bit in `skip`
      four_words(w, [&](auto j, uint32_t v) {
        const uint32_t out = skip >> (2 * j) & 3u;
        v &= (out & 1u ? 0u : 0xffffu) | (out & 2u ? 0u : 0xffff0000u);
        if (TABLES != 0) top = __vmaxu2(top, v & 0x7fff7fffu);
        float2 e1;
        const float2 e = both(j, v, e1);
        acc = __fadd2_rn(acc, make_float2(out & 1u ? 0.f : e.x, out & 2u ? 0.f : e.y));
        if (TWO) acc1 = __fadd2_rn(acc1, make_float2(out & 1u ? 0.f : e1.x, out & 2u ? 0.f : e1.y));
      });
    };
    // (the named logits of a piece that is not the row's as a whole leave the others to the lanes below)
    if (first && at >> 3 >= q.first() && at >> 3 < q.last()) {
      const uint32_t marks = s_named[at >> 3];
      if ((marks & ((1u << (at & 7)) - 1u)) == 0u) add_some(named, marks);
    }
    // the two pieces at the row's ends, an element per lane of the last warp
    const int edge = warp == warps - 1 ? q.edge(lane) : -1;
    const bool edge_mine = edge >= 0 && !(s_map[edge >> 5] >> (edge & 31) & 1u);
    const float x_edge = __uint_as_float(x_end << 16);
    float e_edge = 0.f, e1_edge = 0.f;
    if (edge_mine) {
      e_edge = expf(cap.z_over_t(x_edge));
      e1_edge = TWO ? expf(cap.z(x_edge)) : 0.f;
      acc.x += e_edge;
      if (TWO) acc1.x += e1_edge;
    }
    const int64_t next = row + step;
    const DsRow q_next(p.logits, next < p.rows ? next : row, p.ld, p.vocab);
    if (next < p.rows) fetch_ids(next);
    auto add = [&](const uint4& w, int i) {
      const bool skip = s_named[i] != 0;
      float2 e[4], e1[4];
      four_words(w, [&](auto j, uint32_t v) { e[j] = both(j, v, e1[j]); });
      // (no branch: the look-ups do not wait for the mark)
      const float2 sum = __fadd2_rn(__fadd2_rn(e[0], e[1]), __fadd2_rn(e[2], e[3]));
      acc = __fadd2_rn(acc, make_float2(skip ? 0.f : sum.x, skip ? 0.f : sum.y));
      if (TABLE) top = __vmaxu2(top, C::largest(w));                 // (a NaN that is named is one of the row's all the same)
      if (TWO) {
        const float2 sum1 = __fadd2_rn(__fadd2_rn(e1[0], e1[1]), __fadd2_rn(e1[2], e1[3]));
        acc1 = __fadd2_rn(acc1, make_float2(skip ? 0.f : sum1.x, skip ? 0.f : sum1.y));
      }
    };
    if constexpr (STAGED) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      uint32_t slot = slot0;
#pragma unroll 2
      for (int i = q.first() + tid; i < q.last(); i += nt, slot += uint32_t(nt) * 16u) add(lds128(slot), i);
    } else {
      in.each(q, q.last(), tid, nt, add);
      in.fetch(GRAD ? q : q_next, tid, nt);
    }
    if (next < p.rows) fetch_logits(q_next);
    if (C::is_nan(top)) acc.x = acc1.x = __int_as_float(0x7fffffff);
    // (the entries' sums by the warps that have entries)
    const int entry_warps = (p.k + 31) >> 5;
    float of_row[TWO ? 2 : 1] = {acc.x + acc.y}, of_entries[TWO ? 3 : 2] = {first ? e_here : 0.f, prob};
    if constexpr (TWO) {
      of_row[1] = acc1.x + acc1.y;
      of_entries[2] = first ? e1_here : 0.f;
    }
    ds_warp_sums(of_row, s_red, warp, true);
    ds_warp_sums(of_entries, s_red + 2 * (kDsMaxThreads / 32), warp, warp < entry_warps);
    group.sync();
    ds_add_warps(of_row, s_red, warps);
    ds_add_warps(of_entries, s_red + 2 * (kDsMaxThreads / 32), entry_warps);
    const float tail = of_row[0], kept = of_entries[0], total = tail + kept, inv = __fdiv_rn(1.0f, total);
    const float total1 = TWO ? of_row[TWO ? 1 : 0] + of_entries[TWO ? 2 : 0] : total;
    const float p_rest = expf(rest_here), mass = of_entries[1] + p_rest;
    if (present) s_map[at >> 5] = 0u;          // (last looked at before the sums)
    // ---- the entries' share of the row's loss
    if (warp < entry_warps) {
      float term = 0.f;
      if (prob > 0.f) {
        const float share = e_here * inv;
        term = prob * (lp_here - (share > 1e-30f ? logf(share) : s_here - logf(total)));
      }
      term = ds_warp_sum(term);
      if (lane == 0) s_loss[warp] = term;
    }

    // ---- second pass
    const float soft = w_soft * t;
    const float a = soft == 0.f ? 0.f : soft * (mass * inv - (p_rest > 0.f && tail > 0.f ? __fdiv_rn(p_rest, tail) : 0.f));
    const float b = target_here >= 0 && w_hard != 0.f ? w_hard * __fdiv_rn(1.0f, total1) : 0.f;
    uint16_t* d_base = static_cast<uint16_t*>(p.d) + (q.base - static_cast<const uint16_t*>(p.logits));
    if constexpr (GRAD) {
      const float ab = TWO ? a : a + b;
      const float2 a2 = make_float2(ab, ab), b2 = make_float2(b, b), gs2 = make_float2(-gs, -gs);
      auto body = [&](const uint4& w, int i) {
        uint4 o;
        uint32_t* op = &o.x;
        four_words(w, [&](auto j, uint32_t v) {
          constexpr int J = decltype(j)::value;
          float2 g;
          const float2 nu = cap.template minus_u<J>(v), e = C::ex2_2(C::capped2(v, nu, cap.zt));
          g = __fmul2_rn(a2, e);
          if constexpr (TWO) {
            const float2 e1 = EXPS == 2 ? C::ex2_2(C::capped2(v, nu, z1)) : squared(e);
            g = __ffma2_rn(b2, e1, g);
          }
          g = __fmul2_rn(g, __fmul2_rn(C::minus_sech2(nu), gs2));
          op[J] = pack_bf16x2(g.x, g.y);
        });
        *reinterpret_cast<uint4*>(d_base + i * 8) = o;
      };
      if constexpr (STAGED) {
        // a place that has been read takes the next row's piece, of which there may be one more
        uint32_t slot = slot0;
        const uint4* from = q_next.pieces() + q_next.first() + tid;
        int more = next < p.rows ? q_next.last() - q_next.first() - tid : 0;
#pragma unroll 2
        for (int i = q.first() + tid; i < q.last(); i += nt, slot += uint32_t(nt) * 16u, from += nt, more -= nt) {
          const uint4 w = lds128(slot);
          if (more > 0) cp_async16(slot, from);
          body(w, i);
        }
        if (more > 0) cp_async16(slot, from);
        asm volatile("cp.async.commit_group;" ::: "memory");
      } else {
        in.each(q, q.last(), tid, nt, body);
        in.fetch(q_next, tid, nt);
      }
      if (edge_mine)
        reinterpret_cast<__nv_bfloat16*>(d_base)[edge] = __float2bfloat16_rn((a * e_edge + b * (TWO ? e1_edge : e_edge)) * (cap.sech2(x_edge) * gs));
    }
    group.sync();
    if constexpr (GRAD) {
      auto write = [&](int column, float g, float x_at) {
        reinterpret_cast<__nv_bfloat16*>(d_base)[column + q.off] = __float2bfloat16_rn(g * (cap.sech2(x_at) * gs));
      };
      if (first) {
        float g = (soft == 0.f ? 0.f : soft * (mass * inv * e_here - prob_here)) + b * (TWO ? e1_here : e_here);
        if (id_here == target_here) g -= w_hard;
        write(id_here, g, x);
      }
      if (tid == 0 && target_here >= 0 && !target_named) {
        const float e = expf(cap.z_over_t(xt_here));
        write(target_here, a * e + b * (TWO ? expf(cap.z(xt_here)) : e) - w_hard, xt_here);
      }
    }
    if (tid == 0 && p.row_loss != nullptr) {
      float loss = 0.f;
      for (int i = 0; i * 32 < p.k; ++i) loss += s_loss[i];
      if (p_rest > 0.f) loss += p_rest * (rest_here - log_share(tail, kept));
      loss = w_soft == 0.f ? 0.f : loss * (w_soft * t * t);
      if (target_here >= 0 && w_hard != 0.f) loss += w_hard * (logf(total1) - cap.z(xt_here));
      p.row_loss[row] = loss;
    }
    row = next;
    q = q_next;
  }
  if constexpr (STAGED) asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---------------------------------------------------------------------------------------
// A teacher's top logits.  A group of threads per row.  First a bound that at least k logits reach and few others: the largest logit of every
// group (each of the eight elements of a thread's pieces is one) is found, and the k-th largest of those taken; with 1024 groups about
// 1024 ln(1 / (1 - k / 1024)) logits reach it.  Where a row is long enough the groups come from an eighth of it, eight pieces of every
// 64, and the bound is their `rank`-th largest: k / 8 with four standard deviations and four more, so that one row in some thousand has too
// few.  (All of a row read twice: 8192 x 50304 with 8 logits 316 us instead of 256, 2048 x 131072 with 64 234 us instead of 168.)
// The pass over the row sums exp(z / T) over the pieces without a logit that reaches the bound and marks the others, a bit each; they follow in
// their order, a thread each, so that a warp does not go through a branch for nearly every 32 pieces.  The candidates are then sorted
// by counting into bins of a key or a few, and within their bin.
// Where the bound lets too many or too few through (a row of equal logits, large ones side by side), or a NaN is among them, the k-th largest logit is
// found by bisection on the row's 16-bit keys, from the bound on, and its equals are taken in the row's order: 1024 x 50304 with 64
// kept 160 us with all logits equal and 227 with hundreds equal to the 64th (bisection of all keys: 858 and 562), 43 as a rule.
// 8192 x 50304: 248 us with 8 logits kept, 314 with 256 (2.6 TB/s).  Of a row's 90000 cycles, eight rows at once, the pass over it has 47000, the
// sample and the bound 10000; the rest are the candidates', short steps between barriers.
// ---------------------------------------------------------------------------------------
struct TopArgs {
  const void* logits;
  float cap, temperature;
  int32_t* ids;
  float* logp;
  float* log_rest;
  int rows, vocab, k;
  int64_t ld;
  int rank;                                    // k, or the sample's
  int groups, room;                            // of a block; for candidates
};
constexpr int kTopSampleFrom = 16384 + 16;     // logits of a row that is sampled (at least 256 pieces of it)

// bf16 bits -> an unsigned key of the same order (-0 is 0; NaN above all)
__device__ __forceinline__ uint32_t top_key(uint32_t bits) {
  if ((bits & 0x7fffu) > 0x7f80u) return 0xffffu;
  return bits & 0x8000u ? 0x8000u - (bits & 0x7fffu) : 0x8000u + bits;
}
__device__ __forceinline__ uint32_t top_bits(uint32_t key) { return key >= 0x8000u ? key - 0x8000u : 0x8000u | (0x8000u - key); }

// the larger of each of two pairs of bf16, NaN where one of them is
__device__ __forceinline__ uint32_t top_max_nan(uint32_t a, uint32_t b) {
  const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}

constexpr int kTopBins = 256;
struct TopShared {                             // of a group, followed by room for the candidates, twice, and a bit per piece
  int hist[kTopBins], begin[kTopBins];
  float red[2 * (kDsMaxThreads / 32)];
  int count[2][kDsMaxThreads / 32], n;
  uint32_t bound;
};
static_assert(offsetof(TopShared, hist) % 16 == 0 && sizeof(TopShared) % 8 == 0, "read in 16-byte pieces");
constexpr int top_group_bytes(int64_t vocab, int room) { return int((sizeof(TopShared) + room * 16 + ((vocab + 14) / 8 + 31) / 32 * 4 + 15) / 16 * 16); }

template <bool TABLE>
__global__ void __launch_bounds__(2 * kDsMaxThreads, 1) top_logits_kernel(const TopArgs p) {
  grid_trigger();
  grid_wait();
  extern __shared__ __align__(16) uint8_t s_ds[];
  const int nt = int(blockDim.x) / p.groups, index = int(threadIdx.x) / nt;
  const Group group = {index, int(threadIdx.x) - index * nt, nt};
  const int tid = group.tid, warps = nt >> 5, lane = tid & 31, warp = tid >> 5;
  TopShared& sh = *reinterpret_cast<TopShared*>(s_ds + cap_bytes(TABLE ? kTabE : 0) + index * top_group_bytes(p.vocab, p.room));
  uint64_t *const s_cand = reinterpret_cast<uint64_t*>(&sh + 1), *const s_sorted = s_cand + p.room;
  uint32_t* const s_marks = reinterpret_cast<uint32_t*>(s_sorted + p.room);   // a bit per piece
  uint32_t* const s_list = reinterpret_cast<uint32_t*>(s_sorted);             // the marked ones
  using C = Cap<TABLE ? kTabE : 0>;
  const C cap(p.cap, p.temperature, s_ds);
  const int k = p.k;
  __syncthreads();                             // (the table; from here on the groups go their own ways)
  const int64_t step = int64_t(gridDim.x) * p.groups;
  int64_t row = int64_t(blockIdx.x) * p.groups + index;
  if (row >= p.rows) return;
  DsRow q(p.logits, row, p.ld, p.vocab);
  Pieces in;
  in.fetch(q, tid, nt);
  const bool sampled = p.vocab >= kTopSampleFrom;
  for (int64_t next; row < p.rows; row = next) {
    next = row + step;
    const DsRow q_next(p.logits, next < p.rows ? next : row, p.ld, p.vocab);
    const uint4* src = q.pieces();
    const int pieces = (q.end + 7) >> 3;
    // ---- first pass: the groups' maxima (NaN aside), as keys; 0 for a group of none
    uint32_t top[8], most = 0u;
    {
      const __nv_bfloat162 none = __halves2bfloat162(__ushort_as_bfloat16(0x7fff), __ushort_as_bfloat16(0x7fff));
      __nv_bfloat162 m[4] = {none, none, none, none};
      auto look = [&](const uint4& w) {
        const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(&w);
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = __hmax2(m[j], v[j]);
      };
      if (sampled) {
        const int n = (q.last() - q.first()) / 64 * 8;
#pragma unroll 4
        for (int i = tid; i < n; i += nt) look(ld_stream_v4(src + q.first() + (i >> 3) * 64 + (i & 7)));
      } else {
        in.each(q, q.last(), tid, nt, [&](const uint4& w, int) { look(w); });
        in.fetch(q, tid, nt);
      }
      const int edge = warp == warps - 1 ? q.edge(lane) : -1;
      if (edge >= 0) {
        const __nv_bfloat16 v = __ushort_as_bfloat16(q.base[edge]);
        m[0] = __hmax2(m[0], __halves2bfloat162(v, __ushort_as_bfloat16(0x7fff)));
      }
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        const uint32_t word = *reinterpret_cast<const uint32_t*>(&m[h >> 1]), b = h & 1 ? word >> 16 : word & 0xffffu;
        top[h] = (b & 0x7fffu) > 0x7f80u ? 0u : top_key(b);
        most = max(most, top[h]);
      }
    }
    // how many of the block's `n`s there are (the same value in every thread); two buffers, so that one barrier a call does
    int turn = 0;
    auto count = [&](int n) {
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) sh.count[turn][warp] = n;
      group.sync();
      const int c = __reduce_add_sync(0xffffffffu, lane < warps ? sh.count[turn][lane] : 0);
      turn ^= 1;
      return c;
    };
    // ---- the bound: the rank-th largest of the groups' keys (0: there are not so many), by its upper and then by its lower byte
    uint32_t largest = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) sh.count[turn][warp] = int(largest);
    auto zero = [&] {
      for (int i = tid; i < kTopBins; i += nt) sh.hist[i] = 0;
    };
    zero();
    group.sync();
    largest = __reduce_max_sync(0xffffffffu, lane < warps ? uint32_t(sh.count[turn][lane]) : 0u);
    turn ^= 1;
    // warp 0: the first bin at which the running count reaches `want` and the count before it (kTopBins: none), or all bins' beginnings
    auto scan = [&](int want, bool begins, int& before_it) {
      int v[kTopBins / 32], sum = 0;
#pragma unroll
      for (int j = 0; j < kTopBins / 32; j += 4) {
        const int4 b = reinterpret_cast<const int4*>(sh.hist)[(lane * (kTopBins / 32) + j) / 4];
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
      int found = kTopBins, at_found = 0;
#pragma unroll
      for (int j = 0; j < kTopBins / 32; ++j) {
        if (begins) sh.begin[lane * (kTopBins / 32) + j] = before;
        if (before + v[j] >= want && found == kTopBins) {
          found = lane * (kTopBins / 32) + j;
          at_found = before;
        }
        before += v[j];
      }
      const int first = int(__reduce_min_sync(0xffffffffu, unsigned(found)));
      before_it = int(__reduce_max_sync(0xffffffffu, found == first ? unsigned(at_found) : 0u));
      return first;
    };
#pragma unroll
    for (int h = 0; h < 8; ++h)
      if (top[h] != 0u) atomicAdd(sh.hist + (255 - (top[h] >> 8)), 1);
    group.sync();
    if (warp == 0) {
      int before = 0;
      const int b = scan(p.rank, false, before);
      if (lane == 0) {
        sh.bound = b == kTopBins ? 0u : uint32_t(255 - b) << 8 | 0x80000000u;
        sh.n = p.rank - before;                // of the bin's own
      }
    }
    group.sync();
    uint32_t lo = sh.bound;
    if (lo != 0u) {
      const int want = sh.n;
      zero();
      group.sync();
#pragma unroll
      for (int h = 0; h < 8; ++h)
        if (top[h] != 0u && (top[h] >> 8) == ((lo >> 8) & 0xffu)) atomicAdd(sh.hist + (255 - (top[h] & 0xffu)), 1);
      group.sync();
      if (warp == 0) {
        int before;
        const int b = scan(want, false, before);
        if (lane == 0) sh.bound = (lo & 0xff00u) | uint32_t(255 - b);
      }
      group.sync();
      lo = sh.bound;
    }
    if (tid == 0) sh.n = 0;
    // the candidates' bins: of as many keys as make 256 of them enough down to the bound
    const int shift = max(0, 32 - __clz(int((largest > lo ? largest - lo : 0u) >> 8)));
    auto bin = [&](uint32_t key) { return key > largest ? 0u : min((largest - key) >> shift, uint32_t(kTopBins - 1)); };

    // ---- second pass: the sum over the pieces without a candidate (and wholly of the row), and which ones those are not
    float2 acc = make_float2(0.f, 0.f);
    uint32_t nan = 0u;
    const uint32_t lo_bits = lo == 0u ? 0xff80u : top_bits(lo);          // (no bound: -inf)
    const __nv_bfloat162 bound = __halves2bfloat162(__ushort_as_bfloat16(uint16_t(lo_bits)), __ushort_as_bfloat16(uint16_t(lo_bits)));
    auto reach = [&](uint32_t w) { return __hge2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w), bound); };
    // bit b of the marks is piece first + b (whole warps, for the ballot); the pieces at the row's ends are listed without one
    const int whole = q.last() - q.first(), words = (whole + 31) >> 5;
    in.each(q, q.first() + words * 32, tid, nt, [&](const uint4& w, int i) {
      const uint32_t most = top_max_nan(top_max_nan(w.x, w.y), top_max_nan(w.z, w.w));     // (a NaN marks its piece too)
      const bool skip = __hgeu2_mask(*reinterpret_cast<const __nv_bfloat162*>(&most), bound) != 0u || i >= q.last();
      const uint32_t marks = __ballot_sync(0xffffffffu, skip && i < q.last());
      if (lane == 0) s_marks[(i - q.first()) >> 5] = marks;
      float2 e[4];
      four_words(w, [&](auto j, uint32_t v) { e[j] = cap.template e<decltype(j)::value>(v); });
      const float2 sum = __fadd2_rn(__fadd2_rn(e[0], e[1]), __fadd2_rn(e[2], e[3]));
      acc = __fadd2_rn(acc, make_float2(skip ? 0.f : sum.x, skip ? 0.f : sum.y));
    });
    in.fetch(q_next, tid, nt);
    group.sync();
    // ---- the marked pieces, listed in order
    int marked = 0;
    for (int i0 = 0; i0 < words; i0 += nt) {
      uint32_t m = i0 + tid < words ? s_marks[i0 + tid] : 0u;
      int at = __popc(m);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += x;
      }
      if (lane == 31) sh.count[turn][warp] = at;
      at += marked - __popc(m);
      group.sync();
      const int c = lane < warps ? sh.count[turn][lane] : 0;
      at += __reduce_add_sync(0xffffffffu, lane < warp ? c : 0);
      marked += __reduce_add_sync(0xffffffffu, c);
      turn ^= 1;
      for (; m != 0u; m &= m - 1u, ++at)
        if (at < 2 * p.room - 2) s_list[at] = uint32_t(q.first() + (i0 + tid) * 32 + __ffs(int(m)) - 1);
    }
    const bool crowded = marked > 2 * p.room - 2;
    marked = min(marked, 2 * p.room - 2);
    if (q.first()) {
      if (tid == 0) s_list[marked] = 0u;
      ++marked;
    }
    if (q.last() >= q.first() && (q.end & 7)) {
      if (tid == 0) s_list[marked] = uint32_t(q.last());
      ++marked;
    }
    group.sync();
    // ---- their candidates, a warp's with one addition to the count, and the sum of the others
    auto listed = [&](int l) { return l < marked ? ld_stream_v4(src + s_list[l]) : make_uint4(0u, 0u, 0u, 0u); };
    uint4 w_next = listed(tid);
    for (int l0 = warp * 32; l0 < marked; l0 += nt) {
      const int l = l0 + lane, i = l < marked ? int(s_list[l]) : 0;
      const uint4 w = w_next;
      w_next = listed(l + nt);
      const uint32_t outside = l < marked ? q.outside(i) : 0xffu;
      uint32_t hit = 0u;
      four_words(w, [&](auto j, uint32_t v) {
        const uint32_t ge = reach(v);
        hit |= ((ge & 1u) | (ge >> 31) << 1) << (2 * decltype(j)::value);
      });
      hit &= ~outside;
      const int hits = __popc(hit);
      int before = 0, all = 0;
      for (int t = 1;; ++t) {
        const uint32_t lanes = __ballot_sync(0xffffffffu, hits >= t);
        if (lanes == 0u) break;
        before += __popc(lanes & ((1u << lane) - 1u));
        all += __popc(lanes);
      }
      int at = 0;
      if (lane == 0 && all > 0) at = atomicAdd(&sh.n, all);
      at = __shfl_sync(0xffffffffu, at, 0) + before;
      for (uint32_t rest = hit; rest != 0u; rest &= rest - 1u, ++at) {
        const int h = __ffs(int(rest)) - 1;
        const uint32_t v = h & 4 ? (h & 2 ? w.w : w.z) : (h & 2 ? w.y : w.x);
        if (at < p.room) s_cand[at] = uint64_t(top_key(h & 1 ? v >> 16 : v & 0xffffu)) << 32 | uint32_t(~uint32_t(i * 8 + h - q.off));
      }
      const uint32_t off8 = hit | outside;
      four_words(w, [&](auto j, uint32_t v) {
        const uint32_t off = off8 >> (2 * decltype(j)::value);
        const uint32_t rest = v & ((off & 1u ? 0u : 0xffffu) | (off & 2u ? 0u : 0xffff0000u));
        if (TABLE) nan = __vmaxu2(nan, rest & 0x7fff7fffu);
        const float2 e = cap.template e<decltype(j)::value>(rest);
        acc = __fadd2_rn(acc, make_float2(off & 1u ? 0.f : e.x, off & 2u ? 0.f : e.y));
      });
    }
    if (C::is_nan(nan)) acc.x = __int_as_float(0x7fffffff);
    float others = acc.x + acc.y;
    const bool odd = group.sync_or(isnan(others));
    int n = sh.n;
    float extra = 0.f;                         // the sum of candidates that are not kept
    if (crowded || n > p.room || n < k || odd) {
      // the k-th largest key of the row
      auto keys_of = [&](int i, auto&& f) {
        const uint4 w = ld_stream_v4(src + i);
        const uint32_t wi[4] = {w.x, w.y, w.z, w.w}, skip = q.outside(i);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(skip >> j & 1u)) f(j, top_key(j & 1 ? wi[j >> 1] >> 16 : wi[j >> 1] & 0xffffu));
      };
      auto reached = [&](uint32_t v) {
        int c = 0;
        for (int i = tid; i < pieces; i += nt) keys_of(i, [&](int, uint32_t u) { c += u >= v; });
        return count(c) >= k;
      };
      // it lies at the bound or little above where that lets enough through (steps of 1, 2, 4, ...), else below
      const bool enough = crowded || n >= k;
      uint32_t key = enough ? lo : 0u, step = enough ? 1u : 0x10000u, last = enough || odd ? 0xffffu : lo;
      for (; key + step <= last && reached(key + step); step *= 2u) key += step;
      last = min(last, key + step - 1u);
      while (key < last) {
        const uint32_t mid = (key + last + 1u) >> 1;
        if (reached(mid)) key = mid;
        else last = mid - 1u;
      }
      if (tid == 0) sh.n = 0;
      group.sync();
      // those above it, fewer than k; how many equal it; the sum of those below
      int equal = 0;
      others = 0.f;
      for (int i = tid; i < pieces; i += nt)
        keys_of(i, [&](int j, uint32_t v) {
          if (v > key) s_cand[atomicAdd(&sh.n, 1)] = uint64_t(v) << 32 | uint32_t(~uint32_t(i * 8 + j - q.off));
          else if (v == key) ++equal;
          else others += expf(cap.z_over_t(__uint_as_float(top_bits(v) << 16)));
        });
      const int equals = count(equal), above = sh.n, want = k - above;
      // the first `want` of its equals: block after block of pieces, each thread's in its place by a prefix sum
      int have = 0;
      for (int i0 = 0; have < want; i0 += nt) {
        const int i = i0 + tid;
        uint32_t mine = 0u;
        if (i < pieces) keys_of(i, [&](int j, uint32_t v) { mine |= uint32_t(v == key) << j; });
        int before = __popc(mine);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += v;
        }
        if (lane == 31) sh.count[turn][warp] = before;
        group.sync();
        int all = 0, at = have + before - __popc(mine);
        for (int v = 0; v < warps; ++v) {
          if (v < warp) at += sh.count[turn][v];
          all += sh.count[turn][v];
        }
        turn ^= 1;
        for (; mine != 0u && at < want; mine &= mine - 1u, ++at)
          s_cand[above + at] = uint64_t(key) << 32 | uint32_t(~uint32_t(i * 8 + __ffs(int(mine)) - 1 - q.off));
        have += all;
      }
      group.sync();
      if (tid == 0 && equals > want) extra = float(equals - want) * expf(cap.z_over_t(__uint_as_float(top_bits(key) << 16)));
      n = k;
    }
    // ---- each candidate's place; from there on all in the order of places, so that results do not depend on that of the atomics
    for (int i = tid; i < kTopBins; i += nt) sh.hist[i] = 0;
    group.sync();
    for (int i = tid; i < n; i += nt) atomicAdd(sh.hist + bin(uint32_t(s_cand[i] >> 32)), 1);
    group.sync();
    if (warp == 0) {
      int unused;
      scan(0, true, unused);
    }
    group.sync();
    for (int i = tid; i < n; i += nt) {
      const uint64_t c = s_cand[i];
      s_sorted[atomicAdd(sh.begin + bin(uint32_t(c >> 32)), 1)] = c;      // (a bin's beginning becomes its end)
    }
    group.sync();
    for (int i = tid; i < n; i += nt) {
      const uint64_t mine = s_sorted[i];
      const uint32_t b = bin(uint32_t(mine >> 32));
      const int end = sh.begin[b], begin = end - sh.hist[b];
      int r = begin;
      for (int j = begin; j < end; ++j) r += s_sorted[j] > mine;
      s_cand[r] = mine;
    }
    group.sync();
    auto z_of = [&](int r) { return cap.z_over_t(__uint_as_float(top_bits(uint32_t(s_cand[r] >> 32)) << 16)); };
    float sums[2] = {others + extra, 0.f};
    for (int r = tid; r < n; r += nt) sums[r < k] += expf(z_of(r));
    ds_warp_sums(sums, sh.red, warp, true);
    group.sync();
    ds_add_warps(sums, sh.red, warps);
    const float lse = logf(sums[0] + sums[1]);
    for (int r = tid; r < k; r += nt) {
      p.ids[row * k + r] = int32_t(~uint32_t(s_cand[r]));
      p.logp[row * k + r] = z_of(r) - lse;
    }
    if (tid == 0) p.log_rest[row] = log_share(sums[0], sums[1]);
    group.sync();
    q = q_next;
  }
}

// The same for rows of at most PIECES 16-byte pieces a lane: a warp per row, which takes the largest k times.  A logit is a number whose order is that of
// the answer, its key above its place's complement.
template <int PIECES>
__global__ void __launch_bounds__(128) top_logits_short_kernel(const TopArgs p) {
  grid_trigger();
  grid_wait();
  const int lane = threadIdx.x & 31, k = p.k;
  const Cap<0> cap(p.cap, p.temperature, nullptr);
  for (int64_t row = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5); row < p.rows; row += int64_t(gridDim.x) * 4) {
    const DsRow q(p.logits, row, p.ld, p.vocab);
    const int pieces = (q.end + 7) >> 3;
    uint32_t v[PIECES * 8], most = 0u;         // (0: none, or taken)
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
      const int i = lane + c * 32;
      const uint4 w = i < pieces ? ld_stream_v4(q.pieces() + i) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t wi[4] = {w.x, w.y, w.z, w.w}, out = i < pieces ? q.outside(i) : 0xffu;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t key = top_key(j & 1 ? wi[j >> 1] >> 16 : wi[j >> 1] & 0xffffu);
        v[c * 8 + j] = out >> j & 1u ? 0u : key << 16 | uint32_t(0xffff - (i * 8 + j - q.off));
        most = max(most, v[c * 8 + j]);
      }
    }
    uint32_t mine[2] = {0u, 0u};               // what this lane's places (lane, 32 + lane) got
#pragma unroll 1
    for (int r = 0; r < k; ++r) {
      const uint32_t best = __reduce_max_sync(0xffffffffu, most);
      mine[0] = lane == r ? best : mine[0];
      mine[1] = lane + 32 == r ? best : mine[1];
      most = 0u;
#pragma unroll
      for (int j = 0; j < PIECES * 8; ++j) {   // (every lane looks for it: no branch)
        v[j] = v[j] == best ? 0u : v[j];
        most = max(most, v[j]);
      }
    }
    float tail = 0.f, kept = 0.f, s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < PIECES * 8; j += 2) {
      const uint32_t w = (v[j] ? top_bits(v[j] >> 16) : 0u) | (v[j + 1] ? top_bits(v[j + 1] >> 16) : 0u) << 16;
      const float2 e = cap.template e<3>(w);
      tail += (v[j] ? e.x : 0.f) + (v[j + 1] ? e.y : 0.f);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (mine[h]) {
        s[h] = cap.z_over_t(__uint_as_float(top_bits(mine[h] >> 16) << 16));
        kept += expf(s[h]);
      }
    tail = ds_warp_sum(tail);
    kept = ds_warp_sum(kept);
    const float lse = logf(tail + kept);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (mine[h]) {
        p.ids[row * k + 32 * h + lane] = int32_t(0xffffu - (mine[h] & 0xffffu));
        p.logp[row * k + 32 * h + lane] = s[h] - lse;
      }
    if (lane == 0) p.log_rest[row] = log_share(tail, kept);
  }
}

// Threads for a row of `pieces` 16-byte pieces: two pieces each, at least `least` and at most `most` of them.
static int ds_threads(int64_t pieces, int least, int most) {
  const int64_t want = std::max<int64_t>((pieces + 63) / 64 * 32, (least + 31) / 32 * 32);
  return int(std::min<int64_t>(std::max<int64_t>(want, 32), most));
}

// Whether the logits that a block meets pay for its table: 128 rows of 8192 with the gradient 7.7 us with it and 7.6 without, of 16384 8.15 and
// 8.25, of 32768 11.0 and 12.2; 2000 of 4096 27.3 and 28.9 (evaluated 14.0 and 15.8).
static bool ds_table(int64_t rows, int64_t vocab) { return std::max<int64_t>(1, rows / (2 * sm_count())) * vocab >= 16384; }

// Blocks of `threads` that an SM holds of `kern`, whose registers and static shared memory are looked up once per device.
struct DsKernelInfo {
  std::atomic<int> registers[64];
  std::atomic<int> smem[64];
};
template <typename K>
static int ds_blocks(K kern, DsKernelInfo& info, int64_t smem, int threads, int64_t* per_sm) {
  int dev = 0;
  TG_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return TG_ERR_SHAPE;
  if (info.registers[dev].load(std::memory_order_acquire) == 0) {
    cudaFuncAttributes a;
    TG_CUDA_CHECK(cudaFuncGetAttributes(&a, kern));
    TG_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kDsSmemMax - int64_t(a.sharedSizeBytes))));
    info.smem[dev].store(int(a.sharedSizeBytes), std::memory_order_relaxed);
    info.registers[dev].store(a.numRegs, std::memory_order_release);
  }
  const int per_warp = (info.registers[dev].load(std::memory_order_acquire) * 32 + 255) / 256 * 256;
  const int64_t by_registers = 65536 / (int64_t(per_warp) * (threads / 32));
  const int64_t by_smem = (228 * 1024) / (smem + info.smem[dev].load(std::memory_order_relaxed) + 1024);
  *per_sm = std::max<int64_t>(1, std::min<int64_t>({by_registers, by_smem, 2048 / threads, 32}));
  return TG_OK;
}

constexpr int64_t kDsStatic = 3 * 1024;                       // (the loss's; the selection has none)
constexpr int64_t kDsDynamicMax = kDsSmemMax - kDsStatic;
// Whether two blocks of `smem` dynamic bytes do not fit on an SM (1 KB of each is the system's).
constexpr bool ds_alone(int64_t smem) { return 2 * (smem + kDsStatic + 1024) > 228 * 1024; }

// Threads and groups for rows that are not kept.  A row alone has phases in which little is on its way, so several are in work on an SM: eight by 128
// threads each where that is enough for one (`least`).  Fewer and larger groups cost 1.08 and 1.25 times as much a row and may have the better last round.
// Rows with fewer than `least_group` threads have a block each (128 where there is no table to share: 500 x 500 4.8 us, in groups 6.1).
static void ds_groups(int64_t rows, int64_t pieces, int least, int block, int least_group, int* nt, int* groups) {
  const int64_t sms = sm_count();
  double best = 0.0;
  *groups = 1;
  for (int g = kDsMaxGroups; g >= 2; g /= 2) {
    if (block / g < std::max(least, 128) || rows <= sms * (g / 2)) continue;
    const double cost = double((rows + sms * g - 1) / (sms * g) * g) * (g == 8 ? 1.0 : g == 4 ? 1.08 : 1.25);
    if (best == 0.0 || cost < best) {
      best = cost;
      *groups = g;
    }
  }
  *nt = ds_threads(pieces, least, block / std::max(*groups, 2));
  if (*nt < least_group) *groups = 1;
}

template <int EXPS, bool GRAD, bool TABLE, bool STAGED>
static int launch_distill(DistillArgs a, int nt, cudaStream_t st) {
  static DsKernelInfo info;
  auto kern = softcap_distill_kernel<EXPS, GRAD, TABLE, STAGED>;
  const int64_t table = TABLE ? cap_bytes(distill_table(EXPS, GRAD)) : 0, bytes = ds_map_bytes(a.vocab) + (STAGED ? ds_row_bytes(a.vocab) : 0);
  // groups that share a block's table where a row has less than 128 threads (16384 x 1024 88 us, a table each 149; from 128 on 1.03 times the
  // time) and where two blocks do not fit on an SM beside each other (from 46002 logits on).  Beyond 50457 a row is alone on its SM, with its 256
  // threads (up to 100937, which still are kept): 1.04 ps a logit at 8192 x 50304, 1.25 at 4096 x 65536 (336 us), 1.15 at 4096 x 100277 (474)
  if (STAGED && TABLE && nt < 128) a.groups = int(std::max<int64_t>(1, std::min<int64_t>({kDsMaxGroups, ds_block_threads(true) / nt, a.rows / sm_count()})));
  else if (STAGED) a.groups = ds_alone(table + bytes) && table + 2 * bytes <= kDsDynamicMax && a.rows > sm_count() ? 2 : 1;
  while (a.groups > 1 && table + a.groups * bytes > kDsDynamicMax) --a.groups;
  a.group_bytes = int(bytes);
  const int64_t smem = table + a.groups * bytes;
  int64_t per_sm;
  if (int rc = ds_blocks(kern, info, smem, nt * a.groups, &per_sm)) return rc;
  const int blocks = int(std::min<int64_t>((int64_t(a.rows) + a.groups - 1) / a.groups, sm_count() * per_sm));
  TG_CUDA_CHECK(launch_if_short(int64_t(a.rows) * a.vocab <= 1 << 20, kern, dim3(unsigned(blocks)), nt * a.groups, size_t(smem), st, a));
  return TG_OK;
}
template <int EXPS, bool GRAD>
static int launch_distill(const DistillArgs& a, cudaStream_t st) {
  const bool table = ds_table(a.rows, a.vocab);
  const int64_t pieces = (a.vocab + 14) / 8;
  if constexpr (GRAD) {
    if (cap_bytes(kTabU) + ds_map_bytes(a.vocab) + ds_row_bytes(a.vocab) <= kDsDynamicMax) {
      const int nt = ds_threads(pieces, a.k, ds_block_threads(true) / 2);
      return table ? launch_distill<EXPS, true, true, true>(a, nt, st) : launch_distill<EXPS, true, false, true>(a, nt, st);
    }
  }
  DistillArgs b = a;
  int nt;
  ds_groups(a.rows, pieces, (a.k + 31) / 32 * 32, ds_block_threads(false), table ? 32 : 128, &nt, &b.groups);
  return table ? launch_distill<EXPS, GRAD, true, false>(b, nt, st) : launch_distill<EXPS, GRAD, false, false>(b, nt, st);
}

template <bool TABLE>
static int launch_top(TopArgs a, int nt, cudaStream_t st) {
  static DsKernelInfo info;
  const int64_t table = TABLE ? cap_bytes(kTabE) : 0, bytes = top_group_bytes(a.vocab, a.room);
  while (a.groups > 1 && table + a.groups * bytes > kDsDynamicMax) --a.groups;
  const int64_t smem = table + a.groups * bytes;
  int64_t per_sm;
  if (int rc = ds_blocks(top_logits_kernel<TABLE>, info, smem, nt * a.groups, &per_sm)) return rc;
  const int blocks = int(std::min<int64_t>((int64_t(a.rows) + a.groups - 1) / a.groups, sm_count() * per_sm));
  TG_CUDA_CHECK(launch_if_short(int64_t(a.rows) * a.vocab <= 1 << 20, top_logits_kernel<TABLE>, dim3(unsigned(blocks)), nt * a.groups, size_t(smem), st, a));
  return TG_OK;
}
template <int PIECES>
static int launch_top_short(const TopArgs& a, cudaStream_t st) {
  const int64_t warps = std::min<int64_t>(a.rows, int64_t(sm_count()) * 32);
  TG_CUDA_CHECK(launch_if_short(int64_t(a.rows) * a.vocab <= 1 << 20, top_logits_short_kernel<PIECES>, dim3(unsigned((warps + 3) / 4)), 128, 0, st, a));
  return TG_OK;
}
static int launch_top(TopArgs a, cudaStream_t st) {
  const int64_t pieces = (a.vocab + 14) / 8;
  // where a warp's turns, k of them, take no longer than the general kernel's steps: 8192 x 240 with 64 kept 34 us (the latter 44), x 500 with 48 45
  // (45), x 1000 with 20 41 (41), with 8 26 (39)
  if (pieces <= 32 && a.k <= 64) return launch_top_short<1>(a, st);
  if (pieces <= 64 && a.k <= 48) return launch_top_short<2>(a, st);
  if (pieces <= 128 && a.k <= 20) return launch_top_short<4>(a, st);
  int nt;
  // many short rows, eight to a block with two warps each: 8192 x 4000 with 64 kept 70 us, four warps 77, with 128 94 and 88; x 2000 53 and 72, 79 and 82
  if (pieces <= 512 && pieces * a.k <= 48 * 1024 && a.rows > 8 * sm_count()) {
    a.groups = kDsMaxGroups;
    return launch_top<false>(a, 64, st);
  }
  ds_groups(a.rows, pieces, 32, 2 * kDsMaxThreads, 128, &nt, &a.groups);
  return ds_table(a.rows, a.vocab) ? launch_top<true>(a, nt, st) : launch_top<false>(a, nt, st);
}

// Whether two sets of rows of one pitch have an element in common.  (Rows between each other's, in one buffer of twice the pitch, have none.)
static bool ds_rows_overlap(const void* a, const void* b, int64_t rows, int64_t vocab, int64_t ld) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  const int64_t apart = int64_t((x < y ? y - x : x - y) / 2), q = apart / ld, m = apart % ld;
  return (m < vocab && q < rows) || (ld - m < vocab && q + 1 < rows);
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
  if (logits == nullptr) return TG_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(logits) & 1u) != 0) return TG_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  const bool sampled = vocab >= kTopSampleFrom;
  const int rank = sampled ? int(std::ceil(k / 8.0 + 4.0 * std::sqrt(k / 8.0))) + 4 : k;
  const TopArgs a = {logits, cap, temperature, ids, logp, log_rest, int(rows), int(vocab), k, ld, rank, 1, k <= 64 ? kTopMaxCandidates / 2 : kTopMaxCandidates};
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
  if (g.logits == nullptr) return TG_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(g.logits) & 1u) != 0) return TG_ERR_ALIGN;
  if (g.dlogits != nullptr && ((reinterpret_cast<uintptr_t>(g.logits) ^ reinterpret_cast<uintptr_t>(g.dlogits)) & 15u) != 0) return TG_ERR_ALIGN;
  if (g.dlogits != nullptr && ds_rows_overlap(g.logits, g.dlogits, g.rows, g.vocab, g.ld)) return TG_ERR_SHAPE;
  if (int rc = check_arch()) return rc;
  // One sum does where there is one temperature.  exp(z) is exp(z / T) squared at the two temperatures that are powers of two above 1 and in use, for a
  // product or two; at any other it is an exponential of its own, the other pipe that is short (8192 x 50257 465 and 603 us, the loss alone 197 and 289)
  const bool soft = g.weight > 0.f, hard = g.weight < 1.f && g.targets != nullptr;
  const float t = soft ? g.temperature : 1.0f;
  const int exps = !(soft && hard) || t == 1.0f ? 1 : t == 2.0f ? 3 : t == 4.0f ? 4 : 2;
  const DistillArgs a = {g.logits, g.ids, g.logp, g.log_rest, hard ? g.targets : nullptr, g.ids_64, g.targets_64, g.cap, t,
                         g.weight, g.dlogits, g.gscale, g.only_if_scaled, g.row_loss, int(g.rows), int(g.vocab), g.k, g.ld, 1, 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool grad = g.dlogits != nullptr;
  if (exps == 1) return grad ? launch_distill<1, true>(a, st) : launch_distill<1, false>(a, st);
  if (exps == 2) return grad ? launch_distill<2, true>(a, st) : launch_distill<2, false>(a, st);
  if (exps == 3) return grad ? launch_distill<3, true>(a, st) : launch_distill<3, false>(a, st);
  return grad ? launch_distill<4, true>(a, st) : launch_distill<4, false>(a, st);
}
