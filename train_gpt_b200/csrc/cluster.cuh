// What kernels on pairs of SMs (clusters of two CTAs, tcgen05 cta_group::2) share: PTX wrappers, and the order in which the pairs of a
// launch take up the items of one or two problems.
#pragma once

#include "umma.cuh"

namespace tg {

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// the same shared-memory offset in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster_if(uint32_t bar, uint32_t pred) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t}"
               ::"r"(bar), "r"(pred) : "memory");
}
// a load into this CTA's shared memory whose bytes are counted by a barrier of either CTA of the pair
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
// arrives on the barrier at this offset in both CTAs once the MMAs issued before are done
__device__ __forceinline__ void umma_commit_both(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"(uint16_t(3)) : "memory");
}
__device__ __forceinline__ void umma_commit_here(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// all of tensor memory, in both CTAs of a pair; every CTA of the pair makes the call with a whole warp
__device__ __forceinline__ void tmem_take_pair(uint32_t dst_smem) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(uint32_t(kTmemCols)) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
// the same for one CTA, which may share its SM with others that take columns
__device__ __forceinline__ void tmem_take(uint32_t dst_smem, uint32_t cols) {
  tmem_alloc(dst_smem, cols);
  tmem_relinquish();
}
__device__ __forceinline__ void tmem_give_pair(uint32_t addr) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(uint32_t(kTmemCols)) : "memory");
}

// The items of a problem that one unit (a CTA or a pair) works on: from `first` on in steps of `early_step` below early_end and of `step`
// from there on, while they are below n.
struct Walk {
  int first, early_step, early_end, step, n;
  __device__ __forceinline__ int next(int item) const { return item + (item < early_end ? early_step : step); }
};
__device__ __forceinline__ Walk walk_alone(int unit, int units, int n) { return Walk{unit, 0, 0, units, n}; }
// Two problems on the same units: the first one's items go round, and the units that its last round leaves idle take `rounds` rounds of the
// second one's meanwhile, before all take it up, the idle ones first.
__device__ __forceinline__ Walk walk_second(int unit, int units, int n1, int n2, int rounds) {
  const int busy = n1 % units, idle = units - busy, early_end = rounds * idle;
  if (busy == 0) return walk_alone(unit, units, n2);
  return Walk{unit >= busy ? unit - busy : early_end + idle + unit, idle, early_end, units, n2};
}

}  // namespace tg
