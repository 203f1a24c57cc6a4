// Wrappers for kernels on CTA pairs (two SMs working on one tile, tcgen05 with cta_group::2).
#pragma once
#include "common.cuh"

namespace jb {

// ---- cta_group::2 forms of the wrappers in common.cuh ----
__device__ __forceinline__ void pair_tmem_alloc(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols) : "memory");
}
__device__ __forceinline__ void pair_tmem_relinquish() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void pair_umma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on the barrier at this offset in both CTAs once all previously issued MMAs of this thread retire.
__device__ __forceinline__ void pair_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"(uint16_t(3)) : "memory");
}
// Tile load into this CTA whose bytes are counted by a barrier of the pair's leader.
__device__ __forceinline__ void pair_tma_load_2d(uint32_t dst_smem, const void* tmap, int c0, int c1, uint32_t leader_bar) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst_smem), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(leader_bar) : "memory");
}
// (with .release.cluster every arrival waits for the warp's outstanding memory operations: 1400 cycles per K-block)
__device__ __forceinline__ void cluster_mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Bounded wait that also orders what the other CTA did before its arrival.
__device__ __forceinline__ bool cluster_mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}"
      : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0;
}
__device__ __forceinline__ bool cluster_mbar_wait(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, unsigned int* status,
                                                  unsigned int code) {
  if (cluster_mbar_try(bar, parity)) return true;
  const unsigned long long t0 = globaltimer_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (cluster_mbar_try(bar, parity)) return true;
    if (*abort_flag) return false;
    if (globaltimer_ns() - t0 > JB_WAIT_LIMIT_NS) {
      *abort_flag = 1u;
      atomicCAS(status, 0u, code);
      return false;
    }
  }
}

__device__ __forceinline__ void st_global_256(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Control block of a persistent CTA pair whose operands both come by TMA: a ring of `STAGES` K-blocks and two accumulators.  The pair's
// leader (cluster rank 0) issues every MMA; its `full` barriers count its own expectation and the bytes of both CTAs' loads, `empty`
// and `acc_full` are committed to both CTAs, `acc_empty` counts the epilogue warps of both that drain a tile.
template <int STAGES>
struct PairRing {
  uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2];
  uint32_t tmem_base, abort_flag;
};
constexpr uint32_t PAIR_TMEM_COLS = 512;

// Barriers and tensor memory (its address in ctl->tmem_base); all threads of both CTAs.
template <int STAGES>
__device__ __forceinline__ void pair_ring_init(PairRing<STAGES>* ctl, int warp, int drain_warps) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&ctl->full[s]), 1);
      mbar_init(smem_u32(&ctl->empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&ctl->acc_full[a]), 1);
      mbar_init(smem_u32(&ctl->acc_empty[a]), drain_warps);
    }
    ctl->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    __syncwarp();                 // tcgen05.alloc is warp-collective: lane 0 rejoins from the barrier set-up first
    pair_tmem_alloc(smem_u32(&ctl->tmem_base), PAIR_TMEM_COLS);
    pair_tmem_relinquish();
  }
  __syncwarp();
  tc_fence_before_sync();
  cluster_arrive();               // both CTAs' barriers are initialised before either arrives on the other's
  cluster_wait();
  tc_fence_after_sync();
}
// Neither CTA leaves while the other's MMAs, commits or arrivals may still reach it.
__device__ __forceinline__ void pair_ring_close(uint32_t tmem, int warp) {
  __syncwarp();
  tc_fence_before_sync();
  cluster_arrive();
  cluster_wait();
  if (warp == 0) {
    tc_fence_after_sync();
    pair_tmem_dealloc(tmem, PAIR_TMEM_COLS);
  }
}

// Shared-memory descriptor of an MN-major bf16 operand in the 128-byte swizzle: blocks of [K rows][64 MN-elements], `block` bytes
// apart.  (K-major operands: umma_desc_k_sw128.)  A K-step of 16 is 2048 bytes further.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr, uint32_t block) {
  return (umma_desc_k_sw128(smem_addr) & ~(uint64_t(0x3FFF) << 16)) | uint64_t(block >> 4) << 16;
}
constexpr uint32_t IDESC_F16 = 0u - (1u << 7) - (1u << 10);         // added to umma_idesc_bf16: both operands f16
constexpr uint32_t IDESC_A_MN = 1u << 15, IDESC_B_MN = 1u << 16;      // operand read MN-major (with umma_idesc_bf16)

}  // namespace jb
