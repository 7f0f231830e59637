// Thin wrappers over the PTX the matrix-product kernel is built from: mbarriers,
// tiled TMA copies, tensor memory and tcgen05.mma (sm_100a).
//
// Every wait is bounded: a wait that runs out marks the block as failed and
// returns false, the roles of the block then leave their loops, drain what
// they have in flight (again bounded) and release tensor memory.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace affb {
namespace tc5 {

// A wait gives up after this long: seconds beyond any real wait of these kernels.
constexpr unsigned long long WAIT_NS = 4000000000ull;

__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Address of the same shared-memory location in block `rank` of the cluster.
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
// Every thread of both blocks of a pair.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrival at a barrier of any block of the cluster (address from peer_addr).
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_poll(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// True once the barrier's phase of this parity has completed; false when the
// block has failed or the wait ran out (which marks the block as failed).
// The timer is read only by a wait that has already polled long: one read
// takes longer than a stage of the pipeline does.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* failed,
                                         unsigned long long limit = WAIT_NS) {
#pragma unroll 1
  for (int i = 0; i < 4096; ++i)
    if (bar_poll(bar, parity)) return true;
  const unsigned long long t0 = now_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i)
      if (bar_poll(bar, parity)) return true;
    if (*failed) return false;
    if (now_ns() - t0 > limit) break;
  }
  *failed = 1;
  return false;
}
// The same for a whole warp, with an answer that is uniform for the compiler:
// what the loops around it count then stays in uniform registers, from which
// the copies and products take their operands.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* failed) {
#pragma unroll 1
  for (int i = 0; i < 4096; ++i)
    if (__all_sync(0xffffffffu, bar_poll(bar, parity))) return true;
  return __all_sync(0xffffffffu, bar_wait(bar, parity, failed));
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
// Time for copies in flight to land (microseconds) while a failed block shuts
// down and the barrier they signal is another block's.
__device__ __forceinline__ void settle() {
  const unsigned long long t0 = now_ns();
  while (now_ns() - t0 < 2000000ull) {}
}
// Last wait on a copy or product in flight while a failed block shuts down.
__device__ __forceinline__ void bar_drain(uint32_t bar, uint32_t parity) {
  const unsigned long long t0 = now_ns();
  while (!bar_poll(bar, parity))
    if (now_ns() - t0 > WAIT_NS) return;
}

// CG: blocks that work on one tile.  With 2 the barrier may be the other
// block's (an address from peer_addr); the data always lands in this block.
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void tma_load4(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                          uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x),
               "r"(y), "r"(z), "r"(src)
               : "memory");
}
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// At most N of this thread's store groups still reading shared memory.
template <int N>
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void store_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// Makes this thread's shared-memory writes visible to the TMA engine.
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ------------------------------------------------------- tensor memory --
// All 512 columns; one full warp (of each block of a pair).
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t slot) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {  // the warp that allocated
  if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 consecutive fp32 columns of this warp's 32 lanes (lane = accumulator row).
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ------------------------------------------------------------- products --
// Shared-memory operand descriptor, 128-byte swizzle.  K-major operand: rows
// of 128 bytes, `stride` = bytes between groups of 8 rows.  MN-major operand:
// per k a row of 64 elements, `stride` = bytes between groups of 8 k,
// `lead` = bytes between blocks of 64 rows of the operand.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)((lead & 0x3FFFF) >> 4) << 16) |
         ((uint64_t)((stride & 0x3FFFF) >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: fp32 accumulator of m x n, no negation.
__host__ __device__ inline uint32_t instr_desc(uint32_t type, bool a_mn, bool b_mn, uint32_t m, uint32_t n) {
  return (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((n >> 3) << 17) |
         ((m >> 4) << 24);
}
// One thread (of the pair's first block); F8: e4m3 operands, else 16-bit.
template <int CG, bool F8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
#define AFFB_MMA(GROUP, KIND)                                                                       \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                  \
               "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;\n\t}" ::"r"(d), \
               "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)                                \
               : "memory")
  if constexpr (CG == 1 && F8) AFFB_MMA("1", "f8f6f4");
  else if constexpr (CG == 1) AFFB_MMA("1", "f16");
  else if constexpr (F8) AFFB_MMA("2", "f8f6f4");
  else AFFB_MMA("2", "f16");
#undef AFFB_MMA
}
// The barrier (of both blocks of a pair) completes a phase once every product
// issued so far has finished.
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}

}  // namespace tc5
}  // namespace affb
