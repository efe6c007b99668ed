// Thin inline-PTX layer for tensor-core products by a pair of CTAs (a cluster of two, cta_group::2), beside umma.cuh:
// tensor memory, MMA, commit to both CTAs' barriers, TMA loads that count on the leader's barrier, and the cluster
// barrier.  The leader is the CTA of rank 0; the pair's tile has 256 rows, of which each CTA's tensor memory holds its own
// 128, and each CTA's shared memory holds its own 128 rows of A and its own half of B.
#pragma once

#include <cuda.h>

#include "umma.cuh"

namespace frwkv {
namespace umma2 {

using umma::smem_u32;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// true in one lane; the whole warp calls it.  Tensor-core and TMA instructions take their operands from uniform registers: a
// warp that runs its loop together and elects a lane for the instruction alone keeps them there, where a loop of one lane
// moves every operand over (656 cycles per block of four MMAs against the 512 they run).
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(e));
  return e != 0;
}
// the address of the same shared-memory object in the leader CTA
__device__ __forceinline__ uint32_t in_leader(const void* p) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(0u));
  return r;
}

__device__ __forceinline__ void tmem_alloc(uint32_t* smem_result, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_result)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// D[tmem of both CTAs] (+)= A * B over K = 16; one thread of the leader issues it
__device__ __forceinline__ void mma_bf16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// all MMAs issued so far arrive on this barrier in both CTAs when they complete
__device__ __forceinline__ void commit_both(uint64_t* mbar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(mbar)),
      "h"((uint16_t)3)
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// the same product by one CTA alone, 128 rows
__device__ __forceinline__ void mma_bf16_alone(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// A tile into this CTA's shared memory, its bytes counted on a barrier of its own
__device__ __forceinline__ void tma_load_2d_alone(uint32_t smem_dst, const CUtensorMap* map, int x, int y, uint32_t mbar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_dst),
      "l"(map), "r"(x), "r"(y), "r"(mbar)
      : "memory");
}
// A tile into this CTA's shared memory, its bytes counted on `mbar` (a cluster address: the leader's barrier)
__device__ __forceinline__ void tma_load_2d(uint32_t smem_dst, const CUtensorMap* map, int x, int y, uint32_t mbar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(smem_dst),
      "l"(map), "r"(x), "r"(y), "r"(mbar)
      : "memory");
}

// a tile from shared memory (128-byte swizzle) to global memory, clipped at the map's edges; one thread, then a commit
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t smem_src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
               "r"(smem_src)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void arrive_cluster(uint32_t mbar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(mbar) : "memory");
}
// Shared-memory descriptors of the two 16-bit operand forms that TMA writes with 128-byte swizzle: rows of 64 contraction
// values ("K-major": eight rows are 1024 bytes), or rows that run along the other axis and are indexed by the contraction
// ("MN-major": boxes of 64 columns x 64 rows, 8192 bytes apart).
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
  return uint64_t((addr & 0x3ffffu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr) {
  return uint64_t((addr & 0x3ffffu) >> 4) | (uint64_t(8192 >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
// bf16 operands, fp32 accumulator, `rows` (256 by a pair, 128 by one CTA) x `columns` (a multiple of 32 up to 256); bits 15 /
// 16: A / B is MN-major
__host__ __device__ constexpr uint32_t idesc_bf16(int rows, int columns, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) | (uint32_t(columns >> 3) << 17) |
         (uint32_t(rows >> 4) << 24);
}

}  // namespace umma2
}  // namespace frwkv
