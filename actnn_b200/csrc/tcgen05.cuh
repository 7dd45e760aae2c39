// The 5th-generation tensor core, tensor memory and tiled bulk copies, as thin wrappers of the PTX instructions.
#pragma once

#include <cuda.h>

#include "cluster.cuh"

namespace actnn {
#ifdef __CUDACC__

// ------------------------------------------------------------------ barriers
ACTNN_DEV void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory"); }

// ------------------------------------------------------------------ tiled copies
// A box of a rank-2 tensor to shared memory; x (elements of the contiguous dimension) starts on 16 bytes.
ACTNN_DEV void tile_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
// A box from shared memory; what reaches past the tensor is not written.  Stores of a thread are counted in groups.
ACTNN_DEV void tile_store(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
               :: "l"(map), "r"(x), "r"(y), "r"(src) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Until all but LEFT of the thread's groups have read their shared memory; and until all are written.
template <int LEFT> ACTNN_DEV void tile_store_read() { asm volatile("cp.async.bulk.wait_group.read %0;" :: "n"(LEFT) : "memory"); }
ACTNN_DEV void tile_store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// Ordinary writes to shared memory before, seen by copies after.
ACTNN_DEV void tile_store_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The same by one of a pair of blocks that computes together: the bytes are counted on a barrier of either, `bar` an address in
// the cluster.
ACTNN_DEV void tile_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

// ------------------------------------------------------------------ tensor memory
// One whole warp allocates (a power of two of columns, 32 at least), and the same warp frees; of a PAIR, one in each block.
template <bool PAIR> ACTNN_DEV void tmem_alloc(uint32_t dst_smem, uint32_t columns) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(dst_smem), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(dst_smem), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
}
template <bool PAIR> ACTNN_DEV void tmem_free(uint32_t addr, uint32_t columns) {
  if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(addr), "r"(columns));
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(addr), "r"(columns));
}
ACTNN_DEV void tmem_fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
ACTNN_DEV void tmem_fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 16 columns of the warp's 32 lanes (the quarter that its number modulo four names): column i of lane l in r[i] of lane l.
ACTNN_DEV void tmem_load16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                 "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(addr));
}
ACTNN_DEV void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// ------------------------------------------------------------------ matrix instructions
// Shared-memory operand whose rows of 128 bytes run along the reduction, swizzled in 128-byte lines: eight rows are 1024
// bytes, and 1024 bytes further come the next eight.  `addr` on 1024 bytes (plus the offset along the reduction).
ACTNN_DEV uint64_t rows128_descriptor(uint32_t addr) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
// Signed 8-bit operands, 32-bit integer sums: m rows of A (128, or 256 of a pair), n rows of B (16, or 32 to 256 in steps of 16; of
// a pair in steps of 32).
ACTNN_DEV uint32_t int8_instruction(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// D[m, n] (+)= A[m, 32] B[n, 32]^T, issued by one thread.  Of a PAIR by the first block alone: each holds half of the rows of A, of
// those of B, and of D, at the same places.
template <bool PAIR> ACTNN_DEV void mma_int8(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool add) {
  if constexpr (PAIR)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                 :: "r"(d), "l"(a), "l"(b), "r"(instruction), "r"((uint32_t)add) : "memory");
}
// The barrier (of a PAIR that of both blocks) is arrived at once all matrix instructions that this thread issued before are done.
template <bool PAIR> ACTNN_DEV void mma_commit(uint32_t bar) {
  if constexpr (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 :: "r"(bar), "h"((uint16_t)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
#endif
}  // namespace actnn
