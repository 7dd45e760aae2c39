// Thread-block clusters: barriers and distributed shared memory; and launches that overlap with the one before.
#pragma once

#include "common.cuh"

namespace actnn {
#ifdef __CUDACC__
ACTNN_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
ACTNN_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// The two halves, for work in between.
ACTNN_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
ACTNN_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// From the shared memory of block `rank`, at the place that `addr` is in this block's.
ACTNN_DEV uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  return remote;
}
// Arrives at a barrier of the cluster.
ACTNN_DEV void peer_arrive(uint32_t remote) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(remote) : "memory");
}
ACTNN_DEV void peer_store1(uint32_t addr, uint32_t rank, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" :: "r"(peer_addr(addr, rank)), "r"(v) : "memory");
}
// Sends 16 bytes to block `rank`, whose barrier counts them as they arrive.
ACTNN_DEV void peer_send4(uint32_t addr, uint32_t bar, uint32_t rank, const float4& v) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1,%2,%3,%4}, [%5];"
               :: "r"(peer_addr(addr, rank)), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(peer_addr(bar, rank)) : "memory");
}
ACTNN_DEV int4 peer_load4i(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  int4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(remote) : "memory");
  return v;
}
ACTNN_DEV float4 peer_load4(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
  return v;
}

// ------------------------------------------------------------------ launches that overlap
// The next launch of the stream may begin (where it was launched to); and: all launches before this one are over.
ACTNN_DEV void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
ACTNN_DEV void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
#endif
}  // namespace actnn
