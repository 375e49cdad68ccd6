// Thread-block clusters: rank, barrier, and reads of another CTA's shared memory.
#pragma once

#include <stdint.h>

namespace speckv {

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of CTA `rank`'s copy of a shared variable.
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t local = (uint32_t)__cvta_generic_to_shared(p), at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
  return at;
}
__device__ __forceinline__ float remote_float(const void* p, uint32_t rank) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(remote(p, rank)) : "memory");
  return x;
}
__device__ __forceinline__ float4 remote_float4(const void* p, uint32_t rank) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
               : "r"(remote(p, rank))
               : "memory");
  return x;
}
__device__ __forceinline__ unsigned long long remote_u64(const void* p, uint32_t rank) {
  unsigned long long x;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(remote(p, rank)) : "memory");
  return x;
}

}  // namespace speckv
