// Thread-block clusters whose blocks share numbers through one another's shared memory.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace moba {

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
// All threads of all blocks; what was written before, to global or any block's shared memory, is visible behind it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// In front of the first access to another block's shared memory (which exists once that block runs) lies a cluster_sync; so does one behind the last
// access, before a block ends.
// The place in block `rank` of what lies at `p` in this block's shared memory.
__device__ __forceinline__ uint32_t cluster_place(const void* p, uint32_t rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ void cluster_store(uint32_t at, uint64_t x) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(at), "l"(x) : "memory");
}
__device__ __forceinline__ void cluster_store(uint32_t at, uint32_t x) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at), "r"(x) : "memory");
}

// A launch behind the kernel before it (see launch_pdl), in clusters of `size` blocks.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_clusters(void (*kernel)(KArgs...), int size, dim3 grid, int threads, size_t smem, cudaStream_t st, const Args&... args) {
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = (unsigned)size;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attrs;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace moba
