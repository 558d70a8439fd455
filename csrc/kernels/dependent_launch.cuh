// Kernels of one stream that start before the one ahead of them has ended: what a kernel sets up for itself (barriers, tensor memory, its launch)
// then overlaps with the other's last blocks.  A kernel launched with this attribute touches no global memory before wait_for_previous(), in any
// thread that does, and every thread block calls it; let_next_start() comes after everything that a block of the next kernel could
// otherwise take away (tensor memory).  A neighbour launched without the attribute is kept apart as ever.
#pragma once
#include <cuda_runtime.h>

namespace mnccl {

// The kernels ahead in the stream have ended and what they wrote is there.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// What the kernels ahead wrote is read through pointers without __restrict__ (which would let the compiler take loads from before the wait, or through
// a cache that is not kept coherent), vectors by load_vector() from a pointer that since_wait() hands on behind it.
template <typename T>
__device__ __forceinline__ const T* since_wait(const T* p) {
  asm volatile("" : "+l"(p)::"memory");
  return p;
}
__device__ __forceinline__ uint4 load_vector(const void* p) {
  uint4 v;
  asm("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// The next kernel may start its blocks, once all blocks of this one have come here.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

inline cudaLaunchAttribute early_start() {
  cudaLaunchAttribute a = {};
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  return a;
}

template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, dim3 block, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attr[1] = {early_start()};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

}  // namespace mnccl
