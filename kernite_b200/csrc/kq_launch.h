// kq_launch.h -- kernel launches with programmatic dependent launch: a kernel's blocks may start once every
// block of the one before it on the stream has called pdl_launch_dependents() (or ended), and wait in
// pdl_wait() until that one's memory is visible. A kernel launched this way touches no memory of its
// callers before its pdl_wait().
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace kq {

template <typename T>
struct SameType {
  using Type = T;
};

template <typename... P>
cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, uint32_t threads, size_t shared, cudaStream_t stream,
                       const typename SameType<P>::Type&... args) {
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  void* list[] = {const_cast<void*>(static_cast<const void*>(&args))...};
  return cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kernel), list);
}

}  // namespace kq
