// Launch of a kernel before the one ahead of it in the stream has ended (programmatic launch), so
// that its blocks are in place when that one's last has left. Such a kernel begins with
// wait_for_stream() in every thread, before it reads or writes memory.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

namespace ta {

template <class... Params, class... Args>
inline cudaError_t launch_overlapped(void (*kernel)(Params...), dim3 grid, int threads, size_t smem,
                                     cudaStream_t stream, Args&&... args) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args&&>(args)...);
}

__device__ __forceinline__ void wait_for_stream() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// From here on the next kernel's blocks may take free places.
__device__ __forceinline__ void let_next_kernel_in() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace ta
