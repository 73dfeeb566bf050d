// Kernel launches that overlap the one before them.
#pragma once

#include "common.cuh"

namespace kda {

// `args...` launched so that its CTAs may take their places while the launch
// before it drains; the kernels wait (griddepcontrol.wait) before they read
// what that launch wrote.
template <typename... P, typename... A>
kda_status launch_after(const char* what, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                        A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  return launch_status(what);
}

}  // namespace kda
