// pdl_launch.h -- launch configuration with the programmatic stream-serialisation
// attribute (sm100_ptx.cuh: grid_dependency_wait).
#pragma once

#include <cuda_runtime.h>

namespace clove {
namespace rt {

// `la` must outlive the launch.
inline cudaLaunchConfig_t pdl_config(dim3 grid, int threads, int smem, cudaStream_t stream,
                                     cudaLaunchAttribute* la) {
  la->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  la->val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cfg.attrs = la;
  cfg.numAttrs = 1;
  return cfg;
}

}  // namespace rt
}  // namespace clove
