// Kernel launches of the library's entry points (host side).
#pragma once

#include <cuda_runtime.h>

#include <cstdlib>

namespace cfm {

// Launch with programmatic stream serialisation: the kernel may be scheduled while its
// predecessor in the stream is finishing and waits for it at grid_dependency_wait().
// Used for every launch of a whole call (measured for two of them: 0.6 to 1.3 us per call).  CFM_PDL=0 in the environment makes these ordinary
// launches.  `cluster` CTAs, consecutive in x, share a cluster.
template <typename... Params, typename... Args>
static void launch_clusters(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, int cluster,
                            cudaStream_t stream, Args... args) {
  static const bool on = [] {
    const char* v = std::getenv("CFM_PDL");
    return !v || std::atoi(v) != 0;
  }();
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  config.attrs = attributes;
  if (on) {
    attributes[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attributes[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attributes[config.numAttrs].val.clusterDim.x = cluster;
    attributes[config.numAttrs].val.clusterDim.y = 1;
    attributes[config.numAttrs++].val.clusterDim.z = 1;
  }
  (void)cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
}

template <typename... Params, typename... Args>
static void launch_dependent(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem,
                             cudaStream_t stream, Args... args) {
  launch_clusters(kernel, grid, block, smem, 1, stream, args...);
}

static int launched() {
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? 0 : static_cast<int>(err);
}

}  // namespace cfm
