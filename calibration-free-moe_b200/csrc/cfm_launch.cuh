// Kernel launches of the library's entry points (host side).
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstdlib>

namespace cfm {

// Lets a kernel have as much shared memory, and clusters of as many CTAs, as the device has.  Once per kernel and
// device (of the first 64): the two calls take 1.5 us of a launch.
template <auto KERNEL>
static int allow_everything(bool large_clusters) {
  static std::atomic<uint64_t> done{0};
  int device = 0;
  cudaError_t code = cudaGetDevice(&device);
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (code != cudaSuccess || (done.load(std::memory_order_relaxed) & bit)) return static_cast<int>(code);
  cudaFuncAttributes attributes;
  int most = 0;
  code = cudaFuncGetAttributes(&attributes, KERNEL);
  if (code == cudaSuccess) code = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, device);
  if (code == cudaSuccess)
    code = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, most - static_cast<int>(attributes.sharedSizeBytes));
  if (code == cudaSuccess && large_clusters) code = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (code == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return static_cast<int>(code);
}

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
