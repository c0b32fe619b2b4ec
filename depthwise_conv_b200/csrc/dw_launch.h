// dw_launch.h -- kernel launches with programmatic dependent launch (PDL).
//
// Every engine kernel is launched with the programmatic stream-serialization
// attribute: it may start (barrier set-up, tensor-map prefetch) while the
// previous kernel of the stream drains, and waits in griddep_wait() before it
// touches global memory.  DWB_PDL=0 in the environment launches without the
// attribute (plain stream order), for comparisons.
#pragma once

#include <cuda_runtime.h>
#include <stdlib.h>

namespace dwb {

inline bool pdl_enabled() {
  static const bool on = [] {
    const char* v = getenv("DWB_PDL");
    return !(v && v[0] == '0');
  }();
  return on;
}

// cluster > 1: thread-block clusters of that many CTAs along x.
inline cudaError_t launch_kernel(const void* fn, dim3 grid, dim3 block, void** args, size_t smem,
                                 cudaStream_t stream, unsigned cluster = 1) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelExC(&cfg, fn, args);
}

}  // namespace dwb
