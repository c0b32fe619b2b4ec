// dw_groupnorm_cluster.h -- the resident group-norm kernels' plan and launch,
// shared by dw_groupnorm.cu (entry points) and dw_groupnorm_cluster.cu.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace dwb {

struct GnShape;

// A cluster of CTAs holds one sample's channels [slab] in shared memory.
struct GnResident {
  int slab;          // channels of a cluster: whole groups, whole checkpoint blocks
  int slabs;         // clusters a sample
  int lanes;         // threads along a pixel (a multiple of 4)
  int rl;            // pixels a CTA handles at once
  int threads;       // lanes * rl, rounded up to a warp
  unsigned lane_mul; // thread / lanes = thread * lane_mul >> 16
  int cluster;       // CTAs that share the sample's pixels: 1 << cluster_log
  int cluster_log;
  int rows_per_cta;
  int iters;         // pixels a thread handles
  int smem;
};

enum class GnPass { kForward, kBackward16, kBackward8 };

// Whether the resident kernels take this shape, and how.
bool gn_resident_plan(const GnShape& s, GnPass pass, GnResident* p);

template <typename T>
int gn_resident_forward(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, void* codes,
                        void* scales, const GnShape& s, const GnResident& p, int act, cudaStream_t stream);

// sums: [B][C] float2 (sum g, sum g xh) of every sample.
template <typename T>
int gn_resident_backward(const void* dy, const void* x, const void* codes, const void* scales, const float* mean,
                         const float* rstd, const void* weight, const void* bias, void* dx, float2* sums, const GnShape& s,
                         const GnResident& p, int act, cudaStream_t stream);

}  // namespace dwb
