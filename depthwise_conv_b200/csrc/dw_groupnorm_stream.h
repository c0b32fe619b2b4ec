// dw_groupnorm_stream.h -- the two-pass group-norm kernels' plan and launch,
// shared by dw_groupnorm.cu (entry points) and dw_groupnorm_stream.cu.
#pragma once

#include <cuda_runtime.h>

namespace dwb {

struct GnShape;

struct GnStream {
  // first pass: a CTA takes a tile of channels and a chunk of rows
  int tile, tiles;            // channels; tiles of a sample
  int tiles_per_group;        // > 1: a group larger than a tile
  int entries_per_group;      // partial results of a group in a chunk
  int entries;                // of a sample in a chunk
  int sub;                    // channels of a vector that surely share a segment (8, 4 or 1)
  int lanes, rl;              // threads along a pixel, pixels at once
  unsigned lane_mul;          // thread / lanes = thread * lane_mul >> 16
  int rows, chunks;
  // second pass
  int apply_lanes, apply_rl, apply_tiles;
  unsigned apply_lane_mul;
  int apply_rows, apply_chunks;
  int samples;                // of a launch
  // one launch: what it does
  int first_sample, second_sample;
  unsigned first_ctas, second_ctas;
  int early;                  // its inputs are ready whatever the launch before it does
};

// bytes_per_value: what the two passes read of a value.  False: too many CTAs for a grid.
bool gn_stream_plan(const GnShape& s, int bytes_per_value, GnStream* q);

// part: [B][chunks][entries] float2.
template <typename T>
int gn_stream_forward(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, void* codes,
                      void* scales, float2* part, const GnShape& s, const GnStream& q, int act, cudaStream_t stream);

// part: as above; chan: [B][chunks][C] float2 (sum g, sum g xh).
template <typename T>
int gn_stream_backward(const void* dy, const void* x, const void* codes, const void* scales, const float* mean,
                       const float* rstd, const void* weight, const void* bias, void* dx, float2* part, float2* chan,
                       const GnShape& s, const GnStream& q, int act, cudaStream_t stream);

}  // namespace dwb
