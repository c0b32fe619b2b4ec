// dw_wgrad_act8.cu -- the depthwise weight gradient from the 8-bit checkpoint of
// the convolution's input (dw_act8.cuh):
//   dw[kh][kw][c] = sum over b, h, w of dy[b][h][w][c] * x[b][h + kh - K/2][w + kw - K/2][c]
//
// One CTA per (32 channels, kernel row, chunk of output rows); lane = channel,
// warp = every 8th kernel column.  The chunks' sums go to slices of the
// workspace and a second kernel adds them in order.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/dwconv_b200.h"
#include "dw_act8.cuh"
#include "dw_host.h"
#include "dw_launch.h"

namespace dwb {

struct Wgrad8Params {
  int B, H, W, C, K;
  long long rows_per_chunk;
  int chunks;
};

__global__ void __launch_bounds__(256) wgrad8_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                     const __half* __restrict__ dy, float* __restrict__ part,
                                                     const Wgrad8Params p) {
  griddep_wait();
  griddep_launch_dependents();
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), warp = threadIdx.x >> 5;
  if (c >= p.C) return;
  const int kh = blockIdx.y, pad = p.K / 2;
  const long long r0 = blockIdx.z * p.rows_per_chunk;
  const long long all = static_cast<long long>(p.B) * p.H;
  const long long r1 = r0 + p.rows_per_chunk < all ? r0 + p.rows_per_chunk : all;
  const int sblocks = (p.C + kAct8Block - 1) / kAct8Block;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (long long r = r0; r < r1; ++r) {
    const long long b = r / p.H;
    const int ih = static_cast<int>(r - b * p.H) + kh - pad;
    if (ih < 0 || ih >= p.H) continue;
    const long long drow = r * p.W, xrow = (b * p.H + ih) * p.W;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int kw = warp + 8 * j;
      if (kw >= p.K) break;
      const int w0 = pad - kw > 0 ? pad - kw : 0, w1 = p.W < p.W + pad - kw ? p.W : p.W + pad - kw;
      for (int w = w0; w < w1; ++w) {
        const long long xp = xrow + w + kw - pad;
        const float x = static_cast<float>(codes[xp * p.C + c]) * act8_step(scales[xp * sblocks + c / kAct8Block]);
        acc[j] += __half2float(dy[(drow + w) * p.C + c]) * x;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int kw = warp + 8 * j;
    if (kw < p.K) part[((static_cast<long long>(blockIdx.z) * p.K + kh) * p.K + kw) * p.C + c] = acc[j];
  }
}

// dw[i] = the slices' values added in slice order (n4 groups of 4).
__global__ void __launch_bounds__(256) wgrad8_reduce_kernel(const float4* __restrict__ part, float4* __restrict__ dw,
                                                            long long n4, int slices) {
  griddep_wait();
  griddep_launch_dependents();
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n4) return;
  float4 a = part[i];
  for (int s = 1; s < slices; ++s) {
    const float4 v = part[s * n4 + i];
    a.x += v.x;
    a.y += v.y;
    a.z += v.z;
    a.w += v.w;
  }
  dw[i] = a;
}

static int wgrad8_plan(int64_t B, int64_t H, int64_t W, int64_t C, int K, Wgrad8Params* p) {
  if (K < 1 || K > 31 || (K % 2) == 0 || B < 0 || H < 1 || W < 1 || C < 8 || (C % 8) != 0) return DWB_ERR_BAD_SHAPE;
  if (B > (1 << 30) || H > (1 << 24) || W > (1 << 24) || C > (1 << 20)) return DWB_ERR_BAD_SHAPE;
  p->B = static_cast<int>(B);
  p->H = static_cast<int>(H);
  p->W = static_cast<int>(W);
  p->C = static_cast<int>(C);
  p->K = K;
  const long long rows = B * H > 0 ? B * H : 1;
  const long long base = (C + 31) / 32 * K;
  long long chunks = (8LL * kSmCount + base - 1) / base;
  chunks = chunks < rows ? chunks : rows;
  p->rows_per_chunk = (rows + chunks - 1) / chunks;
  p->chunks = static_cast<int>((rows + p->rows_per_chunk - 1) / p->rows_per_chunk);
  return DWB_OK;
}

static int64_t wgrad8_workspace(const Wgrad8Params& p) {
  return static_cast<int64_t>(p.chunks) * p.K * p.K * p.C * static_cast<int64_t>(sizeof(float));
}

}  // namespace dwb

extern "C" int dwb_conv2d_nhwc_bwd_weight_act8_workspace(int64_t B, int64_t H, int64_t W, int64_t C, int K, int64_t* bytes) {
  using namespace dwb;
  if (!bytes) return DWB_ERR_NULL_POINTER;
  Wgrad8Params p;
  const int rc = wgrad8_plan(B, H, W, C, K, &p);
  if (rc != DWB_OK) return rc;
  *bytes = B == 0 ? 0 : wgrad8_workspace(p);
  return DWB_OK;
}

extern "C" int dwb_conv2d_nhwc_bwd_weight_act8(const void* codes, const void* scales, const void* dy, float* dw,
                                               void* workspace, int64_t workspace_bytes, int64_t B, int64_t H, int64_t W,
                                               int64_t C, int K, void* stream) {
  using namespace dwb;
  Wgrad8Params p;
  int rc = wgrad8_plan(B, H, W, C, K, &p);
  if (rc != DWB_OK) return rc;
  if (!dw) return DWB_ERR_NULL_POINTER;
  if (B > 0) {
    if (!codes || !scales || !dy || !workspace) return DWB_ERR_NULL_POINTER;
    if (workspace_bytes < wgrad8_workspace(p)) return DWB_ERR_BAD_ARG;
  }
  if (!is_aligned(codes, 8) || !is_aligned(dy, 16) || !is_aligned(dw, 16) || !is_aligned(workspace, 16))
    return DWB_ERR_BAD_ALIGN;
  rc = require_device();
  if (rc != DWB_OK) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (B == 0) {
    const cudaError_t e = cudaMemsetAsync(dw, 0, static_cast<size_t>(K) * K * C * 4, st);
    return e == cudaSuccess ? DWB_OK : record_cuda_failure("cudaMemsetAsync(dw)", e);
  }
  float* part = static_cast<float*>(workspace);
  void* a1[] = {&codes, &scales, &dy, &part, &p};
  cudaError_t e = launch_kernel(reinterpret_cast<const void*>(&wgrad8_kernel),
                                dim3(static_cast<unsigned>((C + 31) / 32), K, p.chunks), dim3(256), a1, 0, st);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return record_cuda_failure("wgrad8_kernel", e);
  }
  long long n4 = static_cast<long long>(K) * K * C / 4;
  void* a2[] = {&part, &dw, &n4, &p.chunks};
  e = launch_kernel(reinterpret_cast<const void*>(&wgrad8_reduce_kernel), dim3(static_cast<unsigned>((n4 + 255) / 256)),
                    dim3(256), a2, 0, st);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return record_cuda_failure("wgrad8_reduce_kernel", e);
  }
  return DWB_OK;
}
