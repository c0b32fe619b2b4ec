// dw_groupnorm.cu -- group normalisation with an activation, channels last:
// the C entry points.  The formulas stand in dw_groupnorm.cuh, the kernels in
// dw_groupnorm_cluster.cu (small tensors) and dw_groupnorm_stream.cu (large ones).
#include <cuda_runtime.h>
#include <math.h>

#include "../../include/dwconv_b200.h"
#include "dw_groupnorm.cuh"
#include "dw_groupnorm_cluster.h"
#include "dw_groupnorm_stream.h"
#include "dw_host.h"
#include "dw_launch.h"

namespace dwb {

// a += v, with what the rounding of the sum leaves behind collected in `low` (an exact two-term sum): the error of a sum
// does not grow with its length.
__device__ __forceinline__ void add_exactly(float& a, float& low, float v) {
  const float sum = a + v, of_v = sum - a;
  low += (a - (sum - of_v)) + (v - of_v);
  a = sum;
}
// Where the sum is an infinity or a NaN, nothing else can be said of it.
__device__ __forceinline__ float sum_of(float a, float low) { return fabsf(a) < INFINITY ? a + low : a; }

// dweight[c] and dbias[c]: the rows of sums added up, 32 threads a channel, each over every 32nd row in order (the
// rows of a large batch are one round of loads then: the gradient at 32x32x1536, B = 16, 67.1 us with 8, 65.9 with 32).
// A row is a sample or a chunk of one, so a thread may have thousands of them: 70000 samples are 2188.
constexpr int kParamChannels = 8, kParamParts = 32;
template <typename T>
__global__ void __launch_bounds__(kParamChannels * kParamParts)
    gn_grad_params_kernel(const float2* __restrict__ sums, long long rows, void* __restrict__ dweight, void* __restrict__ dbias,
                          const GnShape s) {
  __shared__ float2 ent[kParamParts][kParamChannels + 1];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x % kParamChannels, part = threadIdx.x / kParamChannels;
  const int c = blockIdx.x * kParamChannels + lane;  // C is a multiple of 8
  float2 a = make_float2(0.0f, 0.0f), low = a;
#pragma unroll 8
  for (long long r = part; r < rows; r += kParamParts) {
    const float2 e = sums[r * s.C + c];
    add_exactly(a.x, low.x, e.x);
    add_exactly(a.y, low.y, e.y);
  }
  a = make_float2(sum_of(a.x, low.x), sum_of(a.y, low.y));
  ent[part][lane] = a;
  __syncthreads();
  if (part != 0) return;
  a = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < kParamParts; ++i) {
    a.x += ent[i][lane].x;
    a.y += ent[i][lane].y;
  }
  // one rounding to the parameters' own type
  if (dbias) {
    if (s.param_f32) static_cast<float*>(dbias)[c] = a.x;
    else static_cast<T*>(dbias)[c] = static_cast<T>(a.x);
  }
  if (dweight) {
    if (s.param_f32) static_cast<float*>(dweight)[c] = a.y;
    else static_cast<T*>(dweight)[c] = static_cast<T>(a.y);
  }
}

// ---- host -----------------------------------------------------------------------------------------

static int gn_shape(int64_t B, int64_t H, int64_t W, int64_t C, int G, double eps, int act, int dtype, int param_dtype,
                    GnShape* s) {
  if (dtype != DWB_F16 && dtype != DWB_BF16) return DWB_ERR_BAD_ARG;
  if (param_dtype != dtype && param_dtype != DWB_F32) return DWB_ERR_BAD_ARG;
  if (act < DWB_ACT_NONE || act > DWB_ACT_SILU) return DWB_ERR_BAD_ARG;
  if (!(eps >= 0.0) || !(eps < 1e30)) return DWB_ERR_BAD_ARG;
  // B * channels: grid x; H * W: the row index; C: 32-bit channel arithmetic
  if (B < 0 || B > (1 << 30) || H < 1 || W < 1 || H > (1 << 30) || W > (1 << 30) || C < 8 || C > 65536 || (C % 8) != 0)
    return DWB_ERR_BAD_SHAPE;
  if (H * W > 0x7fffffffLL) return DWB_ERR_BAD_SHAPE;
  if (G < 1 || G > C || (C % G) != 0) return DWB_ERR_BAD_SHAPE;
  s->P = H * W;
  s->B = static_cast<int>(B);
  s->C = static_cast<int>(C);
  s->G = G;
  s->Cg = static_cast<int>(C / G);
  s->eps = static_cast<float>(eps);
  s->param_f32 = param_dtype == DWB_F32;
  s->param_vec = 0;
  return DWB_OK;
}

// How a call runs: in the shared memory of clusters (gn_resident_plan has the rule) or in two streaming passes.
struct GnPlan {
  bool resident;
  GnResident cluster;
  GnStream stream;
};

static bool gn_plan(const GnShape& s, GnPass pass, GnPlan* p) {
  p->resident = gn_resident_plan(s, pass, &p->cluster);
  return p->resident || gn_stream_plan(s, pass == GnPass::kForward ? 2 : pass == GnPass::kBackward16 ? 4 : 3, &p->stream);
}

// float2 values of workspace.  Forward: the streaming passes' entries.  Backward: the channels' sums (of every
// sample, or of every sample's chunks), then the entries.
static int64_t gn_workspace(const GnShape& s, const GnPlan& p, GnPass pass) {
  const int64_t rows = p.resident ? s.B : static_cast<int64_t>(s.B) * p.stream.chunks;
  const int64_t entries = p.resident ? 0 : rows * p.stream.entries;
  return pass == GnPass::kForward ? entries : rows * s.C + entries;
}

static int gn_launch(const void* fn, const char* what, dim3 grid, int threads, void** args, cudaStream_t stream) {
  const cudaError_t e = launch_kernel(fn, grid, dim3(threads), args, 0, stream);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return record_cuda_failure(what, e);
  }
  return DWB_OK;
}

template <typename T>
static int gn_forward(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, void* codes,
                      void* scales, void* workspace, const GnShape& s, const GnPlan& p, int act, cudaStream_t stream) {
  if (p.resident) return gn_resident_forward<T>(x, weight, bias, y, mean, rstd, codes, scales, s, p.cluster, act, stream);
  return gn_stream_forward<T>(x, weight, bias, y, mean, rstd, codes, scales, static_cast<float2*>(workspace), s, p.stream, act,
                              stream);
}

template <typename T>
static int gn_backward(const void* dy, const void* x, const void* codes, const void* scales, const float* mean,
                       const float* rstd, const void* weight, const void* bias, void* dx, void* dweight, void* dbias,
                       void* workspace, GnShape s, const GnPlan& p, int act, cudaStream_t stream) {
  float2* sums = static_cast<float2*>(workspace);
  long long rows = s.B;
  int rc;
  if (p.resident) {
    rc = gn_resident_backward<T>(dy, x, codes, scales, mean, rstd, weight, bias, dx, sums, s, p.cluster, act, stream);
  } else {
    rows *= p.stream.chunks;
    rc = gn_stream_backward<T>(dy, x, codes, scales, mean, rstd, weight, bias, dx, sums + rows * s.C, sums, s, p.stream, act,
                               stream);
  }
  if (rc != DWB_OK || (!dweight && !dbias)) return rc;
  void* args[] = {&sums, &rows, &dweight, &dbias, &s};
  return gn_launch(reinterpret_cast<const void*>(&gn_grad_params_kernel<T>), "gn_grad_params_kernel",
                   dim3(s.C / kParamChannels), kParamChannels * kParamParts, args, stream);
}

}  // namespace dwb

extern "C" int dwb_group_norm_act_workspace(int64_t B, int64_t H, int64_t W, int64_t C, int G, int backward, int64_t* bytes) {
  using namespace dwb;
  if (!bytes) return DWB_ERR_NULL_POINTER;
  GnShape s;
  const int rc = gn_shape(B, H, W, C, G, 0.0, DWB_ACT_NONE, DWB_F16, DWB_F16, &s);
  if (rc != DWB_OK) return rc;
  int64_t most = 0;
  for (GnPass pass : {GnPass::kForward, GnPass::kBackward16, GnPass::kBackward8}) {
    if ((pass != GnPass::kForward) != (backward != 0) || B == 0) continue;
    GnPlan p;
    if (!gn_plan(s, pass, &p)) return DWB_ERR_BAD_SHAPE;
    const int64_t n = gn_workspace(s, p, pass);
    most = n > most ? n : most;
  }
  *bytes = most * static_cast<int64_t>(sizeof(float2));
  return DWB_OK;
}

extern "C" int dwb_group_norm_act_nhwc_fwd(const void* x, const void* weight, const void* bias, void* y, float* mean,
                                           float* rstd, void* codes, void* scales, void* workspace, int64_t workspace_bytes,
                                           int64_t B, int64_t H, int64_t W, int64_t C, int G, double eps, int act, int dtype,
                                           int param_dtype, void* stream) {
  using namespace dwb;
  GnShape s;
  int rc = gn_shape(B, H, W, C, G, eps, act, dtype, param_dtype, &s);
  if (rc != DWB_OK || B == 0) return rc;
  if (!x || !y || !mean || !rstd || (codes == nullptr) != (scales == nullptr)) return DWB_ERR_NULL_POINTER;
  GnPlan p;
  if (!gn_plan(s, GnPass::kForward, &p)) return DWB_ERR_BAD_SHAPE;
  const int64_t need = gn_workspace(s, p, GnPass::kForward) * static_cast<int64_t>(sizeof(float2));
  if (need > 0 && !workspace) return DWB_ERR_NULL_POINTER;
  if (workspace_bytes < need) return DWB_ERR_BAD_ARG;
  const uintptr_t pa = param_dtype == DWB_F32 ? 4 : 2;
  if (!is_aligned(x, 16) || !is_aligned(y, 16) || !is_aligned(codes, 8) || !is_aligned(mean, 4) || !is_aligned(rstd, 4) ||
      !is_aligned(weight, pa) || !is_aligned(bias, pa) || !is_aligned(workspace, 16))
    return DWB_ERR_BAD_ALIGN;
  rc = require_device();
  if (rc != DWB_OK) return rc;
  s.param_vec = is_aligned(weight, 16) && is_aligned(bias, 16);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == DWB_F16 ? gn_forward<__half>(x, weight, bias, y, mean, rstd, codes, scales, workspace, s, p, act, st)
                          : gn_forward<__nv_bfloat16>(x, weight, bias, y, mean, rstd, codes, scales, workspace, s, p, act, st);
}

extern "C" int dwb_group_norm_act_nhwc_bwd(const void* dy, const void* x, const void* codes, const void* scales,
                                           const float* mean, const float* rstd, const void* weight, const void* bias, void* dx,
                                           void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, int64_t B,
                                           int64_t H, int64_t W, int64_t C, int G, int act, int dtype, int param_dtype,
                                           void* stream) {
  using namespace dwb;
  GnShape s;
  int rc = gn_shape(B, H, W, C, G, 0.0, act, dtype, param_dtype, &s);
  if (rc != DWB_OK) return rc;
  const uintptr_t pa = param_dtype == DWB_F32 ? 4 : 2;
  const GnPass pass = codes ? GnPass::kBackward8 : GnPass::kBackward16;
  GnPlan p;
  if (B > 0) {
    if (!dy || !dx || !mean || !rstd || (codes == nullptr) != (scales == nullptr)) return DWB_ERR_NULL_POINTER;
    if ((x == nullptr) == (codes == nullptr)) return x ? DWB_ERR_BAD_ARG : DWB_ERR_NULL_POINTER;  // one of the two
    if (!gn_plan(s, pass, &p)) return DWB_ERR_BAD_SHAPE;
    const int64_t need = gn_workspace(s, p, pass) * static_cast<int64_t>(sizeof(float2));
    if (!workspace) return DWB_ERR_NULL_POINTER;
    if (workspace_bytes < need) return DWB_ERR_BAD_ARG;
  }
  if (!is_aligned(dy, 16) || !is_aligned(x, 16) || !is_aligned(dx, 16) || !is_aligned(codes, 8) || !is_aligned(mean, 4) ||
      !is_aligned(rstd, 4) || !is_aligned(weight, pa) || !is_aligned(bias, pa) || !is_aligned(dweight, pa) ||
      !is_aligned(dbias, pa) || !is_aligned(workspace, 16))
    return DWB_ERR_BAD_ALIGN;
  if (B == 0 && !dweight && !dbias) return DWB_OK;
  rc = require_device();
  if (rc != DWB_OK) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (B == 0) {  // no sample: the parameters' gradients are zero
    const size_t n = static_cast<size_t>(C) * pa;
    cudaError_t e = cudaSuccess;
    if (dweight) e = cudaMemsetAsync(dweight, 0, n, st);
    if (e == cudaSuccess && dbias) e = cudaMemsetAsync(dbias, 0, n, st);
    return e == cudaSuccess ? DWB_OK : record_cuda_failure("cudaMemsetAsync(dweight, dbias)", e);
  }
  s.param_vec = is_aligned(weight, 16) && is_aligned(bias, 16);
  return dtype == DWB_F16 ? gn_backward<__half>(dy, x, codes, scales, mean, rstd, weight, bias, dx, dweight, dbias, workspace,
                                                s, p, act, st)
                          : gn_backward<__nv_bfloat16>(dy, x, codes, scales, mean, rstd, weight, bias, dx, dweight, dbias,
                                                       workspace, s, p, act, st);
}
