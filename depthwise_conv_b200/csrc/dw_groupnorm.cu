// dw_groupnorm.cu -- group normalisation with an activation, channels last:
// the C entry points, and the split kernels (statistics, combination,
// application as separate launches over row chunks) for groups that are too
// large for the shared memory of a cluster (dw_groupnorm_cluster.cu takes all
// others).  The formulas stand in dw_groupnorm.cuh.
#include <cuda_runtime.h>
#include <math.h>

#include "../../include/dwconv_b200.h"
#include "dw_groupnorm.cuh"
#include "dw_groupnorm_cluster.h"
#include "dw_host.h"
#include "dw_launch.h"

namespace dwb {

constexpr int kGnThreads = 256;
constexpr int kGnTileVecs = 16;  // 128 channels = 256 bytes of a pixel a CTA

// Split of one call: CTA (sample, row chunk, channel tile).
struct GnSplit {
  long long rows_per_chunk;
  int chunks;
  int lanes;   // threads along a pixel (a multiple of 4: the quads of the checkpoint's blocks)
  int rl;      // pixels a CTA handles at once
  int tiles;
};

struct GnThread {
  int c, lane_row;
  bool active;
  long long r0, r1;  // rows of the chunk
  long long sample;
  __device__ __forceinline__ GnThread(const GnShape& s, const GnSplit& p) {
    sample = blockIdx.x;
    const int t = threadIdx.x;
    lane_row = t / p.lanes;
    c = (static_cast<int>(blockIdx.z) * p.lanes + (t - lane_row * p.lanes)) * 8;
    active = lane_row < p.rl && c < s.C;
    r0 = blockIdx.y * p.rows_per_chunk;
    r1 = r0 + p.rows_per_chunk < s.P ? r0 + p.rows_per_chunk : s.P;
  }
};

// ---- forward ------------------------------------------------------------------------------------

// part[sample][chunk][c] = (mean, M2) of the chunk's rows of channel c.
template <typename T>
__global__ void __launch_bounds__(kGnThreads) gn_stats_kernel(const uint4* __restrict__ x, float2* __restrict__ part,
                                                              const GnShape s, const GnSplit p) {
  __shared__ float2 ent[kGnThreads * 8];
  griddep_wait();
  griddep_launch_dependents();
  const GnThread th(s, p);
  const int width = p.lanes * 8;
  if (th.active) {
    const uint4* base = x + (th.sample * s.P * s.C + th.c) / 8;
    const long long step = s.C / 8;
    const long long r = th.r0 + th.lane_row;
    if (r < th.r1) {
      GnSums sums;
      f32x2 f[4];
      gn_unpack<T>(base[r * step], f);
      sums.start(f);
      const int n = static_cast<int>((th.r1 - r + p.rl - 1) / p.rl);
      for (int i = 1; i < n; i += 4) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j < n) v[j] = base[(r + static_cast<long long>(i + j) * p.rl) * step];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j < n) {
            gn_unpack<T>(v[j], f);
            sums.add(f);
          }
      }
      f32x2 mean[4], m2[4];
      sums.moments(n, mean, m2);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = bits_f2(mean[i]), q = bits_f2(m2[i]);
        ent[threadIdx.x * 8 + 2 * i] = make_float2(a.x, q.x);
        ent[threadIdx.x * 8 + 2 * i + 1] = make_float2(a.y, q.y);
      }
    }
  }
  __syncthreads();
  const int rows = static_cast<int>(th.r1 - th.r0);
  for (int j = threadIdx.x; j < width; j += kGnThreads) {
    const int c = static_cast<int>(blockIdx.z) * width + j;
    if (c >= s.C) break;
    float sum = 0.0f, m2 = 0.0f;
    for (int i = 0; i < p.rl && i < rows; ++i) sum += static_cast<float>((rows - i + p.rl - 1) / p.rl) * ent[i * width + j].x;
    const float mean = sum / static_cast<float>(rows);
    for (int i = 0; i < p.rl && i < rows; ++i) {
      const float d = ent[i * width + j].x - mean;
      m2 += ent[i * width + j].y + static_cast<float>((rows - i + p.rl - 1) / p.rl) * d * d;
    }
    part[(th.sample * p.chunks + blockIdx.y) * s.C + c] = make_float2(mean, m2);
  }
}

// One CTA a group: the channels' and chunks' moments merged into mean and rstd.
__global__ void __launch_bounds__(128) gn_combine_kernel(const float2* __restrict__ part, float* __restrict__ mean_out,
                                                         float* __restrict__ rstd_out, const GnShape s, const GnSplit p) {
  __shared__ float scratch[33];
  griddep_wait();
  griddep_launch_dependents();
  const long long sample = blockIdx.x;
  const int g = blockIdx.y;
  const float2* base = part + sample * p.chunks * s.C + static_cast<long long>(g) * s.Cg;
  const long long entries = static_cast<long long>(p.chunks) * s.Cg;
  const float n = static_cast<float>(s.P) * static_cast<float>(s.Cg);
  const float last = static_cast<float>(s.P - (p.chunks - 1) * p.rows_per_chunk), full = static_cast<float>(p.rows_per_chunk);
  float sum = 0.0f;
  for (long long j = threadIdx.x; j < entries; j += 128) {
    const int chunk = static_cast<int>(j / s.Cg);
    sum += (chunk == p.chunks - 1 ? last : full) * base[static_cast<long long>(chunk) * s.C + (j - static_cast<long long>(chunk) * s.Cg)].x;
  }
  const float mean = block_sum(sum, scratch) / n;
  float m2 = 0.0f;
  for (long long j = threadIdx.x; j < entries; j += 128) {
    const int chunk = static_cast<int>(j / s.Cg);
    const float2 e = base[static_cast<long long>(chunk) * s.C + (j - static_cast<long long>(chunk) * s.Cg)];
    const float d = e.x - mean;
    m2 += e.y + (chunk == p.chunks - 1 ? last : full) * d * d;
  }
  m2 = block_sum(m2, scratch);
  if (threadIdx.x == 0) {
    mean_out[sample * s.G + g] = mean;
    rstd_out[sample * s.G + g] = 1.0f / sqrtf(m2 / n + s.eps);
  }
}

// mean and rstd of a thread's 8 channels
__device__ __forceinline__ void gn_load_stats(const float* __restrict__ mean, const float* __restrict__ rstd, long long sample,
                                              int c, const GnShape& s, f32x2 (&m)[4], f32x2 (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long a = sample * s.G + (c + 2 * i) / s.Cg, b = sample * s.G + (c + 2 * i + 1) / s.Cg;
    m[i] = f2_bits(make_float2(mean[a], mean[b]));
    r[i] = f2_bits(make_float2(rstd[a], rstd[b]));
  }
}

template <typename T, int ACT, bool CKPT>
__global__ void __launch_bounds__(kGnThreads) gn_apply_kernel(const uint4* __restrict__ x, const void* __restrict__ weight,
                                                              const void* __restrict__ bias, const float* __restrict__ mean,
                                                              const float* __restrict__ rstd, uint4* __restrict__ y,
                                                              uint2* __restrict__ codes, uint8_t* __restrict__ scales,
                                                              const GnShape s, const GnSplit p) {
  griddep_wait();
  griddep_launch_dependents();
  const GnThread th(s, p);
  const long long step = s.C / 8, sblocks = (s.C + kAct8Block - 1) / kAct8Block;
  f32x2 w[4], b[4], m[4], rs[4];
  if (th.active) {
    gn_load_params<T>(weight, bias, th.c, s, w, b);
    gn_load_stats(mean, rstd, th.sample, th.c, s, m, rs);
  }
  // the trip count is the same for the whole CTA: the block maxima are warp shuffles
  for (long long row = th.r0; row < th.r1; row += 2LL * p.rl) {
    uint4 v[2];
    long long pix[2];
    bool on[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long r = row + static_cast<long long>(i) * p.rl + th.lane_row;
      on[i] = th.active && r < th.r1;
      pix[i] = th.sample * s.P + r;
      v[i] = on[i] ? x[pix[i] * step + th.c / 8] : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (CKPT) {
        const uint32_t E = act8_exponent<T>(act8_block_amax(v[i]));
        if (on[i]) {
          codes[pix[i] * step + th.c / 8] = act8_codes<T>(v[i], E);
          if ((th.c & (kAct8Block - 1)) == 0) scales[pix[i] * sblocks + th.c / kAct8Block] = static_cast<uint8_t>(E);
        }
      }
      if (on[i]) {
        f32x2 f[4];
        gn_unpack<T>(v[i], f);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = act_value2<ACT>(fma2(fmul2(fsub2(f[j], m[j]), rs[j]), w[j], b[j]));
        y[pix[i] * step + th.c / 8] = gn_pack<T>(f);
      }
    }
  }
}

// ---- backward -----------------------------------------------------------------------------------

// 8 saved values of the norm's input: 16 bits, or codes and an exponent byte.
template <typename T, bool SRC8>
__device__ __forceinline__ void gn_load_saved(const void* __restrict__ src, const uint8_t* __restrict__ scales, long long pixel,
                                              int c, const GnShape& s, f32x2 (&f)[4]) {
  const long long at = pixel * (s.C / 8) + c / 8;
  if constexpr (SRC8) {
    const float step = act8_step(scales[pixel * ((s.C + kAct8Block - 1) / kAct8Block) + c / kAct8Block]);
    act8_values(static_cast<const uint2*>(src)[at], step, f);
  } else {
    gn_unpack<T>(static_cast<const uint4*>(src)[at], f);
  }
}

// part[sample][chunk][c] = (sum g, sum g xh) over the chunk's rows.
template <typename T, int ACT, bool SRC8>
__global__ void __launch_bounds__(kGnThreads) gn_grad_sums_kernel(const uint4* __restrict__ dy, const void* __restrict__ src,
                                                                  const uint8_t* __restrict__ scales,
                                                                  const void* __restrict__ weight, const void* __restrict__ bias,
                                                                  const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                  float2* __restrict__ part, const GnShape s, const GnSplit p) {
  __shared__ float2 ent[kGnThreads * 8];
  griddep_wait();
  griddep_launch_dependents();
  const GnThread th(s, p);
  const int width = p.lanes * 8;
  if (th.active) {
    f32x2 w[4], b[4], m[4], rs[4], sg[4], sx[4];
    gn_load_params<T>(weight, bias, th.c, s, w, b);
    gn_load_stats(mean, rstd, th.sample, th.c, s, m, rs);
#pragma unroll
    for (int i = 0; i < 4; ++i) sg[i] = sx[i] = f32x2_zero();
#pragma unroll 2
    for (long long r = th.r0 + th.lane_row; r < th.r1; r += p.rl) {
      const long long pixel = th.sample * s.P + r;
      f32x2 d[4], f[4];
      gn_unpack<T>(dy[pixel * (s.C / 8) + th.c / 8], d);
      gn_load_saved<T, SRC8>(src, scales, pixel, th.c, s, f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2 xh = fmul2(fsub2(f[i], m[i]), rs[i]);
        const f32x2 g = fmul2(d[i], act_slope2<ACT>(fma2(xh, w[i], b[i])));
        fadd2(sg[i], g);
        ffma2(sx[i], g, xh);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = bits_f2(sg[i]), q = bits_f2(sx[i]);
      ent[threadIdx.x * 8 + 2 * i] = make_float2(a.x, q.x);
      ent[threadIdx.x * 8 + 2 * i + 1] = make_float2(a.y, q.y);
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < width; j += kGnThreads) {
    const int c = static_cast<int>(blockIdx.z) * width + j;
    if (c >= s.C) break;
    float2 sum = make_float2(0.0f, 0.0f);
    for (int i = 0; i < p.rl; ++i) {
      sum.x += ent[i * width + j].x;
      sum.y += ent[i * width + j].y;
    }
    part[(th.sample * p.chunks + blockIdx.y) * s.C + c] = sum;
  }
}

// One CTA a group: sums[sample][c] over the chunks, and the group's m1, m2.
template <typename T>
__global__ void __launch_bounds__(128) gn_grad_combine_kernel(const float2* __restrict__ part, const void* __restrict__ weight,
                                                              float2* __restrict__ sums, float2* __restrict__ m12,
                                                              const GnShape s, const GnSplit p) {
  __shared__ float scratch[33];
  griddep_wait();
  griddep_launch_dependents();
  const long long sample = blockIdx.x;
  const int g = blockIdx.y;
  float m1 = 0.0f, m2 = 0.0f;
  for (int j = threadIdx.x; j < s.Cg; j += 128) {
    const int c = g * s.Cg + j;
    float2 a = make_float2(0.0f, 0.0f);
    for (int k = 0; k < p.chunks; ++k) {
      const float2 e = part[(sample * p.chunks + k) * s.C + c];
      a.x += e.x;
      a.y += e.y;
    }
    sums[sample * s.C + c] = a;
    const float w = gn_param<T>(weight, c, s.param_f32, 1.0f);
    m1 += a.x * w;
    m2 += a.y * w;
  }
  const float inv = 1.0f / (static_cast<float>(s.P) * static_cast<float>(s.Cg));
  m1 = block_sum(m1, scratch) * inv;
  m2 = block_sum(m2, scratch) * inv;
  if (threadIdx.x == 0) m12[sample * s.G + g] = make_float2(m1, m2);
}

template <typename T, int ACT, bool SRC8>
__global__ void __launch_bounds__(kGnThreads) gn_grad_apply_kernel(const uint4* __restrict__ dy, const void* __restrict__ src,
                                                                   const uint8_t* __restrict__ scales,
                                                                   const void* __restrict__ weight, const void* __restrict__ bias,
                                                                   const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                   const float2* __restrict__ m12, uint4* __restrict__ dx,
                                                                   const GnShape s, const GnSplit p) {
  griddep_wait();
  griddep_launch_dependents();
  const GnThread th(s, p);
  if (!th.active) return;
  f32x2 w[4], b[4], m[4], rs[4], m1[4], m2[4];
  gn_load_params<T>(weight, bias, th.c, s, w, b);
  gn_load_stats(mean, rstd, th.sample, th.c, s, m, rs);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 lo = m12[th.sample * s.G + (th.c + 2 * i) / s.Cg], hi = m12[th.sample * s.G + (th.c + 2 * i + 1) / s.Cg];
    m1[i] = f2_bits(make_float2(lo.x, hi.x));
    m2[i] = f2_bits(make_float2(-lo.y, -hi.y));
  }
#pragma unroll 2
  for (long long r = th.r0 + th.lane_row; r < th.r1; r += p.rl) {
    const long long pixel = th.sample * s.P + r;
    f32x2 d[4], f[4];
    gn_unpack<T>(dy[pixel * (s.C / 8) + th.c / 8], d);
    gn_load_saved<T, SRC8>(src, scales, pixel, th.c, s, f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 xh = fmul2(fsub2(f[i], m[i]), rs[i]);
      const f32x2 g = fmul2(d[i], act_slope2<ACT>(fma2(xh, w[i], b[i])));
      // the product rounded by itself, so that a group whose m1 is that product leaves exactly nothing
      f[i] = fmul2(rs[i], fma2(xh, m2[i], fsub2(fmul2(g, w[i]), m1[i])));
    }
    dx[pixel * (s.C / 8) + th.c / 8] = gn_pack<T>(f);
  }
}

// dweight[c] and dbias[c]: the samples' sums, 8 lanes a channel, each over its own samples in order.
template <typename T>
__global__ void __launch_bounds__(256) gn_grad_params_kernel(const float2* __restrict__ sums, void* __restrict__ dweight,
                                                             void* __restrict__ dbias, const GnShape s) {
  __shared__ float2 ent[8][33];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float2 a = make_float2(0.0f, 0.0f);
  if (c < s.C)
    for (int b = part; b < s.B; b += 8) {
      const float2 e = sums[static_cast<long long>(b) * s.C + c];
      a.x += e.x;
      a.y += e.y;
    }
  ent[part][lane] = a;
  __syncthreads();
  if (part != 0 || c >= s.C) return;
  a = make_float2(0.0f, 0.0f);
  for (int i = 0; i < 8; ++i) {
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

static GnSplit gn_split(const GnShape& s) {
  GnSplit p;
  const int vecs = s.C / 8;
  const int whole = (vecs + 3) / 4 * 4;
  p.lanes = whole < kGnTileVecs ? whole : kGnTileVecs;
  p.rl = kGnThreads / p.lanes;
  p.tiles = (vecs + p.lanes - 1) / p.lanes;
  // about 8 CTAs an SM, and at least 4 pixels a thread
  const long long base = static_cast<long long>(s.B) * p.tiles;
  long long chunks = (8LL * kSmCount + base - 1) / base;
  const long long most = (s.P + 4LL * p.rl - 1) / (4LL * p.rl);
  chunks = chunks < most ? chunks : most;
  chunks = chunks < 1 ? 1 : chunks > 4096 ? 4096 : chunks;
  p.rows_per_chunk = (s.P + chunks - 1) / chunks;
  p.chunks = static_cast<int>((s.P + p.rows_per_chunk - 1) / p.rows_per_chunk);
  return p;
}

static int gn_shape(int64_t B, int64_t H, int64_t W, int64_t C, int G, double eps, int act, int dtype, int param_dtype,
                    GnShape* s) {
  if (dtype != DWB_F16 && dtype != DWB_BF16) return DWB_ERR_BAD_ARG;
  if (param_dtype != dtype && param_dtype != DWB_F32) return DWB_ERR_BAD_ARG;
  if (act < DWB_ACT_NONE || act > DWB_ACT_SILU) return DWB_ERR_BAD_ARG;
  if (!(eps >= 0.0) || !(eps < 1e30)) return DWB_ERR_BAD_ARG;
  // B: grid x; H * W: the row index; C: 32-bit channel arithmetic; groups of a call: grid y
  if (B < 0 || B > (1 << 30) || H < 1 || W < 1 || H > (1 << 30) || W > (1 << 30) || C < 8 || C > 65536 || (C % 8) != 0)
    return DWB_ERR_BAD_SHAPE;
  if (H * W > 0x7fffffffLL) return DWB_ERR_BAD_SHAPE;
  if (G < 1 || G > C || (C % G) != 0 || G > 65535) return DWB_ERR_BAD_SHAPE;
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

// Workspace: the chunks' partial sums; for the backward pass also the samples' sums and the groups' means.
// Resident kernels need the samples' sums only.
static int64_t gn_workspace(const GnShape& s, bool backward) {
  GnResident r;
  if (backward ? gn_resident_plan(s, GnPass::kBackward16, &r) && gn_resident_plan(s, GnPass::kBackward8, &r)
               : gn_resident_plan(s, GnPass::kForward, &r))
    return backward ? static_cast<int64_t>(s.B) * s.C * static_cast<int64_t>(sizeof(float2)) : 0;
  const GnSplit p = gn_split(s);
  int64_t n = static_cast<int64_t>(s.B) * p.chunks * s.C;
  if (backward) n += static_cast<int64_t>(s.B) * s.C + static_cast<int64_t>(s.B) * s.G;
  return n * static_cast<int64_t>(sizeof(float2));
}

static int gn_launch(const void* fn, const char* what, dim3 grid, int threads, void** args, cudaStream_t stream) {
  const cudaError_t e = launch_kernel(fn, grid, dim3(threads), args, 0, stream);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return record_cuda_failure(what, e);
  }
  return DWB_OK;
}

template <typename T, bool CKPT>
static const void* apply_fn(int act) {
  switch (act) {
    case kActRelu: return reinterpret_cast<const void*>(&gn_apply_kernel<T, kActRelu, CKPT>);
    case kActGelu: return reinterpret_cast<const void*>(&gn_apply_kernel<T, kActGelu, CKPT>);
    case kActSilu: return reinterpret_cast<const void*>(&gn_apply_kernel<T, kActSilu, CKPT>);
    default: return reinterpret_cast<const void*>(&gn_apply_kernel<T, kActNone, CKPT>);
  }
}
template <typename T, bool SRC8>
static const void* grad_sums_fn(int act) {
  switch (act) {
    case kActRelu: return reinterpret_cast<const void*>(&gn_grad_sums_kernel<T, kActRelu, SRC8>);
    case kActGelu: return reinterpret_cast<const void*>(&gn_grad_sums_kernel<T, kActGelu, SRC8>);
    case kActSilu: return reinterpret_cast<const void*>(&gn_grad_sums_kernel<T, kActSilu, SRC8>);
    default: return reinterpret_cast<const void*>(&gn_grad_sums_kernel<T, kActNone, SRC8>);
  }
}
template <typename T, bool SRC8>
static const void* grad_apply_fn(int act) {
  switch (act) {
    case kActRelu: return reinterpret_cast<const void*>(&gn_grad_apply_kernel<T, kActRelu, SRC8>);
    case kActGelu: return reinterpret_cast<const void*>(&gn_grad_apply_kernel<T, kActGelu, SRC8>);
    case kActSilu: return reinterpret_cast<const void*>(&gn_grad_apply_kernel<T, kActSilu, SRC8>);
    default: return reinterpret_cast<const void*>(&gn_grad_apply_kernel<T, kActNone, SRC8>);
  }
}

template <typename T>
static int gn_forward(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, void* codes,
                      void* scales, void* workspace, GnShape s, int act, cudaStream_t stream) {
  GnResident res;
  if (gn_resident_plan(s, GnPass::kForward, &res))
    return gn_resident_forward<T>(x, weight, bias, y, mean, rstd, codes, scales, s, res, act, stream);
  GnSplit p = gn_split(s);
  const dim3 grid(s.B, p.chunks, p.tiles);
  void* part = workspace;
  void* a1[] = {&x, &part, &s, &p};
  int rc = gn_launch(reinterpret_cast<const void*>(&gn_stats_kernel<T>), "gn_stats_kernel", grid, kGnThreads, a1, stream);
  if (rc != DWB_OK) return rc;
  void* a2[] = {&part, &mean, &rstd, &s, &p};
  rc = gn_launch(reinterpret_cast<const void*>(&gn_combine_kernel), "gn_combine_kernel", dim3(s.B, s.G), 128, a2, stream);
  if (rc != DWB_OK) return rc;
  void* a3[] = {&x, &weight, &bias, &mean, &rstd, &y, &codes, &scales, &s, &p};
  return gn_launch(codes ? apply_fn<T, true>(act) : apply_fn<T, false>(act), "gn_apply_kernel", grid, kGnThreads, a3, stream);
}

template <typename T>
static int gn_backward(const void* dy, const void* x, const void* codes, const void* scales, const float* mean,
                       const float* rstd, const void* weight, const void* bias, void* dx, void* dweight, void* dbias,
                       void* workspace, GnShape s, int act, cudaStream_t stream) {
  float2* sums = static_cast<float2*>(workspace);
  int rc;
  GnResident res;
  if (gn_resident_plan(s, codes ? GnPass::kBackward8 : GnPass::kBackward16, &res)) {
    rc = gn_resident_backward<T>(dy, x, codes, scales, mean, rstd, weight, bias, dx, sums, s, res, act, stream);
  } else {
    GnSplit p = gn_split(s);
    const dim3 grid(s.B, p.chunks, p.tiles);
    float2* m12 = sums + static_cast<int64_t>(s.B) * s.C;
    float2* part = m12 + static_cast<int64_t>(s.B) * s.G;
    const void* src = codes ? codes : x;
    void* a1[] = {&dy, &src, &scales, &weight, &bias, &mean, &rstd, &part, &s, &p};
    rc = gn_launch(codes ? grad_sums_fn<T, true>(act) : grad_sums_fn<T, false>(act), "gn_grad_sums_kernel", grid, kGnThreads,
                   a1, stream);
    if (rc != DWB_OK) return rc;
    void* a2[] = {&part, &weight, &sums, &m12, &s, &p};
    rc = gn_launch(reinterpret_cast<const void*>(&gn_grad_combine_kernel<T>), "gn_grad_combine_kernel", dim3(s.B, s.G), 128,
                   a2, stream);
    if (rc != DWB_OK) return rc;
    void* a3[] = {&dy, &src, &scales, &weight, &bias, &mean, &rstd, &m12, &dx, &s, &p};
    rc = gn_launch(codes ? grad_apply_fn<T, true>(act) : grad_apply_fn<T, false>(act), "gn_grad_apply_kernel", grid,
                   kGnThreads, a3, stream);
  }
  if (rc != DWB_OK || (!dweight && !dbias)) return rc;
  void* a4[] = {&sums, &dweight, &dbias, &s};
  return gn_launch(reinterpret_cast<const void*>(&gn_grad_params_kernel<T>), "gn_grad_params_kernel", dim3((s.C + 31) / 32), 256,
                   a4, stream);
}

}  // namespace dwb

extern "C" int dwb_group_norm_act_workspace(int64_t B, int64_t H, int64_t W, int64_t C, int G, int backward, int64_t* bytes) {
  using namespace dwb;
  if (!bytes) return DWB_ERR_NULL_POINTER;
  GnShape s;
  const int rc = gn_shape(B, H, W, C, G, 0.0, DWB_ACT_NONE, DWB_F16, DWB_F16, &s);
  if (rc != DWB_OK) return rc;
  *bytes = B == 0 ? 0 : gn_workspace(s, backward != 0);
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
  const int64_t need = gn_workspace(s, false);
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
  return dtype == DWB_F16 ? gn_forward<__half>(x, weight, bias, y, mean, rstd, codes, scales, workspace, s, act, st)
                          : gn_forward<__nv_bfloat16>(x, weight, bias, y, mean, rstd, codes, scales, workspace, s, act, st);
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
  if (B > 0) {
    if (!dy || !dx || !mean || !rstd || (codes == nullptr) != (scales == nullptr)) return DWB_ERR_NULL_POINTER;
    if ((x == nullptr) == (codes == nullptr)) return x ? DWB_ERR_BAD_ARG : DWB_ERR_NULL_POINTER;  // one of the two
    const int64_t need = gn_workspace(s, true);
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
                                                s, act, st)
                          : gn_backward<__nv_bfloat16>(dy, x, codes, scales, mean, rstd, weight, bias, dx, dweight, dbias,
                                                       workspace, s, act, st);
}
