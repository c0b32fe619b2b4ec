// dw_groupnorm_cluster.cu -- group normalisation in one pass over memory: a
// cluster of CTAs holds the pixels of one sample and a slab of channels (whole
// groups) in shared memory, so that the statistics and the normalisation read
// global memory once.  The formulas stand in dw_groupnorm.cuh.
//
// Bound by memory: forward 4 bytes a value (5.03 with a checkpoint), backward 6
// (5.03 from a checkpoint).  Every thread copies its own vectors to shared
// memory (cp.async, 16 bytes; 8 for codes) and is the only one that reads them,
// so the copies need no barrier: all of a CTA's loads are in flight at once, and
// the sums begin when the first quarter has landed.  Two CTAs an SM (110 KB
// each) let one load while the other computes or stores.  The moments (forward)
// or the channel sums (backward) of the cluster's CTAs are exchanged through
// distributed shared memory, and every CTA adds them up in rank order: the same
// bits in every CTA and on every run.
#include <cuda_runtime.h>

#include "../../include/dwconv_b200.h"
#include "dw_groupnorm.cuh"
#include "dw_groupnorm_cluster.h"
#include "dw_host.h"
#include "dw_launch.h"

namespace dwb {

constexpr int kGnForwardThreads = 512;
constexpr int kGnBackwardThreads = 256;

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Wait until all but the `3 - part` newest of four groups have landed.
__device__ __forceinline__ void cp_async_wait_part(int part) {
  if (part == 0) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (part == 1) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (part == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The aligned forms: the warp comes together first.
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The float2 at the same shared-memory place of another CTA of the cluster.
__device__ __forceinline__ float2 cluster_load(const float2* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}

struct GnPlace {
  int rank, c_base, width;   // rank in the cluster; first channel; channels of this slab
  int lane_row, vec, c;
  bool active;
  long long sample, r0;
  int rows;                  // pixels of this CTA
  __device__ __forceinline__ GnPlace(const GnShape& s, const GnResident& p) {
    const int cl = blockIdx.x / p.cluster;
    rank = blockIdx.x - cl * p.cluster;
    sample = cl / p.slabs;
    c_base = (cl - static_cast<int>(sample) * p.slabs) * p.slab;
    width = s.C - c_base < p.slab ? s.C - c_base : p.slab;
    lane_row = threadIdx.x / p.lanes;
    vec = threadIdx.x - lane_row * p.lanes;
    c = c_base + vec * 8;
    active = lane_row < p.rl && vec * 8 < width;
    r0 = static_cast<long long>(rank) * p.rows_per_cta;
    rows = rows_of(s, p, rank);
  }
  static __device__ __forceinline__ int rows_of(const GnShape& s, const GnResident& p, int rank) {
    const long long first = static_cast<long long>(rank) * p.rows_per_cta, left = s.P - first;
    return left <= 0 ? 0 : left < p.rows_per_cta ? static_cast<int>(left) : p.rows_per_cta;
  }
};

// Pixels of a CTA that lane row `lr` handles.
__device__ __forceinline__ int gn_lane_rows(int rows, int lr, int rl) { return rows > lr ? (rows - lr + rl - 1) / rl : 0; }

// ONE: C / G is a multiple of 8, so that a thread's vector lies in one group.
template <typename T, int ACT, bool CKPT, bool ONE>
__global__ void __launch_bounds__(kGnForwardThreads, 2)
    gn_resident_kernel(const T* __restrict__ x, const void* __restrict__ weight, const void* __restrict__ bias,
                       T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                       int8_t* __restrict__ codes, uint8_t* __restrict__ scales, const GnShape s, const GnResident p) {
  extern __shared__ __align__(16) unsigned char smem[];
  uint4* stage = reinterpret_cast<uint4*>(smem);  // [iters][threads]: a thread's own vectors
  float2* ent = reinterpret_cast<float2*>(stage + p.iters * p.threads);
  float2* grp = ent + p.threads * (ONE ? 1 : 8);
  const int groups = p.slab / s.Cg;
  float2* fin = grp + groups;
  griddep_wait();
  griddep_launch_dependents();
  const GnPlace at(s, p);
  const int tid = threadIdx.x;
  const long long first = (at.sample * s.P + at.r0 + at.lane_row) * s.C + at.c;  // this thread's first value
  const long long step = static_cast<long long>(p.rl) * s.C;
  const int mine = at.active ? gn_lane_rows(at.rows, at.lane_row, p.rl) : 0;
  const int quarter = (p.iters + 3) / 4;
  for (int part = 0; part < 4; ++part) {
    const int end = min(mine, (part + 1) * quarter);
    for (int i = part * quarter; i < end; ++i) cp_async16(stage + i * p.threads + tid, x + first + i * step);
    cp_async_commit();
  }
  GnSums sums;
  for (int part = 0; part < 4; ++part) {
    cp_async_wait_part(part);
    const int end = min(mine, (part + 1) * quarter);
    for (int i = part * quarter; i < end; ++i) {
      f32x2 f[4];
      gn_unpack<T>(stage[i * p.threads + tid], f);
      sums.add(f);
    }
  }
  if (sums.n) {
    float mean[8], m2[8];
    sums.moments(mean, m2);
    if constexpr (ONE) {
      float m = 0.0f, q = 0.0f, d2 = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m += mean[i];
      m *= 0.125f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        q += m2[i];
        d2 += (mean[i] - m) * (mean[i] - m);
      }
      ent[tid] = make_float2(m, q + static_cast<float>(sums.n) * d2);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) ent[tid * 8 + i] = make_float2(mean[i], m2[i]);
    }
  }
  __syncthreads();
  // one warp a group: the moments of this CTA's pixels
  const int lane = tid & 31, warps = blockDim.x >> 5, here = at.width / s.Cg;
  for (int g = tid >> 5; g < here; g += warps) {
    const int per_row = ONE ? s.Cg / 8 : s.Cg;
    const int live = min(at.rows, p.rl), entries = per_row * live;
    auto entry = [&](int e, float& n) {
      const int lr = e / per_row, k = g * per_row + (e - lr * per_row);
      n = static_cast<float>(gn_lane_rows(at.rows, lr, p.rl) * (ONE ? 8 : 1));
      return ONE ? ent[lr * p.lanes + k] : ent[lr * p.lanes * 8 + k];
    };
    float sum = 0.0f, m2 = 0.0f, n;
    for (int e = lane; e < entries; e += 32) {
      const float2 v = entry(e, n);
      sum += n * v.x;
    }
    const float total = static_cast<float>(at.rows) * static_cast<float>(s.Cg);
    const float mean = at.rows ? warp_sum(sum) / total : 0.0f;
    for (int e = lane; e < entries; e += 32) {
      const float2 v = entry(e, n);
      m2 += v.y + n * (v.x - mean) * (v.x - mean);
    }
    m2 = warp_sum(m2);
    if (lane == 0) grp[g] = make_float2(mean, m2);
  }
  if (p.cluster > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  for (int g = tid; g < here; g += blockDim.x) {
    const float n = static_cast<float>(s.P) * static_cast<float>(s.Cg);
    float mean, m2;
    if (p.cluster == 1) {
      mean = grp[g].x;
      m2 = grp[g].y;
    } else {
      float sum = 0.0f;
      for (int r = 0; r < p.cluster; ++r)
        sum += static_cast<float>(GnPlace::rows_of(s, p, r)) * cluster_load(grp + g, r).x;
      mean = sum / static_cast<float>(s.P);
      m2 = 0.0f;
      for (int r = 0; r < p.cluster; ++r) {
        const float2 v = cluster_load(grp + g, r);
        m2 += v.y + static_cast<float>(GnPlace::rows_of(s, p, r)) * static_cast<float>(s.Cg) * (v.x - mean) * (v.x - mean);
      }
    }
    const float rstd = 1.0f / sqrtf(m2 / n + s.eps);
    fin[g] = make_float2(mean, rstd);
    if (at.rank == 0) {
      const long long o = at.sample * s.G + at.c_base / s.Cg + g;
      mean_out[o] = mean;
      rstd_out[o] = rstd;
    }
  }
  if (p.cluster > 1) cluster_arrive();  // this CTA has read the others' moments
  __syncthreads();
  f32x2 w[4], b[4], m[4], rs[4];
  if (at.active) {
    gn_load_params<T>(weight, bias, at.c, s.param_f32, w, b);
    if constexpr (ONE) {
      const float2 f = fin[at.vec * 8 / s.Cg];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[i] = splat2(f.x);
        rs[i] = splat2(f.y);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 lo = fin[(at.vec * 8 + 2 * i) / s.Cg], hi = fin[(at.vec * 8 + 2 * i + 1) / s.Cg];
        m[i] = f2_bits(make_float2(lo.x, hi.x));
        rs[i] = f2_bits(make_float2(lo.y, hi.y));
      }
    }
  }
  const long long sblocks = (s.C + kAct8Block - 1) / kAct8Block;
  // a checkpoint's block maximum is a warp shuffle: every lane goes through every turn
  const int turns = CKPT ? gn_lane_rows(at.rows, 0, p.rl) : mine;
  for (int i = 0; i < turns; ++i) {
    const bool on = i < mine;
    const uint4 v = on ? stage[i * p.threads + tid] : make_uint4(0u, 0u, 0u, 0u);
    if constexpr (CKPT) {
      const uint32_t E = act8_exponent<T>(act8_block_amax(v));
      if (on) {
        *reinterpret_cast<uint2*>(codes + first + i * step) = act8_codes<T>(v, E);
        if ((at.vec & 3) == 0)
          scales[(at.sample * s.P + at.r0 + at.lane_row + static_cast<long long>(i) * p.rl) * sblocks + at.c / kAct8Block] =
              static_cast<uint8_t>(E);
      }
    }
    if (on) {
      f32x2 f[4];
      gn_unpack<T>(v, f);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = act_value2<ACT>(fma2(fmul2(fsub2(f[j], m[j]), rs[j]), w[j], b[j]));
      *reinterpret_cast<uint4*>(y + first + i * step) = gn_pack<T>(f);
    }
  }
  if (p.cluster > 1) cluster_wait();  // nobody reads this CTA's shared memory any more
}

template <typename T, int ACT, bool SRC8, bool ONE>
__global__ void __launch_bounds__(kGnBackwardThreads, 2)
    gn_resident_grad_kernel(const T* __restrict__ dy, const void* __restrict__ src, const uint8_t* __restrict__ scales,
                            const void* __restrict__ weight, const void* __restrict__ bias, const float* __restrict__ mean,
                            const float* __restrict__ rstd, T* __restrict__ dx, float2* __restrict__ sums_out,
                            const GnShape s, const GnResident p) {
  extern __shared__ __align__(16) unsigned char smem[];
  uint4* stage = reinterpret_cast<uint4*>(smem);  // dy
  unsigned char* saved = reinterpret_cast<unsigned char*>(stage + p.iters * p.threads);
  constexpr int kSaved = SRC8 ? 8 : 16;
  float2* ent = reinterpret_cast<float2*>(saved + p.iters * p.threads * kSaved);
  float2* chan = ent + p.threads * 8;
  float2* total = chan + p.slab;
  float2* fin = total + p.slab;
  griddep_wait();
  griddep_launch_dependents();
  const GnPlace at(s, p);
  const int tid = threadIdx.x;
  const long long pixel0 = at.sample * s.P + at.r0 + at.lane_row;
  const long long first = pixel0 * s.C + at.c;
  const long long step = static_cast<long long>(p.rl) * s.C;
  const long long sblocks = (s.C + kAct8Block - 1) / kAct8Block;
  const int mine = at.active ? gn_lane_rows(at.rows, at.lane_row, p.rl) : 0;
  const int quarter = (p.iters + 3) / 4;
  for (int part = 0; part < 4; ++part) {
    const int end = min(mine, (part + 1) * quarter);
    for (int i = part * quarter; i < end; ++i) {
      cp_async16(stage + i * p.threads + tid, dy + first + i * step);
      if constexpr (SRC8)
        cp_async8(saved + (i * p.threads + tid) * kSaved, static_cast<const int8_t*>(src) + first + i * step);
      else
        cp_async16(saved + (i * p.threads + tid) * kSaved, static_cast<const T*>(src) + first + i * step);
    }
    cp_async_commit();
  }
  f32x2 w[4], b[4], m[4], rs[4];
  if (at.active) {
    gn_load_params<T>(weight, bias, at.c, s.param_f32, w, b);
    if constexpr (ONE) {
      const long long o = at.sample * s.G + at.c / s.Cg;
      const f32x2 mv = splat2(mean[o]), rv = splat2(rstd[o]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[i] = mv;
        rs[i] = rv;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long long lo = at.sample * s.G + (at.c + 2 * i) / s.Cg, hi = at.sample * s.G + (at.c + 2 * i + 1) / s.Cg;
        m[i] = f2_bits(make_float2(mean[lo], mean[hi]));
        rs[i] = f2_bits(make_float2(rstd[lo], rstd[hi]));
      }
    }
  }
  // x_hat and g = dy act'(u) of this thread's vector i
  auto normalised = [&](int i, uint32_t E, f32x2(&xh)[4], f32x2(&g)[4]) {
    f32x2 d[4];
    gn_unpack<T>(stage[i * p.threads + tid], d);
    if constexpr (SRC8)
      act8_values(*reinterpret_cast<const uint2*>(saved + (i * p.threads + tid) * kSaved), act8_step(E), xh);
    else
      gn_unpack<T>(*reinterpret_cast<const uint4*>(saved + (i * p.threads + tid) * kSaved), xh);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      xh[j] = fmul2(fsub2(xh[j], m[j]), rs[j]);
      g[j] = fmul2(d[j], act_slope2<ACT>(fma2(xh[j], w[j], b[j])));
    }
  };
  const uint8_t* sc = SRC8 ? scales + pixel0 * sblocks + at.c / kAct8Block : nullptr;
  f32x2 sg[4], sx[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) sg[j] = sx[j] = f32x2_zero();
  for (int part = 0; part < 4; ++part) {
    cp_async_wait_part(part);
    const int end = min(mine, (part + 1) * quarter);
    for (int i = part * quarter; i < end; ++i) {
      f32x2 xh[4], g[4];
      normalised(i, SRC8 ? sc[static_cast<long long>(i) * p.rl * sblocks] : 0u, xh, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        fadd2(sg[j], g[j]);
        ffma2(sx[j], g[j], xh[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 a = bits_f2(sg[j]), q = bits_f2(sx[j]);
    ent[tid * 8 + 2 * j] = make_float2(a.x, q.x);
    ent[tid * 8 + 2 * j + 1] = make_float2(a.y, q.y);
  }
  __syncthreads();
  for (int j = tid; j < at.width; j += blockDim.x) {
    float2 a = make_float2(0.0f, 0.0f);
#pragma unroll 4
    for (int r = 0; r < p.rl; ++r) {
      const float2 e = ent[r * p.lanes * 8 + j];
      a.x += e.x;
      a.y += e.y;
    }
    chan[j] = a;
  }
  if (p.cluster > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  for (int j = tid; j < at.width; j += blockDim.x) {
    float2 a = chan[j];
    if (p.cluster > 1) {
      a = make_float2(0.0f, 0.0f);
      for (int r = 0; r < p.cluster; ++r) {
        const float2 e = cluster_load(chan + j, r);
        a.x += e.x;
        a.y += e.y;
      }
    }
    if (at.rank == 0) sums_out[at.sample * s.C + at.c_base + j] = a;
    const float wj = gn_param<T>(weight, at.c_base + j, s.param_f32, 1.0f);
    total[j] = make_float2(a.x * wj, a.y * wj);
  }
  if (p.cluster > 1) cluster_arrive();
  __syncthreads();
  const float inv = 1.0f / (static_cast<float>(s.P) * static_cast<float>(s.Cg));
  const int lane = tid & 31, warps = blockDim.x >> 5, here = at.width / s.Cg;
  for (int g = tid >> 5; g < here; g += warps) {
    float m1 = 0.0f, m2 = 0.0f;
    for (int j = lane; j < s.Cg; j += 32) {
      m1 += total[g * s.Cg + j].x;
      m2 += total[g * s.Cg + j].y;
    }
    m1 = warp_sum(m1);
    m2 = warp_sum(m2);
    if (lane == 0) fin[g] = make_float2(m1 * inv, -m2 * inv);
  }
  __syncthreads();
  f32x2 m1[4], m2[4];
  if (at.active) {
    if constexpr (ONE) {
      const float2 f = fin[at.vec * 8 / s.Cg];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m1[i] = splat2(f.x);
        m2[i] = splat2(f.y);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 lo = fin[(at.vec * 8 + 2 * i) / s.Cg], hi = fin[(at.vec * 8 + 2 * i + 1) / s.Cg];
        m1[i] = f2_bits(make_float2(lo.x, hi.x));
        m2[i] = f2_bits(make_float2(lo.y, hi.y));
      }
    }
  }
  for (int i = 0; i < mine; ++i) {
    f32x2 xh[4], g[4];
    normalised(i, SRC8 ? sc[static_cast<long long>(i) * p.rl * sblocks] : 0u, xh, g);
    // the product rounded by itself, so that a group whose m1 is that product leaves exactly nothing
#pragma unroll
    for (int j = 0; j < 4; ++j) xh[j] = fmul2(rs[j], fma2(xh[j], m2[j], fsub2(fmul2(g[j], w[j]), m1[j])));
    *reinterpret_cast<uint4*>(dx + first + i * step) = gn_pack<T>(xh);
  }
  if (p.cluster > 1) cluster_wait();
}

// ---- host -----------------------------------------------------------------------------------------

static int gcd_int(int a, int b) { return b == 0 ? a : gcd_int(b, a % b); }

static bool gn_resident_fill(const GnShape& s, GnPass pass, int slab, int cluster, int limit, GnResident* p) {
  const int most = pass == GnPass::kForward ? kGnForwardThreads : kGnBackwardThreads;
  const int bytes = pass == GnPass::kForward ? 16 : pass == GnPass::kBackward16 ? 32 : 24;
  p->slab = slab;
  p->slabs = (s.C + slab - 1) / slab;
  p->lanes = (slab / 8 + 3) / 4 * 4;
  if (p->lanes > most) return false;
  const long long rows = (s.P + cluster - 1) / cluster;
  if (rows > (1 << 20)) return false;
  p->cluster = cluster;
  p->rows_per_cta = static_cast<int>(rows);
  p->rl = most / p->lanes;
  if (p->rl > p->rows_per_cta) p->rl = p->rows_per_cta;
  p->threads = (p->lanes * p->rl + 31) / 32 * 32;
  p->iters = (p->rows_per_cta + p->rl - 1) / p->rl;
  const bool one = s.Cg % 8 == 0;
  const long long extra = pass == GnPass::kForward
                              ? 8LL * (p->threads * (one ? 1 : 8) + 2 * (slab / s.Cg))
                              : 8LL * (p->threads * 8 + 2 * slab + slab / s.Cg);
  const long long need = static_cast<long long>(p->iters) * p->threads * bytes + extra;
  if (need > limit) return false;
  p->smem = static_cast<int>(need);
  return static_cast<long long>(s.B) * p->slabs * cluster <= 0x7fffffffLL;
}

bool gn_resident_plan(const GnShape& s, GnPass pass, GnResident* p) {
  constexpr int kTwo = 113 * 1024;  // two CTAs an SM: (228 KB - 2 x 1 KB) / 2
  constexpr int kOne = 227 * 1024;
  const long long unit_ll = static_cast<long long>(s.Cg) / gcd_int(s.Cg, kAct8Block) * kAct8Block;
  const int unit = unit_ll < s.C ? static_cast<int>(unit_ll) : s.C;
  // whole 128-byte lines of a pixel where that costs no occupancy
  int slab = unit;
  while (slab < 64 && slab < s.C) slab = slab + unit < s.C ? slab + unit : s.C;
  for (int limit : {kTwo, kOne})
    for (int width : {slab, unit})
      for (int cluster = 1; cluster <= 16; cluster *= 2)
        if (gn_resident_fill(s, pass, width, cluster, limit, p)) {
          // few clusters: more CTAs share a sample, as long as each thread keeps a few pixels
          GnResident wider;
          while (static_cast<long long>(s.B) * p->slabs * p->cluster < 2 * kSmCount && p->cluster < 8 && p->iters > 4 &&
                 gn_resident_fill(s, pass, width, p->cluster * 2, limit, &wider))
            *p = wider;
          return true;
        }
  return false;
}

static int gn_resident_launch(const void* fn, const char* what, const GnShape& s, const GnResident& p, void** args,
                              cudaStream_t stream) {
  cudaError_t e = allow_large_cta(fn);
  if (e == cudaSuccess)
    e = launch_kernel(fn, dim3(static_cast<unsigned>(static_cast<long long>(s.B) * p.slabs * p.cluster)), dim3(p.threads), args,
                      p.smem, stream, p.cluster);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return record_cuda_failure(what, e);
  }
  return DWB_OK;
}

template <typename T, bool CKPT, bool ONE>
static const void* resident_fn(int act) {
  switch (act) {
    case kActRelu: return reinterpret_cast<const void*>(&gn_resident_kernel<T, kActRelu, CKPT, ONE>);
    case kActGelu: return reinterpret_cast<const void*>(&gn_resident_kernel<T, kActGelu, CKPT, ONE>);
    case kActSilu: return reinterpret_cast<const void*>(&gn_resident_kernel<T, kActSilu, CKPT, ONE>);
    default: return reinterpret_cast<const void*>(&gn_resident_kernel<T, kActNone, CKPT, ONE>);
  }
}
template <typename T, bool SRC8, bool ONE>
static const void* resident_grad_fn(int act) {
  switch (act) {
    case kActRelu: return reinterpret_cast<const void*>(&gn_resident_grad_kernel<T, kActRelu, SRC8, ONE>);
    case kActGelu: return reinterpret_cast<const void*>(&gn_resident_grad_kernel<T, kActGelu, SRC8, ONE>);
    case kActSilu: return reinterpret_cast<const void*>(&gn_resident_grad_kernel<T, kActSilu, SRC8, ONE>);
    default: return reinterpret_cast<const void*>(&gn_resident_grad_kernel<T, kActNone, SRC8, ONE>);
  }
}

template <typename T>
int gn_resident_forward(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, void* codes,
                        void* scales, const GnShape& s, const GnResident& p, int act, cudaStream_t stream) {
  const bool one = s.Cg % 8 == 0;
  const void* fn = codes ? (one ? resident_fn<T, true, true>(act) : resident_fn<T, true, false>(act))
                         : (one ? resident_fn<T, false, true>(act) : resident_fn<T, false, false>(act));
  GnShape sv = s;
  GnResident pv = p;
  void* args[] = {&x, &weight, &bias, &y, &mean, &rstd, &codes, &scales, &sv, &pv};
  return gn_resident_launch(fn, "gn_resident_kernel", s, p, args, stream);
}

template <typename T>
int gn_resident_backward(const void* dy, const void* x, const void* codes, const void* scales, const float* mean,
                         const float* rstd, const void* weight, const void* bias, void* dx, float2* sums, const GnShape& s,
                         const GnResident& p, int act, cudaStream_t stream) {
  const bool one = s.Cg % 8 == 0;
  const void* fn = codes ? (one ? resident_grad_fn<T, true, true>(act) : resident_grad_fn<T, true, false>(act))
                         : (one ? resident_grad_fn<T, false, true>(act) : resident_grad_fn<T, false, false>(act));
  const void* src = codes ? codes : x;
  GnShape sv = s;
  GnResident pv = p;
  void* args[] = {&dy, &src, &scales, &weight, &bias, &mean, &rstd, &dx, &sums, &sv, &pv};
  return gn_resident_launch(fn, "gn_resident_grad_kernel", s, p, args, stream);
}

#define DWB_GN_RESIDENT(T)                                                                                             \
  template int gn_resident_forward<T>(const void*, const void*, const void*, void*, float*, float*, void*, void*,      \
                                      const GnShape&, const GnResident&, int, cudaStream_t);                           \
  template int gn_resident_backward<T>(const void*, const void*, const void*, const void*, const float*, const float*, \
                                       const void*, const void*, void*, float2*, const GnShape&, const GnResident&,    \
                                       int, cudaStream_t);
DWB_GN_RESIDENT(__half)
DWB_GN_RESIDENT(__nv_bfloat16)
#undef DWB_GN_RESIDENT

}  // namespace dwb
