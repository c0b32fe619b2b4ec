// dw_groupnorm_cluster.cu -- group normalisation in one pass over memory: a
// cluster of CTAs holds the pixels of one sample and a slab of channels (whole
// groups) in shared memory, so that the statistics and the normalisation read
// global memory once.  The formulas stand in dw_groupnorm.cuh.
//
// Bound by memory: forward 4 bytes a value (5.03 with a checkpoint), backward 6
// (5.03 from a checkpoint).  Every thread copies its own vectors to shared
// memory (cp.async) and is the only one that reads them, so the copies need no
// barrier: all of a CTA's loads are in flight at once, and the sums begin when
// the first quarter has landed.  Four CTAs an SM let one load while another
// computes or stores.  The moments (forward)
// or the channel sums (backward) of the cluster's CTAs are exchanged through
// distributed shared memory, and every CTA adds them up in rank order: the same
// bits in every CTA and on every run.
//
// Measured, forward: 31.9 us at 16x32x32x1536, 32 groups, GELU (3.2 TB/s; a plain
// copy of that size takes 19 to 21), 93 to 100 us at 32x56x56x1024, 64 groups, SiLU,
// bf16 (4.1 to 4.4 TB/s), 45 us with a checkpoint at 64x56x56x128 (2.9 TB/s).  What
// bounds it then is issue: 25 instructions a value, 36 with a checkpoint's block
// maxima, exponents and codes, and CTAs of one wave that load and compute in step.
#include <cuda_runtime.h>

#include "../../include/dwconv_b200.h"
#include "dw_groupnorm.cuh"
#include "dw_groupnorm_cluster.h"
#include "dw_host.h"
#include "dw_launch.h"

namespace dwb {

constexpr int kGnThreads = 256;

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
// For a barrier that orders nothing but the end of this CTA's reads.
__device__ __forceinline__ void cluster_arrive_relaxed() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
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
  int r0, rows;              // pixels of this CTA
  long long sample;
  __device__ __forceinline__ GnPlace(const GnShape& s, const GnResident& p, int channels) {  // of a thread
    rank = blockIdx.x & (p.cluster - 1);
    sample = blockIdx.y;
    c_base = (blockIdx.x >> p.cluster_log) * p.slab;
    width = min(s.C - c_base, p.slab);
    lane_row = threadIdx.x * p.lane_mul >> 16;
    vec = threadIdx.x - lane_row * p.lanes;
    c = c_base + vec * channels;
    active = lane_row < p.rl && vec * channels < width;
    r0 = rank * p.rows_per_cta;
    rows = rows_of(s, p, rank);
  }
  static __device__ __forceinline__ int rows_of(const GnShape& s, const GnResident& p, int rank) {
    return max(0, min(p.rows_per_cta, static_cast<int>(s.P) - rank * p.rows_per_cta));
  }
};

// Pixels of a CTA that lane row `lr` handles.
__device__ __forceinline__ int gn_lane_rows(int rows, int lr, int rl) { return rows > lr ? (rows - lr + rl - 1) / rl : 0; }

template <typename T, int ACT, bool CKPT, int SUB>
__global__ void __launch_bounds__(kGnThreads, 4)
    gn_resident_kernel(const T* __restrict__ x, const void* __restrict__ weight, const void* __restrict__ bias,
                       T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out,
                       int8_t* __restrict__ codes, uint8_t* __restrict__ scales, const GnShape s, const GnResident p) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int kEnt = 8 / SUB;                   // moments a thread hands over
  constexpr int kParts = SUB == 8 ? 1 : SUB == 4 ? 2 : 4;
  uint4* stage = reinterpret_cast<uint4*>(smem);  // [iters][threads]: a thread's own vectors
  float2* ent = reinterpret_cast<float2*>(stage + p.iters * p.threads);
  float2* grp = ent + p.threads * kEnt;
  float2* fin = grp + p.slab / s.Cg;
  griddep_wait();
  griddep_launch_dependents();
  const GnPlace at(s, p, 8);
  const int tid = threadIdx.x, nt = p.threads;
  const long long first = (at.sample * s.P + at.r0 + at.lane_row) * s.C + at.c;  // this thread's first value
  const long long step = static_cast<long long>(p.rl) * s.C;
  const int mine = at.active ? gn_lane_rows(at.rows, at.lane_row, p.rl) : 0;
  const int quarter = (p.iters + 3) / 4;
  {
    const T* src = x + first;
    uint4* dst = stage + tid;
    for (int part = 0; part < 4; ++part) {
      const int end = min(mine, (part + 1) * quarter);
#pragma unroll 4
      for (int i = part * quarter; i < end; ++i, src += step, dst += nt) cp_async16(dst, src);
      cp_async_commit();
    }
  }
  // the parameters come in while the pixels do
  f32x2 w[4], b[4];
  if (at.active) gn_load_params<T>(weight, bias, at.c, s, w, b);
  if (mine) {
    GnSums sums;
    f32x2 f[4];
    const uint4* v = stage + tid;
    cp_async_wait_part(0);
    gn_unpack<T>(*v, f);
    sums.start(f);
    v += nt;
    int i = 1;
    for (int part = 0; part < 4; ++part) {
      cp_async_wait_part(part);
      const int end = min(mine, (part + 1) * quarter);
#pragma unroll 4
      for (; i < end; ++i, v += nt) {
        gn_unpack<T>(*v, f);
        sums.add(f);
      }
    }
    f32x2 mean[4], m2[4];
    sums.moments(mine, mean, m2);
    gn_hand_over<SUB>(mean, m2, static_cast<float>(mine), ent + tid * kEnt);
  }
  __syncthreads();
  // one warp a group: the moments of this CTA's pixels
  const int lane = tid & 31, warps = nt >> 5, here = at.width / s.Cg;
  {
    const GnMerge merge(lane, s.Cg / SUB, at.rows, p.rl, p.lanes * kEnt);
    for (int g = tid >> 5; g < here; g += warps) {
      const float2 m = merge.run<SUB>(ent + g * (s.Cg / SUB), at.rows, s.Cg);
      if (lane == 0) grp[g] = m;
    }
  }
  if (p.cluster > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  // a lane a rank, four groups a warp: all of the cluster's moments of a group at once, added up the same way in every
  // CTA (one group a warp: 37.9 us at 64x56x56x128 with 32 groups, so 34.7)
  const int rank = lane & 7;
  const float all = static_cast<float>(s.P) * static_cast<float>(s.Cg);
  for (int g0 = (tid >> 5) * 4; g0 < here; g0 += warps * 4) {
    const int g = g0 + (lane >> 3);
    const bool on = g < here;
    float mean = 0.0f, m2 = 0.0f;
    if (p.cluster > 1) {
      // about rank 0's mean (rank 0 always has pixels)
      const bool has = on && rank < p.cluster;
      const float n = has ? static_cast<float>(GnPlace::rows_of(s, p, rank)) * static_cast<float>(s.Cg) : 0.0f;
      const float2 v = has ? cluster_load(grp + g, rank) : make_float2(0.0f, 0.0f);
      const float pivot = __shfl_sync(0xffffffffu, v.x, lane & 24), d = v.x - pivot;
      // a CTA without pixels has no weight
      float s0 = n * v.x, s1 = n > 0.0f ? n * d : 0.0f, s2 = n > 0.0f ? v.y + n * d * d : 0.0f;
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) {
        s0 += __shfl_xor_sync(0xffffffffu, s0, o);
        s1 += __shfl_xor_sync(0xffffffffu, s1, o);
        s2 += __shfl_xor_sync(0xffffffffu, s2, o);
      }
      const float off = s1 / all;
      mean = gn_mean(pivot, off, s0 / all);
      m2 = not_negative(s2 - s1 * off);
    } else if (on) {
      mean = grp[g].x;
      m2 = grp[g].y;
    }
    const float rstd = 1.0f / sqrtf(m2 / all + s.eps);
    if (on && rank == 0) {
      fin[g] = make_float2(mean, rstd);
      if (at.rank == 0) {
        const long long o = at.sample * s.G + at.c_base / s.Cg + g;
        mean_out[o] = mean;
        rstd_out[o] = rstd;
      }
    }
  }
  if (p.cluster > 1) cluster_arrive_relaxed();  // this CTA has read the others' moments
  __syncthreads();
  f32x2 m[kParts];
  if (at.active) {
    f32x2 rs[kParts];
    gn_read_groups<SUB>(fin, at.vec * 8, s.Cg, 0, m, rs);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = fmul2(w[j], gn_of<SUB>(rs, j));
  }
  const uint4* v = stage + tid;
  T* yp = y + first;
  if constexpr (CKPT) {
    const long long sblocks = (s.C + kAct8Block - 1) / kAct8Block;
    int8_t* qp = codes + first;
    uint8_t* sp = scales + (at.sample * s.P + at.r0 + at.lane_row) * sblocks + at.c / kAct8Block;
    const long long sstep = p.rl * sblocks;
    // a block's maximum is a warp shuffle: every lane goes through every turn
    const int turns = gn_lane_rows(at.rows, 0, p.rl);
#pragma unroll 2
    for (int i = 0; i < turns; ++i, v += nt, yp += step, qp += step, sp += sstep) {
      const bool on = i < mine;
      const uint4 u = on ? *v : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t E = act8_exponent<T>(act8_block_amax(u));
      if (on) {
        *reinterpret_cast<uint2*>(qp) = act8_codes<T>(u, E);
        if ((at.vec & 3) == 0) *sp = static_cast<uint8_t>(E);
        f32x2 f[4];
        gn_unpack<T>(u, f);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = act_value2<ACT>(fma2(fsub2(f[j], gn_of<SUB>(m, j)), w[j], b[j]));
        *reinterpret_cast<uint4*>(yp) = gn_pack<T>(f);
      }
    }
  } else {
#pragma unroll 2
    for (int i = 0; i < mine; ++i, v += nt, yp += step) {
      f32x2 f[4];
      gn_unpack<T>(*v, f);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = act_value2<ACT>(fma2(fsub2(f[j], gn_of<SUB>(m, j)), w[j], b[j]));
      *reinterpret_cast<uint4*>(yp) = gn_pack<T>(f);
    }
  }
  if (p.cluster > 1) cluster_wait();  // nobody reads this CTA's shared memory any more
}

// A thread owns 4 channels here (8 bytes of dy): with its sums and parameters it stays within 64 registers, so that
// four CTAs share an SM.  The slope of the activation costs most of the arithmetic, so g = dy act'(u) is computed
// once and kept in fp32 where dy lay (dy lands in the second half of g's place) for the second use.
// SUB: 4 where C / G is a multiple of 4 (a thread's channels share a group), else 1.
template <typename T, int ACT, bool SRC8, int SUB>
__global__ void __launch_bounds__(kGnThreads, 4)
    gn_resident_grad_kernel(const T* __restrict__ dy, const void* __restrict__ src, const uint8_t* __restrict__ scales,
                            const void* __restrict__ weight, const void* __restrict__ bias, const float* __restrict__ mean,
                            const float* __restrict__ rstd, T* __restrict__ dx, float2* __restrict__ sums_out,
                            const GnShape s, const GnResident p) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int kParts = SUB == 4 ? 1 : 2;
  constexpr int kSaved = SRC8 ? 4 : 8;
  const int nt = p.threads, tid = threadIdx.x;
  uint4* const gs = reinterpret_cast<uint4*>(smem) + tid;  // [iters][threads] g of 4 channels; dy in the second half
  unsigned char* const saved = smem + 16 * p.iters * nt + tid * kSaved;
  float2* const ent = reinterpret_cast<float2*>(smem + (16 + kSaved) * p.iters * nt);
  float2* const chan = ent + nt * 4;
  float2* const total = chan + p.slab;
  float2* const fin = total + p.slab;
  griddep_wait();
  griddep_launch_dependents();
  const GnPlace at(s, p, 4);
  const long long pixel0 = at.sample * s.P + at.r0 + at.lane_row;
  const long long first = pixel0 * s.C + at.c;
  const long long step = static_cast<long long>(p.rl) * s.C;
  const long long sblocks = (s.C + kAct8Block - 1) / kAct8Block;
  const int mine = at.active ? gn_lane_rows(at.rows, at.lane_row, p.rl) : 0;
  const int quarter = (p.iters + 3) / 4;
  {
    const T* a = dy + first;
    const unsigned char* q = static_cast<const unsigned char*>(src) + first * (SRC8 ? 1 : 2);
    unsigned char* da = reinterpret_cast<unsigned char*>(gs) + 8;
    unsigned char* dq = saved;
    for (int part = 0; part < 4; ++part) {
      const int end = min(mine, (part + 1) * quarter);
#pragma unroll 4
      for (int i = part * quarter; i < end; ++i, a += step, q += step * (SRC8 ? 1 : 2), da += nt * 16, dq += nt * kSaved) {
        cp_async8(da, a);
        if constexpr (SRC8) cp_async4(dq, q);
        else cp_async8(dq, q);
      }
      cp_async_commit();
    }
  }
  f32x2 w[2], m[kParts], rs[kParts];
  const uint8_t* const sp0 = SRC8 ? scales + pixel0 * sblocks + at.c / kAct8Block : nullptr;
  const long long sstep = p.rl * sblocks;
  auto x_hat = [&](const unsigned char* place, uint32_t E, f32x2(&xh)[2]) {
    if constexpr (SRC8) {
      act8_values4(*reinterpret_cast<const uint32_t*>(place), act8_step(E), xh);
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(place);
      xh[0] = Type16<T>::to_f32x2(v.x);
      xh[1] = Type16<T>::to_f32x2(v.y);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) xh[j] = fmul2(fsub2(xh[j], m[SUB == 4 ? 0 : j]), rs[SUB == 4 ? 0 : j]);
  };
  {
    f32x2 b[2], sg[2], sx[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) sg[j] = sx[j] = f32x2_zero();
    if (at.active) {
      gn_load_param4<T>(weight, at.c, s, 1.0f, w);
      gn_load_param4<T>(bias, at.c, s, 0.0f, b);
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        const long long row = at.sample * s.G, lo = row + (at.c + 2 * i) / s.Cg;
        const long long hi = SUB == 4 ? lo : row + (at.c + 2 * i + 1) / s.Cg;
        m[i] = f2_bits(make_float2(mean[lo], mean[hi]));
        rs[i] = f2_bits(make_float2(rstd[lo], rstd[hi]));
      }
    }
    const unsigned char* q = saved;
    uint4* g_at = gs;
    const uint8_t* sp = sp0;
    for (int part = 0; part < 4; ++part) {
      cp_async_wait_part(part);
      const int end = min(mine, (part + 1) * quarter);
#pragma unroll 2
      for (int i = part * quarter; i < end; ++i, q += nt * kSaved, g_at += nt) {
        uint32_t E = 0;
        if constexpr (SRC8) {
          E = *sp;
          sp += sstep;
        }
        f32x2 xh[2], g[2];
        x_hat(q, E, xh);
        const uint2 v = reinterpret_cast<const uint2*>(g_at)[1];
        g[0] = Type16<T>::to_f32x2(v.x);
        g[1] = Type16<T>::to_f32x2(v.y);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          g[j] = fmul2(g[j], act_slope2<ACT>(fma2(xh[j], w[j], b[j])));
          fadd2(sg[j], g[j]);
          ffma2(sx[j], g[j], xh[j]);
        }
        *reinterpret_cast<ulonglong2*>(g_at) = make_ulonglong2(g[0], g[1]);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 a = bits_f2(sg[j]), c = bits_f2(sx[j]);
      *reinterpret_cast<float4*>(ent + tid * 4 + 2 * j) = make_float4(a.x, c.x, a.y, c.y);
    }
  }
  __syncthreads();
  for (int j = tid; j < at.width; j += nt) {
    float2 a = make_float2(0.0f, 0.0f);
#pragma unroll 8
    for (int r = 0; r < p.rl; ++r) {
      const float2 e = ent[r * p.lanes * 4 + j];
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
  for (int j = tid; j < at.width; j += nt) {
    float2 a = chan[j];
    if (p.cluster > 1) {
      a = make_float2(0.0f, 0.0f);
#pragma unroll 8
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
  if (p.cluster > 1) cluster_arrive_relaxed();
  __syncthreads();
  const float inv = 1.0f / (static_cast<float>(s.P) * static_cast<float>(s.Cg));
  const int lane = tid & 31, warps = nt >> 5, here = at.width / s.Cg;
  for (int g = tid >> 5; g < here; g += warps) {
    float m1 = 0.0f, m2 = 0.0f;
    for (int j = lane; j < s.Cg; j += 32) {
      m1 += total[g * s.Cg + j].x;
      m2 += total[g * s.Cg + j].y;
    }
    warp_sum2(m1, m2);
    if (lane == 0) fin[g] = make_float2(m1 * inv, -m2 * inv);
  }
  __syncthreads();
  f32x2 m1[kParts], m2[kParts];
  if (at.active) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int c = at.vec * 4 + 2 * i;
      const float2 lo = fin[c / s.Cg], hi = SUB == 4 ? lo : fin[(c + 1) / s.Cg];
      m1[i] = f2_bits(make_float2(lo.x, hi.x));
      m2[i] = f2_bits(make_float2(lo.y, hi.y));
    }
  }
  const unsigned char* q = saved;
  const uint4* g_at = gs;
  const uint8_t* sp = sp0;
  T* out = dx + first;
#pragma unroll 2
  for (int i = 0; i < mine; ++i, q += nt * kSaved, g_at += nt, out += step) {
    uint32_t E = 0;
    if constexpr (SRC8) {
      E = *sp;
      sp += sstep;
    }
    f32x2 xh[2];
    x_hat(q, E, xh);
    const ulonglong2 gv = *reinterpret_cast<const ulonglong2*>(g_at);
    const f32x2 g[2] = {gv.x, gv.y};
    // the product rounded by itself, so that a group whose m1 is that product leaves exactly nothing
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      constexpr int kStep = SUB == 4 ? 0 : 1;
      xh[j] = fmul2(rs[j * kStep], fma2(xh[j], m2[j * kStep], fsub2(fmul2(g[j], w[j]), m1[j * kStep])));
    }
    *reinterpret_cast<uint2*>(out) = make_uint2(Type16<T>::from_f32x2(xh[0]), Type16<T>::from_f32x2(xh[1]));
  }
  if (p.cluster > 1) cluster_wait();
}

// ---- host -----------------------------------------------------------------------------------------

static int gcd_int(int a, int b) { return b == 0 ? a : gcd_int(b, a % b); }

static int gn_sub(const GnShape& s) { return s.Cg % 8 == 0 ? 8 : s.Cg % 4 == 0 ? 4 : 1; }

static bool gn_resident_fill(const GnShape& s, GnPass pass, int slab, int cluster, int most, int limit, GnResident* p) {
  // a thread's 8 (forward) or 4 channels of a pixel
  const int bytes = pass == GnPass::kForward ? 16 : pass == GnPass::kBackward16 ? 24 : 20;
  p->slab = slab;
  p->slabs = (s.C + slab - 1) / slab;
  p->lanes = pass == GnPass::kForward ? (slab / 8 + 3) / 4 * 4 : slab / 4;  // forward: the checkpoint's quads
  if (p->lanes > most) return false;
  const long long rows = (s.P + cluster - 1) / cluster;
  if (rows > (1 << 20)) return false;
  p->cluster = cluster;
  p->cluster_log = 0;
  while ((1 << p->cluster_log) < cluster) ++p->cluster_log;
  // exact for thread < 256, lanes <= 256: the product is too large by thread / 65536 < 1 / lanes at most
  p->lane_mul = 65536u / p->lanes + 1;
  p->rows_per_cta = static_cast<int>(rows);
  p->rl = most / p->lanes;
  if (p->rl > p->rows_per_cta) p->rl = p->rows_per_cta;
  p->threads = (p->lanes * p->rl + 31) / 32 * 32;
  p->iters = (p->rows_per_cta + p->rl - 1) / p->rl;
  const long long extra = pass == GnPass::kForward
                              ? 8LL * (p->threads * (8 / gn_sub(s)) + 2 * (slab / s.Cg))
                              : 8LL * (p->threads * 4 + 2 * slab + slab / s.Cg);
  const long long need = static_cast<long long>(p->iters) * p->threads * bytes + extra;
  if (need > limit) return false;
  p->smem = static_cast<int>(need);
  return s.B <= 65535;  // grid y
}

// The rule.  A unit's pixels are shared by the fewest CTAs (1 to 8) that hold them four to an SM, else two to an SM:
// 32x32x1536, 32 groups, B = 16, forward: 32 us with 4 CTAs of 49 KB, 34 with 2 of 98 KB, 39 with 8 of 25 KB and as many
// threads.  Where that makes eight CTAs an SM or more, CTAs of half the threads, seven or eight to
// an SM: 31.8 us there, 95 against 97.5 us at 56x56x1024, B = 32, 47.5 against 51.3 us with a checkpoint at 56x56x128,
// B = 64.  What needs more goes to the streaming passes (one group over 32x32x768, B = 8: 8 CTAs of 196 KB 14.2 us, 16 of 98 KB
// 11.4 us, streaming 11.2 us).
// Backward, the streaming passes are faster where clusters have more than about 1.75 turns of the CTAs that run at
// once, because a cluster's exchange (3.7 us) is too long for the little that two or four CTAs an SM bring along.
// Four an SM: 32x32x1536 with B = 2 / 4 / 8 / 16, resident 12.3 / 23.8 / 42.1 / 81 us, streaming 16.2 / 24.1 / 37.2 /
// 63 us; two an SM, from a checkpoint: 56x56x768 with B = 2 / 4 / 8, 18.6 / 41.7 / 81.4 and 24.0 / 38.6 / 57.8 us.
// CTAs by themselves have no exchange: 14x14x512 with B = 128 / 512, GELU, 35.0 / 122 and 41.0 / 136 us (at worst, B = 256
// without activation, 56.5 and 53.1 us).
// Forward the resident kernels stay ahead at every size (56x56x1024, B = 32: 97 against 119 us): they move two thirds
// of the data.
bool gn_resident_plan(const GnShape& s, GnPass pass, GnResident* p) {
  // shared memory of seven, four and two CTAs an SM: 228 KB less 1 KB each
  constexpr int kSmall = 31 * 1024 + 512, kFour = 56 * 1024, kTwo = 113 * 1024;
  // whole groups; forward: whole blocks of a checkpoint (with and without one: the same plan, the same bits), backward:
  // whole vectors and, where it can be, 64 bytes of a pixel
  const int align = pass == GnPass::kForward ? kAct8Block : 8;
  const long long unit_ll = static_cast<long long>(s.Cg) / gcd_int(s.Cg, align) * align;
  int unit = unit_ll < s.C ? static_cast<int>(unit_ll) : s.C;
  for (int k = unit; unit < 32 && unit < s.C;) unit = unit + k < s.C ? unit + k : s.C;
  // few pixels: more units a CTA, until it has 512 vectors of 8 channels or an SM would go without (7x7x1024, 32 groups,
  // B = 256: forward 35.7 us with one unit of 32 channels, 20.3 so, gradient 59 and 34.5; with 1024 vectors the gradient
  // 70.2).  At most 1024 channels, a thread for every vector of a pixel.
  for (const int k = unit; unit + k <= s.C && unit + k <= 8 * kGnThreads / 2 && s.P * unit < 8 * 512 &&
                           static_cast<long long>(s.B) * ((s.C + unit + k - 1) / (unit + k)) >= kSmCount;)
    unit += k;
  // many units: small CTAs that are seldom in the same phase
  if (pass == GnPass::kForward)
    for (int cluster = 1; cluster <= 8; cluster *= 2)
      if (gn_resident_fill(s, pass, unit, cluster, kGnThreads / 2, kSmall, p)) {
        if (static_cast<long long>(s.B) * p->slabs * cluster < 8 * kSmCount) break;
        return true;
      }
  for (int limit : {kFour, kTwo})
    for (int cluster = 1; cluster <= 8; cluster *= 2)
      if (gn_resident_fill(s, pass, unit, cluster, kGnThreads, limit, p)) {
        // few clusters: more CTAs share a sample, as long as each thread keeps a few pixels
        GnResident wider;
        while (static_cast<long long>(s.B) * p->slabs * p->cluster < 2 * kSmCount && p->cluster < 8 && p->iters > 4 &&
               gn_resident_fill(s, pass, unit, p->cluster * 2, kGnThreads, limit, &wider))
          *p = wider;
        return pass == GnPass::kForward || p->cluster == 1 ||
               static_cast<long long>(s.B) * p->slabs * p->cluster * 4 <= 7LL * kSmCount * (p->smem <= kFour ? 4 : 2);
      }
  return false;
}

static int gn_resident_launch(const void* fn, const char* what, const GnShape& s, const GnResident& p, void** args,
                              cudaStream_t stream) {
  cudaError_t e = allow_large_cta(fn);
  if (e == cudaSuccess)
    e = launch_kernel(fn, dim3(static_cast<unsigned>(p.slabs * p.cluster), static_cast<unsigned>(s.B)), dim3(p.threads), args,
                      p.smem, stream, p.cluster);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return record_cuda_failure(what, e);
  }
  return DWB_OK;
}

template <typename T, bool CKPT, int SUB>
static const void* resident_fn(int act) {
  switch (act) {
    case kActRelu: return reinterpret_cast<const void*>(&gn_resident_kernel<T, kActRelu, CKPT, SUB>);
    case kActGelu: return reinterpret_cast<const void*>(&gn_resident_kernel<T, kActGelu, CKPT, SUB>);
    case kActSilu: return reinterpret_cast<const void*>(&gn_resident_kernel<T, kActSilu, CKPT, SUB>);
    default: return reinterpret_cast<const void*>(&gn_resident_kernel<T, kActNone, CKPT, SUB>);
  }
}
template <typename T, bool SRC8, int SUB>
static const void* resident_grad_fn(int act) {
  switch (act) {
    case kActRelu: return reinterpret_cast<const void*>(&gn_resident_grad_kernel<T, kActRelu, SRC8, SUB>);
    case kActGelu: return reinterpret_cast<const void*>(&gn_resident_grad_kernel<T, kActGelu, SRC8, SUB>);
    case kActSilu: return reinterpret_cast<const void*>(&gn_resident_grad_kernel<T, kActSilu, SRC8, SUB>);
    default: return reinterpret_cast<const void*>(&gn_resident_grad_kernel<T, kActNone, SRC8, SUB>);
  }
}
template <typename T, bool CKPT>
static const void* resident_fn(int sub, int act) {
  return sub == 8 ? resident_fn<T, CKPT, 8>(act) : sub == 4 ? resident_fn<T, CKPT, 4>(act) : resident_fn<T, CKPT, 1>(act);
}
template <typename T, bool SRC8>
static const void* resident_grad_fn(int sub, int act) {
  return sub >= 4 ? resident_grad_fn<T, SRC8, 4>(act) : resident_grad_fn<T, SRC8, 1>(act);
}

template <typename T>
int gn_resident_forward(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, void* codes,
                        void* scales, const GnShape& s, const GnResident& p, int act, cudaStream_t stream) {
  const void* fn = codes ? resident_fn<T, true>(gn_sub(s), act) : resident_fn<T, false>(gn_sub(s), act);
  GnShape sv = s;
  GnResident pv = p;
  void* args[] = {&x, &weight, &bias, &y, &mean, &rstd, &codes, &scales, &sv, &pv};
  return gn_resident_launch(fn, "gn_resident_kernel", s, p, args, stream);
}

template <typename T>
int gn_resident_backward(const void* dy, const void* x, const void* codes, const void* scales, const float* mean,
                         const float* rstd, const void* weight, const void* bias, void* dx, float2* sums, const GnShape& s,
                         const GnResident& p, int act, cudaStream_t stream) {
  const void* fn = codes ? resident_grad_fn<T, true>(gn_sub(s), act) : resident_grad_fn<T, false>(gn_sub(s), act);
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
