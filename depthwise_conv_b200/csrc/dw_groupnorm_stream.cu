// dw_groupnorm_stream.cu -- group normalisation of large tensors in two
// streaming passes: partial sums of row chunks, then the normalisation (or its
// gradient), which merges the partial sums it needs first.  The formulas stand
// in dw_groupnorm.cuh.
//
// Measured, gradient: 65.9 us at 16x32x32x1536, 32 groups, GELU; 186 us at
// 32x56x56x1024, SiLU.  Each pass reads dy and the input, 252 MB with dx in the first of
// these, 3.8 TB/s, and issues 24 instructions a value (27 to 30 from a checkpoint),
// most of them for the activation's slope, which both passes compute: keeping it
// would write and read 2 bytes a value more.
//
// The call goes through the batch in groups of samples, so that the second pass
// finds part of its data in L2, and one launch does the second pass of a group
// and the first pass of the next one, so that reading the one overlaps with
// writing the other.  No CTA waits for another: a thread always has 8 or 12
// vectors under way, through places of its own in shared memory.
//
// What a CTA hands over (an entry) is the moments, or the weighted sums, of a
// segment of channels and a chunk of rows.  A segment is a group; a tile of 256
// channels of a larger group (C / G a multiple of 8); or a single channel (other
// large groups).
#include <cuda_runtime.h>

#include "../../include/dwconv_b200.h"
#include "dw_groupnorm.cuh"
#include "dw_groupnorm_stream.h"
#include "dw_host.h"
#include "dw_launch.h"

namespace dwb {

constexpr int kThreads = 256;
constexpr int kBatch = 4;         // vectors that a thread waits for and handles together
constexpr int kForwardBatches = 3, kBackwardBatches = 2;  // of them under way (the gradient has two streams)
constexpr int kApplyLanes = 16;   // 128 channels, 256 bytes of a pixel, a CTA of the second pass
constexpr int kSmallTile = 64;    // channels of a first-pass tile: at least
constexpr int kLargeTile = 256;   // and at most
// Inputs of a group of samples.  Smaller groups find more in L2 (126 MB) and pay for it with launches, each with its
// own ramp: 56x56x1024, B = 32, gradient: 352 us with 40 MB, 204 with 110, 197 with 160 and 210, 202 in one group.
constexpr long long kGroupBytes = 160LL << 20;

// A thread's vectors i = 0 .. n - 1, `step` values apart, through its own places of a ring in shared memory:
// BATCHES batches of kBatch loads are under way while one is handled, without barriers (nobody else reads the
// places) and without registers.
template <int BYTES, int BATCHES>
struct Stream {
  unsigned char* ring;   // this thread's first place; places are kThreads * BYTES apart
  const unsigned char* next;
  long long step;        // bytes
  int left;
  __device__ __forceinline__ Stream(unsigned char* smem, const void* first, long long step_bytes, int n)
      : ring(smem + threadIdx.x * BYTES), next(static_cast<const unsigned char*>(first)), step(step_bytes), left(n) {}
  __device__ __forceinline__ void issue(int batch) {
    unsigned char* at = ring + batch * (kBatch * kThreads * BYTES);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (j < left) {
        if constexpr (BYTES == 16) cp_async16(at + j * kThreads * BYTES, next + j * step);
        else cp_async8(at + j * kThreads * BYTES, next + j * step);
      }
    }
    next += kBatch * step;
    left -= kBatch;
  }
  template <typename V>
  __device__ __forceinline__ V get(int batch, int j) const {
    return *reinterpret_cast<const V*>(ring + (batch * kBatch + j) * kThreads * BYTES);
  }
};
template <int BATCHES>
__device__ __forceinline__ void wait_batch() {
  asm volatile("cp.async.wait_group %0;" ::"n"(BATCHES - 1) : "memory");
}
constexpr int kForwardRing = kForwardBatches * kBatch * kThreads * 16;
constexpr int kBackwardRing = kBackwardBatches * kBatch * kThreads * 16;  // of dy
constexpr int kFinMost = kApplyLanes * 8 + 1;  // groups that 128 channels can belong to
constexpr int kFinBytes = kFinMost * 8 + kThreads / 32 * 3 * 4;  // and the sums of warps that share a group

// The first launch of a call waits for the kernel before it, which may make its inputs.  The others read nothing but
// what that launch could read, and the entries of the launch before them: they begin to load first (q.early), while
// that launch's last CTAs run, and wait for it then.
__device__ __forceinline__ void begin_after_previous() {
  griddep_wait();
  griddep_launch_dependents();
}

// Place of a thread in a tile.
struct StreamThread {
  int lane_row, vec, r0, rows;
  __device__ __forceinline__ StreamThread(const GnStream& q, int lanes, unsigned lane_mul, int rows_per_chunk, int chunk, int P) {
    lane_row = threadIdx.x * lane_mul >> 16;
    vec = threadIdx.x - lane_row * lanes;
    r0 = chunk * rows_per_chunk;
    rows = min(rows_per_chunk, P - r0);
  }
  __device__ __forceinline__ int mine(int rl) const { return lane_row < rl && rows > lane_row ? (rows - lane_row + rl - 1) / rl : 0; }
};

// First-pass tile: its channels and first entry.
struct StreamTile {
  int c0, width, seg, entry;
  __device__ __forceinline__ StreamTile(const GnShape& s, const GnStream& q, int tile) {
    if (q.tiles_per_group > 1) {
      const int g = tile / q.tiles_per_group, sub = tile - g * q.tiles_per_group;
      c0 = g * s.Cg + sub * q.tile;
      width = min(q.tile, s.Cg - sub * q.tile);
      seg = width;
      entry = tile;
    } else {
      c0 = tile * q.tile;
      width = min(q.tile, s.C - c0);
      seg = q.entries_per_group > 1 ? 1 : s.Cg;
      entry = c0 / seg;
    }
  }
};

// Channels of entry k of a group.
__device__ __forceinline__ int entry_width(const GnShape& s, const GnStream& q, int k) {
  return q.tiles_per_group > 1 ? min(q.tile, s.Cg - k * q.tile) : s.Cg / q.entries_per_group;
}

// Moments of every segment of a tile and chunk: part[sample][chunk][entry] = (mean, M2).
template <typename T, int SUB>
__device__ __forceinline__ void stats_cta(const T* __restrict__ x, float2* __restrict__ part, const GnShape& s, const GnStream& q,
                                          int sample, int work, float2* ent, unsigned char* ring) {
  constexpr int kEnt = 8 / SUB;
  const int chunk = work / q.tiles;
  const StreamTile tile(s, q, work - chunk * q.tiles);
  const StreamThread t(q, q.lanes, q.lane_mul, q.rows, chunk, static_cast<int>(s.P));
  const int c = tile.c0 + t.vec * 8, tid = threadIdx.x;
  const int n = t.vec * 8 < tile.width ? t.mine(q.rl) : 0;
  const T* p = x + (static_cast<long long>(sample) * s.P + t.r0 + t.lane_row) * s.C + c;
  const long long step = static_cast<long long>(q.rl) * s.C;
  Stream<16, kForwardBatches> in(ring, p, step * sizeof(T), n);
  for (int k = 0; k < kForwardBatches; ++k) {
    in.issue(k);
    cp_async_commit();
  }
  if (q.early) begin_after_previous();
  if (n) {
    GnSums sums;
    f32x2 f[4];
    wait_batch<kForwardBatches>();
    gn_unpack<T>(in.template get<uint4>(0, 0), f);
    sums.start(f);
    int batch = 0;
    for (int i = 0; i < n; i += kBatch) {
      wait_batch<kForwardBatches>();
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i + j < n) {
          gn_unpack<T>(in.template get<uint4>(batch, j), f);
          sums.add(f);  // the first value once more: a difference of 0
        }
      in.issue(batch);
      cp_async_commit();
      batch = batch + 1 < kForwardBatches ? batch + 1 : 0;
    }
    f32x2 mean[4], m2[4];
    sums.moments(n, mean, m2);
    gn_hand_over<SUB>(mean, m2, static_cast<float>(n), ent + tid * kEnt);
  }
  __syncthreads();
  if constexpr (SUB == 1) {
    if (q.entries_per_group > 1) {  // single channels: a thread each, over the lane rows (a warp each: 22.0 us, so 10.1,
      // at 1x36x18x1208, 4 groups)
      const int live = min(t.rows, q.rl), full = t.rows / q.rl, rest = t.rows - full * q.rl;
      for (int j = tid; j < tile.width; j += kThreads) {
        const float pivot = ent[j].x;
        float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f;
#pragma unroll 4
        for (int r = 0; r < live; ++r) {
          const float2 v = ent[r * q.lanes * kEnt + j];
          const float m = static_cast<float>(full + (r < rest)), d = v.x - pivot;
          s0 += m * v.x;
          s1 += m * d;
          s2 += v.y + m * d * d;
        }
        const float rows = static_cast<float>(t.rows), off = s1 / rows;
        part[(static_cast<long long>(sample) * q.chunks + chunk) * q.entries + tile.entry + j] =
            make_float2(gn_mean(pivot, off, s0 / rows), not_negative(s2 - s1 * off));
      }
      return;
    }
  }
  const int lane = tid & 31, segments = tile.width / tile.seg;
  const GnMerge merge(lane, tile.seg / SUB, t.rows, q.rl, q.lanes * kEnt);
  for (int g = tid >> 5; g < segments; g += kThreads / 32) {
    const float2 m = merge.run<SUB>(ent + g * (tile.seg / SUB), t.rows, tile.seg);
    if (lane == 0) part[(static_cast<long long>(sample) * q.chunks + chunk) * q.entries + tile.entry + g] = m;
  }
}

// How a CTA's warps share the entries of its groups: a warp a group, or with SHARE (an entry may be a channel) `split`
// warps a group where it has few groups of many entries (1x36x18x1208, 4 groups: 302 entries a group and chunk).
template <bool SHARE>
struct EntryShare {
  int split = 1, of, slice = 0;
  __device__ __forceinline__ EntryShare(int groups, int entries) {
    of = threadIdx.x >> 5;
    if constexpr (SHARE) {
      while (split * 2 * groups <= kThreads / 32 && split * 64 <= entries) split *= 2;
      slice = of % split;
      of /= split;
    }
  }
  __device__ __forceinline__ int groups_at_once() const { return kThreads / 32 / split; }  // all of them where split > 1
  // The sums of a group's warps, in order, in the first of them; `sums` has three places a warp.  Every thread of the
  // CTA calls it.
  __device__ __forceinline__ void add(float& a, float& b, float& c, float* sums) const {
    if (!SHARE || split == 1) return;
    float* const mine = sums + 3 * (threadIdx.x >> 5);
    if ((threadIdx.x & 31) == 0) {
      mine[0] = a;
      mine[1] = b;
      mine[2] = c;
    }
    __syncthreads();
    if (slice == 0)
      for (int i = 1; i < split; ++i) {
        a += mine[3 * i];
        b += mine[3 * i + 1];
        c += mine[3 * i + 2];
      }
  }
};

// Mean and rstd of the groups that channels [c0, c0 + width) belong to, from their entries.
template <bool SHARE>
__device__ __forceinline__ void merge_stats(const float2* __restrict__ part, const GnShape& s, const GnStream& q, int sample, int c0,
                                            int width, float2* fin, float* mean_out, float* rstd_out) {
  const int lane = threadIdx.x & 31, g0 = c0 / s.Cg, g1 = (c0 + width - 1) / s.Cg, per = q.entries_per_group;
  const float2* of_sample = part + static_cast<long long>(sample) * q.chunks * q.entries;
  const int last = static_cast<int>(s.P) - (q.chunks - 1) * q.rows;
  const EntryShare<SHARE> share(g1 - g0 + 1, q.chunks * per);
  for (int next = g0; next <= g1; next += share.groups_at_once()) {
    const int g = next + share.of;
    float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f, pivot = 0.0f;
    if (g <= g1) {
      const float2* first = of_sample + g * per;
      // about the first entry's mean: entries are means of many values, nothing cancels in the squares
      pivot = first[0].x;
      for (int e = share.slice * 32 + lane; e < q.chunks * per; e += 32 * share.split) {
        const int chunk = e / per, k = e - chunk * per;
        const float2 v = first[static_cast<long long>(chunk) * q.entries + k];
        const float n = static_cast<float>(chunk == q.chunks - 1 ? last : q.rows) * static_cast<float>(entry_width(s, q, k));
        const float d = v.x - pivot;
        s0 += n * v.x;
        s1 += n * d;
        s2 += v.y + n * d * d;
      }
    }
    if (!SHARE && g > g1) break;
    warp_sum3(s0, s1, s2);
    share.add(s0, s1, s2, reinterpret_cast<float*>(fin + kFinMost));
    const float n = static_cast<float>(s.P) * static_cast<float>(s.Cg), off = s1 / n;
    const float mean = gn_mean(pivot, off, s0 / n), rstd = 1.0f / sqrtf(not_negative(s2 - s1 * off) / n + s.eps);
    if (g <= g1 && share.slice == 0 && lane == 0) {
      fin[g - g0] = make_float2(mean, rstd);
      if (mean_out && g * s.Cg >= c0) {
        mean_out[static_cast<long long>(sample) * s.G + g] = mean;
        rstd_out[static_cast<long long>(sample) * s.G + g] = rstd;
      }
    }
  }
  __syncthreads();
}

template <typename T, int ACT, bool CKPT, int SUB>
__device__ __forceinline__ void apply_cta(const T* __restrict__ x, const void* __restrict__ weight, const void* __restrict__ bias,
                                          const float2* __restrict__ part, T* __restrict__ y, float* __restrict__ mean_out,
                                          float* __restrict__ rstd_out, int8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                          const GnShape& s, const GnStream& q, int sample, int work, float2* fin,
                                          unsigned char* ring) {
  constexpr int kParts = SUB == 8 ? 1 : SUB == 4 ? 2 : 4;
  const int chunk = work / q.apply_tiles, c0 = (work - chunk * q.apply_tiles) * (q.apply_lanes * 8);
  const int width = min(q.apply_lanes * 8, s.C - c0);
  const StreamThread t(q, q.apply_lanes, q.apply_lane_mul, q.apply_rows, chunk, static_cast<int>(s.P));
  const int c = c0 + t.vec * 8;
  const bool active = t.vec * 8 < width;
  const int n = active ? t.mine(q.apply_rl) : 0;
  const long long pixel = static_cast<long long>(sample) * s.P + t.r0 + t.lane_row;
  const long long sblocks = (s.C + kAct8Block - 1) / kAct8Block;
  const long long first = pixel * s.C + c, step = static_cast<long long>(q.apply_rl) * s.C, sstep = q.apply_rl * sblocks;
  Stream<16, kForwardBatches> in(ring, x + first, step * sizeof(T), n);
  for (int k = 0; k < kForwardBatches; ++k) {
    in.issue(k);
    cp_async_commit();
  }
  if (q.early) begin_after_previous();
  f32x2 w[4], b[4], m[kParts];
  if (active) gn_load_params<T>(weight, bias, c, s, w, b);
  // the CTA of a chunk's first rows and of a group's first channels writes the group's mean and rstd
  merge_stats<SUB == 1>(part, s, q, sample, c0, width, fin, chunk == 0 ? mean_out : nullptr, rstd_out);
  if (active) {
    f32x2 rs[kParts];
    gn_read_groups<SUB>(fin, c, s.Cg, c0 / s.Cg, m, rs);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = fmul2(w[j], gn_of<SUB>(rs, j));
  }
  T* yp = y + first;
  int8_t* qp = CKPT ? codes + first : nullptr;
  uint8_t* sp = CKPT ? scales + pixel * sblocks + c / kAct8Block : nullptr;
  // a checkpoint's block maximum is a warp shuffle: every lane goes through every turn
  const int turns = CKPT ? (t.rows + q.apply_rl - 1) / q.apply_rl : n;
  int batch = 0;
  for (int i = 0; i < turns; i += kBatch) {
    wait_batch<kForwardBatches>();
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const bool on = i + j < n;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (on) v = in.template get<uint4>(batch, j);
      if constexpr (CKPT) {
        const uint32_t E = act8_exponent<T>(act8_block_amax(v));
        if (on) {
          *reinterpret_cast<uint2*>(qp) = act8_codes<T>(v, E);
          if ((t.vec & 3) == 0) *sp = static_cast<uint8_t>(E);
        }
        qp += step;
        sp += sstep;
      }
      if (on) {
        f32x2 f[4];
        gn_unpack<T>(v, f);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = act_value2<ACT>(fma2(fsub2(f[k], gn_of<SUB>(m, k)), w[k], b[k]));
        *reinterpret_cast<uint4*>(yp) = gn_pack<T>(f);
      }
      yp += step;
    }
    in.issue(batch);
    cp_async_commit();
    batch = batch + 1 < kForwardBatches ? batch + 1 : 0;
  }
}

// Which CTA of which pass: the two passes' CTAs alternate while both last.
__device__ __forceinline__ bool second_pass(const GnStream& q, unsigned block, unsigned* work) {
  const unsigned both = min(q.first_ctas, q.second_ctas) * 2;
  if (block < both) {
    *work = block >> 1;
    return block & 1;
  }
  *work = block - both / 2;
  return q.second_ctas > q.first_ctas;
}

template <typename T, int ACT, bool CKPT, int SUB>
__global__ void __launch_bounds__(kThreads, 3)
    gn_stream_kernel(const T* __restrict__ x, const void* __restrict__ weight, const void* __restrict__ bias,
                     float2* __restrict__ part, T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd,
                     int8_t* __restrict__ codes, uint8_t* __restrict__ scales, const GnShape s, const GnStream q) {
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char* const ring = smem;
  float2* const ent = reinterpret_cast<float2*>(smem + kForwardRing);
  if (!q.early) begin_after_previous();
  unsigned work;
  if (second_pass(q, blockIdx.x, &work)) {
    const unsigned per = q.apply_tiles * q.apply_chunks, sample = work / per;
    apply_cta<T, ACT, CKPT, SUB>(x, weight, bias, part, y, mean, rstd, codes, scales, s, q, q.second_sample + sample,
                                 work - sample * per, ent, ring);
  } else {
    const unsigned per = q.tiles * q.chunks, sample = work / per;
    stats_cta<T, SUB>(x, part, s, q, q.first_sample + sample, work - sample * per, ent, ring);
  }
}

// ---- backward -----------------------------------------------------------------------------------

template <bool SRC8>
struct RawOf {
  using type = uint4;
};
template <>
struct RawOf<true> {
  using type = uint2;
};

// The saved input of the norm: 8 values in 16 bits, or 8 codes and their exponent byte.
template <typename T, bool SRC8, int SUB>
struct SavedInput {
  static constexpr int kParts = SUB == 8 ? 1 : SUB == 4 ? 2 : 4;
  f32x2 m[kParts], rs[kParts];
  __device__ __forceinline__ void load_stats(const float* mean, const float* rstd, const GnShape& s, int sample, int c) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int at = c + i * (SUB == 1 ? 2 : SUB);
      const long long row = static_cast<long long>(sample) * s.G, lo = row + at / s.Cg, hi = SUB == 1 ? row + (at + 1) / s.Cg : lo;
      m[i] = f2_bits(make_float2(mean[lo], mean[hi]));
      rs[i] = f2_bits(make_float2(rstd[lo], rstd[hi]));
    }
  }
  static constexpr int kBytes = SRC8 ? 8 : 16;
  using Raw = typename RawOf<SRC8>::type;
  __device__ __forceinline__ void x_hat(const Raw& raw, uint32_t E, f32x2 (&xh)[4]) const {
    if constexpr (SRC8) act8_values(raw, act8_step(E), xh);
    else gn_unpack<T>(raw, xh);
#pragma unroll
    for (int j = 0; j < 4; ++j) xh[j] = fmul2(fsub2(xh[j], gn_of<SUB>(m, j)), gn_of<SUB>(rs, j));
  }
};

// The exponent bytes of a thread's vectors, a batch ahead in registers.
struct Exponents {
  const uint8_t* next;
  long long step;
  int left;
  uint32_t now[kBatch], then[kBatch];
  __device__ __forceinline__ void fetch() {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) then[j] = j < left ? next[j * step] : 0u;
    next += kBatch * step;
    left -= kBatch;
  }
  __device__ __forceinline__ void advance() {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) now[j] = then[j];
    fetch();
  }
};

// chan[sample][chunk][c] = (sum g, sum g xh); part[sample][chunk][entry] = the same times the weight, over the segment.
template <typename T, int ACT, bool SRC8, int SUB>
__device__ __forceinline__ void grad_sums_cta(const T* __restrict__ dy, const void* __restrict__ src, const uint8_t* __restrict__ scales,
                                              const void* __restrict__ weight, const void* __restrict__ bias,
                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                              float2* __restrict__ part, float2* __restrict__ chan, const GnShape& s,
                                              const GnStream& q, int sample, int work, unsigned char* ring) {
  const int chunk = work / q.tiles;
  const StreamTile tile(s, q, work - chunk * q.tiles);
  const StreamThread t(q, q.lanes, q.lane_mul, q.rows, chunk, static_cast<int>(s.P));
  const int c = tile.c0 + t.vec * 8, tid = threadIdx.x;
  const int n = t.vec * 8 < tile.width ? t.mine(q.rl) : 0;
  using In = SavedInput<T, SRC8, SUB>;
  const long long pixel = static_cast<long long>(sample) * s.P + t.r0 + t.lane_row;
  const long long sblocks = (s.C + kAct8Block - 1) / kAct8Block, sstep = q.rl * sblocks;
  const long long step = static_cast<long long>(q.rl) * s.C, first = pixel * s.C + c;
  Stream<16, kBackwardBatches> grad(ring, dy + first, step * sizeof(T), n);
  Stream<In::kBytes, kBackwardBatches> saved(ring + kBackwardRing, static_cast<const unsigned char*>(src) + first * (SRC8 ? 1 : 2),
                                             step * (SRC8 ? 1 : 2), n);
  for (int k = 0; k < kBackwardBatches; ++k) {
    grad.issue(k);
    saved.issue(k);
    cp_async_commit();
  }
  if (q.early) begin_after_previous();
  f32x2 sg[4], sx[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) sg[j] = sx[j] = f32x2_zero();
  if (n) {
    Exponents ex{scales + (SRC8 ? pixel * sblocks + c / kAct8Block : 0), sstep, SRC8 ? n : 0};
    if constexpr (SRC8) ex.fetch();
    f32x2 w[4], b[4];
    In in;
    gn_load_params<T>(weight, bias, c, s, w, b);
    in.load_stats(mean, rstd, s, sample, c);
    int batch = 0;
    for (int i = 0; i < n; i += kBatch) {
      if constexpr (SRC8) ex.advance();
      wait_batch<kBackwardBatches>();
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i + j < n) {
          f32x2 xh[4], g[4];
          in.x_hat(saved.template get<typename In::Raw>(batch, j), SRC8 ? ex.now[j] : 0u, xh);
          gn_unpack<T>(grad.template get<uint4>(batch, j), g);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            g[k] = fmul2(g[k], act_slope2<ACT>(fma2(xh[k], w[k], b[k])));
            fadd2(sg[k], g[k]);
            ffma2(sx[k], g[k], xh[k]);
          }
        }
      grad.issue(batch);
      saved.issue(batch);
      cp_async_commit();
      batch = batch + 1 < kBackwardBatches ? batch + 1 : 0;
    }
  }
  // the threads' sums take the place of the ring
  static_assert(kThreads * 8 * sizeof(float2) <= kBackwardRing, "sums of a CTA in the ring's place");
  float2* const ent = reinterpret_cast<float2*>(ring);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 a = bits_f2(sg[j]), e = bits_f2(sx[j]);
    *reinterpret_cast<float4*>(ent + tid * 8 + 2 * j) = make_float4(a.x, e.x, a.y, e.y);
  }
  __syncthreads();
  const long long row = static_cast<long long>(sample) * q.chunks + chunk;
  const bool single = SUB == 1 && q.entries_per_group > 1;  // an entry a channel
  for (int j = tid; j < tile.width; j += kThreads) {
    float2 a = make_float2(0.0f, 0.0f);
#pragma unroll 8
    for (int r = 0; r < q.rl; ++r) {
      const float2 e = ent[r * q.lanes * 8 + j];
      a.x += e.x;
      a.y += e.y;
    }
    chan[row * s.C + tile.c0 + j] = a;
    const float wj = gn_param<T>(weight, tile.c0 + j, s.param_f32, 1.0f);
    a = make_float2(a.x * wj, a.y * wj);
    if (single) part[row * q.entries + tile.entry + j] = a;
    else ent[j] = a;  // lane row 0's place of this channel: this thread has just read it
  }
  if (single) return;
  __syncthreads();
  const int lane = tid & 31, segments = tile.width / tile.seg;
  for (int g = tid >> 5; g < segments; g += kThreads / 32) {
    float m1 = 0.0f, m2 = 0.0f;
    for (int j = lane; j < tile.seg; j += 32) {
      m1 += ent[g * tile.seg + j].x;
      m2 += ent[g * tile.seg + j].y;
    }
    warp_sum2(m1, m2);
    if (lane == 0) part[row * q.entries + tile.entry + g] = make_float2(m1, m2);
  }
}

template <typename T, int ACT, bool SRC8, int SUB>
__device__ __forceinline__ void grad_apply_cta(const T* __restrict__ dy, const void* __restrict__ src,
                                               const uint8_t* __restrict__ scales, const void* __restrict__ weight,
                                               const void* __restrict__ bias, const float* __restrict__ mean,
                                               const float* __restrict__ rstd, const float2* __restrict__ part,
                                               T* __restrict__ dx, const GnShape& s, const GnStream& q, int sample, int work,
                                               float2* fin, unsigned char* ring) {
  constexpr int kParts = SUB == 8 ? 1 : SUB == 4 ? 2 : 4;
  const int chunk = work / q.apply_tiles, c0 = (work - chunk * q.apply_tiles) * (q.apply_lanes * 8);
  const int width = min(q.apply_lanes * 8, s.C - c0);
  const StreamThread t(q, q.apply_lanes, q.apply_lane_mul, q.apply_rows, chunk, static_cast<int>(s.P));
  const int c = c0 + t.vec * 8;
  const bool active = t.vec * 8 < width;
  const int n = active ? t.mine(q.apply_rl) : 0;
  using In = SavedInput<T, SRC8, SUB>;
  const long long pixel = static_cast<long long>(sample) * s.P + t.r0 + t.lane_row;
  const long long sblocks = (s.C + kAct8Block - 1) / kAct8Block, sstep = q.apply_rl * sblocks;
  const long long step = static_cast<long long>(q.apply_rl) * s.C, first = pixel * s.C + c;
  Stream<16, kBackwardBatches> grad(ring, dy + first, step * sizeof(T), n);
  Stream<In::kBytes, kBackwardBatches> saved(ring + kBackwardRing, static_cast<const unsigned char*>(src) + first * (SRC8 ? 1 : 2),
                           step * (SRC8 ? 1 : 2), n);
  for (int k = 0; k < kBackwardBatches; ++k) {
    grad.issue(k);
    saved.issue(k);
    cp_async_commit();
  }
  if (q.early) begin_after_previous();
  Exponents ex{scales + (SRC8 ? pixel * sblocks + c / kAct8Block : 0), sstep, SRC8 ? n : 0};
  if constexpr (SRC8) ex.fetch();
  f32x2 w[4], b[4];
  In in;
  if (active) {
    gn_load_params<T>(weight, bias, c, s, w, b);
    in.load_stats(mean, rstd, s, sample, c);
  }
  {
    const int lane = threadIdx.x & 31, g0 = c0 / s.Cg, g1 = (c0 + width - 1) / s.Cg, per = q.entries_per_group;
    const float inv = 1.0f / (static_cast<float>(s.P) * static_cast<float>(s.Cg));
    const EntryShare<SUB == 1> share(g1 - g0 + 1, q.chunks * per);
    for (int next = g0; next <= g1; next += share.groups_at_once()) {
      const int g = next + share.of;
      float m1 = 0.0f, m2 = 0.0f, none = 0.0f;
      if (g <= g1) {
        const float2* entry = part + static_cast<long long>(sample) * q.chunks * q.entries + g * per;
        for (int e = share.slice * 32 + lane; e < q.chunks * per; e += 32 * share.split) {
          const int k = e / per;
          const float2 v = entry[static_cast<long long>(k) * q.entries + (e - k * per)];
          m1 += v.x;
          m2 += v.y;
        }
      }
      if (SUB != 1 && g > g1) break;  // no warp shares
      warp_sum2(m1, m2);
      share.add(m1, m2, none, reinterpret_cast<float*>(fin + kFinMost));
      if (g <= g1 && share.slice == 0 && lane == 0) fin[g - g0] = make_float2(m1 * inv, -m2 * inv);
    }
    __syncthreads();
  }
  if (!n) return;
  f32x2 m1[kParts], m2[kParts];
  gn_read_groups<SUB>(fin, c, s.Cg, c0 / s.Cg, m1, m2);
  T* out = dx + first;
  int batch = 0;
  for (int i = 0; i < n; i += kBatch) {
    if constexpr (SRC8) ex.advance();
    wait_batch<kBackwardBatches>();
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (i + j < n) {
        f32x2 xh[4], g[4];
        in.x_hat(saved.template get<typename In::Raw>(batch, j), SRC8 ? ex.now[j] : 0u, xh);
        gn_unpack<T>(grad.template get<uint4>(batch, j), g);
        // the product rounded by itself, so that a group whose m1 is that product leaves exactly nothing
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          g[k] = fmul2(g[k], act_slope2<ACT>(fma2(xh[k], w[k], b[k])));
          xh[k] = fmul2(gn_of<SUB>(in.rs, k),
                        fma2(xh[k], gn_of<SUB>(m2, k), fsub2(fmul2(g[k], w[k]), gn_of<SUB>(m1, k))));
        }
        *reinterpret_cast<uint4*>(out) = gn_pack<T>(xh);
      }
      out += step;
    }
    grad.issue(batch);
    saved.issue(batch);
    cp_async_commit();
    batch = batch + 1 < kBackwardBatches ? batch + 1 : 0;
  }
}

template <typename T, int ACT, bool SRC8, int SUB>
__global__ void __launch_bounds__(kThreads, 3)
    gn_stream_grad_kernel(const T* __restrict__ dy, const void* __restrict__ src, const uint8_t* __restrict__ scales,
                          const void* __restrict__ weight, const void* __restrict__ bias, const float* __restrict__ mean,
                          const float* __restrict__ rstd, float2* __restrict__ part, float2* __restrict__ chan,
                          T* __restrict__ dx, const GnShape s, const GnStream q) {
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char* const ring = smem;
  float2* const fin = reinterpret_cast<float2*>(smem + kBackwardRing * (SRC8 ? 3 : 4) / 2);
  if (!q.early) begin_after_previous();
  unsigned work;
  if (second_pass(q, blockIdx.x, &work)) {
    const unsigned per = q.apply_tiles * q.apply_chunks, sample = work / per;
    grad_apply_cta<T, ACT, SRC8, SUB>(dy, src, scales, weight, bias, mean, rstd, part, dx, s, q, q.second_sample + sample,
                                      work - sample * per, fin, ring);
  } else {
    const unsigned per = q.tiles * q.chunks, sample = work / per;
    grad_sums_cta<T, ACT, SRC8, SUB>(dy, src, scales, weight, bias, mean, rstd, part, chan, s, q, q.first_sample + sample,
                                     work - sample * per, ring);
  }
}

// ---- host -----------------------------------------------------------------------------------------

static int gcd_int(int a, int b) { return b == 0 ? a : gcd_int(b, a % b); }

// Row chunks: `n`, with at least 8 pixels a thread.
static void stream_rows(long long P, int rl, long long n, int* rows, int* chunks) {
  const long long most = (P + 8LL * rl - 1) / (8LL * rl);
  n = n < most ? n : most;
  n = n < 1 ? 1 : n;
  *rows = static_cast<int>((P + n - 1) / n);
  *chunks = static_cast<int>((P + *rows - 1) / *rows);
}

bool gn_stream_plan(const GnShape& s, int bytes_per_value, GnStream* q) {
  const int whole = s.Cg / gcd_int(s.Cg, 8) * 8;  // the least channels of whole groups and whole vectors
  if (s.Cg % 8 == 0 && s.Cg > kLargeTile) {
    q->tile = kLargeTile;
    q->tiles_per_group = (s.Cg + kLargeTile - 1) / kLargeTile;
    q->entries_per_group = q->tiles_per_group;
    q->tiles = s.G * q->tiles_per_group;
  } else if (whole <= 2 * kLargeTile) {
    q->tile = whole * ((kSmallTile + whole - 1) / whole);
    if (q->tile > s.C) q->tile = s.C;
    q->tiles_per_group = q->entries_per_group = 1;
    q->tiles = (s.C + q->tile - 1) / q->tile;
  } else {
    q->tile = 2 * kSmallTile;
    q->tiles_per_group = 1;
    q->entries_per_group = s.Cg;
    q->tiles = (s.C + q->tile - 1) / q->tile;
  }
  q->entries = s.G * q->entries_per_group;
  q->sub = s.Cg % 8 == 0 ? 8 : s.Cg % 4 == 0 && q->entries_per_group == 1 ? 4 : 1;
  q->lanes = (q->tile + 7) / 8;
  q->lane_mul = 65536u / q->lanes + 1;  // exact for thread < 256
  q->rl = kThreads / q->lanes;
  // second pass: even tiles of whole checkpoint blocks (168 channels are 96 + 72, not 128 + 40)
  const int blocks = (s.C + kAct8Block - 1) / kAct8Block, most = kApplyLanes / 4;
  q->apply_tiles = (blocks + most - 1) / most;
  q->apply_lanes = (blocks + q->apply_tiles - 1) / q->apply_tiles * 4;
  q->apply_lane_mul = 65536u / q->apply_lanes + 1;
  q->apply_rl = kThreads / q->apply_lanes;
  q->apply_tiles = (s.C + q->apply_lanes * 8 - 1) / (q->apply_lanes * 8);
  const long long per_sample = s.P * s.C * bytes_per_value;
  long long samples = kGroupBytes / (per_sample > 0 ? per_sample : 1);
  samples = samples < 1 ? 1 : samples > s.B ? s.B : samples;
  const long long groups = (s.B + samples - 1) / samples;
  q->samples = static_cast<int>((s.B + groups - 1) / groups);
  // CTAs of a pass: about as many as run at once (3 an SM), long ones: more, shorter ones pay their ramp more often
  // (32x32x1536, B = 16, gradient: 67 us with 2 and 3 an SM, 70 with 3 and 5; forward 39 us with 3, 45 with 9).  Second
  // pass: at most 4 for every SM, of which 3 run at once, and as near to that as can be (56x56x128, B = 64, gradient from a
  // checkpoint: 83.7 us with 448 CTAs, 77.1 with 576; 32x32x1536, B = 8: 39.5 with 480, 37.2 with 576).  Neither pass
  // fills a whole number of turns: 512 and 576 CTAs are 1.15 and 1.3 of them at 32x32x1536, B = 16
  const long long a_chunk = static_cast<long long>(q->tiles) * q->samples, want = (bytes_per_value > 2 ? 2 : 3) * kSmCount;
  stream_rows(s.P, q->rl, (want + a_chunk - 1) / a_chunk, &q->rows, &q->chunks);
  stream_rows(s.P, q->apply_rl, 4 * kSmCount / (static_cast<long long>(q->apply_tiles) * q->samples), &q->apply_rows,
              &q->apply_chunks);
  q->first_sample = q->second_sample = 0;
  q->first_ctas = q->second_ctas = 0;
  q->early = 0;
  // CTAs of a launch: grid x
  const long long a = static_cast<long long>(q->tiles) * q->chunks * q->samples;
  const long long b = static_cast<long long>(q->apply_tiles) * q->apply_chunks * q->samples;
  return a + b <= 0x7fffffffLL;
}

// Launches: first pass of group 0; second pass of group i with the first pass of group i + 1.
template <typename Launch>
static int stream_groups(const GnShape& s, GnStream q, Launch launch) {
  for (int done = -q.samples; done < s.B; done += q.samples) {
    const int next = done + q.samples, left = s.B - next;
    const int second = done < 0 ? 0 : s.B - done < q.samples ? s.B - done : q.samples;
    const int first = left <= 0 ? 0 : left < q.samples ? left : q.samples;
    q.second_sample = done < 0 ? 0 : done;
    q.first_sample = next;
    q.early = done >= 0;
    q.second_ctas = static_cast<unsigned>(second) * q.apply_tiles * q.apply_chunks;
    q.first_ctas = static_cast<unsigned>(first) * q.tiles * q.chunks;
    const int rc = launch(q, dim3(q.first_ctas + q.second_ctas));
    if (rc != DWB_OK) return rc;
  }
  return DWB_OK;
}

static int stream_launch(const void* fn, const char* what, dim3 grid, int smem, void** args, cudaStream_t stream) {
  cudaError_t e = allow_large_cta(fn);
  if (e == cudaSuccess) e = launch_kernel(fn, grid, dim3(kThreads), args, smem, stream);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return record_cuda_failure(what, e);
  }
  return DWB_OK;
}

template <typename T, bool CKPT, int SUB>
static const void* stream_fn(int act) {
  switch (act) {
    case kActRelu: return reinterpret_cast<const void*>(&gn_stream_kernel<T, kActRelu, CKPT, SUB>);
    case kActGelu: return reinterpret_cast<const void*>(&gn_stream_kernel<T, kActGelu, CKPT, SUB>);
    case kActSilu: return reinterpret_cast<const void*>(&gn_stream_kernel<T, kActSilu, CKPT, SUB>);
    default: return reinterpret_cast<const void*>(&gn_stream_kernel<T, kActNone, CKPT, SUB>);
  }
}
template <typename T, bool SRC8, int SUB>
static const void* stream_grad_fn(int act) {
  switch (act) {
    case kActRelu: return reinterpret_cast<const void*>(&gn_stream_grad_kernel<T, kActRelu, SRC8, SUB>);
    case kActGelu: return reinterpret_cast<const void*>(&gn_stream_grad_kernel<T, kActGelu, SRC8, SUB>);
    case kActSilu: return reinterpret_cast<const void*>(&gn_stream_grad_kernel<T, kActSilu, SRC8, SUB>);
    default: return reinterpret_cast<const void*>(&gn_stream_grad_kernel<T, kActNone, SRC8, SUB>);
  }
}
template <typename T, bool CKPT>
static const void* stream_fn(int sub, int act) {
  return sub == 8 ? stream_fn<T, CKPT, 8>(act) : sub == 4 ? stream_fn<T, CKPT, 4>(act) : stream_fn<T, CKPT, 1>(act);
}
template <typename T, bool SRC8>
static const void* stream_grad_fn(int sub, int act) {
  return sub == 8   ? stream_grad_fn<T, SRC8, 8>(act)
         : sub == 4 ? stream_grad_fn<T, SRC8, 4>(act)
                    : stream_grad_fn<T, SRC8, 1>(act);
}

template <typename T>
int gn_stream_forward(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, void* codes,
                      void* scales, float2* part, const GnShape& shape, const GnStream& plan, int act, cudaStream_t stream) {
  const void* fn = codes ? stream_fn<T, true>(plan.sub, act) : stream_fn<T, false>(plan.sub, act);
  GnShape s = shape;
  static_assert(kFinBytes <= kThreads * static_cast<int>(sizeof(float2)), "the second pass in the first one's entries");
  const int smem = kForwardRing + kThreads * (8 / plan.sub) * static_cast<int>(sizeof(float2));
  return stream_groups(shape, plan, [&](GnStream q, dim3 grid) {
    void* args[] = {&x, &weight, &bias, &part, &y, &mean, &rstd, &codes, &scales, &s, &q};
    return stream_launch(fn, "gn_stream_kernel", grid, smem, args, stream);
  });
}

template <typename T>
int gn_stream_backward(const void* dy, const void* x, const void* codes, const void* scales, const float* mean,
                       const float* rstd, const void* weight, const void* bias, void* dx, float2* part, float2* chan,
                       const GnShape& shape, const GnStream& plan, int act, cudaStream_t stream) {
  const void* fn =
      codes ? stream_grad_fn<T, true>(plan.sub, act) : stream_grad_fn<T, false>(plan.sub, act);
  const void* src = codes ? codes : x;
  GnShape s = shape;
  const int smem = kBackwardRing * (codes ? 3 : 4) / 2 + kFinBytes;
  return stream_groups(shape, plan, [&](GnStream q, dim3 grid) {
    void* args[] = {&dy, &src, &scales, &weight, &bias, &mean, &rstd, &part, &chan, &dx, &s, &q};
    return stream_launch(fn, "gn_stream_grad_kernel", grid, smem, args, stream);
  });
}

#define DWB_GN_STREAM(T)                                                                                                  \
  template int gn_stream_forward<T>(const void*, const void*, const void*, void*, float*, float*, void*, void*, float2*, \
                                    const GnShape&, const GnStream&, int, cudaStream_t);                                 \
  template int gn_stream_backward<T>(const void*, const void*, const void*, const void*, const float*, const float*,     \
                                     const void*, const void*, void*, float2*, float2*, const GnShape&, const GnStream&, \
                                     int, cudaStream_t);
DWB_GN_STREAM(__half)
DWB_GN_STREAM(__nv_bfloat16)
#undef DWB_GN_STREAM

}  // namespace dwb
