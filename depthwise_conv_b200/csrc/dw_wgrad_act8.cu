// dw_wgrad_act8.cu -- the depthwise weight gradient from the 8-bit checkpoint of
// the convolution's input (dw_act8.cuh):
//   dw[kh][kw][c] = sum over b, h, w of dy[b][h][w][c] * x[b][h + kh - p][w + kw - p][c],  p = K / 2
//
// The K * K taps of a channel are a small matrix product.  For one row r of x
// and 16 columns w0..w0+15 take
//   A[kw][w] = x[r][w0 + w + kw - p]      (a Hankel matrix of one row of x)
//   B[w][j]  = dy[r + p - (K - 1) + j][w0 + w]  (16 columns of K rows of dy)
// then (A B)[kw][j] is what these columns add to dw[K - 1 - j][kw], and adding
// the products over rows, columns and images in the accumulator of the tensor
// core gives the gradient.  Both operands are exact in fp16 (a checkpoint's
// value is 8 bits times a power of two), so the only roundings are those of the
// fp32 accumulator.  On the CUDA cores the same sum is bound by fp32 FMAs, two
// FLOPs a lane; a 16 x 8 x 16 product does 2048 multiplications a warp
// instruction, of which a 7 x 7 kernel uses 49 / 64, 9 x 9 32%, 31 x 31 94%.
// The warp-level product is the right size: the fifth-generation product takes
// 64 rows or more of one matrix from shared memory in 16-byte rows, where a
// Hankel matrix of one channel has 7 to 31 rows, each one element (2 bytes)
// further than the last.
//
// Tile shapes, by K (one x row gives MT x NT products of 16 taps kw x 8 rows j):
//   K <= 7:   the 16 rows of A are 8 taps of TWO x rows; rows r and r + 1 meet
//             the same 8 rows of dy, so one product serves both;
//   K <= 15:  one 16-row A for each of two x rows against the same 16 rows of dy
//             (each loaded B fragment serves two products);
//   K <= 31:  two A tiles (32 taps) of one x row, 3 or 4 B tiles.
//
// One CTA = 32 channels (one block of the checkpoint) x a tile of columns x a
// range of rows.  A row of x (converted to fp16, transposed to channel-major) is
// kept twice, the second time one element further, so that the pairs (w, w + 1)
// of odd taps are aligned words too; the rows of dy stand in a ring.  A warp owns
// 4 channels and keeps their taps in the accumulators.  While it multiplies, the
// next rows travel from global memory into registers.  Partial sums go to slices
// of the workspace that a second kernel adds in order; a chain of accumulations
// is at most kChain products long, because the tensor core's accumulator rounds
// towards zero, which a long chain would turn into a bias.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/dwconv_b200.h"
#include "dw_act8.cuh"
#include "dw_host.h"
#include "dw_launch.h"

namespace dwb {

constexpr int kWgThreads = 256;
constexpr int kWgChannels = 32;
constexpr int kWgTile = 64;    // most columns of a tile
constexpr int kChain = 128;    // most products added up in one accumulator

struct Wgrad8Params {
  int B, H, W, C, K;
  int tw;           // columns of dy a tile holds (a multiple of 16)
  int col_tiles;
  int units;        // B * ceil(H / ROWS) steps of ROWS rows of x
  int unit_rows;    // ceil(H / ROWS)
  int per_chunk;    // units a CTA takes
  int chunks;
  int xp, dp;       // words of a channel's row of x (one copy) and of dy, both odd
  int ring;         // rows of dy kept
};

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 codes of one pixel as fp16 pairs, exactly.  Byte u = q + 128 under 0x64 is the half 1024 + u.
__device__ __forceinline__ void codes_to_half(const uint2& q, uint32_t E, uint32_t (&out)[4]) {
  const __half2 off = __half2half2(__ushort_as_half(0xe480));  // -1152
  const __half2 step = __float2half2_rn(act8_step(E));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (i < 2 ? q.x : q.y) ^ 0x80808080u;
    const uint32_t u = __byte_perm(w, 0x64646464u, (i & 1) ? 0x4342 : 0x4140);
    const __half2 h = __hmul2(__hadd2(*reinterpret_cast<const __half2*>(&u), off), step);
    out[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Five neighbouring pixels' codes: four columns of the tile and the one behind them.
struct XItem {
  uint2 q[5];
  uint8_t e[5];
};

// MT x NT: 16-tap by 8-row products of one x row; ROWS: x rows a step; PACK: both rows in one product.
template <int MT, int NT, int ROWS, bool PACK>
struct Wgrad8 {
  const Wgrad8Params& p;
  const int8_t* codes;
  const uint8_t* scales;
  const __half* dy;
  uint32_t* xs;   // [2 buffers][ROWS][2 copies][32 channels][xp] (+16 words a copy: the copies' banks differ)
  uint32_t* ds;   // [ring][32 channels][dp] (+4 words a row: 8 rows x 4 words fall in 32 banks)
  int c0, w0, sblocks;

  __device__ __forceinline__ int copy_words() const { return kWgChannels * p.xp + 16; }
  __device__ __forceinline__ int row_words() const { return kWgChannels * p.dp + 4; }
  __device__ __forceinline__ int x_items() const { return ((p.tw + p.K - 1 + 3) / 4) * 4; }  // of one row
  __device__ __forceinline__ int dy_items() const { return p.tw * 2; }                        // of one row

  __device__ __forceinline__ void load_x(XItem& it, int b, int row, int item) const {
    const int c = c0 + (item & 3) * 8, col = w0 - p.K / 2 + (item >> 2) * 4;
    const bool on = row < p.H && c < p.C;
    const long long line = (static_cast<long long>(b) * p.H + row) * p.W;
#pragma unroll
    for (int j = 0; j < 5; ++j) {
      const bool in = on && col + j >= 0 && col + j < p.W;
      it.q[j] = in ? *reinterpret_cast<const uint2*>(codes + (line + col + j) * p.C + c) : make_uint2(0u, 0u);
      it.e[j] = in ? scales[(line + col + j) * sblocks + c / kAct8Block] : static_cast<uint8_t>(127);
    }
  }
  // even copy: words (4i, 4i+1), (4i+2, 4i+3); odd copy: (4i+1, 4i+2), (4i+3, 4i+4)
  __device__ __forceinline__ void store_x(const XItem& it, int buffer, int r, int item) const {
    uint32_t h[5][4];
#pragma unroll
    for (int j = 0; j < 5; ++j) codes_to_half(it.q[j], it.e[j], h[j]);
    uint32_t* even = xs + (buffer * ROWS + r) * 2 * copy_words() + (item & 3) * 8 * p.xp + (item >> 2) * 2;
    uint32_t* odd = even + copy_words();
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t sel = (k & 1) ? 0x7632 : 0x5410;
      even[k * p.xp] = __byte_perm(h[0][k / 2], h[1][k / 2], sel);
      even[k * p.xp + 1] = __byte_perm(h[2][k / 2], h[3][k / 2], sel);
      odd[k * p.xp] = __byte_perm(h[1][k / 2], h[2][k / 2], sel);
      odd[k * p.xp + 1] = __byte_perm(h[3][k / 2], h[4][k / 2], sel);
    }
  }
  __device__ __forceinline__ void load_dy(uint4 (&v)[2], int b, int row, int item) const {
    const int c = c0 + (item & 3) * 8, col = w0 + (item >> 2) * 2;
    const bool on = row >= 0 && row < p.H && c < p.C;
    const long long line = (static_cast<long long>(b) * p.H + row) * p.W;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      v[j] = on && col + j < p.W ? *reinterpret_cast<const uint4*>(dy + (line + col + j) * p.C + c)
                                 : make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void store_dy(const uint4 (&v)[2], int slot, int item) const {
    uint32_t* at = ds + slot * row_words() + (item & 3) * 8 * p.dp + (item >> 2);
    const uint32_t a[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, b[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
    for (int k = 0; k < 8; ++k) at[k * p.dp] = __byte_perm(a[k / 2], b[k / 2], (k & 1) ? 0x7632 : 0x5410);
  }

  // One step: ROWS rows of x in `buffer` against the ring rows first, first + 1, ...
  __device__ __forceinline__ void multiply(float (&acc)[4][PACK ? 1 : ROWS][MT][NT][4], int buffer, int first) const {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t* xa = xs + buffer * ROWS * 2 * copy_words() + (g & 1) * copy_words() + warp * 4 * p.xp + (g >> 1) + t;
    const int used = p.K - 1 + ROWS;
    const uint32_t* db[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int j = n * 8 + g < used ? n * 8 + g : 0;  // rows past the last one feed columns that nothing reads
      const int slot = first + j < p.ring ? first + j : first + j - p.ring;
      db[n] = ds + slot * row_words() + warp * 4 * p.dp + t;
    }
    const int blocks = p.tw / 16;
#pragma unroll
    for (int ch = 0; ch < 4; ++ch) {
      const uint32_t* x0 = xa + ch * p.xp;
      if constexpr (PACK) {
        const uint32_t* x1 = x0 + 2 * copy_words();
#pragma unroll 4
        for (int w = 0; w < blocks; ++w)
          mma_16816(acc[ch][0][0][0], x0[w * 8], x1[w * 8], x0[w * 8 + 4], x1[w * 8 + 4], db[0][ch * p.dp + w * 8],
                    db[0][ch * p.dp + w * 8 + 4]);
      } else {
        // a row's words 8 columns apart: A tile m of a block needs words 2m, 2m + 1, 2m + 1, 2m + 2
        uint32_t a[ROWS][2 * MT + 1];
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
          for (int i = 0; i < 2 * MT - 1; ++i) a[r][i + 2] = x0[r * 2 * copy_words() + i * 4];
#pragma unroll 2
        for (int w = 0; w < blocks; ++w) {
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {  // 16 columns on: all words but two are the last block's
#pragma unroll
            for (int i = 0; i < 2 * MT - 1; ++i) a[r][i] = a[r][i + 2];
            a[r][2 * MT - 1] = x0[r * 2 * copy_words() + w * 8 + (2 * MT - 1) * 4];
            a[r][2 * MT] = x0[r * 2 * copy_words() + w * 8 + 2 * MT * 4];
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint32_t b0 = db[n][ch * p.dp + w * 8], b1 = db[n][ch * p.dp + w * 8 + 4];
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
#pragma unroll
              for (int m = 0; m < MT; ++m)
                mma_16816(acc[ch][r][m][n], a[r][2 * m], a[r][2 * m + 1], a[r][2 * m + 1], a[r][2 * m + 2], b0, b1);
          }
        }
      }
    }
  }

  // Row j of dy and row r of x belong to kh = K - 1 - j + r: the two rows' columns j and j + 1 are added.
  __device__ __forceinline__ void write(float (&acc)[4][PACK ? 1 : ROWS][MT][NT][4], float* slice) const {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int c = c0 + warp * 4;
    if (c >= p.C) return;
    auto put = [&](int kh, int kw, float v0, float v1, float v2, float v3) {
      if (kh >= 0 && kh < p.K && kw < p.K)
        *reinterpret_cast<float4*>(slice + (static_cast<long long>(kh) * p.K + kw) * p.C + c) = make_float4(v0, v1, v2, v3);
    };
    if constexpr (PACK) {
      float lo[4], hi[4];
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        float(&d)[4] = acc[ch][0][0][0];
        lo[ch] = d[0] + d[3];
        hi[ch] = d[1] + __shfl_down_sync(0xffffffffu, d[2], 1);  // column 2t + 2; past the last one kh < 0
      }
      put(p.K - 1 - 2 * t, g, lo[0], lo[1], lo[2], lo[3]);
      put(p.K - 2 - 2 * t, g, hi[0], hi[1], hi[2], hi[3]);
    } else {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float lo[4], hi[4];
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) {
              lo[ch] = acc[ch][0][m][n][half * 2];
              hi[ch] = acc[ch][0][m][n][half * 2 + 1];
              if constexpr (ROWS == 2) {
                lo[ch] += acc[ch][1][m][n][half * 2 + 1];
                // column 2t + 2 of row 1: the next lane's first, or the next tile's
                const float mine = acc[ch][1][m][n][half * 2];
                const float next = n + 1 < NT ? acc[ch][1][m][n + 1 < NT ? n + 1 : n][half * 2] : 0.0f;
                const float from = __shfl_sync(0xffffffffu, t == 0 ? next : mine, (lane & ~3) | ((t + 1) & 3));
                hi[ch] += from;
              }
            }
            const int j = n * 8 + 2 * t, kw = m * 16 + half * 8 + g;
            put(p.K - 1 - j, kw, lo[0], lo[1], lo[2], lo[3]);
            put(p.K - 2 - j, kw, hi[0], hi[1], hi[2], hi[3]);
          }
    }
  }
};

template <int MT, int NT, int ROWS, bool PACK>
__global__ void __launch_bounds__(kWgThreads) wgrad8_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                            const __half* __restrict__ dy, float* __restrict__ part,
                                                            const Wgrad8Params p) {
  extern __shared__ __align__(16) uint32_t smem[];
  griddep_wait();
  griddep_launch_dependents();
  Wgrad8<MT, NT, ROWS, PACK> k{p, codes, scales, dy, smem, nullptr, 0, 0, 0};
  k.ds = smem + 2 * ROWS * 2 * k.copy_words();
  k.c0 = blockIdx.x * kWgChannels;
  k.w0 = static_cast<int>(blockIdx.z) * p.tw;
  k.sblocks = (p.C + kAct8Block - 1) / kAct8Block;
  const int pad = p.K / 2, used = p.K - 1 + ROWS, tid = threadIdx.x;
  const int xi = k.x_items(), di = k.dy_items();
  float acc[4][PACK ? 1 : ROWS][MT][NT][4];
#pragma unroll
  for (int ch = 0; ch < 4; ++ch)
#pragma unroll
    for (int r = 0; r < (PACK ? 1 : ROWS); ++r)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[ch][r][m][n][i] = 0.0f;

  const int u1 = min(p.units, static_cast<int>(blockIdx.y + 1) * p.per_chunk);
  int u = blockIdx.y * p.per_chunk;
  while (u < u1) {  // one image's part of the range at a time
    const int b = u / p.unit_rows;
    const int s0 = u - b * p.unit_rows, steps = min(p.unit_rows - s0, u1 - u);
    const int top = s0 * ROWS + pad - (p.K - 1);  // first row of dy that the first row of x meets
    __syncthreads();                              // the last image's rows have been read
    for (int i = tid; i < used * di; i += kWgThreads) {
      uint4 v[2];
      const int r = i / di;
      k.load_dy(v, b, top + r, i - r * di);
      k.store_dy(v, r, i - r * di);
    }
    if (tid < ROWS * xi) {
      XItem it;
      const int r = tid / xi;
      k.load_x(it, b, s0 * ROWS + r, tid - r * xi);
      k.store_x(it, 0, r, tid - r * xi);
    }
    __syncthreads();
    int first = 0;  // ring slot of the row of dy with j = 0
    for (int s = 0; s < steps; ++s) {
      const bool more = s + 1 < steps;
      XItem it;
      uint4 v[2];
      const int xr = tid / xi, dr = tid / di;
      const bool get_x = more && xr < ROWS, get_dy = more && dr < ROWS;
      if (get_x) k.load_x(it, b, (s0 + s + 1) * ROWS + xr, tid - xr * xi);
      if (get_dy) k.load_dy(v, b, top + s * ROWS + used + dr, tid - dr * di);
      k.multiply(acc, s & 1, first);
      if (get_x) k.store_x(it, (s + 1) & 1, xr, tid - xr * xi);
      if (get_dy) {
        // the ring has ROWS rows more than a step reads: these slots belong to no row of this step
        int slot = first + used + dr;
        slot -= slot >= p.ring ? p.ring : 0;
        k.store_dy(v, slot, tid - dr * di);
      }
      first += ROWS;
      first -= first >= p.ring ? p.ring : 0;
      __syncthreads();
    }
    u += steps;
  }
  const long long slice = static_cast<long long>(blockIdx.z) * p.chunks + blockIdx.y;
  k.write(acc, part + slice * p.K * p.K * p.C);
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

// The kernel for K, with its rows a step.
static const void* wgrad8_fn(int K) {
  if (K <= 7) return reinterpret_cast<const void*>(&wgrad8_kernel<1, 1, 2, true>);
  if (K <= 15) return reinterpret_cast<const void*>(&wgrad8_kernel<1, 2, 2, false>);
  if (K <= 23) return reinterpret_cast<const void*>(&wgrad8_kernel<2, 3, 1, false>);
  return reinterpret_cast<const void*>(&wgrad8_kernel<2, 4, 1, false>);
}
static int wgrad8_rows(int K) { return K <= 15 ? 2 : 1; }

static int wgrad8_smem(const Wgrad8Params& p) {
  return 4 * (2 * wgrad8_rows(p.K) * 2 * (kWgChannels * p.xp + 16) + p.ring * (kWgChannels * p.dp + 4));
}

static int wgrad8_plan(int64_t B, int64_t H, int64_t W, int64_t C, int K, Wgrad8Params* p) {
  if (K < 1 || K > 31 || (K % 2) == 0 || B < 0 || H < 1 || W < 1 || C < 8 || (C % 8) != 0) return DWB_ERR_BAD_SHAPE;
  if (B > (1 << 30) || H > (1 << 24) || W > (1 << 21) || C > (1 << 20) || B * H > (1LL << 30)) return DWB_ERR_BAD_SHAPE;
  const int rows = wgrad8_rows(K);
  p->B = static_cast<int>(B);
  p->H = static_cast<int>(H);
  p->W = static_cast<int>(W);
  p->C = static_cast<int>(C);
  p->K = K;
  p->col_tiles = (p->W + kWgTile - 1) / kWgTile;
  p->tw = ((p->W + p->col_tiles - 1) / p->col_tiles + 15) / 16 * 16;  // even tiles: W = 65 is 48 + 17, not 64 + 1
  p->col_tiles = (p->W + p->tw - 1) / p->tw;
  p->unit_rows = (p->H + rows - 1) / rows;
  p->units = p->B * p->unit_rows;
  p->xp = (p->tw + (K <= 7 ? 8 : K <= 15 ? 16 : 32)) / 2 | 1;
  p->dp = (p->tw / 2) | 1;
  p->ring = K - 1 + 2 * rows;
  // a chain of at most kChain products, and CTAs for every SM, but not ranges shorter than the rows of dy
  // that a range has to bring in before its first product
  const long long base = (C + kWgChannels - 1) / kWgChannels * p->col_tiles;
  long long per = (static_cast<long long>(p->units) * base + 2LL * kSmCount - 1) / (2LL * kSmCount);
  const long long least = (K - 1) / (2 * rows) > 1 ? (K - 1) / (2 * rows) : 1, most = kChain / (p->tw / 16);
  per = per < least ? least : per;
  per = per > most ? most : per;
  p->per_chunk = static_cast<int>(per);
  p->chunks = (p->units + p->per_chunk - 1) / p->per_chunk;
  if (p->chunks < 1) p->chunks = 1;
  if (p->chunks > 65535 || p->col_tiles > 65535) return DWB_ERR_BAD_SHAPE;
  return DWB_OK;
}

// The partial sums: one [K][K][C] slice for every range of rows and tile of columns.
static int64_t wgrad8_workspace(const Wgrad8Params& p) {
  return static_cast<int64_t>(p.chunks) * p.col_tiles * p.K * p.K * p.C * static_cast<int64_t>(sizeof(float));
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
  const void* fn = wgrad8_fn(K);
  const int smem = wgrad8_smem(p);
  cudaError_t e = allow_large_cta(fn);
  if (e == cudaSuccess)
    e = launch_kernel(fn, dim3(static_cast<unsigned>((C + kWgChannels - 1) / kWgChannels), p.chunks, p.col_tiles),
                      dim3(kWgThreads), a1, smem, st);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return record_cuda_failure("wgrad8_kernel", e);
  }
  long long n4 = static_cast<long long>(K) * K * C / 4;
  int slices = p.chunks * p.col_tiles;
  void* a2[] = {&part, &dw, &n4, &slices};
  e = launch_kernel(reinterpret_cast<const void*>(&wgrad8_reduce_kernel), dim3(static_cast<unsigned>((n4 + 255) / 256)),
                    dim3(256), a2, 0, st);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return record_cuda_failure("wgrad8_reduce_kernel", e);
  }
  return DWB_OK;
}
