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
// 4 channels and keeps their taps in the accumulators.  The codes and values of
// the next two steps travel by cp.async into places that only their own thread
// reads, so a step has one barrier.  A CTA's sums go to its slice of the workspace,
// and a second kernel adds the slices in order.  A chain of accumulations is at
// most kChain products long, because the tensor core's accumulator rounds towards
// zero, which a long chain would turn into a bias: then the accumulators are added
// to the slice and begin again at zero, so that the slices are as many as the CTAs,
// however long the batch.
//
// Measured (both kernels; the framework's 16-bit weight gradient on the CUDA
// cores in brackets): 16x32x32x768 k7 36.7 us (64.3), 16x32x32x1536 k9 80.6 (182),
// 8x56x56x1024 k13 112 (310), 8x56x56x128 k31 43 (171), 2x14x14x512 k27 11.7,
// 56x56x1024 k31 242 with 8 images, 1701 with 64 (286 and 1908 when a chain's end was
// a range's: 112 slices, 441 MB of workspace for the 64 images, where 9 are 35 MB).
// What bounds it for small K is latency at two CTAs of 8 warps an SM (one at 64
// columns from K = 9 on): at 16x32x32x768 k7 the issue slots are used 43% of the
// time and the tensor pipe 9%, and warps wait for a step's barrier, the
// shared-memory queue and the copies that a step converts and transposes; the 38 MB
// read need 5.8 us and the products' FMAs on the CUDA cores would need 14.8.  At
// K = 31 the tensor pipe is active 54% of the time.  Items of 4 channels, which
// spread a row over twice the threads, were slower; so was one step of read-ahead.
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
constexpr int kTurns = 12;     // most turns of the CTAs that run at once
constexpr int kFlushes = 256;  // most additions to a slice

struct Wgrad8Params {
  int B, H, W, C, K;
  int tw;           // columns of dy a tile holds (16, 32, 48 or 64)
  int col_tiles;
  int units;        // B * unit_rows steps
  int unit_rows;    // ceil(H / rows of x a step)
  int per_chunk;    // steps a CTA takes
  int chunks;
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

constexpr int kAhead = 2;      // steps that global memory is read ahead

// The exponent bytes of five neighbouring pixels: four columns of the tile and the one behind them.
struct XScales {
  uint8_t e[5];
};

// Asynchronous copies, of zeros where `on` is false (nothing is read then).
__device__ __forceinline__ void copy8(void* dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(on ? 8 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy16(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}

constexpr int up_to(int v, int to, int mod) { return v % mod == to % mod ? v : up_to(v + 1, to, mod); }
constexpr int smaller(int a, int b) { return a < b ? a : b; }

// MT x NT: 16-tap by 8-row products of one x row; ROWS: x rows that meet the same rows of dy at once; PACK: both in one
// product; TW: columns; SETS: sets of ROWS rows a step (narrow tiles: a barrier for more work, and items for more
// threads).
//
// Shared memory, in words of two columns: x [2 buffers][kStep rows][2 copies][32 channels][XP], dy [ring][32 channels][DP].
// In x, channel 8 v + k has place 4 k + v and XP is 8 or 24 modulo 32; in dy, places are channels and DP is odd: the
// stores of a warp (4 vectors of 8 channels times 8 column pairs of x, or 8 words of dy) fall in 32 banks.  The copies
// are 16 banks apart and the rows of dy 4, so that a fragment's 32 words do too.  Behind them, for each step read
// ahead, the codes and values that a thread has under way: each in places of its own, which need no barrier.
template <int MT, int NT, int ROWS, bool PACK, int TW, int SETS>
struct Wgrad8 {
  static constexpr int kStep = SETS * ROWS;  // rows of x a step
  static constexpr int kXWords = (TW + (PACK ? 8 : 16 * MT)) / 2, kDWords = TW / 2;
  static constexpr int XP = smaller(up_to(kXWords, 8, 32), up_to(kXWords, 24, 32));
  static constexpr int DP = kDWords | 1;
  static constexpr int kCopy = kWgChannels * XP + 16, kXRow = 2 * kCopy, kXBuffer = kStep * kXRow;
  static constexpr int kDRow = kWgChannels * DP + 4;
  static constexpr int kDItems = TW * 2;  // of a row of dy: 2 columns x 8 channels
  static constexpr int kBlocks = TW / 16;
  static constexpr int kAcc = PACK ? 1 : ROWS;
  static constexpr int kMost = kChain / (kBlocks * SETS);  // steps of a chain
  static constexpr int kTaps = PACK ? 8 : 16, kSumPitch = kWgChannels + 4;  // of the sums in shared memory
  typedef float Acc[4][kAcc][MT][NT][4];
  static __device__ __forceinline__ void clear(Acc& acc) {
#pragma unroll
    for (int ch = 0; ch < 4; ++ch)
#pragma unroll
      for (int r = 0; r < kAcc; ++r)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[ch][r][m][n][i] = 0.0f;
  }

  static constexpr int ring(int K) { return K - 1 + 2 * kStep; }
  static constexpr int x_items(int K) { return (TW + K - 1 + 3) / 4 * 4; }  // of a row of x
  static constexpr int fixed_words(int K) { return (2 * kXBuffer + ring(K) * kDRow + 3) / 4 * 4; }
  static constexpr int smem(int K) {
    const int rows = 4 * fixed_words(K) + kAhead * kStep * (x_items(K) * 5 * 8 + kDItems * 2 * 16);
    const int sums = 4 * K * kTaps * kSumPitch;
    return rows > sums ? rows : sums;
  }

  // even copy: words (4i, 4i + 1), (4i + 2, 4i + 3); odd copy: (4i + 1, 4i + 2), (4i + 3, 4i + 4)
  static __device__ __forceinline__ void store_x(const uint2 (&q)[5], const XScales& s, uint32_t* row, int item) {
    uint32_t h[5][4];
#pragma unroll
    for (int j = 0; j < 5; ++j) codes_to_half(q[j], s.e[j], h[j]);
    uint32_t* even = row + (item & 3) * XP + (item >> 2) * 2;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t sel = (k & 1) ? 0x7632 : 0x5410;
      *reinterpret_cast<uint2*>(even + k * 4 * XP) =
          make_uint2(__byte_perm(h[0][k / 2], h[1][k / 2], sel), __byte_perm(h[2][k / 2], h[3][k / 2], sel));
      *reinterpret_cast<uint2*>(even + kCopy + k * 4 * XP) =
          make_uint2(__byte_perm(h[1][k / 2], h[2][k / 2], sel), __byte_perm(h[3][k / 2], h[4][k / 2], sel));
    }
  }
  static __device__ __forceinline__ void store_dy(const uint4 (&v)[2], uint32_t* row, int item) {
    uint32_t* at = row + (item & 3) * 8 * DP + (item >> 2);
    const uint32_t a[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, b[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
    for (int k = 0; k < 8; ++k) at[k * DP] = __byte_perm(a[k / 2], b[k / 2], (k & 1) ? 0x7632 : 0x5410);
  }

  // Place in x of this warp's first channel (4 * warp); its channels are 4 places apart.
  static __device__ __forceinline__ int warp_place() {
    const int warp = threadIdx.x >> 5;
    return (warp & 1) * 16 + (warp >> 1);
  }

  // One set: ROWS rows of x at `xs` against the ring rows first, first + 1, ...
  static __device__ __forceinline__ void multiply(Acc& acc, const uint32_t* xs, const uint32_t* ds, int first, int K) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t* xa = xs + (g & 1) * kCopy + warp_place() * XP + (g >> 1) + t;
    const int used = K - 1 + ROWS;
    const uint32_t* db[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int j = n * 8 + g < used ? n * 8 + g : 0;  // rows past the last one feed columns that nothing reads
      const int slot = first + j < ring(K) ? first + j : first + j - ring(K);
      db[n] = ds + slot * kDRow + static_cast<int>(threadIdx.x >> 5) * 4 * DP + t;
    }
#pragma unroll
    for (int ch = 0; ch < 4; ++ch) {
      const uint32_t* x0 = xa + ch * 4 * XP;
      if constexpr (PACK) {
#pragma unroll
        for (int w = 0; w < kBlocks; ++w)
          mma_16816(acc[ch][0][0][0], x0[w * 8], x0[kXRow + w * 8], x0[w * 8 + 4], x0[kXRow + w * 8 + 4],
                    db[0][ch * DP + w * 8], db[0][ch * DP + w * 8 + 4]);
      } else {
        // a row's words 8 columns apart: A tile m of a block needs words 2m, 2m + 1, 2m + 1, 2m + 2
        uint32_t a[ROWS][2 * MT + 1];
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
          for (int i = 0; i < 2 * MT - 1; ++i) a[r][i + 2] = x0[r * kXRow + i * 4];
#pragma unroll
        for (int w = 0; w < kBlocks; ++w) {
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {  // 16 columns on: all words but two are the last block's
#pragma unroll
            for (int i = 0; i < 2 * MT - 1; ++i) a[r][i] = a[r][i + 2];
            a[r][2 * MT - 1] = x0[r * kXRow + w * 8 + (2 * MT - 1) * 4];
            a[r][2 * MT] = x0[r * kXRow + w * 8 + 2 * MT * 4];
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint32_t b0 = db[n][ch * DP + w * 8], b1 = db[n][ch * DP + w * 8 + 4];
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

  // f(j, kw, v) with what this lane has of dw[K - 1 - j][m * kTaps + kw] in the warp's channel ch: row j of dy and row
  // r of x belong to kh = K - 1 - j + r, so the two rows' columns j and j + 1 are added.
  template <typename F>
  static __device__ __forceinline__ void each_sum(Acc& acc, int m, int n, int half, int ch, F f) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if constexpr (PACK) {
      float(&d)[4] = acc[ch][0][0][0];
      f(2 * t, g, d[0] + d[3]);
      f(2 * t + 1, g, d[1] + __shfl_down_sync(0xffffffffu, d[2], 1));  // column 2t + 2; past the last one j >= K
    } else {
      float lo = acc[ch][0][m][n][half * 2], hi = acc[ch][0][m][n][half * 2 + 1];
      if constexpr (ROWS == 2) {
        lo += acc[ch][1][m][n][half * 2 + 1];
        // column 2t + 2 of row 1: the next lane's first, or the next tile's
        const float own = acc[ch][1][m][n][half * 2];
        const float next = n + 1 < NT ? acc[ch][1][m][n + 1 < NT ? n + 1 : n][half * 2] : 0.0f;
        hi += __shfl_sync(0xffffffffu, t == 0 ? next : own, (lane & ~3) | ((t + 1) & 3));
      }
      f(n * 8 + 2 * t, half * 8 + g, lo);
      f(n * 8 + 2 * t + 1, half * 8 + g, hi);
    }
  }
  static constexpr int kHalves = PACK ? 1 : 2;

  // The slice of a range that is one chain, from the accumulators.  c: this warp's first channel.
  static __device__ __forceinline__ void write(Acc& acc, float* slice, int c, int C, int K) {
    if (c >= C) return;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int half = 0; half < kHalves; ++half) {
          float lo[4], hi[4];
          int j = 0, kw = 0;
#pragma unroll
          for (int ch = 0; ch < 4; ++ch)
            each_sum(acc, m, n, half, ch, [&](int row, int tap, float v) {
              if (row & 1) hi[ch] = v;
              else lo[ch] = v;
              j = row & ~1;
              kw = m * kTaps + tap;
            });
          auto put = [&](int kh, const float(&v)[4]) {
            if (kh >= 0 && kw < K)
              *reinterpret_cast<float4*>(slice + (static_cast<long long>(kh) * K + kw) * C + c) = make_float4(v[0], v[1], v[2], v[3]);
          };
          put(K - 1 - j, lo);
          put(K - 2 - j, hi);
        }
  }

  // The same where a range has several chains: `again` adds to what this thread has put there before.  No other thread
  // writes to these places and a thread's operations on one place keep their order, so the sums are the same bits on
  // every run.  The sums go through shared memory (`buf`, the place of x and dy between two images or pieces of one:
  // [K][kTaps][kSumPitch]), since this is inside the loop: written from the accumulators, 4 channels at a time, they
  // would take 60 registers more than there are at K > 23.  A lane's four channels are turned by t, which spreads a
  // warp's stores over all banks.
  static __device__ __forceinline__ void add(Acc& acc, float* buf, float* slice, int c0, int C, int K, bool again) {
    const int t = threadIdx.x & 3;
    float* const mine = buf + (threadIdx.x >> 5) * 4;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int ch = 0; ch < 4; ++ch)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int half = 0; half < kHalves; ++half)
            each_sum(acc, m, n, half, ch, [&](int j, int kw, float v) {
              if (j < K) mine[((K - 1 - j) * kTaps + kw) * kSumPitch + ((ch + t) & 3)] = v;
            });
      __syncthreads();
      const int quad = threadIdx.x & 7, c = c0 + quad * 4;
      for (int at = threadIdx.x >> 3; at < K * kTaps; at += kWgThreads / 8) {
        const int kh = at / kTaps, kw = m * kTaps + at % kTaps, turn = (K - 1 - kh) >> 1;
        float4 v = *reinterpret_cast<const float4*>(buf + at * kSumPitch + quad * 4);
        if (turn & 1) v = make_float4(v.y, v.z, v.w, v.x);
        if (turn & 2) v = make_float4(v.z, v.w, v.x, v.y);
        if (kw >= K || c >= C) continue;
        float* const to = slice + (static_cast<long long>(kh) * K + kw) * C + c;
        if (again)
          asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
        else
          *reinterpret_cast<float4*>(to) = v;
      }
      if (m + 1 < MT) __syncthreads();
    }
  }
};

template <int MT, bool PACK>
constexpr int kWgCtas = PACK ? 3 : MT == 1 ? 2 : 1;

// LONG: ranges of several chains.  A kernel of its own, because what it needs for them costs small calls time (2x2x16 k9,
// B = 8: 5.3 us, 6.0 with it; 1x64x16 k29, B = 7: 10.4 and 12.4); large ones it serves better than ranges that end where
// a chain does (28x28x256 k29, B = 64: 158 us with those, 124 so).
template <int MT, int NT, int ROWS, bool PACK, int TW, int SETS, bool LONG>
__global__ void __launch_bounds__(kWgThreads, kWgCtas<MT, PACK>) wgrad8_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                            const __half* __restrict__ dy, float* __restrict__ part,
                                                            const Wgrad8Params p) {
  using S = Wgrad8<MT, NT, ROWS, PACK, TW, SETS>;
  constexpr int kStep = S::kStep;
  extern __shared__ __align__(16) uint32_t smem[];
  uint32_t* const xs = smem;
  uint32_t* const ds = smem + 2 * S::kXBuffer;
  griddep_wait();
  griddep_launch_dependents();
  const int c0 = blockIdx.x * kWgChannels, w0 = static_cast<int>(blockIdx.z) * TW, tid = threadIdx.x;
  const int sblocks = (p.C + kAct8Block - 1) / kAct8Block, pad = p.K / 2, used = p.K - 1 + kStep, ring = S::ring(p.K);

  // What this thread brings in at every step, a row further each time: one item of x (columns x_col .. x_col + 4, of
  // row x_row of the step's) and one of dy (2 columns of row d_row).
  const int x_items = S::x_items(p.K);
  const int x_row = tid / x_items, x_item = tid - x_row * x_items;
  const int x_c = c0 + (x_item & 3) * 8, x_col = w0 - pad + (x_item >> 2) * 4;
  unsigned x_mask = 0;
#pragma unroll
  for (int j = 0; j < 5; ++j)
    if (x_row < kStep && x_c < p.C && x_col + j >= 0 && x_col + j < p.W) x_mask |= 1u << j;
  // the last warps begin with dy, so that those that convert codes have none of it where the tile is narrow
  const int d_tid = kWgThreads - 1 - tid, d_row = d_tid / S::kDItems, d_item = d_tid - d_row * S::kDItems;
  const int d_c = c0 + (d_item & 3) * 8, d_col = w0 + (d_item >> 2) * 2;
  unsigned d_mask = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (d_row < kStep && d_c < p.C && d_col + j < p.W) d_mask |= 1u << j;
  const long long line = static_cast<long long>(p.W) * p.C, s_line = static_cast<long long>(p.W) * sblocks;
  unsigned char* const raw = reinterpret_cast<unsigned char*>(smem + S::fixed_words(p.K));
  uint2* const x_raw = reinterpret_cast<uint2*>(raw) + tid;                                              // [kAhead][5][items]
  uint4* const d_raw = reinterpret_cast<uint4*>(raw + kAhead * kStep * x_items * 5 * 8) + d_tid;           // [kAhead][2][items]
  const int x_many = kStep * x_items, d_many = kStep * S::kDItems;

  // A row past the image: codes of 0, whatever the step.
  auto load_scales = [&](XScales& s, const uint8_t* e, bool on) {
#pragma unroll
    for (int j = 0; j < 5; ++j) s.e[j] = on && (x_mask >> j & 1) ? e[j * sblocks] : static_cast<uint8_t>(127);
  };
  auto fetch = [&](int place, const int8_t* q, bool x_on, const __half* d, bool d_on) {
    if (x_row < kStep) {
#pragma unroll
      for (int j = 0; j < 5; ++j) {
        const bool on = x_on && (x_mask >> j & 1);
        copy8(x_raw + (place * 5 + j) * x_many, on ? q + j * p.C : codes, on);
      }
    }
    if (d_row < kStep) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bool on = d_on && (d_mask >> j & 1);
        copy16(d_raw + (place * 2 + j) * d_many, on ? d + j * p.C : dy, on);
      }
    }
  };
  auto fetched_x = [&](int place, uint2 (&q)[5]) {
#pragma unroll
    for (int j = 0; j < 5; ++j) q[j] = x_raw[(place * 5 + j) * x_many];
  };

  typename S::Acc acc;
  S::clear(acc);
  int added = 0;         // steps in the accumulators
  bool written = false;  // whether the slice holds sums of steps before them
  auto end_chain = [&] {
    const long long slice = static_cast<long long>(blockIdx.z) * p.chunks + blockIdx.y;
    S::add(acc, reinterpret_cast<float*>(smem), part + slice * p.K * p.K * p.C, c0, p.C, p.K, written);
  };

  const int u1 = min(p.units, static_cast<int>(blockIdx.y + 1) * p.per_chunk);
  int u = blockIdx.y * p.per_chunk;
  while (u < u1) {  // one image's part of the range at a time
    const int b = u / p.unit_rows;
    const int s0 = u - b * p.unit_rows;
    int steps = min(p.unit_rows - s0, u1 - u);
    if constexpr (LONG) {  // in even pieces where it is longer than a chain
      if (steps > S::kMost) {
        const int pieces = (steps + S::kMost - 1) / S::kMost;
        steps = (steps + pieces - 1) / pieces;
      }
      if (added + steps > S::kMost) {
        end_chain();
        S::clear(acc);
        added = 0;
        written = true;
      }
      added += steps;
    }
    const int top = s0 * kStep + pad - (p.K - 1);  // first row of dy that the first row of x meets
    // of x and dy, this thread's next to fetch; of the exponent bytes, its next to load
    int row = s0 * kStep + x_row, drow = top + used + d_row;
    const long long x_at = (static_cast<long long>(b) * p.H + row) * p.W + x_col;
    const int8_t* q = codes + x_at * p.C + x_c;
    const uint8_t* e = scales + x_at * sblocks + x_c / kAct8Block;
    const __half* d = dy + ((static_cast<long long>(b) * p.H + drow) * p.W + d_col) * p.C + d_c;
    // `step` of this image, at place step % kAhead; past the last one nothing is written there
    auto next = [&](int step) {
      if (step < steps) fetch(step & 1, q, row < p.H, d, drow >= 0 && drow < p.H);
      cp_async_commit();
      row += kStep;
      drow += kStep;
      q += kStep * line;
      d += kStep * line;
    };
    __syncthreads();  // the last image's rows have been read
    // the first step: its row of x, and all rows of dy that it meets
    XScales sc[2];
    load_scales(sc[0], e, s0 * kStep + x_row < p.H);
    fetch(0, q, row < p.H, d, false);
    cp_async_commit();
    row += kStep;
    q += kStep * line;
    for (int i = tid; i < used * S::kDItems; i += kWgThreads) {
      const int r = i / S::kDItems, item = i - r * S::kDItems, at = top + r;
      const int c = c0 + (item & 3) * 8, col = w0 + (item >> 2) * 2;
      const __half* from = dy + ((static_cast<long long>(b) * p.H + at) * p.W + col) * p.C + c;
      const bool on = at >= 0 && at < p.H && c < p.C;
      uint4 v[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        v[j] = on && col + j < p.W ? *reinterpret_cast<const uint4*>(from + j * p.C) : make_uint4(0u, 0u, 0u, 0u);
      S::store_dy(v, ds + r * S::kDRow, item);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (x_row < kStep) {
      uint2 v[5];
      fetched_x(0, v);
      S::store_x(v, sc[0], xs + x_row * S::kXRow, x_item);
    }
    e += kStep * s_line;
    load_scales(sc[0], e, steps > 1 && s0 * kStep + kStep + x_row < p.H);  // step 1
    next(1);
    __syncthreads();
    int first = 0;  // ring slot of the row of dy with j = 0
    for (int s = 0; s < steps; ++s) {
      const bool more = s + 1 < steps;
      e += kStep * s_line;
      load_scales(sc[1], e, s + 2 < steps && (s0 + s + 2) * kStep + x_row < p.H);
      next(s + 2);
#pragma unroll 1
      for (int i = 0; i < SETS; ++i) {
        if (SETS > 1 && (s0 + s) * kStep + i * ROWS >= p.H) break;  // rows past the image
        const int at = first + i * ROWS;
        S::multiply(acc, xs + (s & 1) * S::kXBuffer + i * ROWS * S::kXRow, ds, at < ring ? at : at - ring, p.K);
      }
      asm volatile("cp.async.wait_group 1;" ::: "memory");  // step s + 1 is here
      if (more && x_row < kStep) {
        uint2 v[5];
        fetched_x((s + 1) & 1, v);
        S::store_x(v, sc[0], xs + ((s + 1) & 1) * S::kXBuffer + x_row * S::kXRow, x_item);
      }
      if (more && d_row < kStep) {
        // the ring has kStep rows more than a step reads: these slots belong to no row of this step
        int slot = first + used + d_row;
        slot -= slot >= ring ? ring : 0;
        const uint4 v[2] = {d_raw[((s + 1) & 1) * 2 * d_many], d_raw[(((s + 1) & 1) * 2 + 1) * d_many]};
        S::store_dy(v, ds + slot * S::kDRow, d_item);
      }
      sc[0] = sc[1];
      first += kStep;
      first -= first >= ring ? ring : 0;
      __syncthreads();
    }
    u += steps;
  }
  if constexpr (LONG) {
    end_chain();
  } else {
    const long long slice = static_cast<long long>(blockIdx.z) * p.chunks + blockIdx.y;
    S::write(acc, part + slice * p.K * p.K * p.C, c0 + (tid >> 5) * 4, p.C, p.K);
  }
}

// dw[i] = the slices' values added up (n2 pairs).  Row y of a block takes every ROWS-th slice in order, and the rows
// are added in order.  ROWS: 8 from 16 slices on, else 1 (many slices of few taps, 272 of 15 x 15 x 8, are one long
// chain of loads with one row: 35 us for the gradient, 19.5 with 8; four slices of 27 x 27 x 512 are 19.9 us with 8
// rows, 16.1 with one).
constexpr int kReduceThreads = 256;
template <int ROWS>
__global__ void __launch_bounds__(kReduceThreads) wgrad8_reduce_kernel(const float2* __restrict__ part,
                                                                       float2* __restrict__ dw, long long n2, int slices) {
  constexpr int kAcross = kReduceThreads / ROWS;
  __shared__ float2 sums[ROWS][kAcross + 1];
  griddep_wait();
  griddep_launch_dependents();
  const int row = threadIdx.x / kAcross, lane = threadIdx.x % kAcross;
  const long long i = static_cast<long long>(blockIdx.x) * kAcross + lane;
  float2 a = make_float2(0.0f, 0.0f);
  if (i < n2)
#pragma unroll 8
    for (int s = row; s < slices; s += ROWS) {
      const float2 v = part[s * n2 + i];
      a.x += v.x;
      a.y += v.y;
    }
  if constexpr (ROWS > 1) {
    sums[row][lane] = a;
    __syncthreads();
    if (row != 0) return;
#pragma unroll
    for (int r = 1; r < ROWS; ++r) {
      a.x += sums[r][lane].x;
      a.y += sums[r][lane].y;
    }
  }
  if (i < n2) dw[i] = a;
}

// The kernel for K and a tile of columns, its rows a step and its shared memory.
struct Wgrad8Kernel {
  const void *fn, *long_fn;
  int step, most, ctas, smem;  // rows a step; steps of a chain; CTAs an SM, by registers
};
template <int MT, int NT, int ROWS, bool PACK, int TW, int SETS>
static Wgrad8Kernel wgrad8_kernel_of(int K) {
  using S = Wgrad8<MT, NT, ROWS, PACK, TW, SETS>;
  return {reinterpret_cast<const void*>(&wgrad8_kernel<MT, NT, ROWS, PACK, TW, SETS, false>),
          reinterpret_cast<const void*>(&wgrad8_kernel<MT, NT, ROWS, PACK, TW, SETS, true>),
          S::kStep, S::kMost, kWgCtas<MT, PACK>, S::smem(K)};
}
static int wgrad8_room(const Wgrad8Kernel& k) { return 228 * 1024 / (k.smem + 1024); }  // CTAs an SM, by shared memory
// Sets: as many as a step's items of x have threads for.  A step of one set leaves most threads of a narrow tile without
// an item and has a barrier for few products (19x14x8x1424 k9: 40.2 us with one set, 32.4 with two; 8x14x14x512 k27: 21.0
// with one, 17.7 with four; 8x32x32x1536 k27: 165 with one, 146 with two).  From K = 9 on not where the longer ring then
// leaves room for one CTA an SM (16x32x32x1536 k11: 86.0 us with one set and two CTAs, 145 with two sets and one).  Up to
// K = 7 two sets are better with two CTAs an SM than one with three (inputs in L2: 16x32x32x768 k7 34.2 and 37.8 us,
// 8x16x16x1536 k3 12.9 and 15.2, 64x56x28x256 k7 65.4 and 72.7).
template <int TW>
static Wgrad8Kernel wgrad8_kernel_for(int K) {
  constexpr int kPair = TW <= 32 ? 2 : 1, kOne = TW == 16 ? 4 : TW == 32 ? 2 : 1;
  if (K <= 7) return wgrad8_kernel_of<1, 1, 2, true, TW, kPair>(K);
  if (K <= 15) {
    const Wgrad8Kernel k = wgrad8_kernel_of<1, 2, 2, false, TW, kPair>(K);
    return kPair > 1 && wgrad8_room(k) < k.ctas ? wgrad8_kernel_of<1, 2, 2, false, TW, 1>(K) : k;
  }
  if (K <= 23) return wgrad8_kernel_of<2, 3, 1, false, TW, kOne>(K);
  return wgrad8_kernel_of<2, 4, 1, false, TW, kOne>(K);
}
static Wgrad8Kernel wgrad8_kernel_for(int K, int tw) {
  switch (tw) {
    case 16: return wgrad8_kernel_for<16>(K);
    case 32: return wgrad8_kernel_for<32>(K);
    case 48: return wgrad8_kernel_for<48>(K);
    default: return wgrad8_kernel_for<64>(K);
  }
}

static long long min_ll(long long a, long long b) { return a < b ? a : b; }
static long long max_ll(long long a, long long b) { return a > b ? a : b; }

static int wgrad8_plan(int64_t B, int64_t H, int64_t W, int64_t C, int K, Wgrad8Params* p) {
  if (K < 1 || K > 31 || (K % 2) == 0 || B < 0 || H < 1 || W < 1 || C < 8 || (C % 8) != 0) return DWB_ERR_BAD_SHAPE;
  if (B > (1 << 30) || H > (1 << 24) || W > (1 << 21) || C > (1 << 20) || B * H > (1LL << 30)) return DWB_ERR_BAD_SHAPE;
  p->B = static_cast<int>(B);
  p->H = static_cast<int>(H);
  p->W = static_cast<int>(W);
  p->C = static_cast<int>(C);
  p->K = K;
  p->col_tiles = (p->W + kWgTile - 1) / kWgTile;
  p->tw = ((p->W + p->col_tiles - 1) / p->col_tiles + 15) / 16 * 16;  // even tiles: W = 65 is 48 + 17, not 64 + 1
  p->col_tiles = (p->W + p->tw - 1) / p->tw;
  const Wgrad8Kernel k = wgrad8_kernel_for(K, p->tw);
  p->unit_rows = (p->H + k.step - 1) / k.step;
  p->units = p->B * p->unit_rows;
  // As many ranges as CTAs run at once (a range more on some SMs would double the time).  However short: the rows of dy
  // that a range brings in before its first product cost less than idle SMs (14x14x512 k27, B = 2: 28.8 us with ranges
  // of 26 rows, 16.2 with 8, 14.7 with 4).  More turns of shorter ranges only where one leaves too many SMs idle (10
  // tiles of 32 channels on 148 SMs are 14 ranges, but 100 are one): the turns' time is their steps and, for each, a
  // start of about (K - 1) / 3 rows, and another turn has to save a part in 32 of it, since it has slices of its own.
  const long long base = (C + kWgChannels - 1) / kWgChannels * p->col_tiles;
  const int room = wgrad8_room(k);
  const long long at_once = static_cast<long long>(room < k.ctas ? room : k.ctas) * kSmCount;
  // so many steps at most to a range that its slice is added to kFlushes times, as long as a grid takes the ranges
  const long long longest = max_ll(static_cast<long long>(k.most) * kFlushes, (p->units + 65534LL) / 65535);
  long long best = 0;
  p->per_chunk = 1;
  for (int turns = 1; turns <= kTurns; ++turns) {
    const long long ranges = max_ll(turns * at_once / base, 1);
    const long long per = max_ll(min_ll((p->units + ranges - 1) / ranges, longest), 1), chunks = (p->units + per - 1) / per;
    const long long time = (base * chunks + at_once - 1) / at_once * (3LL * k.step * per + K - 1);
    if (turns == 1 || time < best - best / 32) {
      best = time;
      p->per_chunk = static_cast<int>(per);
    }
    if (per == 1) break;  // there are no more ranges than that
  }
  p->chunks = (p->units + p->per_chunk - 1) / p->per_chunk;
  if (p->chunks < 1) p->chunks = 1;
  return DWB_OK;
}

// The partial sums: one [K][K][C] slice for every range of rows and tile of columns.  base * chunks CTAs write one 32
// channels of it each, at most kTurns turns of the CTAs that run at once or one for every tile of columns and channels;
// beyond that only 1 in every kFlushes * kMost steps, 0.5% of the codes and dy that they read at most.
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
  const Wgrad8Kernel k = wgrad8_kernel_for(K, p.tw);
  const void* const fn = p.per_chunk > k.most ? k.long_fn : k.fn;
  cudaError_t e = allow_large_cta(fn);
  if (e == cudaSuccess)
    e = launch_kernel(fn, dim3(static_cast<unsigned>((C + kWgChannels - 1) / kWgChannels), p.chunks, p.col_tiles),
                      dim3(kWgThreads), a1, k.smem, st);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return record_cuda_failure("wgrad8_kernel", e);
  }
  long long n2 = static_cast<long long>(K) * K * C / 2;
  int slices = p.chunks * p.col_tiles;
  void* a2[] = {&part, &dw, &n2, &slices};
  const int rows = slices >= 16 ? 8 : 1;
  e = launch_kernel(rows > 1 ? reinterpret_cast<const void*>(&wgrad8_reduce_kernel<8>)
                             : reinterpret_cast<const void*>(&wgrad8_reduce_kernel<1>),
                    dim3(static_cast<unsigned>((n2 * rows + kReduceThreads - 1) / kReduceThreads)), dim3(kReduceThreads), a2, 0, st);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return record_cuda_failure("wgrad8_reduce_kernel", e);
  }
  return DWB_OK;
}
