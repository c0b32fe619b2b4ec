// dw_groupnorm.cuh -- group normalisation with an activation on channels-last
// 16-bit tensors: the arithmetic that its kernels share.
//
//   x [B, P, C] (P = H * W pixels), G groups of Cg = C / G channels, n = P Cg:
//   mean = sum x / n,  var = sum (x - mean)^2 / n,  rstd = 1 / sqrt(var + eps)
//   xh = (x - mean) rstd,  u = xh weight + bias,  y = act(u)
//
//   backward, from dy and the saved x (16 bits, or its 8-bit checkpoint), mean
//   and rstd:  g = dy act'(u),  dbias = sum g,  dweight = sum g xh,
//   m1 = sum_group(g weight) / n,  m2 = sum_group(g weight xh) / n,
//   dx = rstd ((g weight - m1) - xh m2).
//
// Layout of the work in every kernel: a thread owns one vector of 8 (or 4)
// channels and walks over pixels, so that its parameters and its sums stay in
// registers and every group structure (groups of 1, 3, 9 channels, groups that
// end inside a vector) is a matter of how the per-channel sums are added up.
// Statistics: a thread sums (x - k) and (x - k)^2 with k its own first value,
// which takes out the offset of the data, and the (count, mean, sum of squared
// deviations) triples of threads, CTAs and channels are merged by
// M2 = sum M2_i + sum n_i (mean_i - mean)^2.  All in fp32.
#pragma once

#include "dw_act8.cuh"

namespace dwb {

enum : int { kActSilu = 3 };  // after kActNone, kActRelu, kActGelu

// Q(a) = erfc(a / sqrt 2) / 2 for a >= 0 as 2^P(a): log2 Q is so smooth that a polynomial of degree 8 (a weighted
// least-squares fit on [0, 8], reweighted towards its largest error) has a Q to 7.5e-8 and, up to a = 8, to 1.5e-3 of
// itself: GELU's small values below zero are a Q alone, and half a step of bf16 is 3.9e-3 of a value.  Further out P
// falls faster than log2 Q: 6% of a Q are missing at a = 9, where it is 1e-18.  One special-function operation a value.
__device__ __forceinline__ f32x2 normal_tail2(f32x2 a) {
  f32x2 p = fma2(splat2(-1.86687586e-07f), a, splat2(2.77648019e-06f));
  p = fma2(p, a, splat2(1.80209154e-05f));
  p = fma2(p, a, splat2(-0.000729526568f));
  p = fma2(p, a, splat2(0.0080255894f));
  p = fma2(p, a, splat2(-0.0533717498f));
  p = fma2(p, a, splat2(-0.458785474f));
  p = fma2(p, a, splat2(-1.15119958f));
  const float2 e = bits_f2(fma2(p, a, splat2(-0.999993145f)));
  return f2_bits(make_float2(ex2_approx(e.x), ex2_approx(e.y)));
}

template <int ACT>
__device__ __forceinline__ f32x2 act_value2(f32x2 u) {
  if constexpr (ACT == kActRelu) {
    const float2 f = bits_f2(u);  // a comparison, not fmaxf: NaN stays NaN
    return f2_bits(make_float2(f.x < 0.0f ? 0.0f : f.x, f.y < 0.0f ? 0.0f : f.y));
  } else if constexpr (ACT == kActGelu) {
    // u Phi(u) = max(u, 0) - |u| Q(|u|) on both sides of 0: no selection
    const float2 f = bits_f2(u);
    // |u| stays finite in the product, whose other factor is 0 long before: an infinite u leaves max(u, 0); a NaN goes
    // through Q
    constexpr float kMost = 3.4028235e38f;
    return fma2(f2_bits(make_float2(fmaxf(-fabsf(f.x), -kMost), fmaxf(-fabsf(f.y), -kMost))),
                normal_tail2(u & 0x7fffffff7fffffffull), f2_bits(make_float2(fmaxf(f.x, 0.0f), fmaxf(f.y, 0.0f))));
  } else if constexpr (ACT == kActSilu) {
    const float2 e = bits_f2(fmul2(u, splat2(-1.4426950408889634f)));
    const f32x2 d = fma2(f2_bits(make_float2(ex2_approx(e.x), ex2_approx(e.y))), splat2(1.0f), splat2(1.0f));
    const float2 df = bits_f2(d);
    return fmul2(u, f2_bits(make_float2(rcp_approx(df.x), rcp_approx(df.y))));
  } else {
    return u;
  }
}

// act'(u).  ReLU: 0 at 0.
template <int ACT>
__device__ __forceinline__ f32x2 act_slope2(f32x2 u) {
  if constexpr (ACT == kActRelu) {
    const float2 f = bits_f2(u);
    return f2_bits(make_float2(f.x > 0.0f ? 1.0f : 0.0f, f.y > 0.0f ? 1.0f : 0.0f));
  } else if constexpr (ACT == kActGelu) {
    // Phi(u) + u phi(u).  With k = erfc(|u| / sqrt 2) / 2 - |u| phi(u) it is k below 0 and 1 - k above: 1/2 plus
    // k - 1/2 with its sign turned where u is positive.  erfc from Abramowitz & Stegun 7.1.26, as gelu_erf2 has it
    // (|error| <= 1.5e-7): exp(-u^2 / 2) poly(t) t, t = 1 / (1 + p |u|), whose exponential phi shares.
    const f32x2 na = u | 0x8000000080000000ull;
    const float2 d = bits_f2(fma2(na, splat2(-0.3275911f * 0.70710678118654752f), splat2(1.0f)));
    const f32x2 t = f2_bits(make_float2(rcp_approx(d.x), rcp_approx(d.y)));
    f32x2 poly = fma2(splat2(0.5f * 1.061405429f), t, splat2(0.5f * -1.453152027f));
    poly = fma2(poly, t, splat2(0.5f * 1.421413741f));
    poly = fma2(poly, t, splat2(0.5f * -0.284496736f));
    poly = fma2(poly, t, splat2(0.5f * 0.254829592f));
    const f32x2 k = fma2(poly, t, fmul2(na, splat2(0.3989422804014327f)));
    const float2 x = bits_f2(fmul2(fmul2(u, splat2(-0.5f * 1.4426950408889634f)), u));
    f32x2 r = splat2(0.5f);
    fadd2(r, fma2(k, f2_bits(make_float2(ex2_approx(x.x), ex2_approx(x.y))), splat2(-0.5f)) ^ (~u & 0x8000000080000000ull));
    return r;
  } else if constexpr (ACT == kActSilu) {
    const float2 e = bits_f2(fmul2(u, splat2(-1.4426950408889634f)));
    f32x2 d = splat2(1.0f);
    fadd2(d, f2_bits(make_float2(ex2_approx(e.x), ex2_approx(e.y))));
    const float2 df = bits_f2(d);
    const f32x2 sv = f2_bits(make_float2(rcp_approx(df.x), rcp_approx(df.y)));
    const f32x2 rest = fma2(sv, splat2(-1.0f), splat2(1.0f));  // 1 - s
    return fmul2(sv, fma2(u, rest, splat2(1.0f)));
  } else {
    return splat2(1.0f);
  }
}

// Sizes of one call.
struct GnShape {
  long long P;     // pixels of a sample
  int B, C, G, Cg;
  float eps;
  int param_f32;   // weight and bias: fp32 instead of the tensor's type
  int param_vec;   // both on 16-byte boundaries (or absent)
};

// Weight or bias of channel c (`otherwise` where the vector is absent).
template <typename T>
__device__ __forceinline__ float gn_param(const void* p, int c, int f32, float otherwise) {
  if (!p) return otherwise;
  return f32 ? static_cast<const float*>(p)[c] : Type16<T>::to_float(static_cast<const T*>(p)[c]);
}

template <typename T>
__device__ __forceinline__ void gn_unpack(const uint4& v, f32x2 (&f)[4]) {
  f[0] = Type16<T>::to_f32x2(v.x);
  f[1] = Type16<T>::to_f32x2(v.y);
  f[2] = Type16<T>::to_f32x2(v.z);
  f[3] = Type16<T>::to_f32x2(v.w);
}

// 8 channels of a parameter vector.
template <typename T>
__device__ __forceinline__ void gn_load_param8(const void* p, int c, const GnShape& s, float otherwise, f32x2 (&v)[4]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = splat2(otherwise);
  } else if (s.param_vec && s.param_f32) {
    const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(static_cast<const float*>(p) + c);
    const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(static_cast<const float*>(p) + c + 4);
    v[0] = a.x;
    v[1] = a.y;
    v[2] = b.x;
    v[3] = b.y;
  } else if (s.param_vec) {
    gn_unpack<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(p) + c), v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = f2_bits(make_float2(gn_param<T>(p, c + 2 * i, s.param_f32, otherwise),
                                 gn_param<T>(p, c + 2 * i + 1, s.param_f32, otherwise)));
  }
}

// 4 channels of a parameter vector.
template <typename T>
__device__ __forceinline__ void gn_load_param4(const void* p, int c, const GnShape& s, float otherwise, f32x2 (&v)[2]) {
  if (!p) {
    v[0] = v[1] = splat2(otherwise);
  } else if (s.param_vec && s.param_f32) {
    const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(static_cast<const float*>(p) + c);
    v[0] = a.x;
    v[1] = a.y;
  } else if (s.param_vec) {
    const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const T*>(p) + c);
    v[0] = Type16<T>::to_f32x2(a.x);
    v[1] = Type16<T>::to_f32x2(a.y);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      v[i] = f2_bits(make_float2(gn_param<T>(p, c + 2 * i, s.param_f32, otherwise),
                                 gn_param<T>(p, c + 2 * i + 1, s.param_f32, otherwise)));
  }
}

template <typename T>
__device__ __forceinline__ void gn_load_params(const void* weight, const void* bias, int c, const GnShape& s, f32x2 (&w)[4],
                                               f32x2 (&b)[4]) {
  gn_load_param8<T>(weight, c, s, 1.0f, w);
  gn_load_param8<T>(bias, c, s, 0.0f, b);
}

template <typename T>
__device__ __forceinline__ uint4 gn_pack(const f32x2 (&f)[4]) {
  return make_uint4(Type16<T>::from_f32x2(f[0]), Type16<T>::from_f32x2(f[1]), Type16<T>::from_f32x2(f[2]),
                    Type16<T>::from_f32x2(f[3]));
}

__device__ __forceinline__ f32x2 fsub2(f32x2 a, f32x2 b) { return fma2(b, splat2(-1.0f), a); }

// A sum of squares that rounding may leave below zero (a comparison, not fmaxf: NaN stays NaN).
__device__ __forceinline__ float not_negative(float v) { return v < 0.0f ? 0.0f : v; }

// Sums of one thread about its own first values.
struct GnSums {
  f32x2 k[4], s1[4], s2[4];
  __device__ __forceinline__ void start(const f32x2 (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      k[i] = v[i];
      s1[i] = s2[i] = f32x2_zero();
    }
  }
  __device__ __forceinline__ void add(const f32x2 (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 d = fsub2(v[i], k[i]);
      fadd2(s1[i], d);
      ffma2(s2[i], d, d);
    }
  }
  // per-channel mean and sum of squared deviations of the n >= 1 values seen
  __device__ __forceinline__ void moments(int n, f32x2 (&mean)[4], f32x2 (&m2)[4]) const {
    const f32x2 inv = splat2(rcp_approx(static_cast<float>(n)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 d = fmul2(s1[i], inv);
      mean[i] = k[i];
      fadd2(mean[i], d);
      const float2 q = bits_f2(fsub2(s2[i], fmul2(s1[i], d)));
      m2[i] = f2_bits(make_float2(not_negative(q.x), not_negative(q.y)));
    }
  }
};

// Two or three sums at once: the shuffles of one hide those of the others.
__device__ __forceinline__ void warp_sum2(float& a, float& b) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
}

__device__ __forceinline__ void warp_sum3(float& a, float& b, float& c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
    c += __shfl_xor_sync(0xffffffffu, c, o);
  }
}

// The mean of a group, from its offset to a pivot or from the plain mean of the same values.  The pivot takes out a mean
// that is large against the deviations; but where the mean is small against the pivot, pivot + off has the pivot's
// rounding, and the plain mean that of the values only (7x7x1024, 32 groups: the means' error 1.9e-7 of their size with
// the pivot alone, 7e-8 so).
__device__ __forceinline__ float gn_mean(float pivot, float off, float plain) {
  return fabsf(plain) < 0.5f * fabsf(pivot) ? plain : pivot + off;
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// SUB: channels of a vector that surely share a group (8, 4 or 1: C / G is a multiple of it).
template <int SUB>
__device__ __forceinline__ f32x2 gn_of(const f32x2 (&v)[SUB == 8 ? 1 : SUB == 4 ? 2 : 4], int pair) {
  return v[SUB == 8 ? 0 : SUB == 4 ? pair / 2 : pair];
}

// The two halves of what `fin` holds for the groups (from `first_group` on) of the 8 channels from c on.
template <int SUB>
__device__ __forceinline__ void gn_read_groups(const float2* fin, int c, int Cg, int first_group,
                                               f32x2 (&x)[SUB == 8 ? 1 : SUB == 4 ? 2 : 4],
                                               f32x2 (&y)[SUB == 8 ? 1 : SUB == 4 ? 2 : 4]) {
#pragma unroll
  for (int i = 0; i < (SUB == 8 ? 1 : SUB == 4 ? 2 : 4); ++i) {
    const int at = c + i * (SUB == 1 ? 2 : SUB);
    const float2 lo = fin[at / Cg - first_group], hi = SUB == 1 ? fin[(at + 1) / Cg - first_group] : lo;
    x[i] = f2_bits(make_float2(lo.x, hi.x));
    y[i] = f2_bits(make_float2(lo.y, hi.y));
  }
}

// A thread's moments (n pixels a channel) for the merge of its CTA: one entry for every SUB channels.
template <int SUB>
__device__ __forceinline__ void gn_hand_over(const f32x2 (&mean)[4], const f32x2 (&m2)[4], float n, float2* ent) {
  if constexpr (SUB == 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = bits_f2(mean[j]), q = bits_f2(m2[j]);
      *reinterpret_cast<float4*>(ent + 2 * j) = make_float4(a.x, q.x, a.y, q.y);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8 / SUB; ++e) {
      f32x2 sum = mean[e * SUB / 2], q = m2[e * SUB / 2], d2 = f32x2_zero();
#pragma unroll
      for (int j = 1; j < SUB / 2; ++j) {
        fadd2(sum, mean[e * SUB / 2 + j]);
        fadd2(q, m2[e * SUB / 2 + j]);
      }
      const float2 sf = bits_f2(sum), qf = bits_f2(q);
      const float mid = (sf.x + sf.y) * (1.0f / SUB);
#pragma unroll
      for (int j = 0; j < SUB / 2; ++j) {
        const f32x2 d = fsub2(mean[e * SUB / 2 + j], splat2(mid));
        ffma2(d2, d, d);
      }
      const float2 df = bits_f2(d2);
      ent[e] = make_float2(mid, qf.x + qf.y + n * (df.x + df.y));
    }
  }
}

// A warp's merge of a segment's entries [lane row][per_row] in shared memory.  Lanes go along a lane row first.
struct GnMerge {
  int per_row, live, full, rest, row_words, k0, k_step, r0, r_step;
  __device__ __forceinline__ GnMerge(int lane, int entries_per_row, int rows, int rl, int words) {
    per_row = entries_per_row;
    live = min(rows, rl);
    full = rows / rl;
    rest = rows - full * rl;  // lane rows below `rest` have a pixel more
    row_words = words;
    const bool fits = per_row <= 32;
    k0 = fits ? lane % per_row : lane;
    k_step = fits ? per_row : 32;
    r_step = fits ? 32 / per_row : 1;
    r0 = fits ? lane / per_row : 0;
  }
  // (mean, M2) over `rows` pixels of `channels`; (0, 0) without pixels.
  template <int SUB>
  __device__ __forceinline__ float2 run(const float2* first, int rows, int channels) const {
    // about one thread's mean, which is a mean of its values already: nothing cancels in the squares
    const float pivot = live ? first[0].x : 0.0f;
    float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f;
    if (r0 < r_step)
#pragma unroll 4
      for (int r = r0; r < live; r += r_step) {
        const float n = static_cast<float>((full + (r < rest)) * SUB);
        for (int k = k0; k < per_row; k += k_step) {
          const float2 v = first[r * row_words + k];
          const float d = v.x - pivot;
          s0 += n * v.x;
          s1 += n * d;
          s2 += v.y + n * d * d;
        }
      }
    warp_sum3(s0, s1, s2);
    if (!rows) return make_float2(0.0f, 0.0f);
    const float n = static_cast<float>(rows) * static_cast<float>(channels), d = s1 / n;
    return make_float2(gn_mean(pivot, d, s0 / n), not_negative(s2 - s1 * d));
  }
};

}  // namespace dwb
