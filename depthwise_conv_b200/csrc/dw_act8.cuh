// dw_act8.cuh -- the 8-bit activation checkpoint: codec arithmetic on one
// 16-byte vector (8 channels) per lane, four neighbouring lanes per block.
//
// A checkpoint keeps, for every pixel and block of 32 channels, one exponent
// byte E and 32 signed codes q; the value is q * 2^(E - 127).  With amax the
// block's largest magnitude, E - 127 is the smallest exponent e with
// amax <= 127 * 2^e, so the codes use at least 64 of their 127 steps and a
// value is off by at most 2^(e-1) <= amax / 127 (half a step, the step at
// most 2 amax / 127).  A power of two (and not amax / 127 itself) costs up to
// one bit of the codes, and buys three things: one byte of overhead per block
// instead of four, values that are exact in the 16-bit type they came from
// (8 significant bits), and so products that 16-bit tensor-core operands take
// without another rounding.
//
// e stays within the range where q * 2^e is exact in the type: fp16 from -24
// (its finest step) to 9 (127 * 2^9 = 65024; a larger amax saturates there,
// off by at most 480 = less than half of the next exponent's step), bf16 from
// -127 to 121.  A block that holds a NaN or an infinity gets E = 255 and reads
// back as NaN everywhere, so an overflow still reaches the gradients.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "dw_device.cuh"

namespace dwb {

constexpr int kAct8Block = 32;  // channels that share an exponent byte

template <typename T>
struct Type16;

template <>
struct Type16<__half> {
  static constexpr int kExpLow = 127 - 24, kExpHigh = 127 + 9;
  static constexpr uint32_t kInfBits = 0x7c00u;
  static __device__ __forceinline__ f32x2 to_f32x2(uint32_t u) { return h2_to_f32x2(*reinterpret_cast<__half2*>(&u)); }
  static __device__ __forceinline__ uint32_t from_f32x2(f32x2 v) {
    const float2 f = bits_f2(v);
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  // min(max(v, -limit), limit) with limit = 127 * 2^9, the largest value a code stands for
  static __device__ __forceinline__ uint32_t clamp_pair(uint32_t u) {
    const __half2 lim = __half2half2(__ushort_as_half(0x7bf0));
    const __half2 h = __hmax2(__hmin2(*reinterpret_cast<__half2*>(&u), lim), __hneg2(lim));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float to_float(__half h) { return __half2float(h); }
  static __device__ __forceinline__ uint32_t abs_to_f32_bits(uint32_t a) {
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(a))));
  }
};

template <>
struct Type16<__nv_bfloat16> {
  static constexpr int kExpLow = 0, kExpHigh = 127 + 121;
  static constexpr uint32_t kInfBits = 0x7f80u;
  static __device__ __forceinline__ f32x2 to_f32x2(uint32_t u) {
    return (static_cast<unsigned long long>(u & 0xffff0000u) << 32) | (u << 16);
  }
  static __device__ __forceinline__ uint32_t from_f32x2(f32x2 v) {
    const float2 f = bits_f2(v);
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  // limit = 127 * 2^121
  static __device__ __forceinline__ uint32_t clamp_pair(uint32_t u) {
    const __nv_bfloat162 lim = __bfloat162bfloat162(__ushort_as_bfloat16(0x7f7e));
    const __nv_bfloat162 h = __hmax2(__hmin2(*reinterpret_cast<__nv_bfloat162*>(&u), lim), __hneg2(lim));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float to_float(__nv_bfloat16 h) { return __bfloat162float(h); }
  static __device__ __forceinline__ uint32_t abs_to_f32_bits(uint32_t a) { return a << 16; }
};

// Exponent byte of the block whose largest magnitude has the 16-bit pattern `amax`
// (patterns of one sign order like the numbers, infinities and NaN above all).
template <typename T>
__device__ __forceinline__ uint32_t act8_exponent(uint32_t amax) {
  if (amax >= Type16<T>::kInfBits) return 255u;
  // amax = 1.f * 2^k: e = k - 6 where 1.f <= 127 / 64, else k - 5; adding 0x1ffff to the bits carries
  // into the exponent exactly where the fraction is above 63 / 64
  const int e = static_cast<int>((Type16<T>::abs_to_f32_bits(amax) + 0x1ffffu) >> 23) - 6;
  return static_cast<uint32_t>(min(max(e, Type16<T>::kExpLow), Type16<T>::kExpHigh));
}

// 2^(E - 127), NaN for E = 255.
__device__ __forceinline__ float act8_step(uint32_t E) {
  return __uint_as_float((E << 23) | ((E == 0u || E == 255u) ? 0x400000u : 0u));
}

// Largest magnitude (16-bit pattern) of a lane's 8 values and its three neighbours' of the block.
// Every lane of the quad takes part; `v` must be zero in lanes past the last channel.
__device__ __forceinline__ uint32_t act8_block_amax(const uint4& v) {
  const uint32_t m = 0x7fff7fffu;
  uint32_t a = __vmaxu2(__vmaxu2(v.x & m, v.y & m), __vmaxu2(v.z & m, v.w & m));
  a = __vmaxu2(a, __shfl_xor_sync(0xffffffffu, a, 1));
  a = __vmaxu2(a, __shfl_xor_sync(0xffffffffu, a, 2));
  return max(a & 0xffffu, a >> 16);
}

// rint(x * 2^(127 - E)) through the magic number 1.5 * 2^23, whose unit is 1 (ties to even, as rint): the
// code stands in the low byte.  The values are clamped in their own type first, two at a time; below that
// limit every amax has an exponent that 127 steps reach.
template <typename T>
__device__ __forceinline__ uint2 act8_codes(const uint4& v, uint32_t E) {
  if (E == 255u) return make_uint2(0u, 0u);
  const f32x2 inv = splat2(__uint_as_float((254u - E) << 23));  // 2^(127 - E), E <= 248
  const uint32_t* w = &v.x;
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // the product is exact (or so small that it rounds to 0), so one fma rounds as a product and a sum do
    const float2 r = bits_f2(fma2(Type16<T>::to_f32x2(Type16<T>::clamp_pair(w[i])), inv, splat2(12582912.0f)));
    b[i] = __byte_perm(__float_as_uint(r.x), __float_as_uint(r.y), 0x0040);
  }
  return make_uint2(__byte_perm(b[0], b[1], 0x5410), __byte_perm(b[2], b[3], 0x5410));
}

// 4 codes as fp32 pairs times `step`.  Byte u = q + 128 under 0x4b000000 is the float 2^23 + u.
__device__ __forceinline__ void act8_values4(uint32_t q, float step, f32x2 (&out)[2]) {
  const f32x2 off = splat2(-8388736.0f);  // -(2^23 + 128)
  const f32x2 s = splat2(step);
  const uint32_t w = q ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __byte_perm(w, 0x4b000000u, i ? 0x7442 : 0x7440);
    const uint32_t hi = __byte_perm(w, 0x4b000000u, i ? 0x7443 : 0x7441);
    f32x2 f = (static_cast<unsigned long long>(hi) << 32) | lo;
    fadd2(f, off);
    out[i] = fmul2(f, s);
  }
}

__device__ __forceinline__ void act8_values(const uint2& q, float step, f32x2 (&out)[4]) {
  f32x2 a[2], b[2];
  act8_values4(q.x, step, a);
  act8_values4(q.y, step, b);
  out[0] = a[0];
  out[1] = a[1];
  out[2] = b[0];
  out[3] = b[1];
}

}  // namespace dwb
