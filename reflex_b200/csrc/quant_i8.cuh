// int8 symmetric rounding shared by the KV quantizer and the row quantizers.
#pragma once
#include "ptx.cuh"

namespace rfx {

// Packed fp32x2 arithmetic (sm_100): two round-to-nearest fp32 operations per
// instruction, each lane exactly as the scalar one.
__device__ __forceinline__ unsigned long long pack_f32x2(float lo, float hi) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float lo_f32(unsigned long long v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float hi_f32(unsigned long long v) {
  return __uint_as_float(static_cast<uint32_t>(v >> 32));
}
// max that returns NaN when either operand is NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ unsigned long long mul_f32x2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long fma_f32x2(unsigned long long a, unsigned long long b,
                                                        unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add_f32x2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long sub_f32x2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// int8 symmetric quantization of one lane's 8 values of a row, packed little
// endian into two words: q = clamp(rne(x / scale), -127, 127), exactly as with
// rintf(__fdiv_rn(x, scale)), but from a product with rcp = __frcp_rn(scale),
// the correctly rounded 1 / scale.
//
// Error bound: |x| <= absmax and scale = fl(absmax / 127) is a normal float,
// so the exact quotient q has |q| <= 127 (1 + 2^-23); then y = fl(x * rcp)
// and fl(q) both lie within |q| * (3 * 2^-24 + 2^-48) + 2^-149, under 2.3e-5,
// of q.  Hence |y| < 127.5 (rne(y) needs no clamp), and whenever y is at least
// 2^-14 (6.1e-5) away from every half-integer, fl(q) is on the same side of
// all of them and on none, so both round to the same integer.  Values closer
// than that (bf16 inputs put about 0.2 % of the quotients there, most on a
// tie) are divided in a second pass; a denormal scale divides all 8.
//
// Rounding: t = y + 1.5 * 2^23 holds rne(y) in its low mantissa bits, so the
// low byte of t's bit pattern is the two's-complement int8 and t - 1.5 * 2^23
// is rne(y) as a float; y - rne(y) is exact (Sterbenz).  A NaN input fails
// the distance test and takes the divide, as before.
__device__ __forceinline__ void quant8_i8(const float (&v)[8], float scale, float rcp, uint32_t (&packed)[2]) {
  constexpr float kMagic = 12582912.0f;     // 1.5 * 2^23
  constexpr float kFar = 0.5f - 0x1p-14f;   // |y - rne(y)| <= kFar: 2^-14 or more from a half-integer
  uint32_t tb[8];
  if (scale >= 0x1p-126f) {
    // two values per instruction (packed fp32x2, each lane rounded as the
    // scalar op); the largest distance to a rounded value decides the pass
    const unsigned long long r2 = pack_f32x2(rcp, rcp), m2 = pack_f32x2(kMagic, kMagic);
    float dmax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const unsigned long long y = mul_f32x2(pack_f32x2(v[i], v[i + 1]), r2);
      const unsigned long long t = add_f32x2(y, m2);
      const unsigned long long d = sub_f32x2(y, sub_f32x2(t, m2));
      dmax = max_nan(dmax, max_nan(fabsf(lo_f32(d)), fabsf(hi_f32(d))));
      tb[i] = __float_as_uint(lo_f32(t));
      tb[i + 1] = __float_as_uint(hi_f32(t));
    }
    // a NaN distance (NaN input) fails the test and takes the divide
    const bool near = !(dmax <= kFar);
    if (near) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = __fmul_rn(v[i], rcp);
        const float t = __uint_as_float(tb[i]);
        if (!(fabsf(__fsub_rn(y, __fsub_rn(t, kMagic))) <= kFar))
          tb[i] = __float_as_uint(__fadd_rn(fminf(fmaxf(rintf(__fdiv_rn(v[i], scale)), -127.f), 127.f), kMagic));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float r = fminf(fmaxf(rintf(__fdiv_rn(v[i], scale)), -127.f), 127.f);
      tb[i] = __float_as_uint(__fadd_rn(r, kMagic));
    }
  }
  packed[0] = __byte_perm(__byte_perm(tb[0], tb[1], 0x0040), __byte_perm(tb[2], tb[3], 0x0040), 0x5410);
  packed[1] = __byte_perm(__byte_perm(tb[4], tb[5], 0x0040), __byte_perm(tb[6], tb[7], 0x0040), 0x5410);
}

}  // namespace rfx
