// Rows to 4-bit floating point numbers (e2m1) with a scale per block, and back.
//
// A thread takes units of 16 consecutive values: an NV block, or half of an MX
// one, whose other half is its neighbour's.  An MX block needs nothing but
// itself; an NV row's power of two comes from the whole row, which stays in the
// registers of its threads until then (rows above 16384 values are read twice).
// The 4 scale bytes of neighbouring blocks lie together in the tiles that the
// tensor cores take, and are gathered by shuffles into one 4-byte store.
//
// Bound by memory traffic: 2 bytes per value in (bf16), 9/16 out.  768 x 16384 (NV): 9.3 us,
// 3.5 TB/s, whole rows of 5 or 6 per SM; MX 7.5 us; 4096 x 4096 9.6 us, 4.5 TB/s.  Back:
// 6.7 us, 4.8 TB/s.  Single rows take 1.3 us, a launch.
#include "quant_i8.cuh"
#include "rfx_internal.h"

#include <algorithm>

namespace rfx {
namespace {

constexpr int kMaxK = 65536;
constexpr int kMaxRows = 1 << 30;
constexpr int kUnit = 16;

// Where the scale tiles of row t begin: bytes from the start, without block j's
// part ((j / 4) * 512 + j % 4).
struct ScaleTiles {
  int per_part, tiles_per_part, k_tiles;  // rows and row tiles of a part, tiles along K
  __device__ __forceinline__ long row(int t) const {
    const int part = t / per_part, r = t - part * per_part;
    return (static_cast<long>(part * tiles_per_part + r / 128) * k_tiles) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4;
  }
};

struct QuantFp4Params {
  int T, K;
  const void* x;
  long ldx;
  uint8_t* q;
  long ldq;
  uint8_t* scale;
  float* row_scale;
  ScaleTiles tiles;
};

__device__ __forceinline__ void load_32(const void* from, uint4& a, uint4& b) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
               : "l"(from));
}
__device__ __forceinline__ void store_32(void* to, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
               "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// 16 values as they lie in memory.
template <typename T>
struct Unit {
  static constexpr int kVecs = static_cast<int>(sizeof(T));  // 16-byte vectors
  static constexpr int kPer = 8 / static_cast<int>(sizeof(T)) * 2;  // values of a vector
  uint4 v[kVecs];

  // Values k .. k+15 of a row, zeros past K.  VEC: bytes that the row's start and
  // stride are multiples of (32, 16, or 0 for the type's own).
  template <int VEC>
  __device__ __forceinline__ void load(const T* row, int k, int K) {
    if (VEC == 32 && k + kUnit <= K) {
#pragma unroll
      for (int i = 0; i < kVecs; i += 2) load_32(row + k + i * kPer, v[i], v[i + 1]);
      return;
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int at = k + i * kPer;
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (VEC && at + kPer <= K) {
        v[i] = *reinterpret_cast<const uint4*>(row + at);
      } else if (at < K) {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          if (at + e < K) {
            if constexpr (sizeof(T) == 2)
              w[e >> 1] |= static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(row + at + e)) << (16 * (e & 1));
            else
              w[e] = __float_as_uint(row[at + e]);
          }
        }
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  // Pair i (values 2i, 2i + 1) as fp32.
  __device__ __forceinline__ unsigned long long pair(int i) const {
    if constexpr (sizeof(T) == 2) {
      const uint4& a = v[i >> 2];
      const uint32_t w = (i & 3) == 0 ? a.x : (i & 3) == 1 ? a.y : (i & 3) == 2 ? a.z : a.w;
      return pack_f32x2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    } else {
      const uint4& a = v[i >> 1];
      return (i & 1) ? pack_f32x2(__uint_as_float(a.z), __uint_as_float(a.w))
                     : pack_f32x2(__uint_as_float(a.x), __uint_as_float(a.y));
    }
  }
  // The largest magnitude's fp32 bits (NaN above infinity above numbers).
  __device__ __forceinline__ uint32_t absmax() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      if constexpr (sizeof(T) == 2) {
        const uint32_t a = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu),
                                    __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
        m = max(m, max(a & 0xffff0000u, a << 16));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max(m, w[e] & 0x7fffffffu);
      }
    }
    return m;
  }
};

// 8 fp32 values as e2m1 codes, the first in the lowest 4 bits.
__device__ __forceinline__ uint32_t pack_e2m1(const unsigned long long (&y)[4]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(lo_f32(y[0])), "f"(hi_f32(y[0])), "f"(lo_f32(y[1])), "f"(hi_f32(y[1])), "f"(lo_f32(y[2])),
        "f"(hi_f32(y[2])), "f"(lo_f32(y[3])), "f"(hi_f32(y[3])));
  return r;
}
// e4m3 code of a number from 0 to 448, and what a code stands for.
__device__ __forceinline__ uint32_t to_e4m3(float v) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
  return r & 0xffu;
}
__device__ __forceinline__ float from_e4m3(uint32_t code) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<unsigned short>(code)));
  return __low2float(*reinterpret_cast<const __half2*>(&h));
}

// An NV row's power of two: 2^max(floor(log2 absmax) - 10, -100), so that absmax
// / 6 is 170 to 341 of it, inside e4m3.
struct RowStep {
  float value, inverse;
  bool plain;
  __device__ __forceinline__ explicit RowStep(uint32_t absmax) {
    const int e = static_cast<int>(absmax >> 23);
    plain = e != 255;
    const int f = max(e - 10, 27);
    value = plain ? __uint_as_float(static_cast<uint32_t>(f) << 23) : __uint_as_float(0x7fffffffu);
    inverse = __uint_as_float(static_cast<uint32_t>(254 - f) << 23);
  }
};

// One unit's 8 bytes of codes; its block's scale byte.
template <int FMT, typename Tin>
__device__ __forceinline__ uint2 quantize(const Unit<Tin>& x, const RowStep& row, uint32_t* byte) {
  uint32_t m = x.absmax();
  uint2 out = make_uint2(0u, 0u);
  unsigned long long y[2][4];
  if (FMT == RFX_FP4_MX) {
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    const int e = static_cast<int>(m >> 23);
    *byte = e == 255 ? 255u : static_cast<uint32_t>(max(e - 2, 0));
    // x / 2^e is exact
    const float inv = __uint_as_float((254u - (e == 255 ? 127u : *byte)) << 23);
    const unsigned long long inv2 = pack_f32x2(inv, inv);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i >> 2][i & 3] = mul_f32x2(x.pair(i), inv2);
    if (e != 255) out = make_uint2(pack_e2m1(y[0]), pack_e2m1(y[1]));
  } else {
    *byte = row.plain ? to_e4m3(__fmul_rn(__fdiv_rn(__uint_as_float(m), 6.f), row.inverse)) : 0u;
    const float d = __fmul_rn(from_e4m3(*byte), row.value);
    // x / d, correctly rounded: a product with the correctly rounded 1 / d,
    // then one step with the exact remainder (Markstein 1990).  d lies in
    // 2^-109 .. 2^126; a quotient so small that its remainder underflows is 0.
    const float r = __frcp_rn(d);
    const unsigned long long r2 = pack_f32x2(r, r), nd2 = pack_f32x2(-d, -d);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned long long v = x.pair(i), q = mul_f32x2(v, r2);
      y[i >> 2][i & 3] = fma_f32x2(fma_f32x2(q, nd2, v), r2, q);
    }
    if (*byte != 0) out = make_uint2(pack_e2m1(y[0]), pack_e2m1(y[1]));
  }
  return out;
}

// Stores a unit's codes (k its first value) and, gathered over the lanes, scale
// bytes; every lane of a warp takes part.
template <int FMT>
__device__ __forceinline__ void store_unit(const QuantFp4Params& p, uint8_t* q, uint8_t* scale, int u, uint2 codes,
                                           uint32_t byte) {
  constexpr int kLanes = FMT == RFX_FP4_MX ? 8 : 4;  // lanes of 4 blocks
  const int lane = threadIdx.x & 31, k = u * kUnit;
  uint32_t w = byte << (FMT == RFX_FP4_MX ? 8 * ((lane >> 1) & 3) : 8 * (lane & 3));
  if (FMT == RFX_FP4_MX) {
    w |= __shfl_xor_sync(0xffffffffu, w, 2);
    w |= __shfl_xor_sync(0xffffffffu, w, 4);
  } else {
    w |= __shfl_xor_sync(0xffffffffu, w, 1);
    w |= __shfl_xor_sync(0xffffffffu, w, 2);
  }
  const int group = u / kLanes;
  if (u % kLanes == 0 && group < p.tiles.k_tiles) *reinterpret_cast<uint32_t*>(scale + group * 512l) = w;
  if (k + kUnit <= p.K) {
    *reinterpret_cast<uint2*>(q + k / 2) = codes;
  } else if (k < p.K) {
    const int n = (p.K - k + 1) / 2;  // bytes
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) q[k / 2 + i] = static_cast<uint8_t>((i < 4 ? codes.x : codes.y) >> (8 * (i & 3)));
  }
}

constexpr int kWarpRows = 4;  // rows of a CTA at a time where a warp has one
constexpr int rows_at_a_time(int tpr) { return tpr == 32 ? kWarpRows : 1; }
// The longest rows that are held: 64 registers a thread, so that 768 of 16384 values are
// under way at once (left to itself the compiler takes 116, and 10.8 us instead of 9.3);
// shorter ones lose more by it than they gain (4304 values: 5.7 us instead of 4.9).
constexpr int ctas_per_sm(int tpr, int nu, int bytes) { return tpr == 256 && nu == 4 && bytes == 2 ? 4 : 0; }

// NU units per thread of a row's TPR threads; NU = 0: rows of any length, read
// a second time where NV needs their maximum first.
template <typename Tin, int FMT, int TPR, int NU, int VEC>
__global__ void __launch_bounds__(TPR* rows_at_a_time(TPR), ctas_per_sm(TPR, NU, sizeof(Tin)))
    quant_fp4_kernel(const QuantFp4Params p) {
  __shared__ uint32_t part[2][TPR / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const long step = static_cast<long>(gridDim.x) * rows_at_a_time(TPR);
  long t = static_cast<long>(blockIdx.x) * rows_at_a_time(TPR) + (TPR == 32 ? threadIdx.x >> 5 : 0);
  for (int i = 0; t < p.T; t += step, i ^= 1) {
    const Tin* x = static_cast<const Tin*>(p.x) + t * p.ldx;
    uint8_t* q = p.q + t * p.ldq;
    uint8_t* scale = p.scale + p.tiles.row(t);
    constexpr int kHeld = NU == 0 ? 1 : NU;
    Unit<Tin> v[kHeld];
    uint32_t m = 0;
    const int turns = NU == 0 ? (p.K + TPR * kUnit - 1) / (TPR * kUnit) : 0;
    if (NU > 0) {
#pragma unroll
      for (int c = 0; c < kHeld; ++c) v[c].template load<VEC>(x, (c * TPR + tid) * kUnit, p.K);
    }
    if (FMT == RFX_FP4_NV) {
      if (NU > 0) {
#pragma unroll
        for (int c = 0; c < kHeld; ++c) m = max(m, v[c].absmax());
      } else {
        for (int c = 0; c < turns; ++c) {
          v[0].template load<VEC>(x, (c * TPR + tid) * kUnit, p.K);
          m = max(m, v[0].absmax());
        }
      }
      m = __reduce_max_sync(0xffffffffu, m);
      if (TPR > 32) {
        if ((threadIdx.x & 31) == 0) part[i][threadIdx.x >> 5] = m;
        __syncthreads();
        m = part[i][0];
#pragma unroll
        for (int w = 1; w < TPR / 32; ++w) m = max(m, part[i][w]);
      }
    }
    const RowStep row(m);
    if (NU > 0) {
#pragma unroll
      for (int c = 0; c < kHeld; ++c) {
        uint32_t byte;
        const uint2 codes = quantize<FMT>(v[c], row, &byte);
        store_unit<FMT>(p, q, scale, c * TPR + tid, codes, byte);
      }
    } else {
      for (int c = 0; c < turns; ++c) {
        uint32_t byte;
        v[0].template load<VEC>(x, (c * TPR + tid) * kUnit, p.K);
        const uint2 codes = quantize<FMT>(v[0], row, &byte);
        store_unit<FMT>(p, q, scale, c * TPR + tid, codes, byte);
      }
    }
    if (FMT == RFX_FP4_NV && tid == 0) p.row_scale[t] = row.value;
  }
}

struct DequantFp4Params {
  int T, K, units;  // units of a row
  const uint8_t* q;
  long ldq;
  const uint8_t* scale;
  const float* row_scale;
  void* y;
  long ldy;
  ScaleTiles tiles;
};

// 8 codes as fp32 pairs.
__device__ __forceinline__ void unpack_e2m1(uint32_t codes, float (&v)[8]) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ void put(float* y, float v) { *y = v; }
__device__ __forceinline__ void put(__nv_bfloat16* y, float v) { *y = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put8(float* y, const float (&v)[8]) {
  reinterpret_cast<float4*>(y)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(y)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void put8(__nv_bfloat16* y, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(y) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                            pack_bf16x2(v[6], v[7]));
}
template <int VEC>
__device__ __forceinline__ void put16(float* y, const float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; i += 8) {
    const uint4 a = make_uint4(__float_as_uint(v[i]), __float_as_uint(v[i + 1]), __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3]));
    const uint4 b = make_uint4(__float_as_uint(v[i + 4]), __float_as_uint(v[i + 5]), __float_as_uint(v[i + 6]), __float_as_uint(v[i + 7]));
    if (VEC == 32) {
      store_32(y + i, a, b);
    } else {
      *reinterpret_cast<uint4*>(y + i) = a;
      *reinterpret_cast<uint4*>(y + i + 4) = b;
    }
  }
}
template <int VEC>
__device__ __forceinline__ void put16(__nv_bfloat16* y, const float (&v)[16]) {
  const uint4 a = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  const uint4 b = make_uint4(pack_bf16x2(v[8], v[9]), pack_bf16x2(v[10], v[11]), pack_bf16x2(v[12], v[13]), pack_bf16x2(v[14], v[15]));
  if (VEC == 32) {
    store_32(y, a, b);
  } else {
    *reinterpret_cast<uint4*>(y) = a;
    *reinterpret_cast<uint4*>(y + 8) = b;
  }
}

// a * b of a few bits by a float, rounded once to the output type: for bf16 to fp32 so
// that the last bit is odd where bits are lost (of the two neighbours one is), which keeps
// the second rounding from seeing a tie that is none.
template <typename Tout>
__device__ __forceinline__ float product(float a, float b) {
  if (sizeof(Tout) == 4) return __fmul_rn(a, b);
  const float lo = __fmul_rd(a, b), hi = __fmul_ru(a, b);
  return (__float_as_uint(lo) & 1u) ? lo : hi;
}
// 16 values of a row whose scale is no power of two (`left`: those before the row's end),
// 8 at a time, so that the rows that the quantizer makes lose no registers to it.
template <typename Tout, int VEC>
__device__ __forceinline__ void dequant_any_scale(Tout* y, int left, uint2 codes, float block_scale, float row_scale) {
#pragma unroll 1
  for (int h = 0; h < 16; h += 8) {
    float v[8];
    unpack_e2m1(h ? codes.y : codes.x, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = product<Tout>(v[e] * block_scale, row_scale);
    if (VEC && left >= kUnit) {
      put8(y + h, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (h + e < left) put(y + h + e, v[e]);
    }
  }
}

// A CTA takes 256 / TPR rows and kTurn units per thread of them at a time: all codes and
// scales are asked for before the first is used.
template <typename Tout, int FMT, int TPR, int VEC>
__global__ void __launch_bounds__(256) dequant_fp4_kernel(const DequantFp4Params p) {
  constexpr int kRows = 256 / TPR, kTurn = TPR == 256 ? 2 : 1, kChunk = kTurn * TPR;
  // bf16 rows whose scale is no power of two are written a second time, over the first: with
  // the products that they need in one place with the others, 768 x 16384 of the quantizer's
  // rows take 7.0 to 8.1 us instead of 6.7 (fp32 10.8 instead of 10.5: in one place).
  constexpr bool kAgain = FMT == RFX_FP4_NV && sizeof(Tout) == 2;
  pdl_wait();
  pdl_launch_dependents();
  const int chunks = (p.units + kChunk - 1) / kChunk;
  const long total = (static_cast<long>(p.T) + kRows - 1) / kRows * chunks;
  for (long i = blockIdx.x; i < total; i += gridDim.x) {
    const int rows = static_cast<int>(chunks == 1 ? i : i / chunks), t = rows * kRows + static_cast<int>(threadIdx.x) / TPR;
    const int u0 = static_cast<int>(i - static_cast<long>(rows) * chunks) * kChunk + threadIdx.x % TPR;
    if (t >= p.T) continue;
    const uint8_t* q = p.q + t * p.ldq;
    const uint8_t* scale = p.scale + p.tiles.row(t);
    const float row_scale = FMT == RFX_FP4_NV ? p.row_scale[t] : 1.f;
    // a power of two (the quantizer makes no others) that times any block's scale neither
    // overflows nor loses bits: one product per value
    const uint32_t row_bits = __float_as_uint(row_scale);
    const bool power = (row_bits & 0x007fffffu) == 0u && row_bits >= 1u << 23 && row_bits <= (119u + 127u) << 23;
    Tout* y = static_cast<Tout*>(p.y) + t * p.ldy;
    uint2 codes[kTurn];
    uint32_t byte[kTurn];
#pragma unroll
    for (int c = 0; c < kTurn; ++c) {
      const int u = u0 + c * TPR, k = u * kUnit, j = FMT == RFX_FP4_MX ? u >> 1 : u;
      codes[c] = make_uint2(0u, 0u);
      byte[c] = 0;
      if (u >= p.units) continue;
      byte[c] = scale[(j >> 2) * 512l + (j & 3)];
      if (k + kUnit <= p.K) {
        codes[c] = *reinterpret_cast<const uint2*>(q + k / 2);
      } else {
        const int n = (p.K - k + 1) / 2;
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          const uint32_t w = b < n ? static_cast<uint32_t>(q[k / 2 + b]) << (8 * (b & 3)) : 0u;
          (b < 4 ? codes[c].x : codes[c].y) |= w;
        }
      }
    }
#pragma unroll
    for (int c = 0; c < kTurn; ++c) {
      const int u = u0 + c * TPR, k = u * kUnit;
      if (u >= p.units) continue;
      // 2^(byte - 127), of byte 0 a subnormal number; an NV scale's 4 bits times a power of
      // two, and a code's 3 bits times either, are exact
      const float s = FMT == RFX_FP4_MX ? (byte[c] == 255 ? __uint_as_float(0x7fffffffu)
                                           : byte[c] == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte[c] << 23))
                                        : from_e4m3(byte[c]) * (kAgain || power ? row_scale : 1.f);
      const unsigned long long s2 = pack_f32x2(s, s);
      float v[16];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[8];
        unpack_e2m1(h ? codes[c].y : codes[c].x, x);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const unsigned long long y = mul_f32x2(pack_f32x2(x[e], x[e + 1]), s2);
          v[8 * h + e] = lo_f32(y);
          v[8 * h + e + 1] = hi_f32(y);
        }
      }
      if (FMT == RFX_FP4_NV && !kAgain && !power) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = product<Tout>(v[e], row_scale);
      }
      if (VEC && k + kUnit <= p.K) {
        put16<VEC>(y + k, v);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (k + e < p.K) put(y + k + e, v[e]);
      }
    }
    if (kAgain && !power) {
#pragma unroll
      for (int c = 0; c < kTurn; ++c) {
        const int u = u0 + c * TPR, k = u * kUnit;
        if (u < p.units) dequant_any_scale<Tout, VEC>(y + k, p.K - k, codes[c], from_e4m3(byte[c]), row_scale);
      }
    }
  }
}

// ------------------------------------------------------------ host side ---
bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
int block_of(int format) { return format == RFX_FP4_MX ? 32 : 16; }
ScaleTiles tiles_of(int T, int K, int format, int rows_per_part) {
  const int per = rows_per_part > 0 ? rows_per_part : std::max(T, 1);
  return ScaleTiles{per, (per - 1) / 128 + 1, (K - 1) / (4 * block_of(format)) + 1};
}
Rows scale_rows(const void* scale, int T, int K, int format, int rows_per_part) {
  return Rows{scale, 1, 0, fp4_scale_bytes(T, K, format, rows_per_part)};
}

struct FpShape {
  int tpr, nu;
};
// Threads per row: a warp where there are rows enough for every scheduler and
// they are short, else as many as leave each one unit, up to 256.
FpShape fp4_shape(int T, int K) {
  const int units = (K + kUnit - 1) / kUnit;
  if (units > 1024) return {256, 0};
  if (units <= 32 || (units <= 128 && T >= 592)) return {32, units <= 32 ? 1 : units <= 64 ? 2 : 4};
  if (units <= 128 || (units <= 512 && T >= 296)) return {128, units <= 128 ? 1 : units <= 256 ? 2 : 4};
  return {256, units <= 256 ? 1 : units <= 512 ? 2 : 4};
}

template <typename Tin, int FMT, int VEC>
const void* quant_ptr(FpShape s) {
#define RFX_FP4_SHAPE(TPR, NU) \
  if (s.tpr == TPR && s.nu == NU) return reinterpret_cast<const void*>(quant_fp4_kernel<Tin, FMT, TPR, NU, VEC>)
  RFX_FP4_SHAPE(32, 1);
  RFX_FP4_SHAPE(32, 2);
  RFX_FP4_SHAPE(32, 4);
  RFX_FP4_SHAPE(128, 1);
  RFX_FP4_SHAPE(128, 2);
  RFX_FP4_SHAPE(128, 4);
  RFX_FP4_SHAPE(256, 1);
  RFX_FP4_SHAPE(256, 2);
  RFX_FP4_SHAPE(256, 4);
#undef RFX_FP4_SHAPE
  return reinterpret_cast<const void*>(quant_fp4_kernel<Tin, FMT, 256, 0, VEC>);
}
template <typename Tin, int FMT>
const void* quant_vec(int vec, FpShape s) {
  return vec == 32 ? quant_ptr<Tin, FMT, 32>(s) : vec == 16 ? quant_ptr<Tin, FMT, 16>(s) : quant_ptr<Tin, FMT, 0>(s);
}
template <typename Tin>
const void* quant_kernel(int format, int vec, FpShape s) {
  return format == RFX_FP4_MX ? quant_vec<Tin, RFX_FP4_MX>(vec, s) : quant_vec<Tin, RFX_FP4_NV>(vec, s);
}
template <typename Tout, int FMT, int TPR>
const void* dequant_vec(int vec) {
  return vec == 32   ? reinterpret_cast<const void*>(dequant_fp4_kernel<Tout, FMT, TPR, 32>)
         : vec == 16 ? reinterpret_cast<const void*>(dequant_fp4_kernel<Tout, FMT, TPR, 16>)
                     : reinterpret_cast<const void*>(dequant_fp4_kernel<Tout, FMT, TPR, 0>);
}
template <typename Tout, int FMT>
const void* dequant_rows(int tpr, int vec) {
  return tpr == 32 ? dequant_vec<Tout, FMT, 32>(vec) : tpr == 64 ? dequant_vec<Tout, FMT, 64>(vec) : dequant_vec<Tout, FMT, 256>(vec);
}
template <typename Tout>
const void* dequant_kernel(int format, int tpr, int vec) {
  return format == RFX_FP4_MX ? dequant_rows<Tout, RFX_FP4_MX>(tpr, vec) : dequant_rows<Tout, RFX_FP4_NV>(tpr, vec);
}
// Bytes at a time: what the rows' start and stride allow.
int vec_of(const void* p, long stride, int rows) {
  for (int bytes = 32; bytes >= 16; bytes /= 2)
    if (aligned(p, bytes) && (rows == 1 || stride % bytes == 0)) return bytes;
  return 0;
}

// What quantizing and its inverse have in common; `wide` is the bf16 / fp32 side.
int check_rows(const char* what, int T, int K, int format, int dtype, int rows_per_part, const void* wide, long ldw,
               const void* q, long ldq, const void* scale, const float* row_scale) {
  if (T < 0 || T > kMaxRows || K < 1 || K > kMaxK)
    return set_error(RFX_E_INVAL, "%s: need 0<=T<=2^30 and 1<=K<=%d (T=%d K=%d)", what, kMaxK, T, K);
  if (format != RFX_FP4_MX && format != RFX_FP4_NV) return set_error(RFX_E_INVAL, "%s: format must be MX or NV", what);
  if (dtype != kDtypeBF16 && dtype != kDtypeF32) return set_error(RFX_E_INVAL, "%s: dtype must be bf16 or f32", what);
  if (rows_per_part < 0 || (rows_per_part > 0 && T % rows_per_part))
    return set_error(RFX_E_INVAL, "%s: T must be whole parts of rows_per_part rows (T=%d rows_per_part=%d)", what, T,
                     rows_per_part);
  if (T == 0) return RFX_OK;
  if (!wide || !q || !scale) return set_error(RFX_E_INVAL, "%s: null pointer", what);
  if ((format == RFX_FP4_NV) != (row_scale != nullptr))
    return set_error(RFX_E_INVAL, "%s: row_scale goes with RFX_FP4_NV, and only with it", what);
  if (ldw < K || ldq < (K + 1) / 2 || ldq % 16 || !aligned(q, 16) || !aligned(scale, 16))
    return set_error(RFX_E_INVAL,
                     "%s: a row stride below the row, or 4-bit rows or scales off 16-byte boundaries", what);
  if (!aligned(wide, dtype == kDtypeBF16 ? 2 : 4) || !aligned(row_scale, 4))
    return set_error(RFX_E_INVAL, "%s: misaligned pointer", what);
  return RFX_OK;
}

}  // namespace

long fp4_scale_bytes(int T, int K, int format, int rows_per_part) {
  if (T <= 0) return 0;
  const ScaleTiles s = tiles_of(T, K, format, rows_per_part);
  return static_cast<long>((T - 1) / s.per_part + 1) * s.tiles_per_part * s.k_tiles * 512l;
}

int validate_quant_fp4(const rfx_quant_fp4_desc& d) {
  const int rc = check_rows("rfx_quant_fp4", d.T, d.K, d.format, d.in_dtype, d.rows_per_part, d.x, d.ldx, d.q, d.ldq,
                            d.scale, d.row_scale);
  if (rc || d.T == 0) return rc;
  const long esz = d.in_dtype == kDtypeBF16 ? 2 : 4;
  const Rows x{d.x, d.T, d.ldx * esz, d.K * esz}, q{d.q, d.T, d.ldq, (d.K + 1) / 2};
  const Rows s = scale_rows(d.scale, d.T, d.K, d.format, d.rows_per_part), r{d.row_scale, 1, 0, d.T * 4l};
  if (rows_shared(q, x) || rows_shared(s, x) || rows_shared(r, x) || rows_shared(q, s) || rows_shared(q, r) ||
      rows_shared(s, r))
    return set_error(RFX_E_INVAL, "rfx_quant_fp4: x, q, scale and row_scale share memory");
  return RFX_OK;
}

int launch_quant_fp4(const rfx_quant_fp4_desc& d, cudaStream_t stream, bool pdl) {
  const int rc = validate_quant_fp4(d);
  if (rc || d.T == 0) return rc;
  QuantFp4Params p{d.T, d.K, d.x, d.ldx, static_cast<uint8_t*>(d.q), d.ldq, static_cast<uint8_t*>(d.scale), d.row_scale,
                   tiles_of(d.T, d.K, d.format, d.rows_per_part)};
  const long esz = d.in_dtype == kDtypeBF16 ? 2 : 4;
  const int vec = vec_of(d.x, d.ldx * esz, d.T);
  const FpShape s = fp4_shape(d.T, d.K);
  const void* fn = d.in_dtype == kDtypeBF16 ? quant_kernel<__nv_bfloat16>(d.format, vec, s) : quant_kernel<float>(d.format, vec, s);
  int nsm = 148;
  rfx_num_sms(&nsm);
  const int rows = rows_at_a_time(s.tpr), threads = s.tpr * rows;
  const long ctas = (d.T + rows - 1l) / rows;
  return launch_kernel(fn, dim3(static_cast<unsigned>(std::min(ctas, static_cast<long>(nsm) * (2048 / threads)))),
                       dim3(threads), 0, stream, pdl, 1, p);
}

int validate_dequant_fp4(const rfx_dequant_fp4_desc& d) {
  const int rc = check_rows("rfx_dequant_fp4", d.T, d.K, d.format, d.out_dtype, d.rows_per_part, d.y, d.ldy, d.q, d.ldq,
                            d.scale, d.row_scale);
  if (rc || d.T == 0) return rc;
  const long esz = d.out_dtype == kDtypeBF16 ? 2 : 4;
  const Rows y{d.y, d.T, d.ldy * esz, d.K * esz};
  if (rows_shared(y, {d.q, d.T, d.ldq, (d.K + 1) / 2}) ||
      rows_shared(y, scale_rows(d.scale, d.T, d.K, d.format, d.rows_per_part)) ||
      rows_shared(y, {d.row_scale, 1, 0, d.T * 4l}))
    return set_error(RFX_E_INVAL, "rfx_dequant_fp4: y shares memory with an input");
  return RFX_OK;
}

int launch_dequant_fp4(const rfx_dequant_fp4_desc& d, cudaStream_t stream, bool pdl) {
  const int rc = validate_dequant_fp4(d);
  if (rc || d.T == 0) return rc;
  DequantFp4Params p{d.T, d.K, (d.K + kUnit - 1) / kUnit, static_cast<const uint8_t*>(d.q), d.ldq,
                     static_cast<const uint8_t*>(d.scale), d.row_scale, d.y, d.ldy,
                     tiles_of(d.T, d.K, d.format, d.rows_per_part)};
  const long esz = d.out_dtype == kDtypeBF16 ? 2 : 4;
  const int vec = vec_of(d.y, d.ldy * esz, d.T);
  const int tpr = p.units <= 32 ? 32 : p.units <= 64 ? 64 : 256;
  const void* fn = d.out_dtype == kDtypeBF16 ? dequant_kernel<__nv_bfloat16>(d.format, tpr, vec) : dequant_kernel<float>(d.format, tpr, vec);
  int nsm = 148;
  rfx_num_sms(&nsm);
  const long rows = 256 / tpr, chunk = tpr == 256 ? 512 : tpr;
  const long ctas = (d.T + rows - 1) / rows * ((p.units + chunk - 1) / chunk);
  return launch_kernel(fn, dim3(static_cast<unsigned>(std::min(ctas, 8l * nsm))), dim3(256), 0, stream, pdl, 1, p);
}

}  // namespace rfx

extern "C" int rfx_quant_fp4(const rfx_quant_fp4_desc* d, void* stream) {
  using namespace rfx;
  if (!d) return set_error(RFX_E_INVAL, "rfx_quant_fp4: null descriptor");
  return launch_quant_fp4(*d, static_cast<cudaStream_t>(stream), pdl_enabled());
}

extern "C" int rfx_dequant_fp4(const rfx_dequant_fp4_desc* d, void* stream) {
  using namespace rfx;
  if (!d) return set_error(RFX_E_INVAL, "rfx_dequant_fp4: null descriptor");
  return launch_dequant_fp4(*d, static_cast<cudaStream_t>(stream), pdl_enabled());
}
