// What the epilogues of the quantized linears' tiles have in common: activations
// and stores of a warp's outputs.
#pragma once
#include "ptx.cuh"

namespace rfx {

enum { kActNone, kActSilu, kActGelu, kActGeglu };


// GELU-tanh as v * sigmoid(2u), u = sqrt(2/pi) (v + 0.044715 v^3), since
// 0.5 (1 + tanh u) = 1 / (1 + e^-2u): one exponential and one reciprocal, the
// exponent formed in base 2.  An e^-2u that overflows leaves v * 0.
__device__ __forceinline__ float gelu_ex2(float v) {
  constexpr float kA = -2.3022081986f;  // -2 sqrt(2/pi) log2(e)
  constexpr float kB = kA * 0.044715f;
  return v * rcp_approx(1.f + ex2_approx(v * fmaf(kB, v * v, kA)));
}
__device__ __forceinline__ float silu_ex2(float v) {
  return v * rcp_approx(1.f + ex2_approx(v * -1.4426950409f));
}

template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if (ACT == kActSilu) return silu_ex2(v);
  if (ACT == kActGelu) return gelu_ex2(v);
  return v;
}

__device__ __forceinline__ void put1(float* y, float v) { *y = v; }
__device__ __forceinline__ void put1(__nv_bfloat16* y, float v) { *y = __float2bfloat16_rn(v); }

// Whether every epilogue thread's wait succeeded (also a barrier of the 256).
__device__ __forceinline__ bool epi_agree(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(ok ? 1u : 0u)
      : "memory");
  return all != 0;
}

// 16 outputs packed as they are stored.
__device__ __forceinline__ void pack16(const float (&v)[16], uint32_t* w, const __nv_bfloat16*) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void pack16(const float (&v)[16], uint32_t* w, const float*) {
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i]);
}

// 32 staged rows of 64 bytes to global rows of `pitch` bytes, in units of U: a
// lane keeps its column of units and walks the rows, several of them on their way.
template <typename U>
__device__ __forceinline__ void store_units(const uint8_t* st, uint8_t* y, long pitch, int rows, int bytes, int lane) {
  constexpr int kCols = 64 / static_cast<int>(sizeof(U)), kRowsPer = 32 / kCols, kBatch = sizeof(U) == 8 ? 4 : 8;
  const int byte = lane % kCols * static_cast<int>(sizeof(U)), r0 = lane / kCols;
  const int end = byte < bytes ? min(rows, 32) : 0;
  y += r0 * pitch + byte;
#pragma unroll 1
  for (int r = r0; r < 32; r += kBatch * kRowsPer, y += kBatch * kRowsPer * pitch) {
    U v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int q = r + i * kRowsPer;
      v[i] = *reinterpret_cast<const U*>(st + q * 64 + (((byte >> 4) ^ ((q >> 1) & 3)) << 4) + (byte & 15));
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (r + i * kRowsPer < end) *reinterpret_cast<U*>(y + i * kRowsPer * pitch) = v[i];
  }
}

// A warp's 32 rows x 64 bytes of outputs (lane = row) to memory through its own
// 2 KB of shared memory: one TMA store where y's rows begin on 16-byte
// boundaries (`tma`), else in coalesced units of the 2, 4 or 8 bytes that the
// rows allow.  The copy clips rows past T, and columns past F only in units of 16
// bytes, so a last piece that ends inside such a unit goes out that way too.
// `rows` and `n` are the live rows and
// columns from (t, o).
template <typename Tout, typename Params>
__device__ __forceinline__ void store_part(const Params& p, const CUtensorMap* tmY, uint8_t* st,
                                           const uint32_t (&w)[16], int t, int o, int rows, int n, bool tma, int lane) {
  constexpr int kCols = 64 / static_cast<int>(sizeof(Tout));
  if (n <= 0 || rows <= 0) return;
  if (tma) {
    if (lane == 0) bulk_wait_read();  // the previous store has left the buffer
    __syncwarp();
    tma = n >= kCols || n * sizeof(Tout) % 16 == 0;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(st + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  if (tma) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(tmY, st, o, t);
      bulk_commit();
    }
  } else {
    __syncwarp();
    const long pitch = p.ldy * static_cast<long>(sizeof(Tout));
    uint8_t* y = reinterpret_cast<uint8_t*>(static_cast<Tout*>(p.y) + t * p.ldy + o);
    const int bytes = min(n, kCols) * static_cast<int>(sizeof(Tout));
    const uint32_t odd = static_cast<uint32_t>(pitch) | static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p.y)) |
                         static_cast<uint32_t>(bytes);
    if (odd % 8 == 0)
      store_units<uint2>(st, y, pitch, rows, bytes, lane);
    else if (sizeof(Tout) == 4 || odd % 4 == 0)
      store_units<uint32_t>(st, y, pitch, rows, bytes, lane);
    else
      store_units<uint16_t>(st, y, pitch, rows, bytes, lane);
    __syncwarp();
  }
}

}  // namespace rfx
