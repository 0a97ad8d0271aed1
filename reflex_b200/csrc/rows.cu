// Row operators of the int8 layer path: rows to int8 with one scale per row,
// and what lies between two transformer blocks (the norm of a block's output,
// its gate and residual scale, the residual add, the next block's norm).
//
// A row is read from memory once and stays in the registers of the threads
// that read it, through every reduction, until its outputs are written: TPR
// threads per row, NV vectors of 8 elements per thread.
//
// Both operators would be bound by memory traffic; what keeps them from it is
// latency.  With everything on, block_norm of 3200 x 1024 bf16 to int8 has 5
// warps on a scheduler, which issues in 52 % of its active clocks: each warp
// waits for its loads, then for dependent arithmetic (340 instructions in each of
// a row's four warps) and for the shuffles and shared memory of up to three
// reductions in a chain.  768 x 2048 fp32 issues in 29 %, mostly waiting for the
// loads and the reductions of 5 or 6 rows per SM.  Quantizing 768 rows of 16384
// issues in 56 %, and the rows are whole: 296 CTAs take 2 or 3 of them, 6 on the
// busiest SM where 5.2 is the mean (888 rows, 6 on each, take 10.9 us).
// Measured: int8 rows of 768 x 16384 bf16 10.4 us (3.6 TB/s); block_norm 3200 x
// 1024 bf16 to int8 9.3 us (2.5 TB/s), 768 x 2048 fp32 7.8 us (3.2 TB/s), 50 x 1024
// 2.6 us.  Rows off the 16-byte grid take element accesses: 3200 x 1025 25 us.
#include "quant_i8.cuh"
#include "rfx_internal.h"

#include <algorithm>

namespace rfx {
namespace {

constexpr int kMaxRow = 16384;

__device__ __forceinline__ void store_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ void load_vec(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  const float4 b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void store_vec(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// 8 elements as loaded; they become fp32 only where they are used, so that a
// row can be on its way while another one is computed.
template <typename T>
struct Raw;
template <>
struct Raw<__nv_bfloat16> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void set(int e, __nv_bfloat16 x) {
    const uint32_t b = static_cast<uint32_t>(__bfloat16_as_ushort(x)) << (16 * (e & 1));
    uint32_t& w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
    w = (e & 1) ? ((w & 0xffffu) | b) : ((w & 0xffff0000u) | b);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ __forceinline__ void pairs(unsigned long long (&f)[4]) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[i] = pack_f32x2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  __device__ __forceinline__ void round(const unsigned long long (&f)[4]) {
    v = make_uint4(pack_bf16x2(lo_f32(f[0]), hi_f32(f[0])), pack_bf16x2(lo_f32(f[1]), hi_f32(f[1])),
                   pack_bf16x2(lo_f32(f[2]), hi_f32(f[2])), pack_bf16x2(lo_f32(f[3]), hi_f32(f[3])));
  }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = v; }
  __device__ __forceinline__ __nv_bfloat16 at(int e) const {
    const uint32_t w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
    return __ushort_as_bfloat16(static_cast<unsigned short>((e & 1) ? w >> 16 : w & 0xffffu));
  }
  // the largest magnitude's fp32 bit pattern (NaN above infinity above numbers)
  __device__ __forceinline__ uint32_t absmax() const {
    const uint32_t w[4] = {v.x & 0x7fff7fffu, v.y & 0x7fff7fffu, v.z & 0x7fff7fffu, v.w & 0x7fff7fffu};
    const uint32_t m = __vmaxu2(__vmaxu2(w[0], w[1]), __vmaxu2(w[2], w[3]));
    return max(m & 0xffff0000u, m << 16);
  }
};
template <>
struct Raw<float> {
  float f8[8];
  __device__ __forceinline__ void load(const float* p) { load_vec(p, f8); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < 8; ++e) f8[e] = 0.f;
  }
  __device__ __forceinline__ void set(int e, float x) { f8[e] = x; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = f8[e];
  }
  __device__ __forceinline__ void pairs(unsigned long long (&f)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = pack_f32x2(f8[2 * i], f8[2 * i + 1]);
  }
  __device__ __forceinline__ void round(const unsigned long long (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f8[2 * i] = lo_f32(f[i]);
      f8[2 * i + 1] = hi_f32(f[i]);
    }
  }
  __device__ __forceinline__ void store(float* p) const { store_vec(p, f8); }
  __device__ __forceinline__ float at(int e) const { return f8[e]; }
  __device__ __forceinline__ uint32_t absmax() const {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(f8[e]) & 0x7fffffffu);
    return m;
  }
};

// Where element e of vector c of thread `tid` of a row lies.  VEC: 8
// neighbours per thread (16-byte accesses; K % 8 == 0 and aligned rows);
// otherwise threads take single neighbours, so that a warp's accesses stay
// contiguous at any length and alignment.
template <int TPR, bool VEC>
__device__ __forceinline__ int column(int tid, int c, int e) {
  return VEC ? (c * TPR + tid) * 8 + e : (c * 8 + e) * TPR + tid;
}

// Vector c of a thread's part of a row of column values; 0 past the row's end.
template <int TPR, bool VEC>
__device__ __forceinline__ void load_columns(const float* row, int K, int tid, int c, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  if (VEC) {
    const int k = column<TPR, VEC>(tid, c, 0);
    if (k < K) load_vec(row + k, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = column<TPR, VEC>(tid, c, e);
      if (k < K) v[e] = row[k];
    }
  }
}
template <int TPR, bool VEC, typename T>
__device__ __forceinline__ void store_columns(T* row, int K, int tid, int c, const float (&v)[8]) {
  if (VEC) {
    const int k = column<TPR, VEC>(tid, c, 0);
    if (k < K) store_vec(row + k, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = column<TPR, VEC>(tid, c, e);
      if (k < K) store_f(row + k, v[e]);
    }
  }
}
// A thread's part of a row as it lies in memory; 0 past the row's end.
template <int TPR, int NV, bool VEC, typename T>
__device__ __forceinline__ void load_raw(const T* row, int K, int tid, Raw<T> (&v)[NV]) {
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    v[c].zero();
    if (VEC) {
      const int k = column<TPR, VEC>(tid, c, 0);
      if (k < K) v[c].load(row + k);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = column<TPR, VEC>(tid, c, e);
        if (k < K) v[c].set(e, row[k]);
      }
    }
  }
}
// Sum / unsigned maximum over a row's threads; the order of the sum is fixed.
// `part` is this reduction's own slot array, so one barrier is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* part) {
  v = warp_sum(v);
  if (TPR > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) v += part[w];
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* part) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (TPR > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < TPR / 32; ++w) v = max(v, part[w]);
  }
  return v;
}

// A row's scale and its int8 values: scale = absmax / 127, q = clamp(rne(x /
// scale), -127, 127), each as one correctly rounded fp32 operation.
// Magnitudes are compared as bit patterns, which orders NaN above infinity
// above every number: a row that holds either has scale NaN or infinity, and
// q = 0, so that what is computed from it is NaN and not a plausible number.
// A row whose scale is 0 (all zeros, or an absmax that / 127 underflows) has
// q = 0 too.
struct RowScale {
  float scale, rcp;
  bool plain;
  __device__ __forceinline__ explicit RowScale(uint32_t absmax) {
    scale = __fdiv_rn(__uint_as_float(absmax), 127.0f);
    plain = scale > 0.f && scale < __uint_as_float(0x7f800000u);
    rcp = __frcp_rn(scale);
  }
};
template <int TPR, bool VEC>
__device__ __forceinline__ void store_int8(const float (&v)[8], const RowScale& s, int8_t* q, int K, int tid, int c) {
  uint32_t packed[2] = {0u, 0u};
  if (s.plain) quant8_i8(v, s.scale, s.rcp, packed);
  if (VEC) {
    const int k = column<TPR, VEC>(tid, c, 0);
    if (k < K) *reinterpret_cast<uint2*>(q + k) = make_uint2(packed[0], packed[1]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = column<TPR, VEC>(tid, c, e);
      if (k < K) q[k] = static_cast<int8_t>(packed[e >> 2] >> (8 * (e & 3)));
    }
  }
}

// Rows of one CTA: four rows of one warp each, or one row.
template <int TPR>
constexpr int rows_per_cta() {
  return TPR == 32 ? 4 : 1;  // TPR == 32: a row per warp
}

struct QuantRowsParams {
  int T, K;
  const void* x;
  long ldx;
  int8_t* q;
  long ldq;
  float* scale;
};

// Rows t, t + step, ... of a CTA (or warp): the next row is loaded before the
// current one is reduced and stored.
template <typename Tin, int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(TPR* rows_per_cta<TPR>()) quant_rows_kernel(const QuantRowsParams p) {
  __shared__ uint32_t part[2][TPR / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const long step = static_cast<long>(gridDim.x) * rows_per_cta<TPR>();
  long t = static_cast<long>(blockIdx.x) * rows_per_cta<TPR>() + (TPR == 32 ? threadIdx.x >> 5 : 0);
  Raw<Tin> next[NV];
  if (t < p.T) load_raw<TPR, NV, VEC>(static_cast<const Tin*>(p.x) + t * p.ldx, p.K, tid, next);
  for (int i = 0; t < p.T; t += step, i ^= 1) {
    Raw<Tin> v[NV];
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      v[c] = next[c];
      m = max(m, v[c].absmax());
    }
    if (t + step < p.T) load_raw<TPR, NV, VEC>(static_cast<const Tin*>(p.x) + (t + step) * p.ldx, p.K, tid, next);
    const RowScale s(row_max<TPR>(m, part[i]));
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      float f[8];
      v[c].get(f);
      store_int8<TPR, VEC>(f, s, p.q + t * p.ldq, p.K, tid, c);
    }
    if (tid == 0) p.scale[t] = s.scale;
  }
}

struct BlockNormParams {
  int T, K, S;
  const void* h;
  long ldh;
  const void* y;
  long ldy;
  const float* post_w;
  const float* gate;
  long gate_stride;
  float rscale;
  void* h_out;
  long ldho;
  const float* a1;
  const float* a2;
  const float* b2;
  long ab_stride;
  float eps;
  void* z;
  long ldz;
  int8_t* z_q;
  long ldzq;
  float* z_scale;
  int rows;  // per CTA (per warp where a CTA has four rows at a time)
};

// Pairs of neighbouring values, for the two-wide fp32 instructions: these
// kernels issue as many instructions as the memory system leaves time for.
using f32x2 = unsigned long long;
__device__ __forceinline__ void to_pairs(const float (&f)[8], f32x2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pack_f32x2(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ void from_pairs(const f32x2 (&v)[4], float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = lo_f32(v[i]);
    f[2 * i + 1] = hi_f32(v[i]);
  }
}
template <int NV>
__device__ __forceinline__ float sum_squares(const f32x2 (&v)[NV][4]) {
  f32x2 s = 0;
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) s = fma_f32x2(v[c][i], v[c][i], s);
  return lo_f32(s) + hi_f32(s);
}

// The product of two column vectors (absent ones are 1) and k, and a column
// vector that is 0 where absent.
template <int TPR, bool VEC>
__device__ __forceinline__ void column_product(const float* a, const float* b, float k, int K, int tid, int c,
                                               f32x2 (&out)[4]) {
  float f[8];
  f32x2 g[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = pack_f32x2(k, k);
  if (a) {
    load_columns<TPR, VEC>(a, K, tid, c, f);
    to_pairs(f, g);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = mul_f32x2(out[j], g[j]);
  }
  if (b) {
    load_columns<TPR, VEC>(b, K, tid, c, f);
    to_pairs(f, g);
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = mul_f32x2(out[j], g[j]);
  }
}
template <int TPR, bool VEC>
__device__ __forceinline__ void column_shift(const float* b, int K, int tid, int c, f32x2 (&out)[4]) {
  float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (b) load_columns<TPR, VEC>(b, K, tid, c, f);
  to_pairs(f, out);
}

// A CTA's rows are neighbours, and the next row is loaded before the current
// one is computed.  What multiplies a column is one product per stream,
//   h' = h + (u * rstd_u) * [residual_scale * gate * post_w],
//   z  = (h' * rstd_h) * [a1 * a2] + b2,
// which with one vector of 8 per thread stays in registers from row to row and
// with longer rows is formed again from L1.  (The register limit of 768 resident
// threads spills 8 to 20 bytes in four instances: fp32 rows of up to 256, and
// without vector accesses bf16 rows of up to 256 and fp32 rows of 1025 to 2048.)
template <typename T, int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(TPR* rows_per_cta<TPR>(), TPR <= 128 ? 6 : NV == 1 ? 768 / TPR : 1)
    block_norm_kernel(const BlockNormParams p) {
  __shared__ alignas(16) float part[2][2][TPR / 32];
  __shared__ uint32_t part_m[2][TPR / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const long at = (static_cast<long>(blockIdx.x) * rows_per_cta<TPR>() + (TPR == 32 ? threadIdx.x >> 5 : 0)) * p.rows;
  if (at >= p.T) return;
  const int first = static_cast<int>(at);
  const int n = min(p.rows, p.T - first);
  const T* hp = static_cast<const T*>(p.h) + first * p.ldh;
  const T* yp = p.y ? static_cast<const T*>(p.y) + first * p.ldy : nullptr;
  T* ho = p.h_out ? static_cast<T*>(p.h_out) + first * p.ldho : nullptr;
  const float inv_k = 1.f / static_cast<float>(p.K);
  constexpr bool kKeep = NV == 1;
  constexpr bool kAhead = NV <= 2;  // rows above 8192 elements fill the registers by themselves
  Raw<T> hn[NV], yn[NV];
  auto load = [&](int r) {
    load_raw<TPR, NV, VEC>(hp + r * p.ldh, p.K, tid, hn);
    if (yp) load_raw<TPR, NV, VEC>(yp + r * p.ldy, p.K, tid, yn);
  };
  if (kAhead) load(0);
  f32x2 gain[4], a12[4], b2[4];  // of the current stream, when kept
  const float *gate = nullptr, *pa2 = nullptr, *pb2 = nullptr;
  // the stream of the row, and its rows left: one division per CTA
  int b = first / p.S, left = p.S - (first - b * p.S);
  bool fresh = true;
  auto step = [&] {
    if (--left == 0) {
      left = p.S;
      ++b;
      fresh = true;
    }
  };
  for (int r = 0; r < n; ++r, step()) {
    const int i = r & 1;
    if (fresh) {
      fresh = false;
      gate = p.gate ? p.gate + b * p.gate_stride : nullptr;
      pa2 = p.a2 ? p.a2 + b * p.ab_stride : nullptr;
      pb2 = p.b2 ? p.b2 + b * p.ab_stride : nullptr;
      if (kKeep) {
        column_product<TPR, VEC>(p.post_w, gate, p.rscale, p.K, tid, 0, gain);
        column_product<TPR, VEC>(p.a1, pa2, 1.f, p.K, tid, 0, a12);
        column_shift<TPR, VEC>(pb2, p.K, tid, 0, b2);
      }
    }
    if (!kAhead) load(r);
    f32x2 h[NV][4];
#pragma unroll
    for (int c = 0; c < NV; ++c) hn[c].pairs(h[c]);
    if (ho) {
      f32x2 u[NV][4];
#pragma unroll
      for (int c = 0; c < NV; ++c) yn[c].pairs(u[c]);
      if (kAhead && r + 1 < n) load(r + 1);
      float rstd = 1.f;
      if (p.post_w) rstd = rsqrtf(row_sum<TPR>(sum_squares<NV>(u), part[i][0]) * inv_k + p.eps);
      const f32x2 r2 = pack_f32x2(rstd, rstd);
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        if (!kKeep) column_product<TPR, VEC>(p.post_w, gate, p.rscale, p.K, tid, c, gain);
#pragma unroll
        for (int j = 0; j < 4; ++j) h[c][j] = fma_f32x2(mul_f32x2(u[c][j], r2), gain[j], h[c][j]);
        // the stream is rounded to its type here, once, and the next norm reads
        // the rounded values: the same result as with the norm run on its own
        Raw<T> held_row;
        held_row.round(h[c]);
        held_row.pairs(h[c]);
        if (VEC) {
          const int k = column<TPR, VEC>(tid, c, 0);
          if (k < p.K) held_row.store(ho + r * p.ldho + k);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int k = column<TPR, VEC>(tid, c, e);
            if (k < p.K) ho[r * p.ldho + k] = held_row.at(e);
          }
        }
      }
    } else if (kAhead && r + 1 < n) {
      load(r + 1);
    }
    if (!p.z && !p.z_q) continue;
    const float rstd = rsqrtf(row_sum<TPR>(sum_squares<NV>(h), part[i][1]) * inv_k + p.eps);
    const f32x2 r2 = pack_f32x2(rstd, rstd);
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      if (!kKeep) {
        column_product<TPR, VEC>(p.a1, pa2, 1.f, p.K, tid, c, a12);
        column_shift<TPR, VEC>(pb2, p.K, tid, c, b2);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) h[c][j] = fma_f32x2(mul_f32x2(h[c][j], r2), a12[j], b2[j]);
      if (p.z) {
        float f[8];
        from_pairs(h[c], f);
        store_columns<TPR, VEC>(static_cast<T*>(p.z) + (first + r) * p.ldz, p.K, tid, c, f);
      } else {
        // past the row's end h, a12 and b2 hold 0 or, with no vectors, h does
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max_nan(top, max_nan(fabsf(lo_f32(h[c][j])), fabsf(hi_f32(h[c][j]))));
        m = max(m, __float_as_uint(top) & 0x7fffffffu);
      }
    }
    if (p.z_q) {
      const RowScale s(row_max<TPR>(m, part_m[i]));
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        float f[8];
        from_pairs(h[c], f);
        store_int8<TPR, VEC>(f, s, p.z_q + (first + r) * p.ldzq, p.K, tid, c);
      }
      if (tid == 0) p.z_scale[first + r] = s.scale;
    }
  }
}

// Threads per row and vectors per thread for a row of K: one vector per thread
// up to 4096 elements.  (32 elements per thread cost block_norm 16.7 us instead
// of 10.5 at 3200 x 1024: a row's chain of reductions then has too few warps
// beside it.)
struct RowShape {
  int tpr, nv;
};
RowShape row_shape(int K) {
  if (K <= 256) return {32, 1};
  if (K <= 1024) return {128, 1};
  if (K <= 2048) return {256, 1};
  if (K <= 4096) return {512, 1};
  return {512, K <= 8192 ? 2 : 4};
}
// Quantizing many rows: 32 elements per thread, so that the reduction and the
// scale's division weigh less (3200 x 4096: 10.4 us against 12.1; a single
// row of 4096 is quicker with 8 per thread).
RowShape quant_shape(int T, int K) {
  int nsm = 148;
  rfx_num_sms(&nsm);
  if (T < 8 * nsm) return row_shape(K);
  int tpr = 32;
  while (tpr * 32 < K) tpr *= 2;
  return {tpr, 4};
}

template <typename T, bool VEC>
const void* quant_rows_ptr(RowShape s) {
  if (s.nv == 1) {
    if (s.tpr == 32) return reinterpret_cast<const void*>(quant_rows_kernel<T, 32, 1, VEC>);
    if (s.tpr == 128) return reinterpret_cast<const void*>(quant_rows_kernel<T, 128, 1, VEC>);
    if (s.tpr == 256) return reinterpret_cast<const void*>(quant_rows_kernel<T, 256, 1, VEC>);
    return reinterpret_cast<const void*>(quant_rows_kernel<T, 512, 1, VEC>);
  }
  if (s.nv == 2) return reinterpret_cast<const void*>(quant_rows_kernel<T, 512, 2, VEC>);
  if (s.tpr == 32) return reinterpret_cast<const void*>(quant_rows_kernel<T, 32, 4, VEC>);
  if (s.tpr == 64) return reinterpret_cast<const void*>(quant_rows_kernel<T, 64, 4, VEC>);
  if (s.tpr == 128) return reinterpret_cast<const void*>(quant_rows_kernel<T, 128, 4, VEC>);
  if (s.tpr == 256) return reinterpret_cast<const void*>(quant_rows_kernel<T, 256, 4, VEC>);
  return reinterpret_cast<const void*>(quant_rows_kernel<T, 512, 4, VEC>);
}
template <typename T, bool VEC>
const void* block_norm_ptr(RowShape s) {
  if (s.tpr == 32) return reinterpret_cast<const void*>(block_norm_kernel<T, 32, 1, VEC>);
  if (s.tpr == 128) return reinterpret_cast<const void*>(block_norm_kernel<T, 128, 1, VEC>);
  if (s.tpr == 256) return reinterpret_cast<const void*>(block_norm_kernel<T, 256, 1, VEC>);
  if (s.nv == 1) return reinterpret_cast<const void*>(block_norm_kernel<T, 512, 1, VEC>);
  if (s.nv == 2) return reinterpret_cast<const void*>(block_norm_kernel<T, 512, 2, VEC>);
  return reinterpret_cast<const void*>(block_norm_kernel<T, 512, 4, VEC>);
}

bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
// rows of `esz`-byte elements that 8-element vector accesses may walk
bool vec_rows(const void* p, long ld, int esz) { return !p || (aligned(p, esz == 1 ? 8 : 16) && (ld * esz) % (esz == 1 ? 8 : 16) == 0); }
// CTAs of about one wave over the SMs, `threads` threads resident on each
unsigned row_grid(int T, int tpr, int threads) {
  int nsm = 148;
  rfx_num_sms(&nsm);
  const int per_cta = tpr == 32 ? 4 : 1;
  const long all = (static_cast<long>(T) + per_cta - 1) / per_cta;
  return static_cast<unsigned>(std::min<long>(all, static_cast<long>(nsm) * (threads / (tpr * per_cta))));
}
int elem_size(int dtype) { return dtype == kDtypeBF16 ? 2 : 4; }

}  // namespace

int validate_quant_rows(const rfx_quant_rows_desc& d) {
  if (d.T < 0 || d.K < 1 || d.K > kMaxRow)
    return set_error(RFX_E_INVAL, "rfx_quant_rows: need T>=0 and 1<=K<=%d (T=%d K=%d)", kMaxRow, d.T, d.K);
  if (d.in_dtype != kDtypeBF16 && d.in_dtype != kDtypeF32)
    return set_error(RFX_E_INVAL, "rfx_quant_rows: input dtype must be bf16 or f32");
  if (d.T == 0) return RFX_OK;
  if (!d.x || !d.q || !d.scale || d.ldx < d.K || d.ldq < d.K)
    return set_error(RFX_E_INVAL, "rfx_quant_rows: null pointer or a row stride below K");
  if (!aligned(d.x, elem_size(d.in_dtype)) || !aligned(d.scale, 4))
    return set_error(RFX_E_INVAL, "rfx_quant_rows: misaligned pointer");
  const long esz = elem_size(d.in_dtype);
  const Rows x{d.x, d.T, d.ldx * esz, d.K * esz}, q{d.q, d.T, d.ldq, d.K}, scale{d.scale, 1, 0, d.T * 4l};
  if (rows_shared(q, x) || rows_shared(scale, x) || rows_shared(scale, q))
    return set_error(RFX_E_INVAL, "rfx_quant_rows: x, q and scale share memory");
  return RFX_OK;
}

int launch_quant_rows(const rfx_quant_rows_desc& d, cudaStream_t stream, bool pdl) {
  const int rc = validate_quant_rows(d);
  if (rc || d.T == 0) return rc;
  QuantRowsParams p{d.T, d.K, d.x, d.ldx, static_cast<int8_t*>(d.q), d.ldq, d.scale};
  const bool vec = d.K % 8 == 0 && vec_rows(d.x, d.ldx, elem_size(d.in_dtype)) && vec_rows(d.q, d.ldq, 1);
  const RowShape s = quant_shape(d.T, d.K);
  const void* fn = d.in_dtype == kDtypeBF16
                       ? (vec ? quant_rows_ptr<__nv_bfloat16, true>(s) : quant_rows_ptr<__nv_bfloat16, false>(s))
                       : (vec ? quant_rows_ptr<float, true>(s) : quant_rows_ptr<float, false>(s));
  return launch_kernel(fn, dim3(row_grid(d.T, s.tpr, s.nv == 1 ? 1536 : 1024)), dim3(s.tpr == 32 ? 128 : s.tpr), 0, stream, pdl, 1, p);
}

int validate_block_norm(const rfx_block_norm_desc& d) {
  if (d.T < 0 || d.K < 1 || d.K > kMaxRow || d.tokens_per_batch < 1)
    return set_error(RFX_E_INVAL, "rfx_block_norm: need T>=0, 1<=K<=%d, tokens_per_batch>=1 (T=%d K=%d)", kMaxRow,
                     d.T, d.K);
  if (d.dtype != kDtypeBF16 && d.dtype != kDtypeF32)
    return set_error(RFX_E_INVAL, "rfx_block_norm: dtype must be bf16 or f32");
  if (d.T == 0) return RFX_OK;
  const long esz = elem_size(d.dtype);
  if (!d.h || d.ldh < d.K || (d.y && d.ldy < d.K) || (d.h_out && d.ldho < d.K) || (d.z && d.ldz < d.K) ||
      (d.z_q && d.ldzq < d.K))
    return set_error(RFX_E_INVAL, "rfx_block_norm: null h or a row stride below K");
  if (!d.y && (d.post_w || d.gate || d.h_out))
    return set_error(RFX_E_INVAL, "rfx_block_norm: post_w, gate and h_out need the block's output y");
  if (d.y && !d.h_out) return set_error(RFX_E_INVAL, "rfx_block_norm: y needs h_out (h itself for an update in place)");
  if (d.z && d.z_q) return set_error(RFX_E_INVAL, "rfx_block_norm: one of z and z_q");
  if (!d.y && !d.z && !d.z_q)
    return set_error(RFX_E_INVAL, "rfx_block_norm: nothing to compute (no y and no norm output)");
  if (!d.z_q != !d.z_scale) return set_error(RFX_E_INVAL, "rfx_block_norm: z_q and z_scale come together");
  const long w = static_cast<long>(d.K) * esz;
  const Rows h{d.h, d.T, d.ldh * esz, w}, y{d.y, d.T, d.ldy * esz, w}, ho{d.h_out, d.T, d.ldho * esz, w};
  const Rows z{d.z, d.T, d.ldz * esz, w}, q{d.z_q, d.T, d.ldzq, d.K}, zs{d.z_scale, 1, 0, d.T * 4l};
  if ((!rows_same(ho, h) && rows_shared(ho, h)) || rows_shared(ho, y) || (!rows_same(z, h) && rows_shared(z, h)) ||
      (!rows_same(z, y) && rows_shared(z, y)) || rows_shared(z, ho) || rows_shared(q, h) || rows_shared(q, y) ||
      rows_shared(q, ho) || rows_shared(zs, h) || rows_shared(zs, y) || rows_shared(zs, ho) || rows_shared(zs, q))
    return set_error(RFX_E_INVAL, "rfx_block_norm: outputs overlap (in place only h_out or z over h, or z over y, at the same stride)");
  const long B = (static_cast<long>(d.T) - 1) / d.tokens_per_batch + 1;
  const Places vectors[5] = {
      {d.post_w, 4, d.K, {1, 1, 1}, {}},
      {d.gate, 4, d.K, {B, 1, 1}, {d.gate_stride, 0, 0}},
      {d.norm_a1, 4, d.K, {1, 1, 1}, {}},
      {d.norm_a2, 4, d.K, {B, 1, 1}, {d.norm_ab_stride, 0, 0}},
      {d.norm_b2, 4, d.K, {B, 1, 1}, {d.norm_ab_stride, 0, 0}},
  };
  const Places outputs[4] = {
      {d.h_out, esz, d.K, {d.T, 1, 1}, {d.ldho, 0, 0}},
      {d.z, esz, d.K, {d.T, 1, 1}, {d.ldz, 0, 0}},
      {d.z_q, 1, d.K, {d.T, 1, 1}, {d.ldzq, 0, 0}},
      {d.z_scale, 4, d.T, {1, 1, 1}, {}},
  };
  for (const Places& o : outputs)
    for (const Places& v : vectors)
      if (places_shared(o, v))
        return set_error(RFX_E_INVAL, "rfx_block_norm: an output shares memory with post_w, gate or a norm vector");
  if (!d.z && !d.z_q && (d.norm_a1 || d.norm_a2 || d.norm_b2))
    return set_error(RFX_E_INVAL, "rfx_block_norm: norm vectors without a norm output");
  if (!aligned(d.h, elem_size(d.dtype)) || !aligned(d.y, elem_size(d.dtype)) || !aligned(d.h_out, elem_size(d.dtype)) ||
      !aligned(d.z, elem_size(d.dtype)) ||
      !aligned(d.post_w, 4) || !aligned(d.gate, 4) || !aligned(d.norm_a1, 4) || !aligned(d.norm_a2, 4) ||
      !aligned(d.norm_b2, 4) || !aligned(d.z_scale, 4))
    return set_error(RFX_E_INVAL, "rfx_block_norm: misaligned pointer");
  return RFX_OK;
}

int launch_block_norm(const rfx_block_norm_desc& d, cudaStream_t stream, bool pdl) {
  const int rc = validate_block_norm(d);
  if (rc || d.T == 0) return rc;
  BlockNormParams p{d.T,     d.K,       d.tokens_per_batch, d.h,        d.ldh,     d.y,
                    d.ldy,   d.post_w,  d.gate,             d.gate_stride, d.residual_scale, d.h_out,
                    d.ldho,  d.norm_a1, d.norm_a2,          d.norm_b2,  d.norm_ab_stride, d.eps,
                    d.z,     d.ldz,     static_cast<int8_t*>(d.z_q), d.ldzq, d.z_scale, 1};
  const int esz = elem_size(d.dtype);
  const bool vec = d.K % 8 == 0 && vec_rows(d.h, d.ldh, esz) && vec_rows(d.y, d.ldy, esz) &&
                   vec_rows(d.h_out, d.ldho, esz) && vec_rows(d.z, d.ldz, esz) && vec_rows(d.z_q, d.ldzq, 1) &&
                   vec_rows(d.post_w, 0, 4) && vec_rows(d.gate, d.gate_stride, 4) && vec_rows(d.norm_a1, 0, 4) &&
                   vec_rows(d.norm_a2, d.norm_ab_stride, 4) && vec_rows(d.norm_b2, d.norm_ab_stride, 4);
  const RowShape s = row_shape(d.K);
  const void* fn = d.dtype == kDtypeBF16
                       ? (vec ? block_norm_ptr<__nv_bfloat16, true>(s) : block_norm_ptr<__nv_bfloat16, false>(s))
                       : (vec ? block_norm_ptr<float, true>(s) : block_norm_ptr<float, false>(s));
  // neighbouring rows per CTA, so that about one wave of CTAs covers them
  const int per_cta = s.tpr == 32 ? 4 : 1;
  const long slots = static_cast<long>(row_grid(d.T, s.tpr, 768)) * per_cta;
  p.rows = static_cast<int>((d.T + slots - 1) / slots);
  const long ctas = (d.T + static_cast<long>(p.rows) * per_cta - 1) / (static_cast<long>(p.rows) * per_cta);
  return launch_kernel(fn, dim3(static_cast<unsigned>(ctas)), dim3(s.tpr * per_cta), 0, stream, pdl, 1, p);
}

}  // namespace rfx

extern "C" int rfx_quant_rows(const rfx_quant_rows_desc* d, void* stream) {
  if (!d) return rfx::set_error(RFX_E_INVAL, "rfx_quant_rows: null descriptor");
  return rfx::launch_quant_rows(*d, static_cast<cudaStream_t>(stream), rfx::pdl_enabled());
}

extern "C" int rfx_block_norm(const rfx_block_norm_desc* d, void* stream) {
  if (!d) return rfx::set_error(RFX_E_INVAL, "rfx_block_norm: null descriptor");
  return rfx::launch_block_norm(*d, static_cast<cudaStream_t>(stream), rfx::pdl_enabled());
}
