// Row operators of the int8 layer path: rows to int8 with one scale per row,
// and what lies between two transformer blocks (the norm of a block's output,
// its gate and residual scale, the residual add, the next block's norm).
//
// A row is read from memory once and stays in the registers of the threads
// that read it, through every reduction, until its outputs are written: TPR
// threads per row, NV vectors of 8 elements per thread.
#include "quant_i8.cuh"
#include "rfx_internal.h"

namespace rfx {
namespace {

constexpr int kMaxRow = 16384;

__device__ __forceinline__ float load_f(const float* p) { return *p; }
__device__ __forceinline__ float load_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float round_to(const float*, float v) { return v; }
__device__ __forceinline__ float round_to(const __nv_bfloat16*, float v) { return bf16_round(v); }

__device__ __forceinline__ void load_vec(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  const float4 b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void store_vec(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// Where element e of vector c of thread `tid` of a row lies.  VEC: 8
// neighbours per thread (16-byte accesses; K % 8 == 0 and aligned rows);
// otherwise threads take single neighbours, so that a warp's accesses stay
// contiguous at any length and alignment.
template <int TPR, bool VEC>
__device__ __forceinline__ int column(int tid, int c, int e) {
  return VEC ? (c * TPR + tid) * 8 + e : (c * 8 + e) * TPR + tid;
}

// The thread's part of a row as fp32; 0 past the row's end.
template <int TPR, int NV, bool VEC, typename T>
__device__ __forceinline__ void load_row(const T* row, int K, int tid, float (&v)[NV][8]) {
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    if (VEC) {
      const int k = column<TPR, VEC>(tid, c, 0);
      if (k < K) {
        load_vec(row + k, v[c]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = column<TPR, VEC>(tid, c, e);
        v[c][e] = k < K ? load_f(row + k) : 0.f;
      }
    }
  }
}
template <int TPR, int NV, bool VEC, typename T>
__device__ __forceinline__ void store_row(T* row, int K, int tid, const float (&v)[NV][8]) {
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    if (VEC) {
      const int k = column<TPR, VEC>(tid, c, 0);
      if (k < K) store_vec(row + k, v[c]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = column<TPR, VEC>(tid, c, e);
        if (k < K) store_f(row + k, v[c][e]);
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

// A row in registers to int8 and its scale: scale = absmax / 127,
// q = clamp(rne(x / scale), -127, 127), each as one correctly rounded fp32
// operation.  Magnitudes are compared as bit patterns, which orders NaN above
// infinity above every number: a row that holds either has scale NaN or
// infinity, and q = 0, so that what is computed from it is NaN and not a
// plausible number.  A row whose scale is 0 (all zeros, or an absmax that
// / 127 underflows) has q = 0 too.
template <int TPR, int NV, bool VEC>
__device__ __forceinline__ void quantize_row(const float (&v)[NV][8], int8_t* q, float* scale_out, int K, int tid,
                                             uint32_t* part) {
  uint32_t m = 0;
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[c][e]) & 0x7fffffffu);
  m = row_max<TPR>(m, part);
  const float scale = __fdiv_rn(__uint_as_float(m), 127.0f);
  const bool plain = scale > 0.f && scale < __uint_as_float(0x7f800000u);
  const float rcp = __frcp_rn(scale);
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    uint32_t packed[2] = {0u, 0u};
    if (plain) quant8_i8(v[c], scale, rcp, packed);
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
  if (tid == 0) *scale_out = scale;
}

// Rows of one CTA: four rows of one warp each, or one row.
template <int TPR>
constexpr int rows_per_cta() {
  return TPR == 32 ? 4 : 1;
}

struct QuantRowsParams {
  int T, K;
  const void* x;
  long ldx;
  int8_t* q;
  long ldq;
  float* scale;
};

template <typename Tin, int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(TPR* rows_per_cta<TPR>()) quant_rows_kernel(const QuantRowsParams p) {
  __shared__ uint32_t part[TPR / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const long t = TPR == 32 ? static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (t >= p.T) return;
  float v[NV][8];
  load_row<TPR, NV, VEC>(static_cast<const Tin*>(p.x) + t * p.ldx, p.K, tid, v);
  quantize_row<TPR, NV, VEC>(v, p.q + t * p.ldq, p.scale + t, p.K, tid, part);
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
};

template <typename T, int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(TPR* rows_per_cta<TPR>()) block_norm_kernel(const BlockNormParams p) {
  __shared__ float part[2][TPR / 32];
  __shared__ uint32_t part_m[TPR / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const long t = TPR == 32 ? static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (t >= p.T) return;
  const long b = t / p.S;
  float h[NV][8];
  load_row<TPR, NV, VEC>(static_cast<const T*>(p.h) + t * p.ldh, p.K, tid, h);
  if (p.y) {
    float u[NV][8], w[NV][8];
    load_row<TPR, NV, VEC>(static_cast<const T*>(p.y) + t * p.ldy, p.K, tid, u);
    if (p.post_w) {
      load_row<TPR, NV, VEC>(p.post_w, p.K, tid, w);
      float ss = 0.f;
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(u[c][e], u[c][e], ss);
      const float rstd = rsqrtf(row_sum<TPR>(ss, part[0]) / static_cast<float>(p.K) + p.eps);
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) u[c][e] *= rstd * w[c][e];
    }
    if (p.gate) {
      load_row<TPR, NV, VEC>(p.gate + b * p.gate_stride, p.K, tid, w);
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) u[c][e] *= w[c][e];
    }
    // the stream is rounded to its type here, once, and the next norm reads
    // the rounded values: the same result as with the norm run on its own
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[c][e] = round_to(static_cast<const T*>(nullptr), fmaf(p.rscale, u[c][e], h[c][e]));
    if (p.h_out) store_row<TPR, NV, VEC>(static_cast<T*>(p.h_out) + t * p.ldho, p.K, tid, h);
  }
  if (!p.z && !p.z_q) return;
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(h[c][e], h[c][e], ss);
  const float rstd = rsqrtf(row_sum<TPR>(ss, part[1]) / static_cast<float>(p.K) + p.eps);
  float w[NV][8];
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) h[c][e] *= rstd;
  if (p.a1) {
    load_row<TPR, NV, VEC>(p.a1, p.K, tid, w);
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[c][e] *= w[c][e];
  }
  if (p.a2) {
    load_row<TPR, NV, VEC>(p.a2 + b * p.ab_stride, p.K, tid, w);
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[c][e] *= w[c][e];
  }
  if (p.b2) {
    load_row<TPR, NV, VEC>(p.b2 + b * p.ab_stride, p.K, tid, w);
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[c][e] += w[c][e];
  }
  if (p.z) store_row<TPR, NV, VEC>(static_cast<T*>(p.z) + t * p.ldz, p.K, tid, h);
  if (p.z_q) quantize_row<TPR, NV, VEC>(h, p.z_q + t * p.ldzq, p.z_scale + t, p.K, tid, part_m);
}

// Threads per row and vectors per thread for a row of K: the fewest threads
// that hold it, one vector each up to 4096 elements.
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

template <typename T, bool VEC>
const void* quant_rows_ptr(RowShape s) {
  if (s.tpr == 32) return reinterpret_cast<const void*>(quant_rows_kernel<T, 32, 1, VEC>);
  if (s.tpr == 128) return reinterpret_cast<const void*>(quant_rows_kernel<T, 128, 1, VEC>);
  if (s.tpr == 256) return reinterpret_cast<const void*>(quant_rows_kernel<T, 256, 1, VEC>);
  if (s.nv == 1) return reinterpret_cast<const void*>(quant_rows_kernel<T, 512, 1, VEC>);
  if (s.nv == 2) return reinterpret_cast<const void*>(quant_rows_kernel<T, 512, 2, VEC>);
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
unsigned row_grid(int T, int tpr) { return tpr == 32 ? (static_cast<unsigned>(T) + 3) / 4 : static_cast<unsigned>(T); }
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
  return RFX_OK;
}

int launch_quant_rows(const rfx_quant_rows_desc& d, cudaStream_t stream, bool pdl) {
  const int rc = validate_quant_rows(d);
  if (rc || d.T == 0) return rc;
  QuantRowsParams p{d.T, d.K, d.x, d.ldx, static_cast<int8_t*>(d.q), d.ldq, d.scale};
  const bool vec = d.K % 8 == 0 && vec_rows(d.x, d.ldx, elem_size(d.in_dtype)) && vec_rows(d.q, d.ldq, 1);
  const RowShape s = row_shape(d.K);
  const void* fn = d.in_dtype == kDtypeBF16
                       ? (vec ? quant_rows_ptr<__nv_bfloat16, true>(s) : quant_rows_ptr<__nv_bfloat16, false>(s))
                       : (vec ? quant_rows_ptr<float, true>(s) : quant_rows_ptr<float, false>(s));
  return launch_kernel(fn, dim3(row_grid(d.T, s.tpr)), dim3(s.tpr == 32 ? 128 : s.tpr), 0, stream, pdl, 1, p);
}

int validate_block_norm(const rfx_block_norm_desc& d) {
  if (d.T < 0 || d.K < 1 || d.K > kMaxRow || d.tokens_per_batch < 1)
    return set_error(RFX_E_INVAL, "rfx_block_norm: need T>=0, 1<=K<=%d, tokens_per_batch>=1 (T=%d K=%d)", kMaxRow,
                     d.T, d.K);
  if (d.dtype != kDtypeBF16 && d.dtype != kDtypeF32)
    return set_error(RFX_E_INVAL, "rfx_block_norm: dtype must be bf16 or f32");
  if (d.T == 0) return RFX_OK;
  const int esz = elem_size(d.dtype);
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
  if ((d.h_out == d.h && d.h_out && d.ldho != d.ldh) || (d.z && d.z == d.h_out) || (d.z == d.h && d.z && d.ldz != d.ldh) ||
      (d.z && d.z == d.y && d.ldz != d.ldy) || (d.h_out && d.h_out == d.y))
    return set_error(RFX_E_INVAL, "rfx_block_norm: outputs overlap (in place only over h, or z over y, at the same stride)");
  if (!d.z && !d.z_q && (d.norm_a1 || d.norm_a2 || d.norm_b2))
    return set_error(RFX_E_INVAL, "rfx_block_norm: norm vectors without a norm output");
  if (!aligned(d.h, esz) || !aligned(d.y, esz) || !aligned(d.h_out, esz) || !aligned(d.z, esz) ||
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
                    d.z,     d.ldz,     static_cast<int8_t*>(d.z_q), d.ldzq, d.z_scale};
  const int esz = elem_size(d.dtype);
  const bool vec = d.K % 8 == 0 && vec_rows(d.h, d.ldh, esz) && vec_rows(d.y, d.ldy, esz) &&
                   vec_rows(d.h_out, d.ldho, esz) && vec_rows(d.z, d.ldz, esz) && vec_rows(d.z_q, d.ldzq, 1) &&
                   vec_rows(d.post_w, 0, 4) && vec_rows(d.gate, d.gate_stride, 4) && vec_rows(d.norm_a1, 0, 4) &&
                   vec_rows(d.norm_a2, d.norm_ab_stride, 4) && vec_rows(d.norm_b2, d.norm_ab_stride, 4);
  const RowShape s = row_shape(d.K);
  const void* fn = d.dtype == kDtypeBF16
                       ? (vec ? block_norm_ptr<__nv_bfloat16, true>(s) : block_norm_ptr<__nv_bfloat16, false>(s))
                       : (vec ? block_norm_ptr<float, true>(s) : block_norm_ptr<float, false>(s));
  return launch_kernel(fn, dim3(row_grid(d.T, s.tpr)), dim3(s.tpr == 32 ? 128 : s.tpr), 0, stream, pdl, 1, p);
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
