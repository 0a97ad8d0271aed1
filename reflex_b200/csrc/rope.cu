// Rotary positions on the rows of a QKV projection, split on the way into the
// q, k and v that the attention takes.
//
// Pair i of a head (dims i, i + rot/2 in the half layout, 2i, 2i + 1 in the
// interleaved one) of a token at position p turns by the angle p * f_i:
//   (a, b) -> m * (a cos - b sin, b cos + a sin).
// The frequencies f_i come as fp64 radians per position, scaled by the caller
// for long contexts, and there is no table whose length bounds the positions:
// the angle is formed in fp64 turns, p * f_i / (2 pi), of which only the
// fraction goes on to fp32 (a fp32 angle would be off by 0.03 rad at position
// 10^6), once per token and pair; all heads of the token share it through
// shared memory.
#include "rfx_internal.h"

#include <algorithm>

namespace rfx {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kMaxHeadDim = 256;

struct RopeParams {
  int T, S;
  int hq, hr, ha;  // query heads, rotated heads (q and k), all heads (q, k and v)
  int D, rot;
  const void* x;
  long ldx;
  const int* pos;
  const double* freq;
  float mag;
  void* out[3];
  long sb[3], sh[3], ss[3];
  int tokens;  // per CTA
  int items;   // work items per head row
};

template <typename T>
struct Pack;
template <>
struct Pack<__nv_bfloat16> {
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(h[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
  static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
};
template <>
struct Pack<float> {
  static __device__ __forceinline__ void load(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    const float4 b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};

// A work item is what one thread reads and then writes: with VEC 8 dims that
// hold whole pairs (interleaved; also the dims past rot) or 8 dims of the
// first and the matching 8 of the second half (half); without VEC one pair,
// or one dim past rot.  A thread owns every element of a pair, so the output
// may lie over the input.
template <typename T, bool HALF, bool VEC>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams p) {
  extern __shared__ float2 cs[];  // [tokens][rot / 2] cos, sin
  pdl_wait();
  pdl_launch_dependents();
  const int half = p.rot >> 1;
  const int t0 = blockIdx.x * p.tokens;
  const int nt = min(p.tokens, p.T - t0);
  for (int i = threadIdx.x; i < nt * half; i += kRopeThreads) {
    const int tt = i / half, pair = i - tt * half;
    const double turns = static_cast<double>(p.pos[t0 + tt]) * (p.freq[pair] * 0.15915494309189533577);
    const float frac = static_cast<float>(turns - rint(turns));
    float s, c;
    sincospif(2.f * frac, &s, &c);
    cs[i] = make_float2(p.mag * c, p.mag * s);
  }
  __syncthreads();
  const int per = kRopeThreads / p.items;  // head rows per sweep of the CTA
  const int lane = threadIdx.x % p.items;
  int row = threadIdx.x / p.items;  // (token, head) of this CTA
  if (row >= per) return;
  const int rows = nt * p.ha;
  for (; row < rows; row += per) {
    const int tt = row / p.ha, head = row - tt * p.ha;
    const int t = t0 + tt;
    const int b = t / p.S, s = t - b * p.S;
    const int part = head < p.hq ? 0 : head < p.hr ? 1 : 2;
    const int ph = head - (part == 0 ? 0 : part == 1 ? p.hq : p.hr);
    const T* src = static_cast<const T*>(p.x) + t * p.ldx + static_cast<long>(head) * p.D;
    T* dst = static_cast<T*>(p.out[part]) + b * p.sb[part] + ph * p.sh[part] + s * p.ss[part];
    const bool turn = part < 2;
    const float2* a = cs + tt * half;
    if (VEC) {
      if (HALF && lane * 8 < half) {
        float u[8], w[8];
        const int d = lane * 8;
        Pack<T>::load(src + d, u);
        Pack<T>::load(src + half + d, w);
        if (turn) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 r = a[d + e];
            const float x = u[e], y = w[e];
            u[e] = x * r.x - y * r.y;
            w[e] = y * r.x + x * r.y;
          }
        }
        Pack<T>::store(dst + d, u);
        Pack<T>::store(dst + half + d, w);
      } else {
        const int d = HALF ? p.rot + (lane * 8 - half) : lane * 8;
        float u[8];
        Pack<T>::load(src + d, u);
        if (!HALF && turn && d < p.rot) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float2 r = a[(d + e) >> 1];
            const float x = u[e], y = u[e + 1];
            u[e] = x * r.x - y * r.y;
            u[e + 1] = y * r.x + x * r.y;
          }
        }
        Pack<T>::store(dst + d, u);
      }
    } else if (lane < half) {
      const int d0 = HALF ? lane : 2 * lane, d1 = HALF ? lane + half : 2 * lane + 1;
      float x = Pack<T>::get(src + d0), y = Pack<T>::get(src + d1);
      if (turn) {
        const float2 r = a[lane];
        const float u = x * r.x - y * r.y;
        y = y * r.x + x * r.y;
        x = u;
      }
      Pack<T>::put(dst + d0, x);
      Pack<T>::put(dst + d1, y);
    } else {
      const int d = p.rot + (lane - half);
      Pack<T>::put(dst + d, Pack<T>::get(src + d));
    }
  }
}

bool al(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename T>
const void* rope_ptr(bool half, bool vec) {
  if (half)
    return vec ? reinterpret_cast<const void*>(rope_kernel<T, true, true>)
               : reinterpret_cast<const void*>(rope_kernel<T, true, false>);
  return vec ? reinterpret_cast<const void*>(rope_kernel<T, false, true>)
             : reinterpret_cast<const void*>(rope_kernel<T, false, false>);
}

}  // namespace

int validate_rope(const rfx_rope_desc& d) {
  if (d.B < 0 || d.S < 0 || static_cast<long>(d.B) * d.S > 0x7fffffffL - 1024)
    return set_error(RFX_E_INVAL, "rfx_rope: bad B/S (B=%d S=%d)", d.B, d.S);
  if (d.num_q_heads < 1 || d.num_kv_heads < 0 || d.num_q_heads > 1024 || d.num_kv_heads > 1024)
    return set_error(RFX_E_INVAL, "rfx_rope: 1..1024 query heads and 0..1024 KV heads");
  if (d.head_dim < 2 || d.head_dim > kMaxHeadDim || d.rot_dim < 2 || d.rot_dim > d.head_dim || d.rot_dim % 2)
    return set_error(RFX_E_INVAL, "rfx_rope: need 2<=head_dim<=%d and an even rot_dim of 2..head_dim (D=%d rot=%d)",
                     kMaxHeadDim, d.head_dim, d.rot_dim);
  if (d.pairs != RFX_ROPE_HALF && d.pairs != RFX_ROPE_INTERLEAVED) return set_error(RFX_E_INVAL, "rfx_rope: pairs");
  if (d.dtype != kDtypeBF16 && d.dtype != kDtypeF32)
    return set_error(RFX_E_INVAL, "rfx_rope: dtype must be bf16 or f32");
  if (d.B == 0 || d.S == 0) return RFX_OK;
  if (!d.x || !d.positions || !d.inv_freq || !d.q_out || (d.num_kv_heads > 0) != (d.k_out != nullptr) ||
      (d.v_out && !d.k_out))
    return set_error(RFX_E_INVAL, "rfx_rope: null pointer (k_out goes with num_kv_heads > 0, v_out with k_out)");
  const long heads = static_cast<long>(d.num_q_heads) + d.num_kv_heads * (d.v_out ? 2 : 1);
  if (d.ldx < heads * d.head_dim) return set_error(RFX_E_INVAL, "rfx_rope: ldx below the row of all heads");
  const unsigned esz = d.dtype == kDtypeBF16 ? 2 : 4;
  if (!al(d.x, esz) || !al(d.q_out, esz) || !al(d.k_out, esz) || !al(d.v_out, esz) || !al(d.positions, 4) ||
      !al(d.inv_freq, 8))
    return set_error(RFX_E_INVAL, "rfx_rope: misaligned pointer");
  return RFX_OK;
}

int launch_rope(const rfx_rope_desc& d, cudaStream_t stream, bool pdl) {
  const int rc = validate_rope(d);
  if (rc || d.B == 0 || d.S == 0) return rc;
  RopeParams p{};
  p.T = d.B * d.S;
  p.S = d.S;
  p.hq = d.num_q_heads;
  p.hr = d.num_q_heads + d.num_kv_heads;
  p.ha = p.hr + (d.v_out ? d.num_kv_heads : 0);
  p.D = d.head_dim;
  p.rot = d.rot_dim;
  p.x = d.x;
  p.ldx = d.ldx;
  p.pos = d.positions;
  p.freq = d.inv_freq;
  p.mag = d.magnitude;
  p.out[0] = d.q_out; p.sb[0] = d.qs_b; p.sh[0] = d.qs_h; p.ss[0] = d.qs_s;
  p.out[1] = d.k_out; p.sb[1] = d.ks_b; p.sh[1] = d.ks_h; p.ss[1] = d.ks_s;
  p.out[2] = d.v_out; p.sb[2] = d.vs_b; p.sh[2] = d.vs_h; p.ss[2] = d.vs_s;
  const long esz = d.dtype == kDtypeBF16 ? 2 : 4;
  const bool half = d.pairs == RFX_ROPE_HALF;
  // 16-byte accesses: every row, head and half begins on a 16-byte boundary
  bool vec = d.head_dim % 8 == 0 && d.rot_dim % (half ? 16 : 8) == 0 && al(d.x, 16) && (d.ldx * esz) % 16 == 0;
  for (int i = 0; i < 3; ++i)
    vec = vec && (!p.out[i] || (al(p.out[i], 16) && ((p.sb[i] | p.sh[i] | p.ss[i]) * esz) % 16 == 0));
  p.items = vec ? (half ? d.rot_dim / 16 + (d.head_dim - d.rot_dim) / 8 : d.head_dim / 8)
                : d.rot_dim / 2 + (d.head_dim - d.rot_dim);
  int nsm = 148;
  rfx_num_sms(&nsm);
  // enough tokens per CTA for a few sweeps over its rows, while every SM still
  // has some CTAs; their cos / sin stay within 32 KB of shared memory
  const int half_rot = d.rot_dim / 2;
  p.tokens = std::max(1, std::min({p.T / (8 * nsm), 8, 32 * 1024 / (8 * half_rot)}));
  const unsigned grid = static_cast<unsigned>((p.T + p.tokens - 1) / p.tokens);
  const void* fn = d.dtype == kDtypeBF16 ? rope_ptr<__nv_bfloat16>(half, vec) : rope_ptr<float>(half, vec);
  return launch_kernel(fn, dim3(grid), dim3(kRopeThreads), static_cast<size_t>(p.tokens) * half_rot * sizeof(float2),
                       stream, pdl, 1, p);
}

}  // namespace rfx

extern "C" int rfx_rope(const rfx_rope_desc* d, void* stream) {
  if (!d) return rfx::set_error(RFX_E_INVAL, "rfx_rope: null descriptor");
  return rfx::launch_rope(*d, static_cast<cudaStream_t>(stream), rfx::pdl_enabled());
}
