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
// shared memory.  The floor is the rows' one read and one write: 6344 tokens of
// 10 heads x 256 (half of each interleaved) take 15.1 us, 4.3 TB/s, 66 % of the
// measured copy rate, the rest of the time waiting for loads (a thread requests
// two tokens, turns and stores them, and then requests the next two); 3200 tokens
// (64 streams) 11.5 us; one stream's 50 2.2 us.
#include "rfx_internal.h"

#include <algorithm>

namespace rfx {
namespace {

constexpr int kRopeThreads = 512;  // at most
constexpr int kMaxHeadDim = 256;
constexpr int kMaxTokens = 16;  // per CTA

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
struct Item {
  float u[VEC ? 8 : 1], w[VEC ? 8 : 1];

  // whether it has two parts (the halves of pairs), and where the first begins
  static __device__ __forceinline__ bool two(int lane, int half) { return VEC ? HALF && lane * 8 < half : lane < half; }
  static __device__ __forceinline__ int first(int lane, int half, int rot) {
    if (VEC) return !HALF || lane * 8 < half ? lane * 8 : rot + (lane * 8 - half);
    return lane < half ? (HALF ? lane : 2 * lane) : rot + (lane - half);
  }
  static __device__ __forceinline__ int second(int d, int half) { return HALF ? d + half : d + 1; }

  __device__ __forceinline__ void load(const T* src, int d, bool pair, int half) {
    if constexpr (VEC) {
      Pack<T>::load(src + d, u);
      if (pair) Pack<T>::load(src + second(d, half), w);
    } else {
      u[0] = Pack<T>::get(src + d);
      if (pair) w[0] = Pack<T>::get(src + second(d, half));
    }
  }
  // cs: cos, sin of the token's pairs
  __device__ __forceinline__ void turn(const float2* cs, int d, bool pair, int rot) {
    if constexpr (VEC && !HALF) {
      if (d < rot) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float2 r = cs[(d + e) >> 1];
          const float x = u[e], y = u[e + 1];
          u[e] = x * r.x - y * r.y;
          u[e + 1] = y * r.x + x * r.y;
        }
      }
    } else if (pair) {
#pragma unroll
      for (int e = 0; e < (VEC ? 8 : 1); ++e) {
        const float2 r = cs[HALF ? d + e : d >> 1];
        const float x = u[e], y = w[e];
        u[e] = x * r.x - y * r.y;
        w[e] = y * r.x + x * r.y;
      }
    }
  }
  __device__ __forceinline__ void store(T* dst, int d, bool pair, int half) const {
    if constexpr (VEC) {
      Pack<T>::store(dst + d, u);
      if (pair) Pack<T>::store(dst + second(d, half), w);
    } else {
      Pack<T>::put(dst + d, u[0]);
      if (pair) Pack<T>::put(dst + second(d, half), w[0]);
    }
  }
};

// Where the CTA's tokens' q, k and v begin.
__device__ __forceinline__ void token_places(const RopeParams& p, int t0, int nt, long (&at)[3][kMaxTokens]) {
  for (int i = threadIdx.x; i < nt; i += blockDim.x) {
    const int t = t0 + i, b = t / p.S, s = t - b * p.S;
#pragma unroll
    for (int j = 0; j < 3; ++j) at[j][i] = b * p.sb[j] + s * p.ss[j];
  }
}

// cos, sin of the CTA's tokens, [token][pair].
__device__ __forceinline__ void token_angles(const RopeParams& p, int t0, int nt, float2* cs) {
  const int half = p.rot >> 1;
  // a thread keeps its pair: its frequency in turns per position is formed once
  const int width = min(half, static_cast<int>(blockDim.x)), rows = blockDim.x / width;
  for (int pair = threadIdx.x % width; pair < half; pair += width) {
    const double f = p.freq[pair] * 0.15915494309189533577;
    for (int tt = threadIdx.x / width; tt < nt && threadIdx.x < rows * width; tt += rows) {
      const double turns = static_cast<double>(p.pos[t0 + tt]) * f;
      // to the nearest whole turn: |turns| < 2^31, so adding 1.5 * 2^52 rounds it
      const double whole = __dadd_rn(__dadd_rn(turns, 0x1.8p52), -0x1.8p52);
      float s, c;
      sincospif(2.f * static_cast<float>(turns - whole), &s, &c);
      cs[tt * half + pair] = make_float2(p.mag * c, p.mag * s);
    }
  }
}

// Resident threads on an SM, which limit a thread to 64 or 40 registers: a
// half-split item is two loads, an interleaved one is one.  (The bf16 vector kernels
// spill 12 and 16 bytes at these limits.)
template <bool TWO_LOADS>
constexpr int resident_threads() {
  return TWO_LOADS ? 1024 : 1536;
}

// A CTA takes a few neighbouring tokens.  A thread keeps its (head, item) and
// walks the tokens, so that what it adds per 16 bytes is one row stride.
template <typename T, bool HALF, bool VEC>
__global__ void __launch_bounds__(kRopeThreads, resident_threads<HALF && VEC>() / kRopeThreads) rope_kernel(const RopeParams p) {
  constexpr int kBatch = 2;
  extern __shared__ float2 cs[];               // [tokens][rot / 2] cos, sin
  __shared__ long at[3][kMaxTokens];           // where a token's q, k and v begin
  pdl_wait();
  pdl_launch_dependents();
  const int half = p.rot >> 1;
  const int t0 = blockIdx.x * p.tokens;
  const int nt = min(p.tokens, p.T - t0);
  token_places(p, t0, nt, at);
  token_angles(p, t0, nt, cs);
  __syncthreads();
  for (int slot = threadIdx.x; slot < p.items * p.ha; slot += blockDim.x) {
    const int head = slot / p.items, lane = slot - head * p.items;
    const int part = head < p.hq ? 0 : head < p.hr ? 1 : 2;
    const bool pair = Item<T, HALF, VEC>::two(lane, half);
    const int d = Item<T, HALF, VEC>::first(lane, half, p.rot);
    const T* src = static_cast<const T*>(p.x) + t0 * p.ldx + head * p.D;
    T* dst = static_cast<T*>(part == 0 ? p.out[0] : part == 1 ? p.out[1] : p.out[2]) +
             (part == 0 ? head * p.sh[0] : part == 1 ? (head - p.hq) * p.sh[1] : (head - p.hr) * p.sh[2]);
    const long* to = at[part];
    for (int tt = 0; tt < nt; tt += kBatch) {
      Item<T, HALF, VEC> it[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (tt + i < nt) it[i].load(src, d, pair, half);
        src += p.ldx;
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (tt + i < nt) {
          if (part < 2) it[i].turn(cs + (tt + i) * half, d, pair, p.rot);
          it[i].store(dst + to[tt + i], d, pair, half);
        }
      }
    }
  }
}

// Heads that begin on 16-byte boundaries with a rot whose halves (or end) do
// not: the tokens' rows go through shared memory, copied in and out 16 bytes at
// a time, and the pairs are turned in place there.  2400 tokens of 24 heads x
// 128 with 74 dims turned: 11.5 us, element by element from memory 24.2.
constexpr int kStagedThreads = 512;
constexpr int kStagedSmem = 46 * 1024;

template <typename T, bool HALF>
__global__ void __launch_bounds__(kStagedThreads) rope_staged_kernel(const RopeParams p) {
  extern __shared__ uint4 rows4[];  // [tokens][units], then cos, sin [tokens][rot / 2]
  __shared__ long at[3][kMaxTokens];
  pdl_wait();
  pdl_launch_dependents();
  constexpr int kUnit = 16 / static_cast<int>(sizeof(T));
  const int half = p.rot >> 1, units = p.ha * p.D / kUnit;  // 16-byte units of a row
  const int t0 = blockIdx.x * p.tokens;
  const int nt = min(p.tokens, p.T - t0);
  float2* cs = reinterpret_cast<float2*>(rows4 + p.tokens * units);
  for (int tt = 0; tt < nt; ++tt) {
    const T* src = static_cast<const T*>(p.x) + (t0 + tt) * p.ldx;
    for (int u = threadIdx.x; u < units; u += kStagedThreads) cp_async16(rows4 + tt * units + u, src + u * kUnit);
  }
  cp_async_commit();
  token_places(p, t0, nt, at);
  token_angles(p, t0, nt, cs);
  cp_async_wait_all();
  __syncthreads();
  // the threads walk (token, head, pair) in order, kStagedThreads pairs a step
  const int step_h = kStagedThreads / half, step_i = kStagedThreads - step_h * half;
  int i = threadIdx.x % half, head = threadIdx.x / half, tt = 0;
  while (true) {
    while (head >= p.hr) {
      head -= p.hr;
      ++tt;
    }
    if (tt >= nt) break;
    T* row = reinterpret_cast<T*>(rows4 + tt * units) + head * p.D;
    const int d0 = HALF ? i : 2 * i, d1 = HALF ? i + half : 2 * i + 1;
    const float2 c = cs[tt * half + i];
    const float x = Pack<T>::get(row + d0), y = Pack<T>::get(row + d1);
    Pack<T>::put(row + d0, x * c.x - y * c.y);
    Pack<T>::put(row + d1, y * c.x + x * c.y);
    i += step_i;
    head += step_h;
    if (i >= half) {
      i -= half;
      ++head;
    }
  }
  __syncthreads();
  const int per_head = p.D / kUnit;
  for (int tt = 0; tt < nt; ++tt) {
    for (int u = threadIdx.x; u < units; u += kStagedThreads) {
      const int head = u / per_head;
      const int part = head < p.hq ? 0 : head < p.hr ? 1 : 2;
      const long to = part == 0 ? head * p.sh[0] : part == 1 ? (head - p.hq) * p.sh[1] : (head - p.hr) * p.sh[2];
      T* dst = static_cast<T*>(part == 0 ? p.out[0] : part == 1 ? p.out[1] : p.out[2]) + at[part][tt] + to;
      *reinterpret_cast<uint4*>(dst + (u - head * per_head) * kUnit) = rows4[tt * units + u];
    }
  }
}

bool al(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename T>
const void* staged_ptr(bool half) {
  return half ? reinterpret_cast<const void*>(rope_staged_kernel<T, true>)
              : reinterpret_cast<const void*>(rope_staged_kernel<T, false>);
}
template <typename T>
const void* rope_ptr(bool half, bool vec) {
  if (half)
    return vec ? reinterpret_cast<const void*>(rope_kernel<T, true, true>)
               : reinterpret_cast<const void*>(rope_kernel<T, true, false>);
  return vec ? reinterpret_cast<const void*>(rope_kernel<T, false, true>)
             : reinterpret_cast<const void*>(rope_kernel<T, false, false>);
}

}  // namespace

// Whether an output whose first head is head `at` of x lies over it element for element.
static bool over_x(const rfx_rope_desc& d, const Places& out, long at) {
  return (d.S == 1 || out.step[2] == d.ldx) && (d.B == 1 || out.step[0] == static_cast<__int128>(d.S) * d.ldx) &&
         (out.n[1] == 1 || out.step[1] == d.head_dim) &&
         reinterpret_cast<uintptr_t>(out.p) == reinterpret_cast<uintptr_t>(d.x) + at * d.head_dim * out.elem;
}

// The descriptor with the strides of packed outputs written out.
static rfx_rope_desc with_strides(rfx_rope_desc d) {
  auto pack = [&](long H, long& sb, long& sh, long& ss) {
    if (sb || sh || ss) return;
    sb = H * d.S * d.head_dim;
    sh = static_cast<long>(d.S) * d.head_dim;
    ss = d.head_dim;
  };
  pack(d.num_q_heads, d.qs_b, d.qs_h, d.qs_s);
  pack(d.num_kv_heads, d.ks_b, d.ks_h, d.ks_s);
  pack(d.num_kv_heads, d.vs_b, d.vs_h, d.vs_s);
  return d;
}

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
  const rfx_rope_desc s = with_strides(d);
  const Places out[3] = {
      {d.q_out, esz, d.head_dim, {d.B, d.num_q_heads, d.S}, {s.qs_b, s.qs_h, s.qs_s}},
      {d.k_out, esz, d.head_dim, {d.B, d.num_kv_heads, d.S}, {s.ks_b, s.ks_h, s.ks_s}},
      {d.v_out, esz, d.head_dim, {d.B, d.num_kv_heads, d.S}, {s.vs_b, s.vs_h, s.vs_s}},
  };
  for (const Places& o : out)
    if (o.p && places_overlap(o))
      return set_error(RFX_E_INVAL, "rfx_rope: heads or tokens of an output overlap (strides %ld, %ld, %ld)", o.step[0],
                       o.step[1], o.step[2]);
  const long T = static_cast<long>(d.B) * d.S;
  const Places x{d.x, esz, heads * d.head_dim, {T, 1, 1}, {d.ldx, 0, 0}};
  const Places pos{d.positions, 4, T, {1, 1, 1}, {}}, freq{d.inv_freq, 8, d.rot_dim / 2, {1, 1, 1}, {}};
  bool over[3];
  for (int i = 0; i < 3; ++i) {
    over[i] = over_x(d, out[i], i == 0 ? 0 : i == 1 ? d.num_q_heads : d.num_q_heads + d.num_kv_heads);
    if (!over[i] && places_shared(out[i], x))
      return set_error(RFX_E_INVAL, "rfx_rope: an output lies across x (over its own heads exactly, or apart from x)");
    if (places_shared(out[i], pos) || places_shared(out[i], freq))
      return set_error(RFX_E_INVAL, "rfx_rope: an output shares memory with positions or inv_freq");
    // (what lies over x is apart from what does not, and from x's other heads)
    for (int j = 0; j < i; ++j)
      if (!over[i] && !over[j] && places_shared(out[i], out[j]))
        return set_error(RFX_E_INVAL, "rfx_rope: two outputs share memory");
  }
  return RFX_OK;
}

int launch_rope(const rfx_rope_desc& desc, cudaStream_t stream, bool pdl) {
  const int rc = validate_rope(desc);
  if (rc || desc.B == 0 || desc.S == 0) return rc;
  const rfx_rope_desc d = with_strides(desc);
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
  // 16-byte accesses: every row and head begins on a 16-byte boundary; then
  // whole items of 8 dims need the halves (or the end) of rot on one as well
  bool heads = d.head_dim % 8 == 0 && al(d.x, 16) && (d.ldx * esz) % 16 == 0;
  for (int i = 0; i < 3; ++i)
    heads = heads && (!p.out[i] || (al(p.out[i], 16) && ((p.sb[i] | p.sh[i] | p.ss[i]) * esz) % 16 == 0));
  const bool vec = heads && d.rot_dim % (half ? 16 : 8) == 0;
  int nsm = 148;
  rfx_num_sms(&nsm);
  const long token_bytes = static_cast<long>(p.ha) * d.head_dim * esz + 4l * d.rot_dim;
  if (heads && !vec && token_bytes <= kStagedSmem) {
    p.tokens = static_cast<int>(
        std::max(1l, std::min({(p.T - 1l) / (4 * nsm) + 1, static_cast<long>(kMaxTokens), kStagedSmem / token_bytes})));
    return launch_kernel(d.dtype == kDtypeBF16 ? staged_ptr<__nv_bfloat16>(half) : staged_ptr<float>(half),
                         dim3(static_cast<unsigned>((p.T - 1) / p.tokens + 1)), dim3(kStagedThreads),
                         static_cast<size_t>(p.tokens * token_bytes), stream, pdl, 1, p);
  }
  p.items = vec ? (half ? d.rot_dim / 16 + (d.head_dim - d.rot_dim) / 8 : d.head_dim / 8)
                : d.rot_dim / 2 + (d.head_dim - d.rot_dim);
  const int threads = std::min(kRopeThreads, (p.items * p.ha + 31) / 32 * 32);
  // tokens per CTA: one wave of CTAs over all tokens, their cos / sin within
  // 16 KB of shared memory
  const int half_rot = d.rot_dim / 2;
  const int slots = nsm * std::min(16, (half && vec ? resident_threads<true>() : resident_threads<false>()) / threads);
  p.tokens = std::max(1, std::min({(p.T - 1) / slots + 1, kMaxTokens, 16 * 1024 / (8 * half_rot)}));
  const unsigned grid = static_cast<unsigned>((p.T - 1) / p.tokens + 1);
  const void* fn = d.dtype == kDtypeBF16 ? rope_ptr<__nv_bfloat16>(half, vec) : rope_ptr<float>(half, vec);
  return launch_kernel(fn, dim3(grid), dim3(threads), static_cast<size_t>(p.tokens) * half_rot * sizeof(float2),
                       stream, pdl, 1, p);
}

}  // namespace rfx

extern "C" int rfx_rope(const rfx_rope_desc* d, void* stream) {
  if (!d) return rfx::set_error(RFX_E_INVAL, "rfx_rope: null descriptor");
  return rfx::launch_rope(*d, static_cast<cudaStream_t>(stream), rfx::pdl_enabled());
}
