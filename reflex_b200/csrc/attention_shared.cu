// Attention of B streams over one context that they all share, each stream's own
// quantized context of its own length, and its new tokens.
//
// Per KV head the query rows of all streams, B x (heads of the group) x S, are one
// matrix: its tiles of 128 rows (MMA M) cross stream boundaries, so the shared
// keys are multiplied with full tiles whatever a stream's share of rows, and read
// once per tile of rows and not once per stream.  After the shared key blocks a
// tile visits the own keys of each stream that it has rows of, where the other
// streams' rows see nothing.
//
// One unit of work is a 128-key block of one tile.  The units, in tile order, are
// dealt to the CTAs in equal runs, so all SMs work whatever the shape; a tile that
// several CTAs share leaves partial results (O, m, l) that a second kernel joins
// in CTA order (log-sum-exp weights), a whole tile is stored at once.
//
// The keys come as bf16 K and f16 V that a first kernel makes of the rings (exact
// casts of int8 with the scales kept aside; the reference's dequantize for uint8)
// and of the new tokens.  Per unit: S[128 x 128] = Q Kᵀ (fp32 in TMEM), online
// softmax into P (f16, in TMEM over S), O[128 x 256] += P V; S of the next block is
// computed during the softmax.
#include "rfx_internal.h"

#include <algorithm>

namespace rfx {
namespace {

constexpr int kD = 256;
constexpr int kRows = 128;  // query rows per tile
constexpr int kKeys = 128;  // keys per block
constexpr float kLog2e = 1.4426950408889634f;

struct Quantized {  // a ring: quantized rows (bytes), scales and zero points (elements)
  const uint8_t* k;
  const uint8_t* v;
  const void* k_scale;
  const void* v_scale;
  const void* k_zp;
  const void* v_zp;
  long qs_b, qs_h, qs_c;
  long ss_b, ss_h, ss_c;
};

struct SharedAttnParams {
  int B, Hq, Hkv, G, S;  // G = Hq / Hkv
  int mode, scale_bf16;
  int n_shared, own_max, n_new;
  Quantized shared, own;
  const unsigned char* shared_valid;
  const int* own_len;
  const __nv_bfloat16* q;
  long qs_b, qs_h, qs_s;
  const __nv_bfloat16* k_new;
  const __nv_bfloat16* v_new;
  long ks_b, ks_h, ks_s, vs_b, vs_h, vs_s;
  const int* new_block;
  float scale_log2;
  __nv_bfloat16* out;
  long ldo;
  // units: tiles of rows (all heads') x blocks of a tile
  int rows;         // B * G * S
  int tiles;        // Hkv * ceil(rows / 128)
  int head_tiles;   // ceil(rows / 128)
  int shared_blocks, own_blocks;  // of a head / of a stream and head
  int streams;      // that a tile has rows of, at most
  int tile_units;   // shared_blocks + streams * own_blocks
  long units;
  int ctas;
  // dense keys [block][128][256], shared blocks of each head first, then (stream,
  // head, own block); per block the words of its keys: [ks | vs | add | nb][128]
  __nv_bfloat16* kd;
  __half* vd;
  float* words;
  float* part_o;    // [2 * ctas][256 / 16][128][16]
  float2* part_ml;  // [2 * ctas][128]: m (log2 units), l
  int* status;
};

// Block ids: a key is visible to the rows of its stream whose id is not below its
// own.  Ring keys come below every new key's id, other streams' rows below them.
constexpr int kForeignRow = -0x7fffffff - 1;
constexpr int kRingKey = kForeignRow + 1;
__device__ __forceinline__ int block_id(const SharedAttnParams& p, int s) {
  return p.new_block ? max(p.new_block[s], kRingKey) : 0;
}

__device__ __forceinline__ int own_length(const SharedAttnParams& p, int b) {
  if (p.own_max == 0) return 0;
  return p.own_len ? min(max(p.own_len[b], 0), p.own_max) : p.own_max;
}

// The units [first, last) of one tile that a CTA works on.
struct Segment {
  int tile, first, last;
  bool whole;
};
__device__ __forceinline__ long cta_begin(const SharedAttnParams& p, int cta) {
  return p.units * cta / p.ctas;
}
// The CTA that has unit u.
__device__ __forceinline__ int cta_of(const SharedAttnParams& p, long u) {
  return static_cast<int>(((u + 1) * p.ctas - 1) / p.units);
}

// One live block of a tile: where its keys lie and whose rows see them.
struct Block {
  int index;   // of the dense keys
  int stream;  // -1: every row sees them
};
// Walks the blocks of a tile's units that hold keys.
struct Blocks {
  int h, b0, b1;  // KV head; streams of the tile's rows
  __device__ __forceinline__ Blocks(const SharedAttnParams& p, int tile) {
    h = tile / p.head_tiles;
    const int r0 = (tile - h * p.head_tiles) * kRows, per = p.G * p.S;
    b0 = r0 / per;
    b1 = min(r0 + kRows, p.rows) - 1;
    b1 = b1 / per;
  }
  // The first live unit from u on, before `last`; -1 if there is none.
  __device__ __forceinline__ int find(const SharedAttnParams& p, int u, int last, Block* out) const {
    for (; u < last; ++u) {
      if (u < p.shared_blocks) {
        out->index = h * p.shared_blocks + u;
        out->stream = -1;
        return u;
      }
      if (p.own_blocks == 0) return -1;
      const int w = u - p.shared_blocks, s = w / p.own_blocks, j = w - s * p.own_blocks;
      const int b = b0 + s;
      if (b > b1) return -1;
      if (j * kKeys < own_length(p, b) + p.n_new) {
        out->index = p.Hkv * p.shared_blocks + (b * p.Hkv + h) * p.own_blocks + j;
        out->stream = b;
        return u;
      }
    }
    return -1;
  }
};

__device__ __forceinline__ float load_scalar(const void* p, long i, bool bf16) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ float round_to(float x, bool bf16) { return bf16 ? bf16_round(x) : x; }

// ------------------------------------------------------------ dense keys ---
// One CTA per 16 keys of a block.  A key that no row may see has scores of -inf
// and zero rows, so that what its memory holds (a NaN in a scale, say) reaches no
// product.  New keys with values outside f16 (infinities, NaN) get a value scale
// of NaN and zero values: the rows that see them become NaN, the other streams'
// rows in the same tile multiply them by 0.
__global__ void __launch_bounds__(256) shared_dense_kernel(const __grid_constant__ SharedAttnParams p) {
  constexpr int kPer = 16;
  pdl_wait();
  pdl_launch_dependents();
  const int block = blockIdx.x / (kKeys / kPer), q0 = blockIdx.x % (kKeys / kPer) * kPer;
  const bool sbf16 = p.scale_bf16 != 0;
  const int n_sh = p.Hkv * p.shared_blocks;
  const bool is_shared = block < n_sh;
  int h, b, j;
  if (is_shared) {
    h = block / p.shared_blocks;
    j = block - h * p.shared_blocks;
    b = 0;
  } else {
    const int w = block - n_sh, bh = w / p.own_blocks;
    j = w - bh * p.own_blocks;
    b = bh / p.Hkv;
    h = bh - b * p.Hkv;
  }
  const Quantized& ring = is_shared ? p.shared : p.own;
  const int held = is_shared ? p.n_shared : own_length(p, b);
  const int total = is_shared ? held : held + p.n_new;
  if (j * kKeys >= total) return;  // no unit visits it
  __shared__ float dq[4][kPer];    // k scale, v scale, k zp, v zp of ring keys
  __shared__ int seen[kPer];       // 0: no key, 1: of the ring, 2: new
  __shared__ int bad[kPer];
  float* words = p.words + static_cast<long>(block) * 4 * kKeys;
  if (threadIdx.x < kPer) {
    const int t = q0 + threadIdx.x, key = j * kKeys + t;
    int kind = key < held ? 1 : key < total ? 2 : 0;
    if (is_shared && kind == 1 && p.shared_valid && p.shared_valid[key] == 0) kind = 0;
    float ks = 0.f, vs = 0.f;
    int nb = kRingKey;
    if (kind == 1) {
      const long si = b * ring.ss_b + h * ring.ss_h + key * ring.ss_c;
      const bool f32 = p.mode == kQuantI8Sym || !sbf16;
      const float k = load_scalar(ring.k_scale, si, !f32), v = load_scalar(ring.v_scale, si, !f32);
      if (p.mode == kQuantI8Sym) {
        ks = k * p.scale_log2;
        vs = v;
      } else {
        ks = p.scale_log2;
        vs = 1.f;
        dq[0][threadIdx.x] = k;
        dq[1][threadIdx.x] = v;
        dq[2][threadIdx.x] = load_scalar(ring.k_zp, si, sbf16);
        dq[3][threadIdx.x] = load_scalar(ring.v_zp, si, sbf16);
      }
    } else if (kind == 2) {
      ks = p.scale_log2;
      vs = 1.f;
      nb = block_id(p, key - held);
    }
    words[t] = ks;
    words[kKeys + t] = vs;
    words[2 * kKeys + t] = kind ? 0.f : -INFINITY;
    reinterpret_cast<int*>(words)[3 * kKeys + t] = nb;
    seen[threadIdx.x] = kind;
    bad[threadIdx.x] = 0;
  }
  __syncthreads();
  // 16 keys x 16 chunks of 16 dims, K by the first half of the loop and V by the
  // second; a new key's bad values are known only once all of it is looked at
  const int key = q0 + (threadIdx.x >> 4), g = threadIdx.x & 15;
  const int kind = seen[threadIdx.x >> 4];
  const long row = (static_cast<long>(block) * kKeys + key) * kD + g * 16;
  uint32_t wv[8];
#pragma unroll
  for (int isv = 0; isv < 2; ++isv) {
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 0u;
    if (kind == 1) {
      const uint4 raw = *reinterpret_cast<const uint4*>((isv ? ring.v : ring.k) + b * ring.qs_b + h * ring.qs_h +
                                                        static_cast<long>(j * kKeys + key) * ring.qs_c + g * 16);
      const uint8_t* b8 = reinterpret_cast<const uint8_t*>(&raw);
      float f[16];
      if (p.mode == kQuantI8Sym) {
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = static_cast<float>(static_cast<int8_t>(b8[e]));
      } else {
        const float sc = dq[isv ? 1 : 0][threadIdx.x >> 4], zp = dq[isv ? 3 : 2][threadIdx.x >> 4];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float t = round_to(__fsub_rn(static_cast<float>(b8[e]), zp), sbf16);
          f[e] = round_to(__fmul_rn(t, sc), sbf16);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = isv ? pack_f16x2(f[2 * e], f[2 * e + 1]) : pack_bf16x2(f[2 * e], f[2 * e + 1]);
    } else if (kind == 2) {
      const long n = j * kKeys + key - held;
      const __nv_bfloat16* src = isv ? p.v_new + b * p.vs_b + h * p.vs_h + n * p.vs_s : p.k_new + b * p.ks_b + h * p.ks_h + n * p.ks_s;
      const uint4 lo = *reinterpret_cast<const uint4*>(src + g * 16), hi = *reinterpret_cast<const uint4*>(src + g * 16 + 8);
      const uint32_t in[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = isv ? pack_f16x2(__uint_as_float(in[e] << 16), __uint_as_float(in[e] & 0xffff0000u)) : in[e];
    }
    if (isv) {
      bool out_of_range = false;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        out_of_range |= (w[e] & 0x7c00u) == 0x7c00u || (w[e] & 0x7c000000u) == 0x7c000000u;
      if (out_of_range) bad[threadIdx.x >> 4] = 1;
#pragma unroll
      for (int e = 0; e < 8; ++e) wv[e] = w[e];
    } else {
      uint4* dst = reinterpret_cast<uint4*>(p.kd + row);
      dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
      dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  __syncthreads();
  if (bad[threadIdx.x >> 4]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) wv[e] = 0u;
    if (g == 0) words[kKeys + key] = __uint_as_float(0x7fffffffu);
  }
  uint4* dst = reinterpret_cast<uint4*>(p.vd + row);
  dst[0] = make_uint4(wv[0], wv[1], wv[2], wv[3]);
  dst[1] = make_uint4(wv[4], wv[5], wv[6], wv[7]);
}

// ------------------------------------------------------------- attention ---
constexpr int kOffQ = 0;               // 4 x [128 rows x 64 dims] bf16
constexpr int kOffK = 65536;           // 4 x [128 keys x 64 dims] bf16, K-major
constexpr int kOffV = 131072;          // 2 halves x 4 x [64 keys x 64 dims] f16, MN-major
constexpr int kWords = 4 * kKeys;      // of one block
constexpr int kOffWords = 196608;      // 3 stages x kWords words
constexpr int kOffBar = kOffWords + 3 * kWords * 4;
constexpr int kOffXchg = kOffBar + 256;  // 768 floats: row maxima and sums of the two column halves
constexpr int kSmemBytes = kOffXchg + 3072 + 1024;
static_assert(kSmemBytes <= 227 * 1024, "shared memory");
// warp 0 copies, warp 1 issues MMAs, warps 2-9 run the softmax and the epilogue,
// two per TMEM lane quadrant, each on half of a row's columns
constexpr int kWorkers = 256;
constexpr int kThreads = 64 + kWorkers;

// Barrier over the two worker warps of a TMEM lane quadrant that also ANDs a
// flag over them: both leave a loop together when either saw a failed wait.
__device__ __forceinline__ bool pair_all(int quad, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(v ? 1u : 0u), "r"(2 + quad)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ bool workers_all(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(v ? 1u : 0u)
      : "memory");
  return r != 0;
}

__global__ void __launch_bounds__(kThreads, 1)
    attention_shared_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                            const __grid_constant__ SharedAttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* sWords = reinterpret_cast<float*>(smem + kOffWords);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* q_ready = bars + 0;
  uint64_t* k_full = bars + 1;    // [4] per dim block
  uint64_t* k_empty = bars + 5;   // [4]
  uint64_t* v_full = bars + 9;    // [2] per 64-key half
  uint64_t* v_empty = bars + 11;  // [2]
  uint64_t* s_full = bars + 13;   // [2] per S buffer
  uint64_t* w_full = bars + 15;   // [3] per words stage
  uint64_t* p_ready = bars + 18;  // [2] per S buffer
  uint64_t* o_done = bars + 20;
  uint64_t* o_free = bars + 21;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
  if (threadIdx.x == 0) {
    mbar_init(q_ready, kWorkers / 32);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], kWorkers / 32);
    }
    for (int i = 0; i < 3; ++i) mbar_init(&w_full[i], 1);
    mbar_init(o_done, 1);
    mbar_init(o_free, kWorkers / 32);
    fence_mbar_init();
    if (p.shared_blocks + p.own_blocks > 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmO = tmem;  // S buffers at columns 256 and 384, P over each S's own columns
  auto tmS = [&](int j) { return tmem + 256 + static_cast<uint32_t>(j & 1) * kKeys; };
  pdl_launch_dependents();
  pdl_wait();
  const long u0 = cta_begin(p, blockIdx.x), u1 = cta_begin(p, blockIdx.x + 1);
  const int tile0 = static_cast<int>(u0 / p.tile_units), tile1 = static_cast<int>((u1 - 1) / p.tile_units);
  auto segment = [&](int tile) {
    const long t0 = static_cast<long>(tile) * p.tile_units;
    Segment s;
    s.tile = tile;
    s.first = static_cast<int>(max(u0 - t0, 0l));
    s.last = static_cast<int>(min(u1 - t0, static_cast<long>(p.tile_units)));
    s.whole = s.first == 0 && s.last == p.tile_units;
    return s;
  };
  int k_iss = 0, v_iss = 0;  // dim-block / half loads issued (4 / 2 per block)

  if (warp == 0) {
    if (lane == 0) {
      // two queues from one thread, each bounded in time: K dim block a of a block
      // once the scores of the block before over it are done (with dim block 0 the
      // block's words), V half h once P V of the block before over it is done; V
      // never ahead of K
      struct Queue {
        int tile, u;
        Block blk;
        bool more;
      };
      auto advance = [&](Queue& q) {  // the next live block, in whichever tile
        while (q.tile <= tile1) {
          const Segment s = segment(q.tile);
          q.u = Blocks(p, q.tile).find(p, max(q.u, s.first), s.last, &q.blk);
          if (q.u >= 0) return;
          ++q.tile;
          q.u = 0;
        }
        q.more = false;
      };
      Queue kq{tile0, 0, {0, 0}, true}, vq{tile0, 0, {0, 0}, true};
      advance(kq);
      advance(vq);
      unsigned long long t0 = globaltimer_ns();
      while (vq.more) {
        bool moved = false;
        if (kq.more) {
          const int kb = k_iss >> 2, a = k_iss & 3;
          if (kb == 0 || mbar_try_wait(&k_empty[a], (kb - 1) & 1)) {
            if (a == 0) {
              mbar_arrive_expect_tx(&w_full[kb % 3], kWords * 4);
              bulk_load(sWords + (kb % 3) * kWords, p.words + static_cast<long>(kq.blk.index) * kWords, kWords * 4,
                        &w_full[kb % 3]);
            }
            mbar_arrive_expect_tx(&k_full[a], kKeys * 128);
            tma_load_2d(smem + kOffK + a * 16384, &tmK, &k_full[a], a * 64, kq.blk.index * kKeys);
            ++k_iss;
            if ((k_iss & 3) == 0) {
              ++kq.u;
              advance(kq);
            }
            moved = true;
          }
        }
        if (v_iss < 2 * (k_iss >> 2)) {
          const int vb = v_iss >> 1, h = v_iss & 1;
          if (vb == 0 || mbar_try_wait(&v_empty[h], (vb - 1) & 1)) {
            mbar_arrive_expect_tx(&v_full[h], 32768);
            for (int a = 0; a < 4; ++a)
              tma_load_2d(smem + kOffV + h * 32768 + a * 8192, &tmV, &v_full[h], a * 64, vq.blk.index * kKeys + h * 64);
            ++v_iss;
            if ((v_iss & 1) == 0) {
              ++vq.u;
              advance(vq);
            }
            moved = true;
          }
        }
        if (moved) {
          t0 = globaltimer_ns();
        } else if (globaltimer_ns() - t0 > kWaitLimitNs) {
          record_error(p.status, kDevTimeoutStageEmpty);
          break;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = make_idesc_f16(kRows, kKeys, true);
      constexpr uint32_t idesc_o = make_idesc_f16(kRows, kD, false, true);
      bool ok = true;
      int j = 0, seg = 0;
      for (int tile = tile0; tile <= tile1 && ok; ++tile) {
        const Segment s = segment(tile);
        const Blocks blocks(p, tile);
        Block blk;
        int u = blocks.find(p, s.first, s.last, &blk);
        if (u < 0) continue;
        const int j0 = j;
        auto pv = [&](int jp) {  // O += P V of block jp, P from TMEM
          if (!(ok = mbar_wait(&p_ready[jp & 1], (jp >> 1) & 1, p.status, kDevTimeoutConvert))) return;
          if (jp == j0 && seg > 0 && !(ok = mbar_wait(o_free, (seg - 1) & 1, p.status, kDevTimeoutConvert))) return;
          tc_fence_after();
          for (int h = 0; h < 2 && ok; ++h) {
            if (!(ok = mbar_wait(&v_full[h], jp & 1, p.status, kDevTimeoutTmaFull))) return;
            tc_fence_after();
            const uint32_t v_base = smem_u32(smem + kOffV + h * 32768);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              const uint64_t bd = make_sdesc_sw128(v_base + ks * 2048, 8192, 1024);
              umma_f16_ts(tmO, tmS(jp) + static_cast<uint32_t>(h * 64 + ks * 8), bd, idesc_o,
                          (jp > j0 || h > 0 || ks > 0) ? 1u : 0u);
            }
            umma_commit(&v_empty[h]);
          }
          umma_commit(o_done);
        };
        ok = mbar_wait(q_ready, seg & 1, p.status, kDevTimeoutXReady);
        for (; u >= 0 && ok; ++j) {
          // S buffer j % 2 last held P of two blocks before, read by the P V issued
          // before this point (MMAs of one thread run in order)
          for (int a = 0; a < 4 && ok; ++a) {
            if (!(ok = mbar_wait(&k_full[a], j & 1, p.status, kDevTimeoutTmaFull))) break;
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const uint64_t ad = make_sdesc_sw128(smem_u32(smem + kOffQ + a * 16384) + kk * 32, 16, 1024);
              const uint64_t bd = make_sdesc_sw128(smem_u32(smem + kOffK + a * 16384) + kk * 32, 16, 1024);
              umma_f16_ss(tmS(j), ad, bd, idesc_s, (a > 0 || kk > 0) ? 1u : 0u);
            }
            umma_commit(&k_empty[a]);
          }
          if (!ok) break;
          umma_commit(&s_full[j & 1]);
          if (j > j0) pv(j - 1);
          u = blocks.find(p, u + 1, s.last, &blk);
        }
        if (ok) pv(j - 1);
        ++seg;
      }
    }
  } else {
    const int quad = warp & 3;
    const int ch = (threadIdx.x - 64) >> 7;  // this warp's half of the row: 64 score / 128 output columns
    const int r = quad * 32 + lane;          // query row inside the tile == TMEM lane
    float* mx_x = reinterpret_cast<float*>(smem + kOffXchg);  // [2 blocks][2 halves][128] row maxima
    float* l_x = mx_x + 512;                                   // [2 halves][128] row sums
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    constexpr int kHalf = kKeys / 2;
    bool ok = true;
    int j = 0;
    for (int tile = tile0; tile <= tile1; ++tile) {
      const Segment s = segment(tile);
      const Blocks blocks(p, tile);
      const int R = (tile - blocks.h * p.head_tiles) * kRows + r;
      const bool row_valid = R < p.rows;
      const int per = p.G * p.S;
      const int b_row = row_valid ? R / per : -1;
      const int g_row = row_valid ? (R - b_row * per) / p.S : 0;
      const int s_row = row_valid ? R - b_row * per - g_row * p.S : 0;
      const int my_block = row_valid ? block_id(p, s_row) : 0;
      float m_run = -INFINITY, l_run = 0.f;
      Block blk;
      int u = blocks.find(p, s.first, s.last, &blk);
      const bool live = u >= 0;
      const int j0 = j;
      if (live) {
        // Q: each thread a half of its row (every MMA that read the tile before is
        // done: its last o_done)
        const __nv_bfloat16* q = p.q + b_row * p.qs_b + (blocks.h * p.G + g_row) * p.qs_h + s_row * p.qs_s;
#pragma unroll 4
        for (int c = 0; c < 16; ++c) {
          const int col = ch * 16 + c;  // 16-byte chunk of the row
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (row_valid) v = *reinterpret_cast<const uint4*>(q + col * 8);
          *reinterpret_cast<uint4*>(smem + kOffQ + (col >> 3) * 16384 + sw128_offset(r, col & 7)) = v;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_ready);
      }
      for (; u >= 0; ++j) {
        if (ok) ok = mbar_wait(&w_full[j % 3], (j / 3) & 1, p.status, kDevTimeoutTmaFull);
        if (ok) ok = mbar_wait(&s_full[j & 1], (j >> 1) & 1, p.status, kDevTimeoutMmaDone);
        ok = __all_sync(0xffffffffu, ok);
        // this half's keys: score scale (log2 units), value scale, additive mask
        // and block id
        const float* sc = sWords + (j % 3) * kWords + kHalf * ch;
        const float* ks_s = sc;
        const float* vs_s = sc + kKeys;
        const float* kadd_s = sc + 2 * kKeys;
        const int* nb_s = reinterpret_cast<const int*>(sc + 3 * kKeys);
        const bool own = blk.stream >= 0;
        const int upto = blk.stream == b_row ? my_block : kForeignRow;
        float z[kHalf];
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (ok) {
          tc_fence_after();
          {
            uint32_t rr[4][16];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld16(tmS(j) + lane_base + kHalf * ch + 16 * c, rr[c]);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 16; ++e) z[c * 16 + e] = __uint_as_float(rr[c][e]);
          }
#pragma unroll
          for (int c = 0; c < kHalf / 4; ++c) {
            const float4 km = reinterpret_cast<const float4*>(ks_s)[c];
            const float4 ka = reinterpret_cast<const float4*>(kadd_s)[c];
            z[4 * c + 0] = fmaf(z[4 * c + 0], km.x, ka.x);
            z[4 * c + 1] = fmaf(z[4 * c + 1], km.y, ka.y);
            z[4 * c + 2] = fmaf(z[4 * c + 2], km.z, ka.z);
            z[4 * c + 3] = fmaf(z[4 * c + 3], km.w, ka.w);
            if (own) {
              const int4 nb = reinterpret_cast<const int4*>(nb_s)[c];
              if (nb.x > upto) z[4 * c + 0] = -INFINITY;
              if (nb.y > upto) z[4 * c + 1] = -INFINITY;
              if (nb.z > upto) z[4 * c + 2] = -INFINITY;
              if (nb.w > upto) z[4 * c + 3] = -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], z[4 * c + e]);
          }
        }
        // the row's max over both column halves (the partner warp holds the other)
        float* mxb = mx_x + (j & 1) * 256;
        mxb[ch * 128 + r] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        ok = pair_all(quad, ok);
        if (!ok) break;  // both warps of the pair agree
        const float m_new = fmaxf(m_run, fmaxf(mxb[r], mxb[128 + r]));
        bool need = false;
        float m_use;
        if (m_run == -INFINITY) {
          m_use = m_new;
        } else if (m_new > m_run + 8.f) {
          need = true;
          m_use = m_new;
        } else {
          m_use = m_run;
        }
        const float alpha = need ? exp2f(m_run - m_use) : 1.f;
        const float m_sub = m_use == -INFINITY ? 0.f : m_use;
        if (__any_sync(0xffffffffu, need)) {
          // O is final for the rescale once P V of the block before is done
          ok = __all_sync(0xffffffffu, mbar_wait(o_done, (j - 1) & 1, p.status, kDevTimeoutMmaDone));
          if (!ok) {
            u = blocks.find(p, u + 1, s.last, &blk);
            continue;  // and the pair leaves together at the next exchange
          }
          tc_fence_after();
#pragma unroll 1
          for (int c0 = 8 * ch; c0 < 8 * ch + 8; c0 += 2) {
            uint32_t rr[2][16];
#pragma unroll
            for (int q = 0; q < 2; ++q) tmem_ld16(tmO + lane_base + (c0 + q) * 16, rr[q]);
            tmem_wait_ld();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
#pragma unroll
              for (int e = 0; e < 16; ++e) rr[q][e] = __float_as_uint(__uint_as_float(rr[q][e]) * alpha);
              tmem_st16(tmO + lane_base + (c0 + q) * 16, rr[q]);
            }
          }
        }
        // P (times the value scales) as f16 pairs over the first 32 of this
        // half's 64 score columns, which are already read
        float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int hq = 0; hq < 2; ++hq) {
          uint32_t pk[16];
#pragma unroll
          for (int c = 8 * hq; c < 8 * hq + 8; ++c) {
            const float4 vsc = reinterpret_cast<const float4*>(vs_s)[c];
            const float vv[4] = {vsc.x, vsc.y, vsc.z, vsc.w};
            float pe[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              pe[e] = ex2_approx(z[4 * c + e] - m_sub);
              ps[e] += pe[e];
              // a weight of 0 stays 0 whatever another stream's value scale is
              pe[e] = own && z[4 * c + e] == -INFINITY ? 0.f : pe[e] * vv[e];
            }
            pk[(2 * c) & 15] = pack_f16x2(pe[0], pe[1]);
            pk[(2 * c + 1) & 15] = pack_f16x2(pe[2], pe[3]);
          }
          tmem_st16(tmS(j) + lane_base + kHalf * ch + 16 * hq, pk);
        }
        l_run = l_run * alpha + ((ps[0] + ps[1]) + (ps[2] + ps[3]));
        m_run = m_use;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[j & 1]);
        u = blocks.find(p, u + 1, s.last, &blk);
      }
      // ---- epilogue: every pair takes its barrier once, whatever happened ----
      // (P V of the block before the last one may be on its way too: a wait for the
      // last one's parity alone would take the one two before it for done)
      if (live && ok && j > j0 + 1)
        ok = __all_sync(0xffffffffu, mbar_wait(o_done, (j - 2) & 1, p.status, kDevTimeoutMmaDone));
      if (live && ok && j > j0)
        ok = __all_sync(0xffffffffu, mbar_wait(o_done, (j - 1) & 1, p.status, kDevTimeoutMmaDone));
      tc_fence_after();
      l_x[ch * 128 + r] = l_run;
      ok = pair_all(quad, ok);
      if (ok) {
        l_run = l_x[r] + l_x[128 + r];  // in a fixed order
        const float inv_l = l_run > 0.f || l_run != l_run ? 1.f / l_run : 0.f;
        __nv_bfloat16* orow = p.out + (static_cast<long>(b_row) * p.S + s_row) * p.ldo + (blocks.h * p.G + g_row) * kD;
        const int slot = 2 * blockIdx.x + (tile == tile0 ? 0 : 1);
        float* wrow = p.part_o ? p.part_o + (static_cast<long>(slot) * (kD / 16) * kRows + r) * 16 : nullptr;
#pragma unroll 1
        for (int c0 = 8 * ch; c0 < 8 * ch + 8; c0 += 4) {
          uint32_t rr[4][16];
          if (live) {
#pragma unroll
            for (int q = 0; q < 4; ++q) tmem_ld16(tmO + lane_base + (c0 + q) * 16, rr[q]);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int e = 0; e < 16; ++e) rr[q][e] = 0u;
          }
          if (!row_valid) continue;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int c = c0 + q;
            if (s.whole) {
              uint32_t w8[8];
#pragma unroll
              for (int e = 0; e < 8; ++e)
                w8[e] = pack_bf16x2(__uint_as_float(rr[q][2 * e]) * inv_l, __uint_as_float(rr[q][2 * e + 1]) * inv_l);
              *reinterpret_cast<uint4*>(orow + c * 16) = make_uint4(w8[0], w8[1], w8[2], w8[3]);
              *reinterpret_cast<uint4*>(orow + c * 16 + 8) = make_uint4(w8[4], w8[5], w8[6], w8[7]);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                *reinterpret_cast<float4*>(wrow + static_cast<long>(c) * kRows * 16 + 4 * e) =
                    make_float4(__uint_as_float(rr[q][4 * e]), __uint_as_float(rr[q][4 * e + 1]),
                                __uint_as_float(rr[q][4 * e + 2]), __uint_as_float(rr[q][4 * e + 3]));
            }
          }
        }
        if (!s.whole && row_valid && ch == 0) p.part_ml[static_cast<long>(slot) * kRows + r] = make_float2(m_run, l_run);
      }
      if (live) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_free);
      }
      // all workers go on to the next tile or none does (its Q goes where this
      // tile's was)
      if (tile < tile1 && !(ok = workers_all(ok))) break;
    }
  }
  tc_fence_before();
  __syncthreads();
  // every issued load completes before the block leaves (a producer or MMA
  // issuer that stopped early)
  if (warp == 0 && lane == 0) {
    for (int a = 0; a < 4; ++a) {
      const int n = (k_iss - a + 3) / 4;
      if (n > 0) mbar_wait(&k_full[a], (n - 1) & 1, p.status, kDevTimeoutTmaFull);
    }
    for (int h = 0; h < 2; ++h) {
      const int n = (v_iss - h + 1) / 2;
      if (n > 0) mbar_wait(&v_full[h], (n - 1) & 1, p.status, kDevTimeoutTmaFull);
    }
    const int n_w = (k_iss + 3) / 4;
    for (int s = 0; s < 3; ++s) {
      const int n = (n_w - s + 2) / 3;
      if (n > 0) mbar_wait(&w_full[s], (n - 1) & 1, p.status, kDevTimeoutTmaFull);
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the partial results of the tiles that several CTAs had units of, in CTA
// order: one warp per row, lane l holding 8 of the 256 columns.
__global__ void __launch_bounds__(256) shared_combine_kernel(const __grid_constant__ SharedAttnParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long g = static_cast<long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int tile = static_cast<int>(g / kRows), r = static_cast<int>(g % kRows);
  const int h = tile / p.head_tiles, R = (tile - h * p.head_tiles) * kRows + r;
  if (tile >= p.tiles || R >= p.rows) return;
  const long t0 = static_cast<long>(tile) * p.tile_units;
  const int c0 = cta_of(p, t0), c1 = cta_of(p, t0 + p.tile_units - 1);
  if (c0 == c1) return;  // the tile was one CTA's: stored there
  // a CTA's first tile is in its slot 0, its last one in slot 1
  auto slot_of = [&](int c) { return 2 * c + (cta_begin(p, c) / p.tile_units == tile ? 0 : 1); };
  auto load = [&](int slot, float4& a, float4& b) {
    const float* o = p.part_o + ((static_cast<long>(slot) * (kD / 16) + (lane >> 1)) * kRows + r) * 16 + (lane & 1) * 8;
    a = *reinterpret_cast<const float4*>(o);
    b = *reinterpret_cast<const float4*>(o + 4);
  };
  float M = -INFINITY, L = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  constexpr int kBatch = 8;
  for (int c = c0; c <= c1; c += kBatch) {
    float4 a[kBatch], b[kBatch];
    float2 ml[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      ml[i] = make_float2(-INFINITY, 0.f);
      a[i] = b[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c + i <= c1) {
        const int slot = slot_of(c + i);
        ml[i] = p.part_ml[static_cast<long>(slot) * kRows + r];
        load(slot, a[i], b[i]);
      }
    }
    float m = M;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) m = fmaxf(m, ml[i].x);
    if (m == -INFINITY) {
      // nothing seen so far but, perhaps, scores that are NaN
#pragma unroll
      for (int i = 0; i < kBatch; ++i) L += ml[i].y;
      continue;
    }
    const float w0 = exp2f(M - m);
    L *= w0;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= w0;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float w = exp2f(ml[i].x - m);
      L = fmaf(w, ml[i].y, L);
      acc[0] = fmaf(w, a[i].x, acc[0]); acc[1] = fmaf(w, a[i].y, acc[1]);
      acc[2] = fmaf(w, a[i].z, acc[2]); acc[3] = fmaf(w, a[i].w, acc[3]);
      acc[4] = fmaf(w, b[i].x, acc[4]); acc[5] = fmaf(w, b[i].y, acc[5]);
      acc[6] = fmaf(w, b[i].z, acc[6]); acc[7] = fmaf(w, b[i].w, acc[7]);
    }
    M = m;
  }
  const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
  const int per = p.G * p.S, b = R / per, gq = (R - b * per) / p.S, s = R - b * per - gq * p.S;
  __nv_bfloat16* orow = p.out + (static_cast<long>(b) * p.S + s) * p.ldo + (h * p.G + gq) * kD + lane * 8;
  *reinterpret_cast<uint4*>(orow) =
      make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                 pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
}

// ------------------------------------------------------------ host side ---
bool al(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Sizes of a call and where its parts lie in the workspace.
struct Plan {
  SharedAttnParams p;
  long blocks;  // dense key blocks
  size_t kd, vd, words, part_o, part_ml, total;
  bool joined;  // some tile is several CTAs'
};

int plan_shared(const rfx_attn_shared_desc& d, Plan* out) {
  SharedAttnParams& p = out->p;
  p = SharedAttnParams{};
  p.B = d.B;
  p.Hq = d.num_q_heads;
  p.Hkv = d.num_kv_heads;
  p.G = d.num_q_heads / d.num_kv_heads;
  p.S = d.S;
  p.n_shared = d.n_shared;
  p.own_max = d.own_max;
  p.n_new = d.k_new ? d.S : 0;
  const long rows = static_cast<long>(d.B) * p.G * d.S;
  if (rows > (1l << 30)) return set_error(RFX_E_INVAL, "rfx_attention_shared: more than 2^30 query rows per KV head");
  p.rows = static_cast<int>(rows);
  p.head_tiles = (p.rows - 1) / kRows + 1;
  p.tiles = p.Hkv * p.head_tiles;
  p.shared_blocks = (d.n_shared + kKeys - 1) / kKeys;
  p.own_blocks = static_cast<int>((static_cast<long>(d.own_max) + p.n_new + kKeys - 1) / kKeys);
  // streams that a tile of rows can touch
  const long per = static_cast<long>(p.G) * d.S;
  const long touch = per >= kRows ? (per % kRows ? 2 : 1) : kRows % per ? kRows / per + 2 : kRows / per;
  p.streams = static_cast<int>(std::min<long>(touch, d.B));
  const long units = p.shared_blocks + static_cast<long>(p.streams) * p.own_blocks;
  out->blocks = static_cast<long>(p.Hkv) * (p.shared_blocks + static_cast<long>(d.B) * p.own_blocks);
  if (units * p.tiles > (1l << 40) || units > (1l << 28) || out->blocks * kKeys > 0x7fffffffl ||
      out->blocks * (kKeys / 16) > 0x7fffffffl)
    return set_error(RFX_E_INVAL, "rfx_attention_shared: too many keys");
  p.tile_units = static_cast<int>(std::max<long>(units, 1));  // (without keys: one empty unit, rows of zeros)
  p.units = static_cast<long>(p.tile_units) * p.tiles;
  int nsm = 148;
  rfx_num_sms(&nsm);
  p.ctas = static_cast<int>(std::min<long>(p.units, nsm));
  // whole tiles for every CTA?
  out->joined = p.units % p.ctas != 0 || (p.units / p.ctas) % p.tile_units != 0;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = (off + bytes + 1023) & ~size_t(1023);
    return o;
  };
  out->kd = take(static_cast<size_t>(out->blocks) * kKeys * kD * 2);
  out->vd = take(static_cast<size_t>(out->blocks) * kKeys * kD * 2);
  out->words = take(static_cast<size_t>(out->blocks) * kWords * 4);
  out->part_o = take(out->joined ? static_cast<size_t>(2) * p.ctas * kRows * kD * 4 : 0);
  out->part_ml = take(out->joined ? static_cast<size_t>(2) * p.ctas * kRows * 8 : 0);
  out->total = off;
  return RFX_OK;
}

int check_sizes(const rfx_attn_shared_desc& d) {
  if (d.B < 0 || d.S < 0 || d.num_q_heads < 1 || d.num_kv_heads < 1 || d.num_q_heads % d.num_kv_heads ||
      d.head_dim != kD || d.n_shared < 0 || d.own_max < 0)
    return set_error(RFX_E_INVAL,
                     "rfx_attention_shared: need head_dim=256, whole groups of query heads, B, S, n_shared and own_max "
                     ">= 0 (B=%d S=%d heads %d/%d dim %d n_shared=%d own_max=%d)",
                     d.B, d.S, d.num_q_heads, d.num_kv_heads, d.head_dim, d.n_shared, d.own_max);
  if (d.quant_mode != RFX_QUANT_I8_SYM && d.quant_mode != RFX_QUANT_U8_REF)
    return set_error(RFX_E_INVAL, "rfx_attention_shared: quant_mode");
  if (d.scale_dtype != kDtypeBF16 && d.scale_dtype != kDtypeF32)
    return set_error(RFX_E_INVAL, "rfx_attention_shared: scale_dtype");
  if (d.quant_mode == RFX_QUANT_I8_SYM && d.scale_dtype != kDtypeF32)
    return set_error(RFX_E_INVAL, "rfx_attention_shared: RFX_QUANT_I8_SYM rings have fp32 scales");
  if (!d.k_new != !d.v_new) return set_error(RFX_E_INVAL, "rfx_attention_shared: k_new and v_new come together");
  return RFX_OK;
}

int check_ring(const char* name, const rfx_kv_view& r, int mode, int scale_dtype) {
  if (!r.k || !r.v || !r.k_scale || !r.v_scale || (mode == RFX_QUANT_U8_REF && (!r.k_zp || !r.v_zp)))
    return set_error(RFX_E_INVAL, "rfx_attention_shared: null pointer in the %s ring", name);
  if (!al(r.k, 16) || !al(r.v, 16) || r.qs_b % 16 || r.qs_h % 16 || r.qs_c % 16)
    return set_error(RFX_E_INVAL, "rfx_attention_shared: rows of the %s ring must begin on 16-byte boundaries", name);
  const unsigned e = scale_dtype == kDtypeBF16 ? 2 : 4;
  if (!al(r.k_scale, e) || !al(r.v_scale, e) || !al(r.k_zp, e) || !al(r.v_zp, e))
    return set_error(RFX_E_INVAL, "rfx_attention_shared: misaligned scales of the %s ring", name);
  return RFX_OK;
}

Quantized quantized(const rfx_kv_view& r) {
  return Quantized{static_cast<const uint8_t*>(r.k), static_cast<const uint8_t*>(r.v), r.k_scale, r.v_scale, r.k_zp, r.v_zp,
                   r.qs_b, r.qs_h, r.qs_c, r.ss_b, r.ss_h, r.ss_c};
}

int validate(const rfx_attn_shared_desc& d, Plan* plan) {
  int rc = check_sizes(d);
  if (rc || d.B == 0 || d.S == 0) return rc;
  if (!d.q || !d.out) return set_error(RFX_E_INVAL, "rfx_attention_shared: null q or out");
  if (d.n_shared > 0 && (rc = check_ring("shared", d.shared, d.quant_mode, d.scale_dtype))) return rc;
  if (d.own_max > 0 && (rc = check_ring("own", d.own, d.quant_mode, d.scale_dtype))) return rc;
  if (!al(d.q, 16) || d.qs_b % 8 || d.qs_h % 8 || d.qs_s % 8 || !al(d.out, 16) || d.ldo % 8 ||
      d.ldo < static_cast<long>(d.num_q_heads) * kD ||
      (d.k_new && (!al(d.k_new, 16) || !al(d.v_new, 16) || d.ks_b % 8 || d.ks_h % 8 || d.ks_s % 8 || d.vs_b % 8 ||
                   d.vs_h % 8 || d.vs_s % 8)))
    return set_error(RFX_E_INVAL,
                     "rfx_attention_shared: heads of q, out, k_new and v_new must begin on 16-byte boundaries (ldo at "
                     "least a row)");
  if (!al(d.own_len, 4) || !al(d.new_block, 4))
    return set_error(RFX_E_INVAL, "rfx_attention_shared: misaligned own_len or new_block");
  const long heads = d.num_q_heads, kv = d.num_kv_heads;
  const Places o{d.out, 2, heads * kD, {static_cast<long>(d.B) * d.S, 1, 1}, {d.ldo, 0, 0}};
  auto ring = [&](const void* p, const rfx_kv_view& r, long b, long n) {
    return Places{n > 0 ? p : nullptr, 1, kD, {b, kv, n}, {r.qs_b, r.qs_h, r.qs_c}};
  };
  auto scales = [&](const void* p, const rfx_kv_view& r, long b, long n) {
    return Places{n > 0 ? p : nullptr, d.scale_dtype == kDtypeBF16 ? 2 : 4, 1, {b, kv, n}, {r.ss_b, r.ss_h, r.ss_c}};
  };
  auto fresh = [&](const void* p, long sb, long sh, long ss) { return Places{p, 2, kD, {d.B, kv, d.S}, {sb, sh, ss}}; };
  const Places inputs[] = {
      {d.q, 2, kD, {d.B, heads, d.S}, {d.qs_b, d.qs_h, d.qs_s}},
      ring(d.shared.k, d.shared, 1, d.n_shared), ring(d.shared.v, d.shared, 1, d.n_shared),
      ring(d.own.k, d.own, d.B, d.own_max), ring(d.own.v, d.own, d.B, d.own_max),
      scales(d.shared.k_scale, d.shared, 1, d.n_shared), scales(d.shared.v_scale, d.shared, 1, d.n_shared),
      scales(d.shared.k_zp, d.shared, 1, d.n_shared), scales(d.shared.v_zp, d.shared, 1, d.n_shared),
      scales(d.own.k_scale, d.own, d.B, d.own_max), scales(d.own.v_scale, d.own, d.B, d.own_max),
      scales(d.own.k_zp, d.own, d.B, d.own_max), scales(d.own.v_zp, d.own, d.B, d.own_max),
      fresh(d.k_new, d.ks_b, d.ks_h, d.ks_s), fresh(d.v_new, d.vs_b, d.vs_h, d.vs_s),
      {d.shared_valid, 1, d.n_shared, {1, 1, 1}, {}},
      {d.own_len, 4, d.B, {1, 1, 1}, {}},
      {d.new_block, 4, d.S, {1, 1, 1}, {}},
  };
  rc = plan_shared(d, plan);
  if (rc) return rc;
  if (!d.workspace || d.workspace_bytes < plan->total || !al(d.workspace, 1024))
    return set_error(RFX_E_INVAL, "rfx_attention_shared: needs a 1024-byte aligned workspace of %zu bytes", plan->total);
  const Places ws{d.workspace, 1, static_cast<long>(plan->total), {1, 1, 1}, {}};
  if (places_shared(o, ws)) return set_error(RFX_E_INVAL, "rfx_attention_shared: out lies in the workspace");
  for (const Places& in : inputs) {
    if (in.width > 0 && places_shared(o, in)) return set_error(RFX_E_INVAL, "rfx_attention_shared: out shares memory with an input");
    if (in.width > 0 && places_shared(ws, in))
      return set_error(RFX_E_INVAL, "rfx_attention_shared: the workspace shares memory with an input");
  }
  return RFX_OK;
}

}  // namespace

int attention_shared_launches(const rfx_attn_shared_desc& d) {
  Plan plan;
  if (d.B == 0 || d.S == 0 || plan_shared(d, &plan)) return 0;
  return (plan.blocks > 0 ? 1 : 0) + 1 + (plan.joined ? 1 : 0);
}

int validate_attention_shared(const rfx_attn_shared_desc& d) {
  Plan plan;
  return validate(d, &plan);
}

int launch_attention_shared(const rfx_attn_shared_desc& d, cudaStream_t stream, bool pdl) {
  Plan plan;
  int rc = validate(d, &plan);
  if (rc || d.B == 0 || d.S == 0) return rc;
  const void* fn = reinterpret_cast<const void*>(attention_shared_kernel);
  rc = ensure_smem_attr(fn, kSmemBytes);
  if (rc) return rc;
  SharedAttnParams& p = plan.p;
  p.mode = d.quant_mode;
  p.scale_bf16 = d.scale_dtype == RFX_DTYPE_BF16;
  p.shared = quantized(d.shared);
  p.own = quantized(d.own);
  p.shared_valid = d.shared_valid;
  p.own_len = d.own_len;
  p.q = static_cast<const __nv_bfloat16*>(d.q);
  p.qs_b = d.qs_b;
  p.qs_h = d.qs_h;
  p.qs_s = d.qs_s;
  p.k_new = static_cast<const __nv_bfloat16*>(d.k_new);
  p.v_new = static_cast<const __nv_bfloat16*>(d.v_new);
  p.ks_b = d.ks_b;
  p.ks_h = d.ks_h;
  p.ks_s = d.ks_s;
  p.vs_b = d.vs_b;
  p.vs_h = d.vs_h;
  p.vs_s = d.vs_s;
  p.new_block = d.new_block;
  p.scale_log2 = d.softmax_scale * kLog2e;
  p.out = static_cast<__nv_bfloat16*>(d.out);
  p.ldo = d.ldo;
  char* ws = static_cast<char*>(d.workspace);
  p.kd = reinterpret_cast<__nv_bfloat16*>(ws + plan.kd);
  p.vd = reinterpret_cast<__half*>(ws + plan.vd);
  p.words = reinterpret_cast<float*>(ws + plan.words);
  p.part_o = reinterpret_cast<float*>(ws + plan.part_o);
  p.part_ml = reinterpret_cast<float2*>(ws + plan.part_ml);
  p.status = device_status_ptr();
  CUtensorMap k{}, v{};
  if (plan.blocks > 0) {
    const uint64_t keys = static_cast<uint64_t>(plan.blocks) * kKeys;
    rc = make_tmap_2d(&k, p.kd, 2, kD, keys, kD * 2, 64, kKeys, true);
    if (rc) return rc;
    rc = make_tmap_2d(&v, p.vd, 2, kD, keys, kD * 2, 64, 64, true);
    if (rc) return rc;
    rc = launch_kernel(reinterpret_cast<const void*>(shared_dense_kernel),
                       dim3(static_cast<unsigned>(plan.blocks * (kKeys / 16))), dim3(256), 0, stream, pdl, 1, p);
    if (rc) return rc;
  }
  rc = launch_kernel(fn, dim3(p.ctas), dim3(kThreads), kSmemBytes, stream, pdl, 1, k, v, p);
  if (rc || !plan.joined) return rc;
  return launch_kernel(reinterpret_cast<const void*>(shared_combine_kernel), dim3(static_cast<unsigned>(p.tiles * (kRows / 8))),
                       dim3(256), 0, stream, pdl, 1, p);
}

}  // namespace rfx

extern "C" int rfx_attention_shared_workspace_size(const rfx_attn_shared_desc* desc, size_t* bytes) {
  using namespace rfx;
  if (!desc || !bytes) return set_error(RFX_E_INVAL, "rfx_attention_shared_workspace_size: null argument");
  int rc = check_sizes(*desc);
  if (rc) return rc;
  *bytes = 0;
  if (desc->B == 0 || desc->S == 0) return RFX_OK;
  Plan plan;
  rc = plan_shared(*desc, &plan);
  if (rc) return rc;
  *bytes = plan.total;
  return RFX_OK;
}

extern "C" int rfx_attention_shared(const rfx_attn_shared_desc* desc, void* stream) {
  using namespace rfx;
  if (!desc) return set_error(RFX_E_INVAL, "rfx_attention_shared: null descriptor");
  return launch_attention_shared(*desc, static_cast<cudaStream_t>(stream), pdl_enabled());
}
