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
// One unit of work is a 64-key block of one tile: S[128 x 64] = Q Kᵀ (Q from TMEM,
// fp32 into TMEM), online softmax into P (f16, shared memory), O[128 x 256] += P V.
// O takes 256 TMEM columns and Q 128, which leaves two buffers of S for 64 keys.  A
// buffer is free as soon as its softmax has read it, so S runs two blocks ahead of P
// V.  (Q in shared memory would make S wait for operands: 192 bytes a clock.)
//
// What bounds it: a block's MMAs take 1024 clocks, and a block comes about every 2400.  That
// is the chain of one softmax warp, whose two groups take the blocks in turn: 940
// instructions of 64 keys at 2 warps per scheduler, which issues in 27 % of its clocks.
// A third group (152 registers a thread, a tile's end in smaller steps) gained 3 % on the
// first batch below and lost 6 and 9 % on the last and on small ones.  64 streams of 50
// tokens x 8 heads over 818 shared slots: 61 us, 374 TFLOP/s; 16 of 51 over 6344: 75 us,
// 575 TFLOP/s; 64 single tokens over 32768: 51 us.
//
// K (bf16) and V (f16) of a block come by TMA from a dense copy of all keys that a
// first kernel makes (exact casts of int8, whose scales go to the scores and to P; the
// reference's uint8 scheme dequantized as it does).  Few query rows have a form of
// their own that reads the rings itself.
//
// How the units are dealt to CTAs:
//   * a cluster of CTAs per tile, each a run of its units; they leave their (O, m, l)
//     in memory, and after the cluster's barrier each joins a part of the columns;
//   * runs of all tiles' units, equal for all SMs; a tile that several CTAs share
//     leaves partial results that the last of few CTAs, or a second kernel, joins.
// Each adds the parts in CTA order (log-sum-exp weights), whichever CTA is last.
#include "quant_i8.cuh"
#include "rfx_internal.h"

#include <algorithm>
#include <type_traits>

namespace rfx {
namespace {

constexpr int kD = 256;
constexpr int kRows = 128;  // query rows per tile
constexpr int kKeys = 64;   // keys per block
constexpr int kWords = 4 * kKeys + 4;  // of one block (the last 3 fill up 16 bytes)
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
  int tile_rows;    // rows per tile: 128, or 16 in the form for few
  int tiles;        // Hkv * head_tiles
  int head_tiles;   // ceil(rows / tile_rows)
  int shared_blocks, own_blocks;  // of a head / of a stream and head
  int tile_units;   // shared_blocks + own_blocks of each stream that a tile can have rows of
  int cluster;      // CTAs per tile, or 0: runs of units over `ctas` CTAs,
  int ctas;
  int run, longer;  // `run` units each, the first `longer` CTAs one more
  int join;         // of the CTAs of a tile the last to finish joins the parts
  int early;        // q is there once this grid runs: the keys' copy went before
  // dense keys [block][64][256], shared blocks of each head first, then (stream,
  // head, own block); per block the words of its keys: [ks | vs | add | nb][64], and the
  // lift of all of them
  __nv_bfloat16* kd;
  __half* vd;
  float* words;
  // parts of tiles, a slot per CTA of a cluster, or two per CTA
  float* part_o;    // [slot][256 / 4][tile_rows][4]
  float2* part_ml;  // [slot][tile_rows]: m (log2 units), l
  int* arrived;     // [tile] CTAs whose part is there
  int* status;
};

// Block ids: a key is visible to the rows of its stream whose id is not below its
// own.  They may be any numbers, and ring keys have the lowest; that a row is another
// stream's, or that a key's place is empty, is told apart from them.
constexpr int kRingKey = -0x7fffffff - 1;
__device__ __forceinline__ int block_id(const SharedAttnParams& p, int s) { return p.new_block ? p.new_block[s] : 0; }

__device__ __forceinline__ int own_length(const SharedAttnParams& p, int b) {
  if (p.own_max == 0) return 0;
  return p.own_len ? min(max(p.own_len[b], 0), p.own_max) : p.own_max;
}

// Whether a stream's rows see any key (each sees its own new one).
__device__ __noinline__ bool sees_key(const SharedAttnParams& p, int b) {
  if (p.n_new > 0 || own_length(p, b) > 0 || (p.n_shared > 0 && !p.shared_valid)) return true;
  for (int i = 0; i < p.n_shared; ++i)
    if (p.shared_valid[i]) return true;
  return false;
}

// Runs of units.
__device__ __forceinline__ int cta_begin(const SharedAttnParams& p, int cta) { return cta * p.run + min(cta, p.longer); }
// The CTA that has unit u.
__device__ __forceinline__ int cta_of(const SharedAttnParams& p, int u) {
  const int head = p.longer * (p.run + 1);
  return u < head ? u / (p.run + 1) : p.longer + (u - head) / p.run;
}

// The units [first, last) of one tile that a CTA works on.
struct Segment {
  int tile, first, last;
  bool whole;
};
// A CTA's tiles, first to last, and its segment of each.
struct Share {
  int u0, u1, tile0, tile1;
  __device__ __forceinline__ explicit Share(const SharedAttnParams& p) {
    if (p.cluster) {
      const int tile = blockIdx.x / p.cluster, rank = blockIdx.x - tile * p.cluster;
      u0 = tile * p.tile_units + static_cast<int>(static_cast<long>(rank) * p.tile_units / p.cluster);
      u1 = tile * p.tile_units + static_cast<int>(static_cast<long>(rank + 1) * p.tile_units / p.cluster);
      tile0 = tile1 = tile;
    } else {
      u0 = cta_begin(p, blockIdx.x);
      u1 = cta_begin(p, blockIdx.x + 1);
      tile0 = u0 / p.tile_units;
      tile1 = (u1 - 1) / p.tile_units;
    }
  }
  __device__ __forceinline__ Segment segment(const SharedAttnParams& p, int tile) const {
    const int t0 = tile * p.tile_units;
    Segment s;
    s.tile = tile;
    s.first = max(u0 - t0, 0);
    s.last = min(u1 - t0, p.tile_units);
    s.whole = s.first == 0 && s.last == p.tile_units;
    return s;
  }
};

// One block of a tile: where its keys lie and whose rows see them.
struct Block {
  int unit;    // -1: none left
  int stream;  // -1: shared, every row sees them
  int j;       // number among the shared blocks, or the stream's own
  int held, total;  // ring keys, and with the new ones, of the shared or of the stream's own
};
// Walks the blocks of a segment that hold keys: ROWS rows per tile, KEYS per block.
template <int ROWS, int KEYS>
struct Blocks {
  int h, b0, b1;  // KV head; streams of the tile's rows
  int last, shared_end;
  __device__ __forceinline__ Blocks(const SharedAttnParams& p, const Segment& s) {
    h = s.tile / p.head_tiles;
    const int r0 = (s.tile - h * p.head_tiles) * ROWS, per = p.G * p.S;
    b0 = r0 / per;
    b1 = (min(r0 + ROWS, p.rows) - 1) / per;
    last = s.last;
    shared_end = min(last, p.shared_blocks);
  }
  // The first block that holds keys from unit u on.
  __device__ __forceinline__ Block find(const SharedAttnParams& p, int u) const {
    for (; u < last; ++u) {
      if (u < p.shared_blocks) return Block{u, -1, u, p.n_shared, p.n_shared};
      if (p.own_blocks == 0) break;
      const int w = u - p.shared_blocks, s = w / p.own_blocks, j = w - s * p.own_blocks;
      if (b0 + s > b1) break;
      const int held = own_length(p, b0 + s);
      if (j * KEYS < held + p.n_new) return Block{u, b0 + s, j, held, held + p.n_new};
      u += p.own_blocks - j - 1;  // none of the stream's later ones does
    }
    return Block{-1, 0, 0, 0, 0};
  }
  // The block after b: another shared one, as a rule.
  __device__ __forceinline__ void step(const SharedAttnParams& p, Block& b) const {
    const int u = b.unit + 1;
    if (u < shared_end)
      b.unit = b.j = u;
    else
      b = find(p, u);
  }
  // A block's place among the dense keys.
  __device__ __forceinline__ int dense(const SharedAttnParams& p, const Block& b) const {
    return b.stream < 0 ? h * p.shared_blocks + b.j
                        : p.Hkv * p.shared_blocks + (b.stream * p.Hkv + h) * p.own_blocks + b.j;
  }
};

__device__ __forceinline__ float load_scalar(const void* p, long i, bool bf16) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ float round_to(float x, bool bf16) { return bf16 ? bf16_round(x) : x; }

// P times the value scales is f16, a product of the tensor cores' 16-bit kind (with the
// int8 values exact, outputs are 2e-4 from the formula, 2-norm, before their rounding to
// bf16, which is 1.7e-3).  f16's numbers are fine from 2^-14 to 2^16 only.  So a
// row's weights are not taken relative to its largest score, but to the largest sum of
// a block's largest score and its lift: the exponent of its largest value scale (all
// are below 2^that) less 7.  Then the largest products are between 2^7 and 2^15 whatever
// the values' size is, those down to 2^-21 of them have f16's 11 bits, and smaller ones
// steps of 2^-31 of them.  (Scales of 0, NaN and infinity have no say; beyond 2^-64 and
// 2^64 the lift stays what it is there, so that the sums of weights stay in range.)
__device__ __forceinline__ uint32_t lift_bits(float value_scale) {
  const uint32_t b = __float_as_uint(value_scale) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ float lift_of(uint32_t bits) {
  return static_cast<float>(min(max(static_cast<int>((bits + 0x7fffffu) >> 23) - 127, -64), 64) - 7);
}

// ------------------------------------------------------------ dense keys ---
// One CTA per 16 keys of a block (768 blocks, 17 MB in and 50 out, 15 us from cold memory).  A key that no row may see has scores of -inf
// and zero rows, so that what its memory holds (a NaN in a scale, say) reaches no
// product.  New keys with values outside f16 (infinities, NaN) get a value scale
// of NaN and zero values: the rows that see them become NaN, the other streams'
// rows in the same tile multiply them by 0.
__global__ void __launch_bounds__(256) shared_dense_kernel(const __grid_constant__ SharedAttnParams p) {
  constexpr int kPer = 16;
  // (before the grid behind this one may begin: what went before is done, and that
  // grid's early reads of q are safe)
  pdl_wait();
  pdl_launch_dependents();
  if (p.join)
    for (int i = blockIdx.x * 256 + threadIdx.x; i < p.tiles; i += gridDim.x * 256) p.arrived[i] = 0;
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
  // 16 threads per key, 16 dims each.  A key's kind: 0 none, 1 of the ring, 2 new.
  const int key = q0 + (threadIdx.x >> 4), g = threadIdx.x & 15, slot = j * kKeys + key;
  int kind = slot < held ? 1 : slot < total ? 2 : 0;
  uint4 raw[2][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) raw[i >> 1][i & 1] = make_uint4(0u, 0u, 0u, 0u);
  float scale[2] = {0.f, 0.f}, zp[2] = {0.f, 0.f};
  if (kind == 1) {
    const long at = b * ring.qs_b + h * ring.qs_h + slot * ring.qs_c + g * 16;
    raw[0][0] = *reinterpret_cast<const uint4*>(ring.k + at);
    raw[1][0] = *reinterpret_cast<const uint4*>(ring.v + at);
    const long si = b * ring.ss_b + h * ring.ss_h + slot * ring.ss_c;
    const bool f32 = p.mode == kQuantI8Sym || !sbf16;
    scale[0] = load_scalar(ring.k_scale, si, !f32);
    scale[1] = load_scalar(ring.v_scale, si, !f32);
    if (p.mode != kQuantI8Sym) {
      zp[0] = load_scalar(ring.k_zp, si, sbf16);
      zp[1] = load_scalar(ring.v_zp, si, sbf16);
    }
    if (is_shared && p.shared_valid && p.shared_valid[slot] == 0) kind = 0;
  } else if (kind == 2) {
    const long n = slot - held;
#pragma unroll
    for (int isv = 0; isv < 2; ++isv) {
      const __nv_bfloat16* src = isv ? p.v_new + b * p.vs_b + h * p.vs_h + n * p.vs_s : p.k_new + b * p.ks_b + h * p.ks_h + n * p.ks_s;
      raw[isv][0] = *reinterpret_cast<const uint4*>(src + g * 16);
      raw[isv][1] = *reinterpret_cast<const uint4*>(src + g * 16 + 8);
    }
  }
  float* words = p.words + static_cast<long>(block) * kWords;
  bool bad = false;
  const long row = (static_cast<long>(block) * kKeys + key) * kD + g * 16;
#pragma unroll
  for (int isv = 0; isv < 2; ++isv) {
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 0u;
    if (kind == 1) {
      const uint8_t* b8 = reinterpret_cast<const uint8_t*>(&raw[isv][0]);
      float f[16];
      if (p.mode == kQuantI8Sym) {
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = static_cast<float>(static_cast<int8_t>(b8[e]));
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = round_to(__fsub_rn(static_cast<float>(b8[e]), zp[isv]), sbf16);
          f[e] = round_to(__fmul_rn(x, scale[isv]), sbf16);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = isv ? pack_f16x2(f[2 * e], f[2 * e + 1]) : pack_bf16x2(f[2 * e], f[2 * e + 1]);
    } else if (kind == 2) {
      const uint4 lo = raw[isv][0], hi = raw[isv][1];
      const uint32_t in[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = isv ? pack_f16x2(__uint_as_float(in[e] << 16), __uint_as_float(in[e] & 0xffff0000u)) : in[e];
    }
    if (isv) {
#pragma unroll
      for (int e = 0; e < 8; ++e) bad |= (w[e] & 0x7c00u) == 0x7c00u || (w[e] & 0x7c000000u) == 0x7c000000u;
      // (a key's 16 threads are half of a warp)
      const uint32_t all = __ballot_sync(0xffffffffu, bad);
      bad = (all >> (threadIdx.x & 16) & 0xffffu) != 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = bad ? 0u : w[e];
    }
    uint4* dst = reinterpret_cast<uint4*>(isv ? reinterpret_cast<uint16_t*>(p.vd) + row : reinterpret_cast<uint16_t*>(p.kd) + row);
    dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
    dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
  const bool i8 = p.mode == kQuantI8Sym;
  const float vs = kind == 0 ? 0.f : bad ? __uint_as_float(0x7fffffffu) : kind == 1 && i8 ? scale[1] : 1.f;
  if (g == 0) {
    words[key] = kind == 0 ? 0.f : kind == 1 && i8 ? scale[0] * p.scale_log2 : p.scale_log2;
    words[kKeys + key] = vs;
    words[2 * kKeys + key] = kind ? 0.f : -INFINITY;
    reinterpret_cast<int*>(words)[3 * kKeys + key] = kind == 2 ? block_id(p, slot - held) : kRingKey;
  }
  // the block's lift: one warp looks at all of its value scales
  if (q0 == 0 && threadIdx.x < 32) {
    uint32_t most = 0u;
#pragma unroll
    for (int i = 0; i < kKeys; i += 32) {
      const int at = j * kKeys + i + threadIdx.x;
      if (at < held && i8 && !(is_shared && p.shared_valid && p.shared_valid[at] == 0))
        most = max(most, lift_bits(static_cast<const float*>(ring.v_scale)[b * ring.ss_b + h * ring.ss_h + at * ring.ss_c]));
      else if (at < total && !(at < held && i8))
        most = max(most, lift_bits(1.f));
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (threadIdx.x == 0) words[4 * kKeys] = lift_of(most);
  }
}

// ------------------------------------------------------------- attention ---
constexpr int kStages = 3;                   // of K,
constexpr int kStagesV = 2;                  // and of V
constexpr int kTile = kKeys * kD * 2;        // bytes of a block's K, or V
constexpr int kTileP = kRows * kKeys * 2;
constexpr int kOffK = 0;                     // [3] x 4 x [64 keys x 64 dims] bf16, K-major
constexpr int kOffV = kOffK + kStages * kTile;   // [2] x 4 x [64 keys x 64 dims] f16, MN-major
constexpr int kOffP = kOffV + kStagesV * kTile;  // [2] x [128 rows x 64 keys] f16, K-major
constexpr int kWordStages = 6;
constexpr int kOffWords = kOffP + 2 * kTileP;
constexpr int kOffXchg = kOffWords + kWordStages * kWords * 4;  // running maxima [2][128], the groups' sums and maxima [4][128]
constexpr int kOffStage = kOffXchg + 6 * kRows * 4;             // 32 rows x 64 bytes per worker warp
constexpr int kMaxCluster = 8;
constexpr int kOffBar = kOffStage + 8 * 2048;
constexpr int kSmemBytes = kOffBar + 512 + 1024;
static_assert(kSmemBytes <= 227 * 1024, "shared memory");
// TMEM columns
constexpr int kTmQ = 256;
constexpr int kTmS = 384;
// warp 0 copies K, warp 2 V, warp 1 issues MMAs, warps 4-11 run the softmax, two
// groups of four that take the blocks in turn (a thread has a row), and the epilogue
// (a group has half of the columns).  Two groups, because a block's chain from its
// scores to its P takes longer than its MMAs; what they pass on is the running
// maximum.
constexpr int kWorkers = 256;
constexpr int kFirstWorker = 128;
constexpr int kThreads = kFirstWorker + kWorkers;
constexpr int kJoinMost = 3;  // parts of a tile that the last CTA joins, at most
constexpr int kFewMost = 2048;  // rows per KV head up to which the form for few may be taken (its time is above the
                               // other's from about 1000 on, whatever the keys)

// Barrier over the two worker warps of a TMEM lane quadrant that also ANDs a
// flag over them.
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

// 4 int8 as bf16 or f16, exactly.  bf16 holds 8 significant bits: the low 7 over
// 128 and the sign bit over 128 are two numbers whose difference is the value.
// f16 holds 1024 + (q + 128).
__device__ __forceinline__ void i8_to_bf16(uint32_t q, uint32_t& lo, uint32_t& hi) {
  const uint32_t t[2] = {__byte_perm(q, 0u, 0x4140), __byte_perm(q, 0u, 0x4342)};
  uint32_t r[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t a = (t[i] & 0x007f007fu) | 0x43004300u, c = (t[i] & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&c));
    r[i] = *reinterpret_cast<const uint32_t*>(&d);
  }
  lo = r[0];
  hi = r[1];
}
__device__ __forceinline__ void i8_to_f16(uint32_t q, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = q ^ 0x80808080u, bias = 0x64806480u;
  const uint32_t t[2] = {__byte_perm(u, 0x64646464u, 0x4140), __byte_perm(u, 0x64646464u, 0x4342)};
  const __half2 b = *reinterpret_cast<const __half2*>(&bias);
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&t[0]), b), y = __hsub2(*reinterpret_cast<const __half2*>(&t[1]), b);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}
// Barrier wait that may sleep: the waiting warps' polls take issue slots from the
// others'.
__device__ __forceinline__ bool sleep_wait(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ bool wait_long(uint64_t* bar, uint32_t parity, int* status, int code) {
  if (sleep_wait(bar, parity)) return true;
  const unsigned long long t0 = globaltimer_ns();
  while (!sleep_wait(bar, parity)) {
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      record_error(status, code);
      return false;
    }
  }
  return true;
}

// A warp's 32 rows of 64 bytes through its own shared memory: in one direction or
// the other a lane has its row's 4 chunks, and 4 lanes have a row's between them, so
// that global accesses are whole 64-byte pieces.
__device__ __forceinline__ uint8_t* own_chunk(uint8_t* st, int lane, int c) {
  return st + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4);
}
__device__ __forceinline__ uint8_t* shared_chunk(uint8_t* st, int lane, int it) {
  const int row = it * 8 + (lane >> 2);
  return st + row * 64 + (((lane & 3) ^ ((row >> 1) & 3)) << 4);
}

// O, m and l of a row part: part_o [column / 4][row][4] and part_ml [row] of a slot.
__device__ __forceinline__ float4* part_at(const SharedAttnParams& p, long slot, int col4, int r) {
  return reinterpret_cast<float4*>(p.part_o) + (slot * (kD / 4) + col4) * p.tile_rows + r;
}

// 32 columns of a row's O, or zeros where no block was seen.
__device__ __forceinline__ void load_o(bool live, uint32_t at, uint32_t (&o)[2][16]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    if (live) tmem_ld16(at + q * 16, o[q]);
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (!live) o[q][e] = 0u;
  }
  if (live) tmem_wait_ld();
}

__device__ __forceinline__ int ld_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// Columns 8 g .. 8 g + 7 of a row, from parts that are added in order.
template <int BATCH = 8>
struct Joined {
  float M = -INFINITY, L = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  template <typename Slot>
  __device__ __forceinline__ void add(const SharedAttnParams& p, int n, int r, int g, Slot slot) {
    constexpr int kBatch = BATCH;
    for (int i0 = 0; i0 < n; i0 += kBatch) {
      float4 a[kBatch], b[kBatch];
      float2 ml[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        ml[i] = make_float2(-INFINITY, 0.f);
        a[i] = b[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i0 + i < n) {
          const long s = slot(i0 + i);
          ml[i] = __ldcg(p.part_ml + s * p.tile_rows + r);
          a[i] = __ldcg(part_at(p, s, 2 * g, r));
          b[i] = __ldcg(part_at(p, s, 2 * g + 1, r));
        }
      }
      float m = M;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) m = fmaxf(m, ml[i].x);
      // (nothing seen so far, but, perhaps, scores that are NaN: weights of 1)
      const float w0 = M == m ? 1.f : exp2f(M - m);
      L *= w0;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] *= w0;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float w = ml[i].x == m ? 1.f : exp2f(ml[i].x - m);
        L = fmaf(w, ml[i].y, L);
        acc[0] = fmaf(w, a[i].x, acc[0]); acc[1] = fmaf(w, a[i].y, acc[1]);
        acc[2] = fmaf(w, a[i].z, acc[2]); acc[3] = fmaf(w, a[i].w, acc[3]);
        acc[4] = fmaf(w, b[i].x, acc[4]); acc[5] = fmaf(w, b[i].y, acc[5]);
        acc[6] = fmaf(w, b[i].z, acc[6]); acc[7] = fmaf(w, b[i].w, acc[7]);
      }
      M = m;
    }
  }
  __device__ __forceinline__ uint4 result() const {
    const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
    return make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                      pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
  }
};

// Row R of KV head h: its stream, group head and token.
struct RowOf {
  int b, g, s;
  __device__ __forceinline__ RowOf(const SharedAttnParams& p, int R) {
    const int per = p.G * p.S;
    b = R / per;
    const int w = R - b * per;
    g = w / p.S;
    s = w - g * p.S;
  }
};
__device__ __forceinline__ long out_at(const SharedAttnParams& p, int h, const RowOf& w) {
  return (static_cast<long>(w.b) * p.S + w.s) * p.ldo + (h * p.G + w.g) * kD;
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
  uint64_t* k_full = bars + 1;    // [3]
  uint64_t* k_empty = bars + 4;   // [3]
  uint64_t* v_full = bars + 7;    // [2]
  uint64_t* v_empty = bars + 9;   // [2]
  uint64_t* s_free = bars + 11;   // [2] per S buffer
  uint64_t* s_full = bars + 13;   // [2] per S buffer
  uint64_t* p_ready = bars + 15;  // [2] per S buffer
  uint64_t* w_full = bars + 17;   // [6] per words stage
  uint64_t* o_last = bars + 23;   // every P V of a segment is done
  uint64_t* o_free = bars + 24;
  uint64_t* m_set = bars + 25;    // [4 quadrants][2 groups]: the running maxima after a block
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 33);
  volatile int* last_x = reinterpret_cast<volatile int*>(bars + 34);
  if (threadIdx.x == 0) {
    mbar_init(q_ready, kWorkers / 32);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_free[i], kWorkers / 64);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], kWorkers / 64);
      for (int q = 0; q < 4; ++q) mbar_init(&m_set[2 * q + i], 1);
    }
    for (int i = 0; i < kWordStages; ++i) mbar_init(&w_full[i], 1);
    mbar_init(o_last, 1);
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
  const uint32_t tmO = tmem, tmQ = tmem + kTmQ;
  auto tmS = [&](int j) { return tmem + kTmS + static_cast<uint32_t>(j & 1) * kKeys; };
  pdl_launch_dependents();
  const bool worker = threadIdx.x >= kFirstWorker;
  if (!worker || !p.early) pdl_wait();
  const Share share(p);
  int issued = 0;  // blocks whose K (warp 0) or V (warp 2) was requested

  if (warp == 0 || warp == 2) {
    // warp 0 copies K and the words, warp 2 V
    const bool is_v = warp == 2;
    if (is_v && share.tile1 > share.tile0) {
      // the second tile's Q into L2: the CTAs get there at about the same time, and
      // would wait for memory together
      const int tile = share.tile0 + 1, h = tile / p.head_tiles;
#pragma unroll 1
      for (int r = lane; r < kRows; r += 32) {
        const RowOf row(p, min((tile - h * p.head_tiles) * kRows + r, p.rows - 1));
        const __nv_bfloat16* q = p.q + row.b * p.qs_b + (h * p.G + row.g) * p.qs_h + row.s * p.qs_s;
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + 64 * i));
      }
    }
    if (lane == 0) {
      const int stages = is_v ? kStagesV : kStages;
      uint64_t* full = is_v ? v_full : k_full;
      uint64_t* empty = is_v ? v_empty : k_empty;
      const CUtensorMap* map = is_v ? &tmV : &tmK;
      uint8_t* ring = smem + (is_v ? kOffV : kOffK);
      bool ok = true;
      for (int tile = share.tile0; tile <= share.tile1 && ok; ++tile) {
        const Segment s = share.segment(p, tile);
        const Blocks<kRows, kKeys> blocks(p, s);
        for (Block b = blocks.find(p, s.first); b.unit >= 0; blocks.step(p, b)) {
          const int st = issued % stages, n = issued / stages, at = blocks.dense(p, b);
          if (n > 0 && !(ok = wait_long(&empty[st], (n - 1) & 1, p.status, kDevTimeoutStageEmpty))) break;
          if (!is_v) {
            // (the words' stage is that of six blocks before, whose P V was issued before
            // the S of the block that had K's stage: its softmax is done)
            const int ws = issued % kWordStages;
            mbar_arrive_expect_tx(&w_full[ws], kWords * 4);
            bulk_load(sWords + ws * kWords, p.words + static_cast<long>(at) * kWords, kWords * 4, &w_full[ws]);
          }
          mbar_arrive_expect_tx(&full[st], kTile);
          for (int a = 0; a < 4; ++a)
            tma_load_2d(ring + st * kTile + a * (kKeys * 128), map, &full[st], a * 64, at * kKeys);
          ++issued;
        }
      }
    }
  } else if (warp == 1) {
    // the whole warp walks the blocks and one elected lane issues: the loop's values
    // stay uniform
    constexpr uint32_t idesc_s = make_idesc_f16(kRows, kKeys, true);
    constexpr uint32_t idesc_o = make_idesc_f16(kRows, kD, false, true);
    const uint64_t kd0 = make_sdesc_sw128(smem_u32(smem + kOffK), 16, 1024);
    const uint64_t vd0 = make_sdesc_sw128(smem_u32(smem + kOffV), kKeys * 128, 1024);
    const uint64_t pd0 = make_sdesc_sw128(smem_u32(smem + kOffP), 16, 1024);
    bool ok = true;
    int j = 0, seg = 0;
    // stage and parity of the next S, and of the next P V
    int ss = 0, vs = 0;
    uint32_t sp = 0, vp = 0;
    auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
      return __all_sync(0xffffffffu, wait_long(bar, parity, p.status, code));
    };
    for (int tile = share.tile0; tile <= share.tile1 && ok; ++tile) {
      const Segment s = share.segment(p, tile);
      const Blocks<kRows, kKeys> blocks(p, s);
      Block blk = blocks.find(p, s.first);
      if (blk.unit < 0) continue;
      const int j0 = j;
      auto pv = [&](int jp, bool last) {  // O += P V of block jp
        if (!(ok = wait(&v_full[vs], vp, kDevTimeoutTmaFull))) return;
        if (!(ok = wait(&p_ready[jp & 1], (jp >> 1) & 1, kDevTimeoutConvert))) return;
        if (jp == j0 && seg > 0 && !(ok = wait(o_free, (seg - 1) & 1, kDevTimeoutConvert))) return;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = vd0 + static_cast<uint64_t>(vs) * (kTile >> 4);
          const uint64_t pd = pd0 + static_cast<uint64_t>(jp & 1) * (kTileP >> 4);
#pragma unroll
          for (int ks = 0; ks < kKeys / 16; ++ks)
            umma_f16_ss(tmO, pd + ks * 2, vd + ks * (2048 >> 4), idesc_o, (jp > j0 || ks > 0) ? 1u : 0u);
          umma_commit(&v_empty[vs]);
          if (last) umma_commit(o_last);
        }
        __syncwarp();
        if (++vs == kStagesV) {
          vs = 0;
          vp ^= 1;
        }
      };
      ok = wait(q_ready, seg & 1, kDevTimeoutXReady);
      for (; blk.unit >= 0 && ok; ++j) {
        // S runs two blocks ahead of P V
        if (!(ok = wait(&k_full[ss], sp, kDevTimeoutTmaFull))) break;
        if (j >= 2 && !(ok = wait(&s_free[j & 1], ((j >> 1) - 1) & 1, kDevTimeoutConvert))) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t kd = kd0 + static_cast<uint64_t>(ss) * (kTile >> 4);
          const uint32_t st = tmS(j);
#pragma unroll
          for (int ks = 0; ks < kD / 16; ++ks)
            umma_f16_ts(st, tmQ + static_cast<uint32_t>(ks * 8), kd + (ks >> 2) * ((kKeys * 128) >> 4) + (ks & 3) * 2, idesc_s,
                        ks > 0 ? 1u : 0u);
          umma_commit(&k_empty[ss]);
          umma_commit(&s_full[j & 1]);
        }
        __syncwarp();
        if (++ss == kStages) {
          ss = 0;
          sp ^= 1;
        }
        blocks.step(p, blk);
        if (j >= j0 + 2) pv(j - 2, false);
      }
      if (ok && j >= j0 + 2) pv(j - 2, false);
      if (ok) pv(j - 1, true);
      ++seg;
    }
  } else if (worker) {
    const int quad = warp & 3;
    const int ch = (threadIdx.x - kFirstWorker) >> 7;  // this warp's group: blocks in turn, half of the output columns
    const int r = quad * 32 + lane;                    // query row inside the tile == TMEM lane
    float* m_x = reinterpret_cast<float*>(smem + kOffXchg);  // [2][128] running maxima after a block
    float* l_x = m_x + 2 * kRows;                            // [2][128] the groups' sums, and their maxima
    uint64_t* m_bar = m_set + quad * 2;
    uint8_t* st = smem + kOffStage + (warp - kFirstWorker / 32) * 2048;
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    bool ok = true;
    int j = 0, seg = 0, wst = 0;
    uint32_t wph = 0;  // stage and parity of the next block's words
    for (int tile = share.tile0; tile <= share.tile1; ++tile) {
      const Segment s = share.segment(p, tile);
      const Blocks<kRows, kKeys> blocks(p, s);
      const int R = (tile - blocks.h * p.head_tiles) * kRows + r;
      const bool row_valid = R < p.rows;
      const RowOf row(p, min(R, p.rows - 1));
      const int b_row = row_valid ? row.b : -1;
      const int my_block = block_id(p, row.s);
      float m_mine = -INFINITY, l_run = 0.f;  // the maximum that this group's sum is relative to
      Block blk = blocks.find(p, s.first);
      const bool live = blk.unit >= 0;
      const int j0 = j;
      if (live) {
        // Q into TMEM, two dims per column: a warp its 32 rows' half (every MMA that
        // read the tile before is done: its o_last)
        // (rows past the last one repeat it: they are not stored)
        const long at = row.b * p.qs_b + (blocks.h * p.G + row.g) * p.qs_h + row.s * p.qs_s;
        uint4 v[4][4];
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const long from = __shfl_sync(0xffffffffu, at, it * 8 + (lane >> 2));
          const __nv_bfloat16* q = p.q + from + ch * 128 + (lane & 3) * 8;
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c][it] = *reinterpret_cast<const uint4*>(q + c * 32);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int it = 0; it < 4; ++it) *reinterpret_cast<uint4*>(shared_chunk(st, lane, it)) = v[c][it];
          __syncwarp();
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(own_chunk(st, lane, i));
            w[4 * i] = x.x;
            w[4 * i + 1] = x.y;
            w[4 * i + 2] = x.z;
            w[4 * i + 3] = x.w;
          }
          // (a value that is not finite times a masked key's zeros would be NaN: where the
          // row sees no key it counts as 0)
          uint32_t most = 0u;
#pragma unroll
          for (int i = 0; i < 16; ++i) most = __vmaxu2(most, w[i] & 0x7fff7fffu);
          if (max(most & 0xffffu, most >> 16) >= 0x7f80u && !sees_key(p, row.b)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = 0u;
          }
          __syncwarp();
          tmem_st16(tmQ + lane_base + ch * 64 + c * 16, w);
          __syncwarp();
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_ready);
      }
      if (tile == share.tile0 && p.early) pdl_wait();
      for (; blk.unit >= 0 && ok; blocks.step(p, blk), ++j) {
        const int ws = wst;
        const uint32_t wp = wph;
        if (++wst == kWordStages) {
          wst = 0;
          wph ^= 1;
        }
        if ((j & 1) != ch) continue;
        ok = wait_long(&w_full[ws], wp, p.status, kDevTimeoutTmaFull);
        if (ok) ok = wait_long(&s_full[ch], (j >> 1) & 1, p.status, kDevTimeoutMmaDone);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        // the block's keys: score scale (log2 units), value scale, additive mask and
        // block id
        const float* sc = sWords + ws * kWords;
        const float4* ks_s = reinterpret_cast<const float4*>(sc);
        const float4* vs_s = reinterpret_cast<const float4*>(sc + kKeys);
        const float4* kadd_s = reinterpret_cast<const float4*>(sc + 2 * kKeys);
        const int4* nb_s = reinterpret_cast<const int4*>(sc + 3 * kKeys);
        auto softmax = [&](auto of_stream) {
          constexpr bool kOwn = decltype(of_stream)::value;
          unsigned long long z[kKeys / 2];
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          uint32_t rr[kKeys / 16][16];
  #pragma unroll
          for (int c = 0; c < kKeys / 16; ++c) tmem_ld16(tmS(j) + lane_base + 16 * c, rr[c]);
          tmem_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[ch]);
  #pragma unroll
          for (int c = 0; c < kKeys / 4; ++c) {
            const float4 km = ks_s[c], ka = kadd_s[c];
            const uint32_t* s4 = &rr[c >> 2][4 * (c & 3)];
            z[2 * c] = fma_f32x2(pack_f32x2(__uint_as_float(s4[0]), __uint_as_float(s4[1])), pack_f32x2(km.x, km.y),
                                 pack_f32x2(ka.x, ka.y));
            z[2 * c + 1] = fma_f32x2(pack_f32x2(__uint_as_float(s4[2]), __uint_as_float(s4[3])), pack_f32x2(km.z, km.w),
                                     pack_f32x2(ka.z, ka.w));
          }
          if (kOwn) {
  #pragma unroll
            for (int c = 0; c < kKeys / 4; ++c) {
              const int4 nb = nb_s[c];
              z[2 * c] = pack_f32x2(nb.x > my_block ? -INFINITY : lo_f32(z[2 * c]),
                                    nb.y > my_block ? -INFINITY : hi_f32(z[2 * c]));
              z[2 * c + 1] = pack_f32x2(nb.z > my_block ? -INFINITY : lo_f32(z[2 * c + 1]),
                                        nb.w > my_block ? -INFINITY : hi_f32(z[2 * c + 1]));
            }
            // (on its own: as a second condition above it takes more registers)
            if (blk.stream != b_row) {
  #pragma unroll
              for (int c = 0; c < kKeys / 2; ++c) z[c] = pack_f32x2(-INFINITY, -INFINITY);
            }
          }
  #pragma unroll
          for (int c = 0; c < kKeys / 2; ++c) mx[c & 3] = fmaxf(fmaxf(mx[c & 3], lo_f32(z[c])), hi_f32(z[c]));
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) + sc[4 * kKeys];
          // the row's running maximum, from the other group's block before
          float m_prev = -INFINITY;
          if (j > j0) {
            ok = __all_sync(0xffffffffu, wait_long(&m_bar[ch ^ 1], ((j - 1) >> 1) & 1, p.status, kDevTimeoutMmaDone));
            if (!ok) return;
            m_prev = m_x[(ch ^ 1) * kRows + r];
          }
          const float m_new = fmaxf(m_prev, top);
          // (moved by more than 2^8 only: P stays below 2^15, and O is seldom rescaled)
          const bool need = m_prev != -INFINITY && m_new > m_prev + 8.f;
          const float m_use = need || m_prev == -INFINITY ? m_new : m_prev;
          m_x[ch * kRows + r] = m_use;
          __syncwarp();
          if (lane == 0) mbar_arrive(&m_bar[ch]);
          const float m_sub = m_use == -INFINITY ? 0.f : m_use;
          if (__any_sync(0xffffffffu, need)) {
            // O is final for the rescale once P V of the block before is done (that of the
            // two before it went before this block's S: the parity is clear)
            ok = __all_sync(0xffffffffu, wait_long(&v_empty[ch ^ 1], ((j - 1) >> 1) & 1, p.status, kDevTimeoutMmaDone));
            if (!ok) return;
            tc_fence_after();
            const float alpha = need ? exp2f(m_prev - m_use) : 1.f;
  #pragma unroll 1
            for (int c0 = 0; c0 < kD / 16; c0 += 2) {
              uint32_t oo[2][16];
  #pragma unroll
              for (int q = 0; q < 2; ++q) tmem_ld16(tmO + lane_base + (c0 + q) * 16, oo[q]);
              tmem_wait_ld();
  #pragma unroll
              for (int q = 0; q < 2; ++q) {
  #pragma unroll
                for (int e = 0; e < 16; ++e) oo[q][e] = __float_as_uint(__uint_as_float(oo[q][e]) * alpha);
                tmem_st16(tmO + lane_base + (c0 + q) * 16, oo[q]);
              }
            }
            // (the stores are asynchronous: they are done before P is announced, which
            // lets the issuing warp add to O)
            tmem_wait_st();
          }
          // P (times the value scales), where P of this group's block before was, once
          // its P V is done
          if (j >= 2) {
            ok = __all_sync(0xffffffffu, wait_long(&v_empty[ch], ((j >> 1) - 1) & 1, p.status, kDevTimeoutMmaDone));
            if (!ok) return;
          }
          const unsigned long long nm = pack_f32x2(-m_sub, -m_sub);
          unsigned long long sum[2] = {0ull, 0ull};
          uint8_t* pt = smem + kOffP + ch * kTileP;
#pragma unroll
          for (int c = 0; c < kKeys / 8; ++c) {  // 8 keys
            uint32_t pk[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const float4 vsc = vs_s[2 * c + (h >> 1)];
              const unsigned long long zz = z[4 * c + h], d = add_f32x2(zz, nm);
              const unsigned long long e = pack_f32x2(ex2_approx(lo_f32(d)), ex2_approx(hi_f32(d)));
              sum[h & 1] = add_f32x2(sum[h & 1], e);
              const unsigned long long w = mul_f32x2(e, (h & 1) ? pack_f32x2(vsc.z, vsc.w) : pack_f32x2(vsc.x, vsc.y));
              pk[h] = pack_f16x2(lo_f32(w), hi_f32(w));
              // a weight of 0 stays 0 whatever another stream's value scale is
              if (kOwn) {
                if (lo_f32(zz) == -INFINITY) pk[h] &= 0xffff0000u;
                if (hi_f32(zz) == -INFINITY) pk[h] &= 0x0000ffffu;
              }
            }
            *reinterpret_cast<uint4*>(pt + sw128_offset(r, c)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
          }
          fence_proxy_async_smem();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_ready[ch]);
          const unsigned long long both = add_f32x2(sum[0], sum[1]);
          // (2^-inf = 0: nothing seen before)
          l_run = fmaf(l_run, m_mine == m_use ? 1.f : ex2_approx(m_mine - m_use), lo_f32(both) + hi_f32(both));
          m_mine = m_use;
        };
        // (shared blocks, the most, without the masks by row)
        if (blk.stream >= 0)
          softmax(std::true_type{});
        else
          softmax(std::false_type{});
      }
      // ---- epilogue: every pair takes its barrier once, whatever happened ----
      if (live && ok) ok = __all_sync(0xffffffffu, wait_long(o_last, seg & 1, p.status, kDevTimeoutMmaDone));
      tc_fence_after();
      l_x[ch * kRows + r] = l_run;
      l_x[(2 + ch) * kRows + r] = m_mine;
      ok = pair_all(quad, ok);
      // both groups' sums relative to the maximum after the last block (the larger),
      // in a fixed order
      const float m0 = l_x[2 * kRows + r], m1 = l_x[3 * kRows + r], m_run = fmaxf(m0, m1);
      // (where scores were all NaN a maximum is -inf and its sum NaN)
      l_run = (m0 == m_run ? l_x[r] : l_x[r] * exp2f(m0 - m_run)) +
              (m1 == m_run ? l_x[kRows + r] : l_x[kRows + r] * exp2f(m1 - m_run));
      const bool part = p.cluster > 1 || !s.whole;
      const long slot = p.cluster > 1 ? blockIdx.x : 2 * blockIdx.x + (tile == share.tile0 ? 0 : 1);
      // A tile of several CTAs without a cluster: the last of them to get here joins the
      // parts, in their order whichever it is.  It is the last for sure where all others
      // have arrived, and then leaves no part of its own.
      const bool joins = part && p.join;
      int c0 = 0, c1 = 0;
      bool last = false;
      if (joins) {
        c0 = cta_of(p, tile * p.tile_units);
        c1 = cta_of(p, (tile + 1) * p.tile_units - 1);
        if (threadIdx.x == kFirstWorker) *last_x = ld_acquire(p.arrived + tile) == c1 - c0;
        workers_all(true);
        last = *last_x != 0;
      }
      const long at = row_valid ? out_at(p, blocks.h, row) : -1;
      float inv_l = l_run > 0.f || l_run != l_run ? 1.f / l_run : 0.f;
      if (part && !last) {
        if (ok) {
          if (ch == 0) p.part_ml[slot * kRows + r] = make_float2(m_run, l_run);
#pragma unroll 1
          for (int c = 4 * ch; c < 4 * ch + 4; ++c) {  // 32 columns
            uint32_t rr[2][16];
            load_o(live, tmO + lane_base + c * 32, rr);
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                *part_at(p, slot, c * 8 + q * 4 + e, r) =
                    make_float4(__uint_as_float(rr[q][4 * e]), __uint_as_float(rr[q][4 * e + 1]),
                                __uint_as_float(rr[q][4 * e + 2]), __uint_as_float(rr[q][4 * e + 3]));
          }
        }
        if (joins) {
          __threadfence();
          workers_all(true);
          if (threadIdx.x == kFirstWorker) *last_x = atomicAdd(p.arrived + tile, 1) == c1 - c0;
          workers_all(true);
          last = *last_x != 0;
        }
      }
      if (ok && (!part || last)) {
        // weights of the parts before and after this one, and of this one
        const int mine = static_cast<int>(blockIdx.x) - c0;
        const long first = 2l * c0 + (c0 != static_cast<int>(blockIdx.x) && cta_begin(p, c0) >= tile * p.tile_units ? 0 : 1);
        auto slot_of = [&](int q) { return q == 0 ? first : 2l * (c0 + q); };
        float M = m_run;
        if (last) {
          __threadfence();
          for (int q = 0; q <= c1 - c0; ++q)
            if (q != mine) M = fmaxf(M, __ldcg(&p.part_ml[slot_of(q) * kRows + r].x));
          float L = 0.f;
          for (int q = 0; q <= c1 - c0; ++q) {
            const float2 ml = q == mine ? make_float2(m_run, l_run) : __ldcg(p.part_ml + slot_of(q) * kRows + r);
            L = fmaf(ml.x == M ? 1.f : exp2f(ml.x - M), ml.y, L);
          }
          inv_l = L > 0.f || L != L ? 1.f / L : 0.f;
        }
#pragma unroll 1
        for (int c = 4 * ch; c < 4 * ch + 4; ++c) {  // 32 columns
          uint32_t rr[2][16];
          load_o(live, tmO + lane_base + c * 32, rr);
          if (last) {
            float acc[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) acc[e] = 0.f;
#pragma unroll 1
            for (int q = 0; q <= c1 - c0; ++q) {
              float4 x[8];
              float m = m_run;
              if (q == mine) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const uint32_t* o = &rr[e >> 2][4 * (e & 3)];
                  x[e] = make_float4(__uint_as_float(o[0]), __uint_as_float(o[1]), __uint_as_float(o[2]), __uint_as_float(o[3]));
                }
              } else {
                const long from = slot_of(q);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __ldcg(part_at(p, from, c * 8 + e, r));
                m = __ldcg(&p.part_ml[from * kRows + r].x);
              }
              const float w = m == M ? 1.f : exp2f(m - M);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                acc[4 * e] = fmaf(w, x[e].x, acc[4 * e]);
                acc[4 * e + 1] = fmaf(w, x[e].y, acc[4 * e + 1]);
                acc[4 * e + 2] = fmaf(w, x[e].z, acc[4 * e + 2]);
                acc[4 * e + 3] = fmaf(w, x[e].w, acc[4 * e + 3]);
              }
            }
#pragma unroll
            for (int e = 0; e < 32; ++e) rr[e >> 4][e & 15] = __float_as_uint(acc[e]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t* x = &rr[i >> 1][8 * (i & 1)];
            *reinterpret_cast<uint4*>(own_chunk(st, lane, i)) =
                make_uint4(pack_bf16x2(__uint_as_float(x[0]) * inv_l, __uint_as_float(x[1]) * inv_l),
                           pack_bf16x2(__uint_as_float(x[2]) * inv_l, __uint_as_float(x[3]) * inv_l),
                           pack_bf16x2(__uint_as_float(x[4]) * inv_l, __uint_as_float(x[5]) * inv_l),
                           pack_bf16x2(__uint_as_float(x[6]) * inv_l, __uint_as_float(x[7]) * inv_l));
          }
          __syncwarp();
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const long to = __shfl_sync(0xffffffffu, at, it * 8 + (lane >> 2));
            const uint4 x = *reinterpret_cast<const uint4*>(shared_chunk(st, lane, it));
            if (to >= 0) *reinterpret_cast<uint4*>(p.out + to + c * 32 + (lane & 3) * 8) = x;
          }
          __syncwarp();
        }
      }
      if (live) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_free);
        ++seg;
      }
      // all workers go on to the next tile or none does (its Q goes where this
      // tile's was)
      if (tile < share.tile1 && !(ok = workers_all(ok))) break;
    }
  }
  __syncwarp();
  if (p.cluster > 1) {
    // Every CTA of the cluster has left its part of the tile in its slot (in L2, which
    // takes them faster than the SMs' network takes stores into one another); each
    // joins its share of the columns of all rows.
    cluster_sync();
    const int n = p.cluster, rank = static_cast<int>(cluster_ctarank());
    const int h = share.tile0 / p.head_tiles, r = (threadIdx.x - kFirstWorker) & (kRows - 1);
    const int R = (share.tile0 - h * p.head_tiles) * kRows + r;
    if (worker && R < p.rows) {
      const long at = out_at(p, h, RowOf(p, R));
      const int slot0 = blockIdx.x - rank, groups = kD / 8 / n;
#pragma unroll 1
      for (int g = rank * groups + ((threadIdx.x - kFirstWorker) >> 7); g < (rank + 1) * groups; g += 2) {
        Joined<> j;
        j.add(p, n, r, g, [&](int i) { return static_cast<long>(slot0 + i); });
        *reinterpret_cast<uint4*>(p.out + at + g * 8) = j.result();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  // every issued load completes before the block leaves (an MMA issuer that
  // stopped early)
  if ((warp == 0 || warp == 2) && lane == 0) {
    const int stages = warp == 2 ? kStagesV : kStages;
    uint64_t* full = warp == 2 ? v_full : k_full;
    for (int i = max(issued - stages, 0); i < issued; ++i) {
      wait_long(&full[i % stages], (i / stages) & 1, p.status, kDevTimeoutTmaFull);
      if (warp == 0) wait_long(&w_full[i % kWordStages], (i / kWordStages) & 1, p.status, kDevTimeoutTmaFull);
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------- few rows ---
// Tiles of 16 rows on the warps' own matrix instructions (mma.sync): where a batch
// has few query rows, reading the keys and starting up bound the call, and this form
// has no copy of the keys, no barriers between roles and no TMEM to set up.  A warp
// takes 16 keys at a time straight from the ring into registers: a thread's 16-byte
// pieces are its operands, since the order of the dims in a dot product is free if Q
// has the same (K: a thread has 16 dims at a time of key lane / 4), and so is that of
// the output columns (V: 16 dims of 4 keys).  The warps' results are added in shared
// memory, those of a cluster's CTAs through DSMEM, each in order.
// Bound by latency: 16 keys of a warp take 3.3 us, loads, products and softmax in a row.
// 8 rows over 1000 keys 10 us (the other form 16), 256 rows 15 (17), 1024 rows 34 (17).
constexpr int kFewRows = 16;
constexpr int kFewKeys = 16;
constexpr int kFewWarps = 8;
constexpr int kFewMaxCluster = 8;
constexpr int kFewPitch = kD + 8;                                      // floats of a row of a warp's O
constexpr int kFewOffQ = 0;                                            // [16 k steps][32 lanes][4 words]
constexpr int kFewOffO = 16 * 32 * 16;                                 // [8 warps][16 rows][264]
constexpr int kFewOffMl = kFewOffO + kFewWarps * kFewRows * kFewPitch * 4;  // [8 warps][16] (m, l)
constexpr int kFewOffSum = kFewOffMl + kFewWarps * kFewRows * 8;       // the CTA's O [16][256]
constexpr int kFewOffSumMl = kFewOffSum + kFewRows * kD * 4;           // and (m, l) [16]
constexpr int kFewSmem = kFewOffSumMl + kFewRows * 8;
static_assert(kFewSmem <= 227 * 1024, "shared memory");

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// Bytes 0..3 of two keys as four (key a, key b) pairs of f16.
__device__ __forceinline__ void i8_pairs_to_f16(uint32_t a, uint32_t b, uint32_t (&out)[4]) {
  const uint32_t bias = 0x64806480u;
  const uint32_t p[2] = {__byte_perm(a ^ 0x80808080u, b ^ 0x80808080u, 0x5140), __byte_perm(a ^ 0x80808080u, b ^ 0x80808080u, 0x7362)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = __byte_perm(p[i >> 1], 0x64646464u, (i & 1) ? 0x4342 : 0x4140);
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&t), *reinterpret_cast<const __half2*>(&bias));
    out[i] = *reinterpret_cast<const uint32_t*>(&d);
  }
}

// A step's keys as they lie in memory: K of keys g and g + 8 (dims 16 (t + 4 c) ..),
// V and scales of keys 2t, 2t + 1, 2t + 8, 2t + 9 (dims 128 hf + 16 g ..); g = lane / 4,
// t = lane % 4.  Keys past the ring's last one repeat it: they are masked.
struct FewKeys {
  uint4 k[2][4];
  uint4 v[4][2];
  float ks[4], vs[4];
  uint32_t valid;  // bit n
};

__device__ __forceinline__ void add_scaled(float4& a, float f, const float4& x) {
  a.x = fmaf(f, x.x, a.x);
  a.y = fmaf(f, x.y, a.y);
  a.z = fmaf(f, x.z, a.z);
  a.w = fmaf(f, x.w, a.w);
}
__device__ __forceinline__ float at16(const float4 (&a)[4], int e) {  // e a constant where it is unrolled
  const float4& v = a[e >> 2];
  return (e & 3) == 0 ? v.x : (e & 3) == 1 ? v.y : (e & 3) == 2 ? v.z : v.w;
}
// The column of place e of a thread's 16 (see the end of the kernel).
__device__ __forceinline__ int few_column(int cg, int e) {
  const int i = e >> 2;
  return 128 * (i >> 1) + 16 * (4 * (cg & 1) + (e & 3)) + 8 * (i & 1) + (cg >> 1);
}
__device__ __forceinline__ void few_store(__nv_bfloat16* row, int cg, const float4 (&acc)[4], float l) {
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) row[few_column(cg, e)] = __float2bfloat16_rn(at16(acc, e) * inv);
}

// The 16 keys of a step into a warp's shared memory, bf16 K and f16 V (8 dims per
// lane); returns which keys have values beyond f16, whose rows are left 0 (the rows
// that see such a key become NaN by its value scale, the other streams' rows
// multiply it by 0).
__device__ __noinline__ uint32_t few_stage(const SharedAttnParams& p, const Block b, int h, int lane, unsigned short* kt,
                                           unsigned short* vt) {
  uint32_t beyond = 0;
  const long ring_at = b.stream * p.own.qs_b + h * p.own.qs_h + 8 * lane;
#pragma unroll 1
  for (int i = 0; i < kFewKeys; ++i) {
    const int key = b.j * kFewKeys + i;
    uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
    if (key < b.held) {
      const uint2 kq = *reinterpret_cast<const uint2*>(p.own.k + ring_at + key * p.own.qs_c);
      const uint2 vq = *reinterpret_cast<const uint2*>(p.own.v + ring_at + key * p.own.qs_c);
      i8_to_bf16(kq.x, k.x, k.y);
      i8_to_bf16(kq.y, k.z, k.w);
      i8_to_f16(vq.x, v.x, v.y);
      i8_to_f16(vq.y, v.z, v.w);
    } else if (key < b.total) {
      const long n = key - b.held;
      k = *reinterpret_cast<const uint4*>(p.k_new + b.stream * p.ks_b + h * p.ks_h + n * p.ks_s + 8 * lane);
      const uint4 x = *reinterpret_cast<const uint4*>(p.v_new + b.stream * p.vs_b + h * p.vs_h + n * p.vs_s + 8 * lane);
      const uint32_t in[4] = {x.x, x.y, x.z, x.w};
      uint32_t w[4];
      bool bad = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = pack_f16x2(__uint_as_float(in[e] << 16), __uint_as_float(in[e] & 0xffff0000u));
        bad |= (w[e] & 0x7c00u) == 0x7c00u || (w[e] & 0x7c000000u) == 0x7c000000u;
      }
      if (__any_sync(0xffffffffu, bad))
        beyond |= 1u << i;
      else
        v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    *reinterpret_cast<uint4*>(kt + i * kFewPitch + 8 * lane) = k;
    *reinterpret_cast<uint4*>(vt + i * kFewPitch + 8 * lane) = v;
  }
  __syncwarp();
  return beyond;
}

__global__ void __launch_bounds__(32 * kFewWarps, 1) shared_few_kernel(const __grid_constant__ SharedAttnParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  pdl_wait();
  // a CTA's share of a tile's units, and a warp's of that
  const int per_tile = p.cluster;  // CTAs per tile
  const int tile = blockIdx.x / per_tile, rank = blockIdx.x - tile * per_tile;
  const int workers = per_tile * kFewWarps, me = rank * kFewWarps + warp;
  Segment s;
  s.tile = tile;
  s.first = static_cast<int>(static_cast<long>(me) * p.tile_units / workers);
  s.last = static_cast<int>(static_cast<long>(me + 1) * p.tile_units / workers);
  const Blocks<kFewRows, kFewKeys> blocks(p, s);
  const int h = blocks.h, R0 = (tile - h * p.head_tiles) * kFewRows;
  // Q in the order of the A operands
  for (int i = threadIdx.x; i < 16 * 32; i += 32 * kFewWarps) {
    const int step = i >> 5, l = i & 31, dim = 16 * ((l & 3) + 4 * (step >> 2)) + 4 * (step & 3);
    uint2 x[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const RowOf w(p, min(R0 + (l >> 2) + 8 * k, p.rows - 1));  // (rows past the last one are not stored)
      x[k] = *reinterpret_cast<const uint2*>(p.q + w.b * p.qs_b + (h * p.G + w.g) * p.qs_h + w.s * p.qs_s + dim);
    }
    reinterpret_cast<uint4*>(smem + kFewOffQ)[i] = make_uint4(x[0].x, x[1].x, x[0].y, x[1].y);
  }
  __syncthreads();
  int stream[2], upto[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int R = R0 + g + 8 * k;
    const RowOf w(p, min(R, p.rows - 1));
    stream[k] = R < p.rows ? w.b : -1;
    upto[k] = block_id(p, w.s);
  }
  float o[2][16][4];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf)
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[hf][i][e] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  const uint4* qf = reinterpret_cast<const uint4*>(smem + kFewOffQ) + lane;
  unsigned short* kt = reinterpret_cast<unsigned short*>(smem + kFewOffO + warp * kFewRows * kFewPitch * 4);
  unsigned short* vt = kt + kFewKeys * kFewPitch;

  FewKeys raw;
  // where a block's ring rows begin for this head, and the last one that it may read
  auto load_k = [&](const Block& b) {
    const bool shared = b.stream < 0;
    const int most = b.held - 1 - b.j * kFewKeys;
    if (most < 0) return;  // new tokens only
    const long row0 = static_cast<long>(b.j) * kFewKeys;
    const long qc = shared ? p.shared.qs_c : p.own.qs_c, sc = shared ? p.shared.ss_c : p.own.ss_c;
    const uint8_t* k = shared ? p.shared.k + h * p.shared.qs_h : p.own.k + b.stream * p.own.qs_b + h * p.own.qs_h;
    k += row0 * qc + 16 * t;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const uint8_t* row = k + min(8 * n + g, most) * qc;
#pragma unroll
      for (int c = 0; c < 4; ++c) raw.k[n][c] = *reinterpret_cast<const uint4*>(row + 64 * c);
    }
    const long s0 = (shared ? h * p.shared.ss_h : b.stream * p.own.ss_b + h * p.own.ss_h) + row0 * sc;
    const float* ks = static_cast<const float*>(shared ? p.shared.k_scale : p.own.k_scale) + s0;
    const float* vs = static_cast<const float*>(shared ? p.shared.v_scale : p.own.v_scale) + s0;
    raw.valid = 15;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int i = min(2 * t + (n & 1) + 8 * (n >> 1), most);
      raw.ks[n] = ks[i * sc];
      raw.vs[n] = vs[i * sc];
    }
    if (shared && p.shared_valid) {
      unsigned char ok[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) ok[n] = p.shared_valid[row0 + min(2 * t + (n & 1) + 8 * (n >> 1), most)];
      raw.valid = (ok[0] ? 1 : 0) | (ok[1] ? 2 : 0) | (ok[2] ? 4 : 0) | (ok[3] ? 8 : 0);
    }
  };
  auto load_v = [&](const Block& b) {
    const bool shared = b.stream < 0;
    const int most = b.held - 1 - b.j * kFewKeys;
    if (most < 0) return;
    const long qc = shared ? p.shared.qs_c : p.own.qs_c;
    const uint8_t* v = shared ? p.shared.v + h * p.shared.qs_h : p.own.v + b.stream * p.own.qs_b + h * p.own.qs_h;
    v += static_cast<long>(b.j) * kFewKeys * qc + 16 * g;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const uint8_t* row = v + min(2 * t + (n & 1) + 8 * (n >> 1), most) * qc;
      raw.v[n][0] = *reinterpret_cast<const uint4*>(row);
      raw.v[n][1] = *reinterpret_cast<const uint4*>(row + 128);
    }
  };
  Block b = blocks.find(p, s.first);
  if (b.unit >= 0) {
    load_k(b);
    load_v(b);
  }
  while (b.unit >= 0) {
    Block ahead = b;
    blocks.step(p, ahead);
    const int key0 = b.j * kFewKeys;
    const bool has_new = b.total > b.held && key0 + kFewKeys > b.held;
    // score and value scales of the thread's four keys, whether there is such a key, and
    // the block id from which on it is seen
    float ks[4], vs[4];
    int nb[4];
    bool there[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int key = key0 + 2 * t + (n & 1) + 8 * (n >> 1);
      const bool seen = key < b.held && (raw.valid >> n & 1);
      ks[n] = seen ? raw.ks[n] * p.scale_log2 : 0.f;
      vs[n] = seen ? raw.vs[n] : 0.f;
      nb[n] = kRingKey;
      there[n] = seen;
    }
    // a step with new tokens goes through the warp's (still unused) part of shared
    // memory, bf16 K and f16 V
    if (has_new) {
      const uint32_t bad = few_stage(p, b, h, lane, kt, vt);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int i = 2 * t + (n & 1) + 8 * (n >> 1), key = key0 + i;
        if (key >= b.held && key < b.total) {
          ks[n] = p.scale_log2;
          vs[n] = (bad >> i & 1) ? __uint_as_float(0x7fffffffu) : 1.f;
          nb[n] = block_id(p, key - b.held);
          there[n] = true;
        }
      }
    }
    float c[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) c[n][e] = 0.f;
    if (!has_new) {
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
        const uint32_t q0[4] = {raw.k[0][cc].x, raw.k[0][cc].y, raw.k[0][cc].z, raw.k[0][cc].w};
        const uint32_t q1[4] = {raw.k[1][cc].x, raw.k[1][cc].y, raw.k[1][cc].z, raw.k[1][cc].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint4 qa = qf[(4 * cc + e) * 32];
          uint32_t lo, hi;
          i8_to_bf16(q0[e], lo, hi);
          mma_bf16(c[0], qa, lo, hi);
          i8_to_bf16(q1[e], lo, hi);
          mma_bf16(c[1], qa, lo, hi);
        }
      }
    } else {
#pragma unroll 1
      for (int e = 0; e < 16; ++e) {
        const uint4 qa = qf[e * 32];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint2 w = *reinterpret_cast<const uint2*>(kt + (8 * n + g) * kFewPitch + 16 * (t + 4 * (e >> 2)) + 4 * (e & 3));
          mma_bf16(c[n], qa, w.x, w.y);
        }
      }
    }
    if (ahead.unit >= 0) load_k(ahead);
    uint32_t top = max(max(lift_bits(vs[0]), lift_bits(vs[1])), max(lift_bits(vs[2]), lift_bits(vs[3])));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float lift = lift_of(top);
    // c[n]: row g keys 8 n + 2t, + 1, row g + 8 the same
    float z[2][4];  // [row][key]
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const bool ours = b.stream < 0 || b.stream == stream[k];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        z[k][n] = ours && there[n] && nb[n] <= upto[k] ? c[n >> 1][2 * k + (n & 1)] * ks[n] : -INFINITY;
        mx[k] = fmaxf(mx[k], z[k][n]);
      }
      mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], 1));
      mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], 2));
    }
    // (moved by more than 2^8 only, as in the other form)
    float alpha[2];
    bool need = false;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float m_new = fmaxf(m_run[k], mx[k] + lift);
      const bool up = m_run[k] != -INFINITY && m_new > m_run[k] + 8.f;
      const float m_use = up || m_run[k] == -INFINITY ? m_new : m_run[k];
      alpha[k] = up ? ex2_approx(m_run[k] - m_use) : 1.f;
      need |= up;
      m_run[k] = m_use;
    }
    if (__any_sync(0xffffffffu, need)) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[hf][i][e] *= alpha[e >> 1];
      l_run[0] *= alpha[0];
      l_run[1] *= alpha[1];
    }
    float pr[2][4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float m_sub = m_run[k] == -INFINITY ? 0.f : m_run[k];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float e = ex2_approx(z[k][n] - m_sub);
        l_run[k] += e;
        pr[k][n] = z[k][n] == -INFINITY ? 0.f : e * vs[n];  // (a weight of 0 whatever the value scale is)
      }
    }
    const uint4 pa = make_uint4(pack_f16x2(pr[0][0], pr[0][1]), pack_f16x2(pr[1][0], pr[1][1]), pack_f16x2(pr[0][2], pr[0][3]),
                                pack_f16x2(pr[1][2], pr[1][3]));
    if (!has_new) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t b0[4], b1[4];
          auto word = [&](const uint4& x) { return w == 0 ? x.x : w == 1 ? x.y : w == 2 ? x.z : x.w; };
          i8_pairs_to_f16(word(raw.v[0][hf]), word(raw.v[1][hf]), b0);
          i8_pairs_to_f16(word(raw.v[2][hf]), word(raw.v[3][hf]), b1);
#pragma unroll
          for (int i = 0; i < 4; ++i) mma_f16(o[hf][4 * w + i], pa, b0[i], b1[i]);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; i += 2) {  // two columns at a time: their pairs of two keys each
        const unsigned short* src = vt + 2 * t * kFewPitch + 128 * (i >> 4) + 16 * g + (i & 15);
        const uint32_t x0 = *reinterpret_cast<const uint32_t*>(src), x1 = *reinterpret_cast<const uint32_t*>(src + kFewPitch);
        const uint32_t y0 = *reinterpret_cast<const uint32_t*>(src + 8 * kFewPitch), y1 = *reinterpret_cast<const uint32_t*>(src + 9 * kFewPitch);
        mma_f16(o[i >> 4][i & 15], pa, __byte_perm(x0, x1, 0x5410), __byte_perm(y0, y1, 0x5410));
        mma_f16(o[i >> 4][(i & 15) + 1], pa, __byte_perm(x0, x1, 0x7632), __byte_perm(y0, y1, 0x7632));
      }
      __syncwarp();  // (the next step may be staged over it)
    }
    b = ahead;
    if (b.unit >= 0) load_v(b);
  }
  // a row's sum over its 4 lanes; O and (m, l) of the warp
  float* O = reinterpret_cast<float*>(smem + kFewOffO) + warp * kFewRows * kFewPitch;
  float2* ml = reinterpret_cast<float2*>(smem + kFewOffMl);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    l_run[k] += __shfl_xor_sync(0xffffffffu, l_run[k], 1);
    l_run[k] += __shfl_xor_sync(0xffffffffu, l_run[k], 2);
    if (t == 0) ml[warp * kFewRows + g + 8 * k] = make_float2(m_run[k], l_run[k]);
  }
  // column 128 hf + 16 n + i at place (16 hf + i) 8 + n
#pragma unroll
  for (int hf = 0; hf < 2; ++hf)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      *reinterpret_cast<float2*>(O + g * kFewPitch + (hf * 16 + i) * 8 + 2 * t) = make_float2(o[hf][i][0], o[hf][i][1]);
      *reinterpret_cast<float2*>(O + (g + 8) * kFewPitch + (hf * 16 + i) * 8 + 2 * t) = make_float2(o[hf][i][2], o[hf][i][3]);
    }
  __syncthreads();
  // the warps' parts of 16 places of a row, 4 (c + 16 i) .. + 3: columns
  // 128 (i / 2) + 16 n + 8 (i % 2) + c / 2, n = 4 (c % 2) .. + 3
  const int r = threadIdx.x >> 4, cg = threadIdx.x & 15, R = R0 + r;
  const float4* parts = reinterpret_cast<const float4*>(smem + kFewOffO + (r * kFewPitch + cg * 4) * 4);
  float M = -INFINITY, L = 0.f;
  float4 acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  float2 of[kFewWarps];
#pragma unroll
  for (int w = 0; w < kFewWarps; ++w) {
    of[w] = ml[w * kFewRows + r];
    M = fmaxf(M, of[w].x);
  }
#pragma unroll
  for (int w = 0; w < kFewWarps; ++w) {
    const float f = of[w].x == M ? 1.f : ex2_approx(of[w].x - M);
    L = fmaf(f, of[w].y, L);
#pragma unroll
    for (int i = 0; i < 4; ++i) add_scaled(acc[i], f, parts[w * kFewRows * kFewPitch / 4 + 16 * i]);
  }
  if (p.ctas != 0) {  // parts that the joining kernel adds
    if (R < p.rows) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int col = few_column(cg, e);
        reinterpret_cast<float*>(part_at(p, blockIdx.x, col >> 2, r))[col & 3] = at16(acc, e);
      }
      if (cg == 0) p.part_ml[static_cast<long>(blockIdx.x) * p.tile_rows + r] = make_float2(M, L);
    }
    return;
  }
  if (per_tile == 1) {
    if (R < p.rows) few_store(p.out + out_at(p, h, RowOf(p, R)), cg, acc, L);
    return;
  }
  float4* sum = reinterpret_cast<float4*>(smem + kFewOffSum);
  float2* sum_ml = reinterpret_cast<float2*>(smem + kFewOffSumMl);
#pragma unroll
  for (int i = 0; i < 4; ++i) sum[threadIdx.x * 4 + i] = acc[i];
  if (cg == 0) sum_ml[r] = make_float2(M, L);
  __syncwarp();
  cluster_sync();
  // this CTA's share of the tile's 16 x 16 such pieces
  const int share = 256 / per_tile;
  if (threadIdx.x < share) {
    const int i = rank * share + threadIdx.x, row = i >> 4;
    const uint32_t at = smem_u32(sum) + static_cast<uint32_t>(i) * 64u, at_ml = smem_u32(sum_ml) + static_cast<uint32_t>(row) * 8u;
    float top = -INFINITY, l = 0.f;
    float2 from[kFewMaxCluster];
#pragma unroll
    for (int q = 0; q < kFewMaxCluster; ++q) {
      from[q] = make_float2(-INFINITY, 0.f);
      if (q < per_tile)
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(from[q].x), "=f"(from[q].y) : "r"(mapa_shared(at_ml, q)) : "memory");
      top = fmaxf(top, from[q].x);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int q = 0; q < per_tile; ++q) {
      float2 x = from[0];
#pragma unroll
      for (int k = 1; k < kFewMaxCluster; ++k)
        if (k == q) x = from[k];
      const float f = x.x == top ? 1.f : ex2_approx(x.x - top);
      l = fmaf(f, x.y, l);
#pragma unroll
      for (int k = 0; k < 4; ++k) add_scaled(acc[k], f, ld_dsmem_f4(mapa_shared(at + 16u * k, q)));
    }
    if (R0 + row < p.rows) few_store(p.out + out_at(p, h, RowOf(p, R0 + row)), i & 15, acc, l);
  }
  __syncwarp();
  cluster_sync();  // no CTA leaves while another reads its sums
}

// Joins the parts of the tiles that several CTAs had units of: a thread 8 columns of
// every SLICES-th part of a row (lanes along the rows), then the slices in order.
template <int ROWS, int SLICES>
__global__ void __launch_bounds__(ROWS * SLICES < 256 ? 256 : ROWS * SLICES) shared_combine_kernel(const __grid_constant__ SharedAttnParams p) {
  constexpr int kSlices = SLICES, kThreads = ROWS * SLICES < 256 ? 256 : ROWS * SLICES;
  constexpr int kGroups = kThreads / (ROWS * SLICES);  // of 8 columns, in a CTA
  __shared__ float part[10][SLICES > 1 ? kThreads : 1];
  pdl_launch_dependents();
  const int tile = blockIdx.x / (kD / 8 / kGroups), slice = threadIdx.x / ROWS % SLICES, r = threadIdx.x % ROWS;
  const int g = blockIdx.x % (kD / 8 / kGroups) * kGroups + threadIdx.x / (ROWS * SLICES);
  int n, first, rest;  // parts of the tile; slot of the first, and of the following ones
  int step = 1;
  if (ROWS == kFewRows) {
    n = p.cluster;
    first = tile * n;
    rest = first;
  } else {
    const int t0 = tile * p.tile_units;
    const int c0 = cta_of(p, t0), c1 = cta_of(p, t0 + p.tile_units - 1);
    if (c0 == c1) return;  // the tile was one CTA's: stored there
    // a CTA's first tile is in its slot 0, its last one in slot 1: of a tile's CTAs
    // only the first can have begun with another
    n = c1 - c0 + 1;
    first = 2 * c0 + (cta_begin(p, c0) >= t0 ? 0 : 1);
    rest = 2 * c0;
    step = 2;
  }
  const int h = tile / p.head_tiles, R = (tile - h * p.head_tiles) * ROWS + r;
  pdl_wait();
  Joined<kThreads == 1024 ? 4 : 8> j;  // (64 registers a thread)
  if (R < p.rows) {
    const int mine = (n - slice + kSlices - 1) / kSlices;
    j.add(p, mine, r, g, [&](int i) {
      const int q = slice + i * kSlices;
      return static_cast<long>(q == 0 ? first : rest + step * q);
    });
  }
  if (SLICES == 1) {
    if (R < p.rows) *reinterpret_cast<uint4*>(p.out + out_at(p, h, RowOf(p, R)) + g * 8) = j.result();
    return;
  }
  part[8][threadIdx.x] = j.M;
  part[9][threadIdx.x] = j.L;
#pragma unroll
  for (int e = 0; e < 8; ++e) part[e][threadIdx.x] = j.acc[e];
  __syncthreads();
  if (slice > 0 || R >= p.rows) return;
  float M = -INFINITY, L = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < kSlices; ++q) M = fmaxf(M, part[8][q * ROWS + r]);
#pragma unroll 4
  for (int q = 0; q < kSlices; ++q) {
    const float m = part[8][q * ROWS + r], w = m == M ? 1.f : exp2f(m - M);
    L = fmaf(w, part[9][q * ROWS + r], L);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, part[e][q * ROWS + r], acc[e]);
  }
  const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
  *reinterpret_cast<uint4*>(p.out + out_at(p, h, RowOf(p, R)) + g * 8) =
      make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                 pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
}

// ------------------------------------------------------------ host side ---
bool al(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Sizes of a call, how it is cut up and where its parts lie in the workspace.
struct Plan {
  SharedAttnParams p;
  bool few;     // the form for few rows
  long blocks;  // of the dense copy of the keys
  bool joined;  // some tile is several CTAs', without a cluster
  size_t kd, vd, words, part_o, part_ml, arrived, total;
};

// Whole tiles, clusters, or runs of units: what ends soonest by this model, in us, fitted
// to 13 batches at every way.  The keys' copy and the launches cost kCopy and kCopyBlock
// per block of keys, a CTA's start and end on a tile kFix, a unit kUnit.  A cluster's
// exchange is shorter the more CTAs share it.  Where a tile has at most kJoinMost parts the
// last CTA joins them (kJoin), else a kernel of its own (kCombine and kCombineRow per row):
// measured 62 and 70 us for 64 streams of 50 tokens over 818 slots (3 parts), 77 and 73 for
// 16 of 51 over 6344 (4 parts).  Returns the time.
double deal(Plan* out, int nsm) {
  SharedAttnParams& p = out->p;
  constexpr double kCopy = 4.9, kCopyBlock = 0.0138, kFix = 5.5, kUnit = 1.22, kJoin = 13.0, kCombine = 6.0, kCombineRow = 0.0007;
  const long units = static_cast<long>(p.tiles) * p.tile_units;
  double best = 0;
  for (int c = 1; c <= kMaxCluster; c *= 2) {
    if (c > 1 && c > p.tile_units) break;
    const long slots = c == 1 ? nsm : static_cast<long>(max_active_clusters(reinterpret_cast<const void*>(attention_shared_kernel), kThreads, kSmemBytes, c)) * c;
    if (slots <= 0) continue;
    const long waves = (static_cast<long>(p.tiles) * c + slots - 1) / slots;
    const double cost = waves * (kFix + (p.tile_units + c - 1) / c * kUnit + (c > 1 ? 1.5 + 11.0 / c : 0.0));
    if (p.cluster && cost >= best) continue;
    best = cost;
    p.cluster = c;
  }
  const int ctas = static_cast<int>(std::min<long>(units, nsm));
  p.run = static_cast<int>(units / ctas);
  p.longer = static_cast<int>(units % ctas);
  const bool join = p.tile_units <= (kJoinMost - 1) * p.run;
  const double ends = 1.0 + static_cast<double>(p.tiles) / ctas;  // of tiles, per CTA
  const double cost = static_cast<double>((units + ctas - 1) / ctas) * kUnit + ends * kFix +
                      (join ? kJoin : kCombine + kCombineRow * p.tiles * kRows);
  out->joined = cost < best;
  if (out->joined) p.cluster = 0;
  p.join = out->joined && join;
  p.ctas = p.cluster ? p.tiles * p.cluster : ctas;
  return std::min(cost, best) + kCopy + kCopyBlock * out->blocks;
}

// The form for few rows: CTAs per tile (a cluster, or as many as there are SMs for, whose
// parts a second kernel joins).  16 keys of a warp cost kStep us, a CTA's start and end
// kFix.  Returns the time, fitted like the other form's to 8 to 1024 rows of 64 to 16000
// keys.
double deal_few(Plan* out, int nsm) {
  SharedAttnParams& p = out->p;
  constexpr double kFix = 4.0, kStep = 3.27, kJoin = 2.2, kJoinRow = 0.013;
  auto time = [&](int ctas, long slots) {  // per tile, of all tiles at once
    const long waves = (static_cast<long>(p.tiles) * ctas + slots - 1) / slots;
    return waves * (kFix + (p.tile_units + ctas * kFewWarps - 1) / (ctas * kFewWarps) * kStep);
  };
  p.cluster = 1;
  double best = time(1, nsm);
  for (int c = 2; c <= kFewMaxCluster && c <= p.tile_units; c *= 2) {
    const long slots = static_cast<long>(max_active_clusters(reinterpret_cast<const void*>(shared_few_kernel), 32 * kFewWarps, kFewSmem, c)) * c;
    if (slots <= 0) break;
    const double cost = time(c, slots) + 1.8 + 0.1 * c;
    if (cost < best) {
      best = cost;
      p.cluster = c;
    }
  }
  const int most = std::min(std::max(1, nsm / p.tiles), (p.tile_units + kFewWarps - 1) / kFewWarps);
  const double cost = time(most, nsm) + kJoin + kJoinRow * p.tiles * kFewRows;
  if (most > 1 && cost < best) {
    best = cost;
    out->joined = true;
    p.cluster = most;
  }
  p.ctas = out->joined ? p.tiles * p.cluster : 0;
  return best;
}

// One form's plan and its time (few: tiles of 16 rows on the warps' matrix instructions).
int plan_form(const rfx_attn_shared_desc& d, bool few, int nsm, Plan* out, double* time) {
  SharedAttnParams& p = out->p;
  *out = Plan{};
  p.B = d.B;
  p.Hq = d.num_q_heads;
  p.Hkv = d.num_kv_heads;
  p.G = d.num_q_heads / d.num_kv_heads;
  p.S = d.S;
  p.n_shared = d.n_shared;
  p.own_max = d.own_max;
  p.n_new = d.k_new ? d.S : 0;
  const long rows = static_cast<long>(d.B) * p.G * d.S;
  const long per = static_cast<long>(p.G) * d.S;
  out->few = few;
  const int tile_rows = few ? kFewRows : kRows, keys = few ? kFewKeys : kKeys;
  // streams that a tile of rows can touch
  const long touch = per >= tile_rows ? (per % tile_rows ? 2 : 1) : tile_rows % per ? tile_rows / per + 2 : tile_rows / per;
  const long shared_blocks = (static_cast<long>(d.n_shared) + keys - 1) / keys;
  const long own_blocks = (static_cast<long>(d.own_max) + p.n_new + keys - 1) / keys;
  const long units = std::max(shared_blocks + std::min<long>(touch, d.B) * own_blocks, 1l);  // (no keys: one empty unit)
  const long head_tiles = (rows + tile_rows - 1) / tile_rows;
  constexpr long kMost = 1l << 30;
  if (rows > kMost || p.Hkv > kMost / head_tiles || units > kMost / (p.Hkv * head_tiles))
    return set_error(RFX_E_INVAL, "rfx_attention_shared: too many query rows or keys");
  p.rows = static_cast<int>(rows);
  p.tile_rows = tile_rows;
  p.head_tiles = static_cast<int>(head_tiles);
  p.tiles = p.Hkv * p.head_tiles;
  p.shared_blocks = static_cast<int>(shared_blocks);
  p.own_blocks = static_cast<int>(own_blocks);
  p.tile_units = static_cast<int>(units);
  out->blocks = few ? 0 : p.Hkv * (shared_blocks + d.B * own_blocks);
  if (out->blocks > 0x7fffffffl / kKeys) return set_error(RFX_E_INVAL, "rfx_attention_shared: too many keys");
  *time = few ? deal_few(out, nsm) : deal(out, nsm);
  return RFX_OK;
}

int plan_shared(const rfx_attn_shared_desc& d, Plan* out) {
  SharedAttnParams& p = out->p;
  int nsm = 148;
  rfx_num_sms(&nsm);
  double time = 0;
  int rc = plan_form(d, false, nsm, out, &time);
  if (rc) return rc;
  if (d.quant_mode == RFX_QUANT_I8_SYM && p.rows <= kFewMost) {
    Plan few;
    double few_time = 0;
    rc = plan_form(d, true, nsm, &few, &few_time);
    if (rc) return rc;
    if (few_time < time) *out = few;
  }
  const int tile_rows = p.tile_rows;
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = (off + bytes + 1023) & ~size_t(1023);
    return o;
  };
  out->kd = take(static_cast<size_t>(out->blocks) * kTile);
  out->vd = take(static_cast<size_t>(out->blocks) * kTile);
  out->words = take(static_cast<size_t>(out->blocks) * kWords * 4);
  const size_t slots = out->few ? p.ctas : out->joined ? 2 * static_cast<size_t>(p.ctas) : p.cluster > 1 ? p.ctas : 0;
  out->part_o = take(slots * tile_rows * kD * 4);
  out->part_ml = take(slots * tile_rows * 8);
  out->arrived = take(p.join ? static_cast<size_t>(p.tiles) * 4 : 0);
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

// The addresses between which places lie: most pairs are told apart by them.
struct Reach {
  __int128 lo, hi;
  explicit Reach(const Places& a) {
    lo = static_cast<__int128>(reinterpret_cast<uintptr_t>(a.p));
    hi = lo + static_cast<__int128>(a.width) * a.elem;
    for (int i = 0; i < 3; ++i) {
      const __int128 far = a.n[i] > 1 ? static_cast<__int128>(a.n[i] - 1) * a.step[i] * a.elem : 0;
      (far < 0 ? lo : hi) += far;
    }
  }
  bool meets(const Reach& b) const { return lo < b.hi && b.lo < hi; }
};

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
  if (plan->total > 0 && (!d.workspace || d.workspace_bytes < plan->total || !al(d.workspace, 1024)))
    return set_error(RFX_E_INVAL, "rfx_attention_shared: needs a 1024-byte aligned workspace of %zu bytes", plan->total);
  const Places ws{plan->total > 0 ? d.workspace : nullptr, 1, static_cast<long>(plan->total), {1, 1, 1}, {}};
  if (places_shared(o, ws)) return set_error(RFX_E_INVAL, "rfx_attention_shared: out lies in the workspace");
  const Reach out_reach(o), ws_reach(ws);
  for (const Places& in : inputs) {
    if (!in.p || in.width == 0) continue;
    const Reach r(in);
    if (r.meets(out_reach) && places_shared(o, in))
      return set_error(RFX_E_INVAL, "rfx_attention_shared: out shares memory with an input");
    if (r.meets(ws_reach) && places_shared(ws, in))
      return set_error(RFX_E_INVAL, "rfx_attention_shared: the workspace shares memory with an input");
  }
  return RFX_OK;
}

}  // namespace

int attention_shared_launches(const rfx_attn_shared_desc& d) {
  Plan plan;
  if (d.B == 0 || d.S == 0 || plan_shared(d, &plan)) return 0;
  return (plan.blocks > 0 ? 1 : 0) + 1 + (plan.joined && !plan.p.join ? 1 : 0);
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
  if (!plan.few && (rc = ensure_smem_attr(fn, kSmemBytes))) return rc;
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
  p.arrived = reinterpret_cast<int*>(ws + plan.arrived);
  p.early = plan.blocks > 0;
  p.status = device_status_ptr();
  CUtensorMap k{}, v{};
  if (plan.blocks > 0) {
    const uint64_t keys = static_cast<uint64_t>(plan.blocks) * kKeys;
    rc = make_tmap_2d(&k, p.kd, 2, kD, keys, kD * 2, 64, kKeys, true);
    if (rc) return rc;
    rc = make_tmap_2d(&v, p.vd, 2, kD, keys, kD * 2, 64, kKeys, true);
    if (rc) return rc;
    rc = launch_kernel(reinterpret_cast<const void*>(shared_dense_kernel),
                       dim3(static_cast<unsigned>(plan.blocks * (kKeys / 16))), dim3(256), 0, stream, pdl, 1, p);
    if (rc) return rc;
  }
  if (plan.few) {
    const void* few = reinterpret_cast<const void*>(shared_few_kernel);
    rc = ensure_smem_attr(few, kFewSmem);
    if (rc) return rc;
    rc = launch_kernel(few, dim3(p.tiles * p.cluster), dim3(32 * kFewWarps), kFewSmem, stream, pdl, plan.joined ? 1 : p.cluster, p);
    if (rc || !plan.joined) return rc;
    return launch_kernel(reinterpret_cast<const void*>(shared_combine_kernel<kFewRows, 16>), dim3(p.tiles * (kD / 8)), dim3(256), 0,
                         stream, pdl, 1, p);
  }
  rc = launch_kernel(fn, dim3(p.ctas), dim3(kThreads), kSmemBytes, stream, pdl,
                     std::max(p.cluster, 1), k, v, p);
  if (rc || !plan.joined || p.join) return rc;
  // a few parts per tile are added one after another, many by eight threads
  if (p.ctas > 8 * p.tiles)
    return launch_kernel(reinterpret_cast<const void*>(shared_combine_kernel<kRows, 8>), dim3(p.tiles * (kD / 8)), dim3(8 * kRows), 0,
                         stream, pdl, 1, p);
  return launch_kernel(reinterpret_cast<const void*>(shared_combine_kernel<kRows, 1>), dim3(p.tiles * (kD / 16)), dim3(2 * kRows), 0,
                       stream, pdl, 1, p);
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
