// Linear layers in 4-bit floating point: y = act(x_row[t] * w_row[o] * (x · wᵀ) + bias[o])
// with x and w of e2m1 values under a scale per block (rows as rfx_quant_fp4
// makes them).
//
// The tensor cores multiply the values with their block scales and sum in fp32
// (tcgen05.mma kind::mxf4 / kind::mxf4nvf4, 64 values of K per instruction); the
// scales go from global memory by TMA to shared memory and by tcgen05.cp to TMEM,
// as whole tiles of 128 rows x 4 blocks.  The epilogue applies the row scales,
// bias and activation in fp32 and rounds once.
//
// Two forms: CTA-pair tiles of 256 tokens (tokens on the MMA's M side), and tiles
// of 128 weight rows (the weights on the M side) for up to 128 tokens.  Operands
// are K-major rows of 128 bytes (256 values) per K step, staged by TMA with
// 128-byte swizzle; what lies past T, O or K is filled with zeros by the copy or
// not copied, and not stored.  MMAs whose 64 values all lie past K are left out,
// so no scale tile past a row's last one is used.
#include "quant_i8.cuh"
#include "rfx_internal.h"
#include "tile_epilogue.cuh"

#include <algorithm>
#include <cmath>

namespace rfx {
namespace {

constexpr int kTileM = 128;
constexpr int kStepB = 128;            // bytes of K per stage
constexpr int kStepK = 2 * kStepB;     // values of K per stage
constexpr int kMmaK = 64;              // values of K per MMA
constexpr int kSmemMax = 227 * 1024;
constexpr int kMaxRows = 1 << 30;      // of x and of w
constexpr int kMaxK = 65536;
constexpr int kScaleTile = 512;        // bytes: 128 rows x 4 blocks

// Scale tiles of 128 rows per K step, and MMAs that share one.
template <bool MX>
struct Fmt {
  static constexpr int kTiles = MX ? 2 : 4;
  static constexpr int kMmas = MX ? 2 : 1;
  static constexpr int kBytes = kTiles * kScaleTile;  // of 128 rows per K step
};

struct Fp4Params {
  int T;
  int F;            // output columns: O, or O / 2 with GeGLU
  int k_steps;      // of 256 values
  int k_mmas;       // of 64 values
  int k_tiles;      // scale tiles along K
  int up_tiles;     // GeGLU: row tiles of the gate part's scales
  int splits;       // parts of K: pairs, or CTAs, per cluster
  int m_tiles;      // 256-token tiles
  int n_tile;       // weight rows per tile (side: tokens),
  int n_tail;       // of the tiles from column cols_a on
  int cols_a, units;
  int stages;
  const float* x_row;  // NV
  const float* w_row;
  const float* bias;
  void* y;
  long ldy;
  int* status;
};

// ------------------------------------------------------- CTA-pair tiles ---
// A pair of CTAs computes 256 tokens x N weight rows with cta_group::2 MMAs: each
// CTA stages its 128 tokens and half of the weight rows per K step, its tokens'
// scales and the scales of all N weight rows (an MMA reads those from either
// CTA's own TMEM).  With GeGLU half of a tile's weight rows are gate rows and half
// up rows, and a thread of the epilogue finds both halves of its outputs in its own
// TMEM lane.  256 weight rows are one MMA's N, the gate rows from the even CTA and the
// up rows from the odd one, each a whole tile of scales; 128 are two MMAs, since their
// scales lie in halves of two tiles.
//
// TMEM: one accumulator of up to 256 columns, or two of up to 128 that alternate,
// and as many sets of scales as the ring has stages: a stage that has been filled
// again was free, and so is its set.  The 16 epilogue warps take all of their columns
// into registers and free the accumulator at once, so that the epilogue runs under
// the next tile's MMAs also where there is one accumulator.
//
// What bounds it: 256 columns' four MMAs of a K step take 670 clocks and come every 740,
// narrower ones every 600, which is what the issuing and the copying thread spend on a
// step; between tiles of one accumulator 1600 ns pass, and 4.5 to 6 us of a call are
// outside its products (set-up, first copies, last epilogue).  768 x 32768 x 2048 GeGLU 33 us,
// 3.1 PFLOP/s; 3200 x 1024 x 4096 12.3 us, 2.2 PFLOP/s; 4096 x 4096 x 4096 35 us, 3.9 PFLOP/s (MX 31, 4.4).
//
// splits == 1: persistent, the pair walks the tiles.  splits > 1: a cluster of
// `splits` pairs computes one tile, each pair a part of K; at the end each CTA
// pushes the fp32 sums of the columns that another split owns into that CTA's
// (now idle) operand ring through DSMEM, and the owner adds them in split order.
constexpr int kEpiWarps = 16;
constexpr int kPairThreads = 64 + 32 * kEpiWarps;
constexpr int kAcc1 = 128;             // TMEM columns: the second accumulator,
constexpr int kSets = 256;             // the sets of scales,
constexpr int kSetCols = 48;           // each tokens' (16) and weight rows' (32)
constexpr int kPairMaxStages = (512 - kSets) / kSetCols;
constexpr int kPairSmem = kSmemMax;
constexpr int kPairRing = (kPairSmem - 1024 - 256 - kEpiWarps * 2048 - 2 * 2 * 256 * 4) & ~1023;
constexpr int kPairOffVec = kPairRing;                      // [2][w_row | bias][256]
constexpr int kPairOffOut = kPairOffVec + 2 * 2 * 256 * 4;  // output staging, 2 KB per epilogue warp
constexpr int kPairOffBars = kPairOffOut + kEpiWarps * 32 * 64;
constexpr int kMaxSplits = 4;                               // clusters of at most 8 CTAs
static_assert(kPairOffBars + 256 + 1024 <= kPairSmem, "pair tiles fit in shared memory");
static_assert((kPairMaxStages * 2 + 4) * 8 + 4 <= 256, "barriers fit");

using f32x2 = unsigned long long;
__device__ __forceinline__ bool epi_all(bool ok) {  // (also a barrier of the epilogue's warps)
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(ok ? 1u : 0u), "n"(32 * kEpiWarps)
      : "memory");
  return all != 0;
}

// GELU (as in gelu_ex2) and SiLU of two values.
template <int ACT>
__device__ __forceinline__ f32x2 activate2(f32x2 v) {
  if (ACT == kActNone) return v;
  f32x2 e;
  if (ACT == kActSilu) {
    e = mul_f32x2(v, pack_f32x2(-1.4426950409f, -1.4426950409f));
  } else {
    constexpr float kA = -2.3022081986f, kB = kA * 0.044715f;  // -2 sqrt(2/pi) log2(e)
    e = mul_f32x2(v, fma_f32x2(mul_f32x2(v, v), pack_f32x2(kB, kB), pack_f32x2(kA, kA)));
  }
  const f32x2 d = add_f32x2(pack_f32x2(ex2_approx(lo_f32(e)), ex2_approx(hi_f32(e))), pack_f32x2(1.f, 1.f));
  return mul_f32x2(v, pack_f32x2(rcp_approx(lo_f32(d)), rcp_approx(hi_f32(d))));
}

// A row scale as two factors, scale = a * b, that a product sum is multiplied with before
// and after the other row's scale: a sum of 0 or of 2^-20 to 2^39 (those of e2m1 and e4m3
// numbers) times a is in range, and what leaves fp32 after the second product stays
// outside with b.  b is 1 for scales between 2^-80 and 2^80.
struct ScalePair {
  float a, b;
  __device__ __forceinline__ explicit ScalePair(float s) {
    const float m = fabsf(s);
    b = m > 0x1p80f ? s * 0x1p-80f : m < 0x1p-80f && m > 0.f ? s * 0x1p80f : 1.f;
    a = m > 0x1p80f ? 0x1p80f : m < 0x1p-80f && m > 0.f ? 0x1p-80f : s;
  }
};

// 16 outputs of one token: row scales (NV) and bias from shared memory, packed as
// they are stored.  `up`: the up half with GeGLU.  FAR: some lane's b is not 1.
template <int ACT, bool MX, bool FAR, typename Tout>
__device__ __forceinline__ void finish16(const uint32_t (&acc)[16], const uint32_t (&up)[16], const ScalePair& sx,
                                         const float* ws, const float* bs, bool bias, int half, uint32_t* out) {
  const f32x2 sa = pack_f32x2(sx.a, sx.a), sb = pack_f32x2(sx.b, sx.b);
  auto scaled = [&](const uint32_t (&a)[16], int g, int at) {  // values g, g + 1 of 4 at a time
    f32x2 v = pack_f32x2(__uint_as_float(a[g]), __uint_as_float(a[g + 1]));
    if (!MX) v = mul_f32x2(mul_f32x2(v, sa), *reinterpret_cast<const f32x2*>(ws + at + g));
    if (bias) {
      const f32x2 b = *reinterpret_cast<const f32x2*>(bs + at + g);
      return FAR ? fma_f32x2(v, sb, b) : add_f32x2(v, b);
    }
    return FAR ? mul_f32x2(v, sb) : v;
  };
#pragma unroll
  for (int g = 0; g < 16; g += 2) {
    f32x2 v = scaled(acc, g, 0);
    if (ACT == kActGeglu)
      v = mul_f32x2(activate2<kActGelu>(v), scaled(up, g, half));
    else
      v = activate2<ACT>(v);
    if (sizeof(Tout) == 2) {
      out[g >> 1] = pack_bf16x2(lo_f32(v), hi_f32(v));
    } else {
      out[g] = __float_as_uint(lo_f32(v));
      out[g + 1] = __float_as_uint(hi_f32(v));
    }
  }
}

template <int ACT, bool MX, typename Tout>
__global__ void __launch_bounds__(kPairThreads, 1)
    linear_fp4_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                           const __grid_constant__ CUtensorMap tmW2, const __grid_constant__ CUtensorMap tmXS,
                           const __grid_constant__ CUtensorMap tmWS, const __grid_constant__ CUtensorMap tmY,
                           const Fp4Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr bool kGeglu = ACT == kActGeglu;
  using F = Fmt<MX>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* vec = reinterpret_cast<float*>(smem + kPairOffVec);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kPairOffBars);
  uint64_t* empty = full + kPairMaxStages;
  uint64_t* acc_full = empty + kPairMaxStages;  // [2]
  uint64_t* acc_free = acc_full + 2;            // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_free + 2);
  const uint32_t crank = cluster_ctarank();
  const uint32_t rank = crank & 1u;  // in the pair
  const bool leader = rank == 0;
  const int split = static_cast<int>(crank >> 1);
  // Units, m_tiles to a column of tiles: first tiles of N = n_tile, then, from
  // column cols_a on, of N = n_tail, so that the last round of tiles is a narrow
  // one.  A walker keeps its place (tile row, column) and steps without dividing.
  const int ustep = gridDim.x / (2 * p.splits), unit0 = blockIdx.x / (2 * p.splits);
  struct Tile {
    int m, o0, N;
    bool tail;
  };
  struct Walk {
    int un, n, m;
  };
  const int step_n = ustep / p.m_tiles, step_m = ustep - step_n * p.m_tiles;
  const int first_n = unit0 / p.m_tiles;
  const Walk first{unit0, first_n, unit0 - first_n * p.m_tiles};
  auto next = [&](Walk& k) {
    k.un += ustep;
    k.n += step_n;
    k.m += step_m;
    if (k.m >= p.m_tiles) {
      k.m -= p.m_tiles;
      ++k.n;
    }
  };
  auto tile_of = [&](const Walk& k) {
    const int w = kGeglu ? p.n_tile / 2 : p.n_tile, w2 = kGeglu ? p.n_tail / 2 : p.n_tail;
    Tile u;
    u.m = k.m;
    u.tail = k.n >= p.cols_a;
    u.N = u.tail ? p.n_tail : p.n_tile;
    u.o0 = u.tail ? p.cols_a * w + (k.n - p.cols_a) * w2 : k.n * w;
    return u;
  };
  // row tiles of the weights' scales that a tile takes: the gate's and the up's,
  // or those that its rows (from a multiple of 64 on) lie in
  auto w_scale_tiles = [&](const Tile& u) { return kGeglu || (u.o0 & 127) + u.N > 128 ? 2 : 1; };
  const int stages = p.stages;
  const int off_xs = (kTileM + p.n_tile / 2) * kStepB;  // scales: tokens', then weight rows'
  const int stage = off_xs + 3 * F::kBytes;
  const int k0 = static_cast<int>(static_cast<long>(split) * p.k_steps / p.splits);
  const int nk = static_cast<int>(static_cast<long>(split + 1) * p.k_steps / p.splits) - k0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_free[i], 2 * kEpiWarps);  // both CTAs' epilogue warps, on the even CTA's barrier
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmXS);
    tma_prefetch_desc(&tmWS);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // every CTA's barriers are initialised before a remote arrival
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();

  const bool tma_y = (p.ldy * sizeof(Tout)) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15u) == 0;
  constexpr int kPiece = 64 / static_cast<int>(sizeof(Tout));  // output columns that a warp stores at a time
  constexpr int kPieces = 4 * (kGeglu ? 32 : 64) / (4 * kPiece);  // of a warp, at most: every fourth
  const bool one = p.n_tile > kAcc1;                             // one accumulator
  uint8_t* out_st = smem + kPairOffOut + (warp - 2) * 32 * 64;
  bool failed = false;
  int issued = 0;
  if (warp == 0) {
    // as in the MMA warp, the whole warp walks the steps and one lane waits and issues
    const bool lead = elect_one();
    const int leader_lane = __ffs(__ballot_sync(0xffffffffu, lead)) - 1;
    bool ok = true;
    int s = 0;
    uint32_t phase = 0;
    const uint32_t full0 = mapa_shared(smem_u32(full), crank & ~1u);
    for (Walk k = first; k.un < p.units && ok; next(k)) {
      const Tile tile = tile_of(k);
      const int t0 = tile.m * 2 * kTileM + static_cast<int>(rank) * kTileM;
      const CUtensorMap* tw = tile.tail ? &tmW2 : &tmW;
      const int quarter = tile.N / 4;
      const bool halves = kGeglu && tile.N < 256;
      const int wrow = kGeglu && !halves ? tile.o0 + static_cast<int>(rank) * p.F
                                         : tile.o0 + static_cast<int>(rank) * (kGeglu ? quarter : tile.N / 2);
      const int wst = w_scale_tiles(tile);
      // both CTAs' copies count on the even CTA's barrier; a half without
      // tokens copies none (what its rows multiply is not stored)
      const bool has_x = t0 < p.T;
      const int x_halves = has_x && t0 + kTileM < p.T ? 2 : 1;  // (the even CTA's view: it has tokens)
      const uint32_t bytes = static_cast<uint32_t>(x_halves * (kTileM * kStepB + F::kBytes) + tile.N * kStepB +
                                                   2 * wst * F::kBytes);
      const int xs0 = (t0 / kTileM) * p.k_tiles;
      const int ws0 = (tile.o0 / 128) * p.k_tiles, ws1 = ws0 + (kGeglu ? p.up_tiles : 1) * p.k_tiles;
      for (int i = 0; i < nk; i += 2) {
        const bool two = i + 1 < nk;
        const int s1 = s + 1 == stages ? 0 : s + 1;
        const uint32_t phase1 = s1 ? phase : phase ^ 1;
        int done = 0;
        if (lead) {
          auto copy = [&](int sg, int step) {
            uint8_t* st = smem + sg * stage;
            const uint32_t bar = full0 + 8u * sg;
            const int kb = (k0 + step) * kStepB, kt = (k0 + step) * F::kTiles;
            if (leader) mbar_arrive_expect_tx(&full[sg], bytes);
            if (has_x) {
              tma_load_2d_pair(st, &tmX, bar, kb, t0);
              tma_load_2d_pair(st + off_xs, &tmXS, bar, 0, xs0 + kt);
            }
            tma_load_2d_pair(st + kTileM * kStepB, tw, bar, kb, wrow);
            if (halves) tma_load_2d_pair(st + (kTileM + quarter) * kStepB, tw, bar, kb, p.F + wrow);
            tma_load_2d_pair(st + off_xs + F::kBytes, &tmWS, bar, 0, ws0 + kt);
            if (wst == 2) tma_load_2d_pair(st + off_xs + 2 * F::kBytes, &tmWS, bar, 0, ws1 + kt);
          };
          if (issued < stages || mbar_wait(&empty[s], phase ^ 1, p.status, kDevTimeoutStageEmpty)) {
            copy(s, i);
            done = 1;
            if (two && (issued + 1 < stages || mbar_wait(&empty[s1], phase1 ^ 1, p.status, kDevTimeoutStageEmpty))) {
              copy(s1, i + 1);
              done = 2;
            }
          }
        }
        done = __shfl_sync(0xffffffffu, done, leader_lane);
        issued += done;
        if (!(ok = done == (two ? 2 : 1))) break;
        if (two && s1 + 1 < stages) {
          s = s1 + 1;
          phase = phase1;
        } else if (two) {
          s = 0;
          phase = phase1 ^ 1;
        } else {
          s = s1;
          phase = phase1;
        }
      }
    }
  } else if (warp == 1) {
    if (leader) {
      // the whole warp walks the steps and one elected lane issues: the loop's
      // values stay uniform, where a loop inside `if (lane == 0)` spends more
      // clocks on each instruction's operands than the MMA takes
      const uint64_t a0 = make_sdesc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t b0 = make_sdesc_sw128(smem_u32(smem + kTileM * kStepB), 16, 1024);
      const uint64_t s0 = make_sdesc_rows16(smem_u32(smem + off_xs));
      bool ok = true;
      int s = 0, tl = 0;
      uint32_t phase = 0;
      const uint16_t both = static_cast<uint16_t>(3u << crank);
      const bool lead = elect_one();
      for (Walk k = first; k.un < p.units && ok; next(k), ++tl) {
        const int buf = one ? 0 : tl & 1, turn = one ? tl : tl >> 1;
        const Tile tile = tile_of(k);
        const int wst = w_scale_tiles(tile);
        const uint32_t shift = static_cast<uint32_t>(tile.o0 & 127) / 32;  // columns of the first row's scales
        const bool halves = kGeglu && tile.N < 256;
        const int nb = halves ? tile.N / 2 : tile.N;
        const uint32_t n_field = static_cast<uint32_t>(nb >> 3) << 17;
        if (turn > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(&acc_free[buf], (turn - 1) & 1, p.status, kDevTimeoutMmaDone))))
          break;
        tc_fence_after();
        const uint32_t acc = tmem + buf * kAcc1;
        // two K steps at a time: what this warp spends around them (waits, votes, the
        // loop) is otherwise longer than a step's MMAs
        for (int i = 0; i < nk; i += 2) {
          const bool two = i + 1 < nk;
          const int s1 = s + 1 == stages ? 0 : s + 1;
          const uint32_t phase1 = s1 ? phase : phase ^ 1;
          bool fine = true;
          if (lead) {
            auto scales = [&](int st, int mmas) {
              const uint32_t xs = tmem + kSets + st * kSetCols, ws = xs + 16;
              const uint64_t sc0 = s0 + static_cast<uint64_t>((st * stage) >> 4);
#pragma unroll
              for (int c = 0; c < F::kTiles; ++c) {
                if (c * F::kMmas < mmas) {
                  const uint64_t sc = sc0 + c * (kScaleTile >> 4);
                  tmem_copy_scales<true>(xs + c * 4, sc);
                  tmem_copy_scales<true>(ws + c * 8, sc + (F::kBytes >> 4));
                  if (wst == 2) tmem_copy_scales<true>(ws + c * 8 + 4, sc + 2 * (F::kBytes >> 4));
                }
              }
            };
            auto multiply = [&](int st, int mmas, bool first_step, bool last_step) {
              const uint32_t xs = tmem + kSets + st * kSetCols, ws = xs + 16 + shift;
              const uint64_t off = static_cast<uint64_t>((st * stage) >> 4), ad = a0 + off, bd = b0 + off;
#pragma unroll
              for (int kk = 0; kk < kStepK / kMmaK; ++kk) {
                if (kk < mmas) {
                  const int c = kk / F::kMmas;
                  const uint32_t idesc = make_idesc_fp4(2 * kTileM, 0, MX, 2 * (kk % F::kMmas)) | n_field;
                  const uint32_t add = (!first_step || kk > 0) ? 1u : 0u;
                  umma_fp4_ss<MX, true>(acc, ad + kk * 2, bd + kk * 2, idesc, xs + c * 4, ws + c * 8, add);
                  if (halves)
                    umma_fp4_ss<MX, true>(acc + nb, ad + kk * 2, bd + kk * 2 + ((nb / 2 * kStepB) >> 4), idesc, xs + c * 4,
                                          ws + c * 8 + 4, add);
                }
              }
              umma_commit_pair_mask(&empty[st], both);
              if (last_step) umma_commit_pair_mask(&acc_full[buf], both);
            };
            const int left = p.k_mmas - (k0 + i) * (kStepK / kMmaK);
            fine = mbar_wait(&full[s], phase, p.status, kDevTimeoutTmaFull);
            if (fine) {
              scales(s, left);
              multiply(s, left, i == 0, i == nk - 1);
              if (two) {
                fine = mbar_wait(&full[s1], phase1, p.status, kDevTimeoutTmaFull);
                if (fine) {
                  scales(s1, left - kStepK / kMmaK);
                  multiply(s1, left - kStepK / kMmaK, false, i + 1 == nk - 1);
                }
              }
            }
          }
          if (!(ok = __all_sync(0xffffffffu, fine))) break;
          if (two && s1 + 1 < stages) {
            s = s1 + 1;
            phase = phase1;
          } else if (two) {
            s = 0;
            phase = phase1 ^ 1;
          } else {
            s = s1;
            phase = phase1;
          }
        }
      }
    }
  } else {
    const int et = threadIdx.x - 64;
    const int quad = warp & 3;
    const int hw = (warp - 2) >> 2;  // which of the four warps of this TMEM quadrant
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t free_bar = mapa_shared(smem_u32(&acc_free[0]), crank & ~1u);
    const bool bias = p.bias != nullptr;
    int tl = 0;
    // a tile's scales and bias come asynchronously while the tile before it is
    // finished (a short K's products are there at once: the loads would be
    // waited for at every tile's start)
    float sx_next = 0.f;
    auto request = [&](const Tile& tile, int b) {
      if (et < tile.N) {
        const int nh = tile.N / 2;
        const int c = kGeglu ? (et < nh ? et : et - nh) : et;
        const bool in = tile.o0 + c < p.F;
        const int o = tile.o0 + c + (kGeglu && et >= nh ? p.F : 0);
        float* ws = vec + b * 512 + et;
        if (!MX && in)
          cp_async4(ws, p.w_row + o);
        else
          *ws = 1.f;
        if (in && bias)
          cp_async4(ws + 256, p.bias + o);
        else
          ws[256] = 0.f;
      }
      cp_async_commit();
      const int t = tile.m * 2 * kTileM + static_cast<int>(rank) * kTileM + quad * 32 + lane;
      sx_next = !MX && t < p.T ? p.x_row[t] : 1.f;
    };
    if (first.un < p.units) request(tile_of(first), 0);
    for (Walk k = first; k.un < p.units; next(k), ++tl) {
      const int buf = one ? 0 : tl & 1, vbuf = tl & 1;
      const Tile tile = tile_of(k);
      const int N = tile.N, nh = N / 2, oc = kGeglu ? nh : N;  // oc output columns
      const int tw = tile.m * 2 * kTileM + static_cast<int>(rank) * kTileM + quad * 32;  // the warp's first token
      const int o0 = tile.o0;
      const float* ws = vec + vbuf * 512;
      const float* bs = ws + 256;
      const ScalePair sx(sx_next);
      const bool full_ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], (one ? tl : tl >> 1) & 1, p.status, kDevTimeoutMmaDone));
      tc_fence_after();
      const uint32_t acc = tmem + buf * kAcc1 + lane_base;
      // pieces hw, hw + 4, ... of the tile's columns, all of them at once: then the
      // accumulator is free
      uint32_t r[kPieces][kPiece / 16][16], u[kGeglu ? kPieces : 1][kPiece / 16][16];
      if (full_ok && p.splits == 1) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int c = (hw + 4 * i) * kPiece;
          if (c < oc) {
#pragma unroll
            for (int q = 0; q < kPiece / 16; ++q) {
              tmem_ld16(acc + c + 16 * q, r[i][q]);
              if (kGeglu) tmem_ld16(acc + nh + c + 16 * q, u[i][q]);
            }
          }
        }
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(free_bar + 8u * buf);
      }
      cp_async_wait_all();
      // (the scales are there; every epilogue warp agrees before anyone leaves the loop)
      if (!epi_all(full_ok)) {
        failed = true;
        break;
      }
      if (p.splits > 1) break;  // one tile per cluster: summed below
      Walk ahead = k;
      next(ahead);
      if (ahead.un < p.units) request(tile_of(ahead), vbuf ^ 1);
      const bool far = !MX && __any_sync(0xffffffffu, sx.b != 1.f);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int c = (hw + 4 * i) * kPiece;
        if (c < oc) {
          uint32_t w[16];
          // (a branch per piece: a product more per output takes 768 x 32768 x 2048 GeGLU from
          // 33.2 to 33.9 us)
          if (far) {
#pragma unroll
            for (int q = 0; q < kPiece / 16; ++q)
              finish16<ACT, MX, !MX, Tout>(r[i][q], u[kGeglu ? i : 0][q], sx, ws + c + 16 * q, bs + c + 16 * q, bias, nh, w + q * 8);
          } else {
#pragma unroll
            for (int q = 0; q < kPiece / 16; ++q)
              finish16<ACT, MX, false, Tout>(r[i][q], u[kGeglu ? i : 0][q], sx, ws + c + 16 * q, bs + c + 16 * q, bias, nh, w + q * 8);
          }
          store_part<Tout>(p, &tmY, out_st, w, tw, o0 + c, p.T - tw, min(kPiece, p.F - o0 - c), tma_y, lane);
        }
      }
    }
  }
  if (p.splits > 1) {
    // Every CTA's products are summed and its ring is idle: each pushes the
    // groups of 128 output bytes that another split owns (group j: split
    // j % splits) to the CTA of the same token half there, as
    // [group][source][gate | up][4 columns][token].  The owner adds them to its
    // own in split order.
    const Tile tile = tile_of(first);
    const int nh = tile.N / 2, oc = kGeglu ? nh : tile.N;
    constexpr int kGroup = 2 * kPiece;
    const int quad = warp & 3, hw = (warp - 2) >> 2;
    const int rowt = quad * 32 + lane;
    const uint32_t acc = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    constexpr int kParts = kGeglu ? 2 : 1;
    constexpr int kSlot = kGroup / 4 * kTileM * 16;  // bytes of one part of one group
    const int groups = (oc + kGroup - 1) / kGroup, others = p.splits - 1;
    __syncwarp();
    cluster_sync();
    if (warp >= 2 && !failed) {
      const uint32_t base = smem_u32(smem) + static_cast<uint32_t>(rowt) * 16u;
#pragma unroll 1
      for (int j = hw; j < groups * (kGroup / 16); j += 4) {  // 16-column chunks
        const int grp = j / (kGroup / 16), q = j % (kGroup / 16);
        const int owner = grp % p.splits;
        if (owner == split || j * 16 >= oc) continue;
        const int src = split < owner ? split : split - 1;
        const uint32_t dst = mapa_shared(base, static_cast<uint32_t>(owner) * 2u + rank);
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          uint32_t r[16];
          tmem_ld16(acc + part * nh + j * 16, r);
          tmem_wait_ld();
          const int slot = ((grp / p.splits) * others + src) * kParts + part;
#pragma unroll
          for (int g = 0; g < 4; ++g)
            st_dsmem_f4(dst + static_cast<uint32_t>(slot * kSlot + (q * 4 + g) * kTileM * 16), __uint_as_float(r[4 * g]),
                        __uint_as_float(r[4 * g + 1]), __uint_as_float(r[4 * g + 2]), __uint_as_float(r[4 * g + 3]));
        }
      }
    }
    __syncwarp();
    cluster_sync();
    if (warp >= 2 && !failed) {
      const int tw = tile.m * 2 * kTileM + static_cast<int>(rank) * kTileM + quad * 32;
      const int o0 = tile.o0;
      const ScalePair sx(!MX && tw + lane < p.T ? p.x_row[tw + lane] : 1.f);
#pragma unroll 1
      for (int lg = hw >> 1; lg * p.splits + split < groups; lg += 2) {
        const int g0 = (lg * p.splits + split) * kGroup;
        uint32_t w[16];
#pragma unroll
        for (int qq = 0; qq < kPiece / 16; ++qq) {
          const int q = (hw & 1) * (kPiece / 16) + qq;
          const int c = g0 + 16 * q;
          if (c < oc) {
            uint32_t r[kParts][16], sum[kParts][16];
#pragma unroll
            for (int part = 0; part < kParts; ++part) tmem_ld16(acc + part * nh + c, r[part]);
            tmem_wait_ld();
#pragma unroll
            for (int part = 0; part < kParts; ++part)
#pragma unroll
              for (int e = 0; e < 16; ++e) sum[part][e] = 0u;
#pragma unroll 1
            for (int from = 0; from < p.splits; ++from) {
              const int src = from < split ? from : from - 1;
#pragma unroll
              for (int part = 0; part < kParts; ++part) {
                const float4* recv =
                    reinterpret_cast<const float4*>(smem + ((lg * others + max(src, 0)) * kParts + part) * kSlot) +
                    q * 4 * kTileM + rowt;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                  float4 v = make_float4(__uint_as_float(r[part][4 * g]), __uint_as_float(r[part][4 * g + 1]),
                                         __uint_as_float(r[part][4 * g + 2]), __uint_as_float(r[part][4 * g + 3]));
                  if (from != split) v = recv[g * kTileM];
                  const float add[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    sum[part][4 * g + e] = __float_as_uint(__uint_as_float(sum[part][4 * g + e]) + add[e]);
                }
              }
            }
            finish16<ACT, MX, !MX, Tout>(sum[0], sum[kParts - 1], sx, vec + c, vec + 256 + c, p.bias != nullptr, nh, w + qq * 8);
          }
        }
        const int g = g0 + (hw & 1) * kPiece;
        store_part<Tout>(p, &tmY, out_st, w, tw, o0 + g, p.T - tw, min(min(kPiece, oc - g), p.F - o0 - g), tma_y, lane);
      }
    }
    __syncwarp();
  }
  if (warp >= 2 && lane == 0) bulk_wait_all();  // the output's stores are complete
  tc_fence_before();
  // a producer that stopped early waits (bounded) for the pair's copies in flight
  if (warp == 0 && lane == 0 && leader)
    for (int i = (issued > stages ? issued - stages : 0); i < issued; ++i)
      mbar_wait(&full[i % stages], (i / stages) & 1, p.status, kDevTimeoutTmaFull);
  __syncwarp();
  cluster_sync();  // neither CTA leaves while the pair's copies or MMAs may touch it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ------------------------------------------- weights on the MMA's M side ---
// Few tokens leave most of a 256-token tile's TMEM lanes empty.  Here 128 weight
// rows are the MMA's M and the tokens, a multiple of 16 up to kSideTokens, its N:
// every lane of the accumulator holds outputs, lanes lie along a row of y, and the
// tokens are copied once per tile of weight rows at their own size.  With GeGLU a
// tile is 128 gate rows and their 128 up rows in two accumulators, so a thread
// has both of its outputs' halves.
//
// One CTA per tile and part of K; a cluster of `splits` CTAs computes a tile.
// A CTA gives the sums of 4 tokens x 128 rows (group g: CTA g % splits) to the
// CTA that finishes them, as [source][group][gate | up][row][4], through DSMEM into
// memory of their own (not the ring: no CTA has to wait for another's products
// before it sends), and they are added in the order of the sources.
//
// Bound by latency: 1 x 2560 x 2048 3.5 us, 50 x 8192 x 1024 GeGLU 5.3, 128 x 32768 x 2048
// GeGLU 10.5 (3.6 TB/s of weights).  Above 128 tokens pair tiles are taken.
constexpr int kSideTokens = 128;
constexpr int kSideThreads = 320;
constexpr int kSideMaxSplits = 8;
constexpr int kSideMaxStages = 16;

int side_stage(int N, bool geglu, bool mx) {
  return ((geglu ? 2 : 1) * kTileM + N) * kStepB + (geglu ? 3 : 2) * (mx ? Fmt<true>::kBytes : Fmt<false>::kBytes);
}
int side_smem(int N, int splits, bool geglu, bool mx, int stages) {
  const int groups = (N / 4 + splits - 1) / splits;
  return stages * side_stage(N, geglu, mx) + (splits > 1 ? splits * groups * (geglu ? 2 : 1) * kTileM * 16 : 0) + N * 4 +
         (2 * stages + 2) * 8 + 1024;
}
// TMEM columns: the accumulators and two sets of scales.
__host__ __device__ constexpr int side_set(bool geglu, bool mx) { return (geglu ? 3 : 2) * (mx ? 2 : 4) * 4; }
__host__ __device__ constexpr int side_cols(int N, bool geglu, bool mx) {
  const int need = (geglu ? 2 : 1) * N + 2 * side_set(geglu, mx);
  return need <= 64 ? 64 : need <= 128 ? 128 : need <= 256 ? 256 : 512;
}

template <int ACT, bool MX, typename Tout>
__global__ void __launch_bounds__(kSideThreads, 3)
    linear_fp4_side_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                           const __grid_constant__ CUtensorMap tmXS, const __grid_constant__ CUtensorMap tmWS,
                           const Fp4Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr bool kGeglu = ACT == kActGeglu;
  constexpr int kParts = kGeglu ? 2 : 1;
  using F = Fmt<MX>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int N = p.n_tile, splits = p.splits, stages = p.stages;
  const int off_x = kParts * kTileM * kStepB;
  const int off_ws = off_x + N * kStepB;            // scales: weight rows', then tokens'
  const int off_xs = off_ws + kParts * F::kBytes;
  const int stage = off_xs + F::kBytes;
  const int shift = 31 - __clz(splits);             // splits is a power of 2
  const int mine = (N / 4 + splits - 1) >> shift;   // groups of 4 tokens per CTA, at most
  const int ring = stages * stage;
  uint8_t* red = smem + ring;
  float* sx = reinterpret_cast<float*>(red + (splits > 1 ? splits * mine * kParts * kTileM * 16 : 0));
  uint64_t* full = reinterpret_cast<uint64_t*>(sx + N);
  uint64_t* empty = full + stages;
  uint64_t* acc_full = empty + stages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  const int rank = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int o0 = (static_cast<int>(blockIdx.x) >> shift) * kTileM;
  const int k0 = static_cast<int>(static_cast<long>(rank) * p.k_steps / splits);
  const int nk = static_cast<int>(static_cast<long>(rank + 1) * p.k_steps / splits) - k0;
  const uint32_t cols = side_cols(N, kGeglu, MX);

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(acc_full, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmXS);
    tma_prefetch_desc(&tmWS);
  }
  // Waited for before the first store into a peer.  Before TMEM is asked for, and TMEM is
  // given back before the peers' sums are waited for: CTAs that wait for TMEM which
  // others on their SM hold would otherwise wait in a circle.
  if (splits > 1) cluster_arrive_release();
  if (warp == 1) {
    tmem_alloc(tmem_slot, cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();

  const int et = threadIdx.x - 64, quad = warp & 3, hw = (warp - 2) >> 2;
  const uint32_t acc = tmem + (static_cast<uint32_t>(quad * 32) << 16);
  const int rowt = quad * 32 + lane;
  ScalePair ws(1.f), wu(1.f);  // of the row that this thread finishes
  float bs = 0.f, bu = 0.f;
  int o = 0;
  bool summed = false;
  int issued = 0;
  if (warp == 0) {
    bool ok = true;
    int s = 0;
    uint32_t phase = 0;
    const int ws0 = (o0 / 128) * p.k_tiles, ws1 = ws0 + p.up_tiles * p.k_tiles;
    for (int i = 0; i < nk; ++i) {
      if (issued >= stages && !(ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], phase ^ 1, p.status, kDevTimeoutStageEmpty))))
        break;
      if (elect_one()) {
        uint8_t* st = smem + s * stage;
        const int kb = (k0 + i) * kStepB, kt = (k0 + i) * F::kTiles;
        mbar_arrive_expect_tx(&full[s], static_cast<uint32_t>((kParts * kTileM + p.T) * kStepB + (kParts + 1) * F::kBytes));
        tma_load_2d(st, &tmW, &full[s], kb, o0);
        if (kGeglu) tma_load_2d(st + kTileM * kStepB, &tmW, &full[s], kb, p.F + o0);
        tma_load_2d(st + off_ws, &tmWS, &full[s], 0, ws0 + kt);
        if (kGeglu) tma_load_2d(st + off_ws + F::kBytes, &tmWS, &full[s], 0, ws1 + kt);
        tma_load_2d(st + off_x, &tmX, &full[s], kb, 0);
        tma_load_2d(st + off_xs, &tmXS, &full[s], 0, kt);
      }
      __syncwarp();
      ++issued;
      if (++s == stages) {
        s = 0;
        phase ^= 1;
      }
    }
  } else if (warp == 1) {
    const uint64_t a0 = make_sdesc_sw128(smem_u32(smem), 16, 1024);
    const uint64_t b0 = make_sdesc_sw128(smem_u32(smem + off_x), 16, 1024);
    const uint64_t s0 = make_sdesc_rows16(smem_u32(smem + off_ws));
    int s = 0, s2 = 0;  // s2: the stage of two steps before
    uint32_t phase = 0, phase2 = 0;
    for (int i = 0; i < nk; ++i) {
      // The MMAs of two steps before have read this set of scales.  (A ring of one or two
      // stages has been filled again, so they have; waiting for their phase there could
      // miss it, since the next one of that parity may be over.)
      if (i >= 2 && stages > 2) {
        if (!__all_sync(0xffffffffu, mbar_wait(&empty[s2], phase2, p.status, kDevTimeoutMmaDone))) break;
        if (++s2 == stages) {
          s2 = 0;
          phase2 ^= 1;
        }
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&full[s], phase, p.status, kDevTimeoutTmaFull))) break;
      tc_fence_after();
      const uint64_t off = static_cast<uint64_t>((s * stage) >> 4);
      const uint32_t wsc = tmem + kParts * N + (i & 1) * side_set(kGeglu, MX), xsc = wsc + kParts * F::kTiles * 4;
      const int mmas = min(kStepK / kMmaK, p.k_mmas - (k0 + i) * (kStepK / kMmaK));
      if (elect_one()) {
#pragma unroll
        for (int c = 0; c < F::kTiles; ++c) {
          if (c * F::kMmas < mmas) {
            const uint64_t sc = s0 + off + c * (kScaleTile >> 4);
#pragma unroll
            for (int part = 0; part < kParts; ++part)
              tmem_copy_scales<false>(wsc + (part * F::kTiles + c) * 4, sc + part * (F::kBytes >> 4));
            tmem_copy_scales<false>(xsc + c * 4, sc + kParts * (F::kBytes >> 4));
          }
        }
#pragma unroll
        for (int kk = 0; kk < kStepK / kMmaK; ++kk) {
          if (kk < mmas) {
            const int c = kk / F::kMmas;
            const uint32_t idesc = make_idesc_fp4(kTileM, 0, MX, 2 * (kk % F::kMmas)) | (static_cast<uint32_t>(N >> 3) << 17);
#pragma unroll
            for (int part = 0; part < kParts; ++part)
              umma_fp4_ss<MX, false>(tmem + part * N, a0 + off + part * ((kTileM * kStepB) >> 4) + kk * 2, b0 + off + kk * 2,
                                     idesc, wsc + (part * F::kTiles + c) * 4, xsc + c * 4, (i > 0 || kk > 0) ? 1u : 0u);
          }
        }
        umma_commit(&empty[s]);
        if (i == nk - 1) umma_commit(acc_full);
      }
      __syncwarp();
      if (++s == stages) {
        s = 0;
        phase ^= 1;
      }
    }
  } else {
    if (et < N) sx[et] = !MX && et < p.T ? p.x_row[et] : 1.f;
    o = o0 + rowt;
    if (splits > 1) o = o0 + et % kTileM;
    if (o < p.F) {
      if (!MX) ws = ScalePair(p.w_row[o]);
      if (p.bias) bs = p.bias[o];
      if (kGeglu) {
        if (!MX) wu = ScalePair(p.w_row[p.F + o]);
        if (p.bias) bu = p.bias[p.F + o];
      }
    }
    epi_agree(true);  // the scales are in shared memory
    summed = __all_sync(0xffffffffu, mbar_wait(acc_full, 0, p.status, kDevTimeoutMmaDone));
    tc_fence_after();
    if (splits == 1 && summed) {
      for (int j = hw; j < N / 16; j += 2) {
        uint32_t r[kParts][16];
#pragma unroll
        for (int part = 0; part < kParts; ++part) tmem_ld16(acc + part * N + 16 * j, r[part]);
        tmem_wait_ld();
        if (o < p.F) {
          Tout* y = static_cast<Tout*>(p.y) + 16l * j * p.ldy + o;
          float v[16];
#pragma unroll
          for (int q = 0; q < 16; ++q) {
            const float s = sx[16 * j + q];
            v[q] = fmaf(__uint_as_float(r[0][q]) * ws.a * s, ws.b, bs);
            if (kGeglu)
              v[q] = gelu_ex2(v[q]) * fmaf(__uint_as_float(r[kParts - 1][q]) * wu.a * s, wu.b, bu);
            else
              v[q] = activate<ACT>(v[q]);
          }
          // (the values first: behind its own branch each would wait for the one before it)
#pragma unroll
          for (int q = 0; q < 16; ++q, y += p.ldy)
            if (16 * j + q < p.T) put1(y, v[q]);
        }
      }
    }
  }
  if (splits > 1) {
    __syncwarp();
    cluster_wait_acquire();
    if (warp >= 2 && summed) {
      for (int j = hw; j < N / 16; j += 2) {
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          uint32_t r[16];
          tmem_ld16(acc + part * N + 16 * j, r);
          tmem_wait_ld();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int g = 4 * j + q;
            const int owner = g & (splits - 1), slot = ((rank * mine + (g >> shift)) * kParts + part) * kTileM + rowt;
            st_dsmem_f4(mapa_shared(smem_u32(red), static_cast<uint32_t>(owner)) + static_cast<uint32_t>(slot) * 16u,
                        __uint_as_float(r[4 * q]), __uint_as_float(r[4 * q + 1]), __uint_as_float(r[4 * q + 2]),
                        __uint_as_float(r[4 * q + 3]));
          }
        }
      }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem, cols);
    }
    __syncwarp();
    cluster_sync();
    if (warp >= 2 && summed && o < p.F) {
      const float4* in = reinterpret_cast<const float4*>(red) + et % kTileM;
      for (int it = et / kTileM; it < mine && (it * splits + rank) * 4 < p.T; it += 2) {
        const int t = (it * splits + rank) * 4;
        float a[kParts][4];
#pragma unroll
        for (int part = 0; part < kParts; ++part)
#pragma unroll
          for (int q = 0; q < 4; ++q) a[part][q] = 0.f;
        for (int src = 0; src < splits; ++src) {
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            const float4 x = in[((src * mine + it) * kParts + part) * kTileM];
            a[part][0] += x.x;
            a[part][1] += x.y;
            a[part][2] += x.z;
            a[part][3] += x.w;
          }
        }
        const float4 s4 = *reinterpret_cast<const float4*>(sx + t);
        const float sv[4] = {s4.x, s4.y, s4.z, s4.w};
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v[q] = fmaf(a[0][q] * ws.a * sv[q], ws.b, bs);
          if (kGeglu)
            v[q] = gelu_ex2(v[q]) * fmaf(a[kParts - 1][q] * wu.a * sv[q], wu.b, bu);
          else
            v[q] = activate<ACT>(v[q]);
        }
        Tout* y = static_cast<Tout*>(p.y) + static_cast<long>(t) * p.ldy + o;
#pragma unroll
        for (int q = 0; q < 4; ++q, y += p.ldy)
          if (t + q < p.T) put1(y, v[q]);
      }
    }
  }
  tc_fence_before();
  // a producer that stopped early waits (bounded) for its copies in flight
  if (warp == 0 && lane == 0)
    for (int i = (issued > stages ? issued - stages : 0); i < issued; ++i)
      mbar_wait(&full[i % stages], (i / stages) & 1, p.status, kDevTimeoutTmaFull);
  __syncthreads();
  if (warp == 1 && splits == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

// ------------------------------------------------------------ host side ---
bool al(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int out_cols(const rfx_linear_fp4_desc& d) { return d.epilogue == RFX_EPI_GEGLU ? d.O / 2 : d.O; }

template <int ACT, bool MX>
const void* fp4_ptr(int out_dtype, int form) {
  if (form == kFp4Side)
    return out_dtype == kDtypeBF16 ? reinterpret_cast<const void*>(linear_fp4_side_kernel<ACT, MX, __nv_bfloat16>)
                                   : reinterpret_cast<const void*>(linear_fp4_side_kernel<ACT, MX, float>);
  return out_dtype == kDtypeBF16 ? reinterpret_cast<const void*>(linear_fp4_pair_kernel<ACT, MX, __nv_bfloat16>)
                                 : reinterpret_cast<const void*>(linear_fp4_pair_kernel<ACT, MX, float>);
}
template <int ACT>
const void* fp4_act(const rfx_linear_fp4_desc& d, int form) {
  return d.format == RFX_FP4_MX ? fp4_ptr<ACT, true>(d.out_dtype, form) : fp4_ptr<ACT, false>(d.out_dtype, form);
}
const void* fp4_kernel(const rfx_linear_fp4_desc& d, int form) {
  switch (d.epilogue) {
    case RFX_EPI_STORE: return fp4_act<kActNone>(d, form);
    case RFX_EPI_SILU: return fp4_act<kActSilu>(d, form);
    case RFX_EPI_GELU: return fp4_act<kActGelu>(d, form);
    case RFX_EPI_GEGLU: return fp4_act<kActGeglu>(d, form);
  }
  return nullptr;
}

// Tiles with the weights on the M side: the split of K that ends soonest by this model, in
// us, fitted to 10 projections of 1, 16, 50 and 128 tokens at every split.  A K step takes
// kStep (kStepGeglu with two weight rows per output; more where the ring has a stage or
// two), launch and epilogue kFix and kFixToken per token, the exchange kSplit, kSplitStep
// and kSplitToken (twice the sums with two rows per output).
void plan_side(const rfx_linear_fp4_desc& d, int nsm, int k_steps, LinearFp4Plan* c) {
  constexpr double kFix = 1.75, kFixToken = 0.0095, kStep = 0.365, kStepGeglu = 0.55;
  const double kSplit = d.epilogue == RFX_EPI_GEGLU ? 1.6 : 0.6, kSplitStep = 0.12, kSplitToken = d.epilogue == RFX_EPI_GEGLU ? 0.025 : 0.012;
  const bool geglu = d.epilogue == RFX_EPI_GEGLU, mx = d.format == RFX_FP4_MX;
  const void* fn = fp4_kernel(d, kFp4Side);
  const int N = (d.T + 15) / 16 * 16;
  const long tiles = (out_cols(d) - 1) / kTileM + 1;
  c->form = kFp4Side;
  c->nt = N;
  c->clusters = static_cast<int>(tiles);
  double best = 0;
  for (int s = 1; s <= kSideMaxSplits && s <= k_steps; s *= 2) {
    const int n = (k_steps + s - 1) / s;
    int stages = std::min(kSideMaxStages, n);
    while (stages > 1 && side_smem(N, s, geglu, mx, stages) > kSmemMax) --stages;
    const int smem = side_smem(N, s, geglu, mx, stages);
    if (smem > kSmemMax) break;
    double waves = std::max(1.0, static_cast<double>(tiles) / nsm);
    if (s > 1) {
      const long slots = std::min<long>(max_active_clusters(fn, kSideThreads, smem, s), nsm * (512l / side_cols(N, geglu, mx)) / s);
      if (slots <= 0) break;
      waves = std::max<double>((tiles + slots - 1) / slots, static_cast<double>(tiles) * s / nsm);
    }
    const double step = (geglu ? kStepGeglu : kStep) + (n > stages ? (stages == 1 ? 0.8 : stages == 2 ? 0.35 : 0.0) : 0.0);
    // (without clusters CTAs follow one another on an SM, or share it)
    const double cost = s == 1 ? kFix + waves * (kFixToken * d.T + n * step)
                               : waves * (kFix + kFixToken * d.T + n * step + kSplit + kSplitStep * n + kSplitToken * d.T);
    if (s > 1 && cost >= best) continue;
    best = cost;
    c->splits = s;
    c->stages = stages;
  }
}

// Pair tiles, above 128 tokens: the width and the split of K that finish soonest by
// this model, in ns, fitted to measured times of 17 projections of 129 to 4096 tokens
// at every width and split.  Launch, first copies and last epilogue take kBase +
// kBaseRow per weight row; a K step what kStep says of its width, and kHalves more
// where the gate and up rows are MMAs of their own; from one tile to the next kTurn,
// more where one accumulator has to be emptied in between; adding up a split K kSplit
// per split.
LinearFp4Plan plan_fp4(const rfx_linear_fp4_desc& d, int nsm) {
  constexpr double kBase = 4300, kBaseRow = 5.8, kStep[4] = {310, 320, 365, 385}, kHalves = 130;
  constexpr double kTurn[2] = {600, 1600}, kSplit = 1200;
  LinearFp4Plan c{};
  const bool geglu = d.epilogue == RFX_EPI_GEGLU, mx = d.format == RFX_FP4_MX;
  const int div = geglu ? 2 : 1;  // weight rows per output column
  const int F = out_cols(d);
  const int k_steps = (d.K + kStepK - 1) / kStepK;
  if (d.T <= kSideTokens) {
    plan_side(d, nsm, k_steps, &c);
    return c;
  }
  const int m = (d.T - 1) / (2 * kTileM) + 1;
  const int width = 64 * div;  // scale tiles are taken from multiples of 64 rows on
  const void* fn = fp4_kernel(d, kFp4Pair);
  auto tiles_of = [&](int cols, int nt) { return static_cast<int>((static_cast<long>(cols) * div + nt - 1) / nt); };
  auto sum_ns = [&](int nt, int s) {
    return (k_steps + s - 1) / s * (kStep[nt / 64 - 1] + (geglu && nt < 256 ? kHalves : 0.0));
  };
  auto epi_ns = [&](int nt) { return kBase + kBaseRow * nt; };
  auto tile_ns = [&](int nt) { return sum_ns(nt, 1) + kTurn[nt > kAcc1]; };
  double best = 0;
  for (int s = 1; s <= std::min(kMaxSplits, k_steps); ++s) {
    // clusters of 2s CTAs that are resident at once (GPCs hold whole clusters)
    int slots = max_active_clusters(fn, kPairThreads, kPairSmem, 2 * s);
    if (slots <= 0) {
      if (s > 1) break;
      slots = std::max(1, nsm / 2);
    }
    for (int nt = width; nt <= 256; nt += width) {
      const int n = tiles_of(F, nt);
      const long tiles = static_cast<long>(m) * n;
      const long rounds = (tiles + slots - 1) / slots;
      if (s > 1 && rounds > 1) continue;
      // what a CTA is sent has to fit into its ring: groups of 128 output bytes, of which
      // it finishes one in `s`, from each of the other splits
      const int group = 128 / (d.out_dtype == kDtypeBF16 ? 2 : 4), groups = (nt / div + group - 1) / group;
      if (s > 1 && (groups + s - 1) / s * (s - 1) * div * (group / 4 * kTileM * 16) > kPairRing) continue;
      auto consider = [&](double cost, int n_a, int nt2, int n_b) {
        if (c.nt != 0 && cost >= best) return;
        best = cost;
        c.nt = nt;
        c.splits = s;
        c.n_tiles = n_a;
        c.nt2 = nt2;
        c.n_tiles2 = n_b;
        c.clusters = static_cast<int>(std::min<long>(static_cast<long>(m) * (n_a + n_b), slots));
      };
      if (s > 1) {
        consider(sum_ns(nt, s) + epi_ns(nt) + kSplit * s, n, 0, 0);
        continue;
      }
      consider((rounds - 1) * tile_ns(nt) + sum_ns(nt, 1) + epi_ns(nt), n, 0, 0);
      if (rounds < 2) continue;
      // the full rounds at this width, the rest in narrower tiles
      const int n_a = static_cast<int>((rounds - 1) * slots / m);
      if (n_a < 1 || n_a >= n) continue;
      for (int nt2 = width; nt2 < nt; nt2 += width) {
        const int n_b = tiles_of(F - n_a * (nt / div), nt2);
        const long ua = static_cast<long>(n_a) * m, ub = static_cast<long>(n_b) * m;
        // the tiles go round the slots: the busiest slot's time
        const double ta = tile_ns(nt), tb = tile_ns(nt2), end = epi_ns(nt2) - kTurn[nt2 > kAcc1];
        const long qa = ua / slots, ra = ua % slots, first = slots - ra;  // `first` slots have one wide tile less
        double time;
        if (ub <= first) {
          time = std::max(qa * ta + tb, (qa + (ra ? 1 : 0)) * ta);
        } else {
          const long qb = (ub - first) / slots, rb = (ub - first) % slots;
          time = std::max(ra ? (qa + 1) * ta + (qb + (rb ? 1 : 0)) * tb : 0.0, qa * ta + (1 + qb + (rb > ra ? 1 : 0)) * tb);
        }
        // (a gain of a hundredth by this model is none by the clock)
        consider(1.01 * (time + end), n_a, nt2, n_b);
      }
    }
  }
  c.form = kFp4Pair;
  c.m_tiles = m;
  const int stage = (kTileM + c.nt / 2) * kStepB + 3 * (mx ? Fmt<true>::kBytes : Fmt<false>::kBytes);
  c.stages = std::min(kPairMaxStages, kPairRing / stage);
  return c;
}

}  // namespace

int validate_linear_fp4(const rfx_linear_fp4_desc& d) {
  if (d.T < 0 || d.T > kMaxRows || d.O < 1 || d.O > kMaxRows || d.K < 1 || d.K > kMaxK)
    return set_error(RFX_E_INVAL, "rfx_linear_fp4: need 0<=T<=2^30, 1<=O<=2^30, 1<=K<=%d (T=%d O=%d K=%d)", kMaxK, d.T,
                     d.O, d.K);
  if (d.format != RFX_FP4_MX && d.format != RFX_FP4_NV)
    return set_error(RFX_E_INVAL, "rfx_linear_fp4: format must be MX or NV");
  if (d.epilogue != RFX_EPI_STORE && d.epilogue != RFX_EPI_SILU && d.epilogue != RFX_EPI_GELU &&
      d.epilogue != RFX_EPI_GEGLU)
    return set_error(RFX_E_INVAL, "rfx_linear_fp4: epilogue must be STORE, SILU, GELU or GEGLU");
  if (d.epilogue == RFX_EPI_GEGLU && d.O % 2)
    return set_error(RFX_E_INVAL, "rfx_linear_fp4: GEGLU needs an even O (gate rows, then as many up rows)");
  if (d.out_dtype != kDtypeBF16 && d.out_dtype != kDtypeF32)
    return set_error(RFX_E_INVAL, "rfx_linear_fp4: output dtype must be bf16 or f32");
  if (d.T == 0) return RFX_OK;
  if (!d.x || !d.w || !d.x_scale || !d.w_scale || !d.y)
    return set_error(RFX_E_INVAL, "rfx_linear_fp4: null pointer");
  const bool nv = d.format == RFX_FP4_NV;
  if (nv != (d.x_row_scale != nullptr) || nv != (d.w_row_scale != nullptr))
    return set_error(RFX_E_INVAL, "rfx_linear_fp4: row scales go with RFX_FP4_NV, and only with it");
  const long kb = (d.K + 1) / 2;
  if (!al(d.x, 16) || !al(d.w, 16) || !al(d.x_scale, 16) || !al(d.w_scale, 16) || d.ldx < kb || d.ldw < kb ||
      d.ldx % 16 || d.ldw % 16)
    return set_error(RFX_E_INVAL,
                     "rfx_linear_fp4: 4-bit rows and scales must begin on 16-byte boundaries (ldx and ldw at least half "
                     "of K and multiples of 16)");
  if (d.ldy < out_cols(d) || !al(d.y, d.out_dtype == kDtypeBF16 ? 2 : 4) || !al(d.x_row_scale, 4) ||
      !al(d.w_row_scale, 4) || !al(d.bias, 4))
    return set_error(RFX_E_INVAL, "rfx_linear_fp4: ldy below the output's columns, or a misaligned pointer");
  const long esz = d.out_dtype == kDtypeBF16 ? 2 : 4;
  const int part = d.epilogue == RFX_EPI_GEGLU ? d.O / 2 : 0;
  const long xs = fp4_scale_bytes(d.T, d.K, d.format, 0), ws = fp4_scale_bytes(d.O, d.K, d.format, part);
  const Rows y{d.y, d.T, d.ldy * esz, out_cols(d) * esz};
  if (rows_shared(y, {d.x, d.T, d.ldx, kb}) || rows_shared(y, {d.w, d.O, d.ldw, kb}) ||
      rows_shared(y, {d.x_scale, 1, 0, xs}) || rows_shared(y, {d.w_scale, 1, 0, ws}) ||
      rows_shared(y, {d.x_row_scale, 1, 0, d.T * 4l}) || rows_shared(y, {d.w_row_scale, 1, 0, d.O * 4l}) ||
      rows_shared(y, {d.bias, 1, 0, d.O * 4l}))
    return set_error(RFX_E_INVAL, "rfx_linear_fp4: y shares memory with an input");
  if ((static_cast<long>(d.T) / kTileM + 1) * (d.O / 32 + 1) > 0x7fffffffL / 8 || xs / kScaleTile > 0x3fffffffL ||
      ws / kScaleTile > 0x3fffffffL)
    return set_error(RFX_E_INVAL, "rfx_linear_fp4: too many tiles (T=%d O=%d K=%d)", d.T, d.O, d.K);
  return RFX_OK;
}

int build_linear_fp4_maps(const rfx_linear_fp4_desc& d, LinearFp4Maps* maps) {
  int rc = validate_linear_fp4(d);
  if (rc || d.T == 0) return rc;
  int nsm = 148;
  rfx_num_sms(&nsm);
  maps->plan = plan_fp4(d, nsm);
  const LinearFp4Plan& c = maps->plan;
  const bool geglu = d.epilogue == RFX_EPI_GEGLU;
  const int kb = (d.K + 1) / 2, tiles = d.format == RFX_FP4_MX ? Fmt<true>::kTiles : Fmt<false>::kTiles;
  rc = make_tmap_2d(&maps->x, d.x, 1, kb, d.T, d.ldx, kStepB, c.form == kFp4Side ? d.T : kTileM, true);
  if (rc) return rc;
  // scale tiles as rows of 512 bytes
  const long xs = fp4_scale_bytes(d.T, d.K, d.format, 0), ws = fp4_scale_bytes(d.O, d.K, d.format, geglu ? d.O / 2 : 0);
  rc = make_tmap_2d(&maps->xs, d.x_scale, 4, kScaleTile / 4, xs / kScaleTile, kScaleTile, kScaleTile / 4, tiles, false);
  if (rc) return rc;
  rc = make_tmap_2d(&maps->ws, d.w_scale, 4, kScaleTile / 4, ws / kScaleTile, kScaleTile, kScaleTile / 4, tiles, false);
  if (rc) return rc;
  if (c.form == kFp4Side) return make_tmap_2d(&maps->w, d.w, 1, kb, d.O, d.ldw, kStepB, kTileM, true);
  auto box = [&](int nt) { return geglu && nt < 256 ? nt / 4 : nt / 2; };
  rc = make_tmap_2d(&maps->w, d.w, 1, kb, d.O, d.ldw, kStepB, box(c.nt), true);
  if (rc) return rc;
  maps->w2 = maps->w;
  if (c.n_tiles2 > 0) {
    rc = make_tmap_2d(&maps->w2, d.w, 1, kb, d.O, d.ldw, kStepB, box(c.nt2), true);
    if (rc) return rc;
  }
  const int esz = d.out_dtype == kDtypeBF16 ? 2 : 4;
  maps->y = maps->w;  // not used where y's rows are not 16-byte aligned
  if (al(d.y, 16) && (d.ldy * esz) % 16 == 0)
    rc = make_tmap_2d_swizzle(&maps->y, d.y, esz, out_cols(d), d.T, d.ldy * esz, 64 / esz, 32, 64);
  return rc;
}

int launch_linear_fp4(const rfx_linear_fp4_desc& d, const LinearFp4Maps& maps, cudaStream_t stream, bool pdl) {
  if (d.T == 0) return RFX_OK;
  const LinearFp4Plan& c = maps.plan;
  const bool geglu = d.epilogue == RFX_EPI_GEGLU, mx = d.format == RFX_FP4_MX;
  const void* fn = fp4_kernel(d, c.form);
  const int rc = ensure_smem_attr(fn, kSmemMax);
  if (rc) return rc;
  const int per_step = mx ? Fmt<true>::kTiles : Fmt<false>::kTiles;
  Fp4Params p{};
  p.T = d.T;
  p.F = out_cols(d);
  p.k_steps = (d.K + kStepK - 1) / kStepK;
  p.k_mmas = (d.K + kMmaK - 1) / kMmaK;
  p.k_tiles = (d.K + kStepK / per_step - 1) / (kStepK / per_step);
  p.up_tiles = geglu ? (d.O / 2 - 1) / 128 + 1 : 0;
  p.splits = c.splits;
  p.m_tiles = c.m_tiles;
  p.n_tile = c.nt;
  p.n_tail = c.nt2;
  p.cols_a = c.n_tiles;
  p.units = c.m_tiles * (c.n_tiles + c.n_tiles2);
  p.stages = c.stages;
  p.x_row = d.x_row_scale;
  p.w_row = d.w_row_scale;
  p.bias = d.bias;
  p.y = d.y;
  p.ldy = d.ldy;
  p.status = device_status_ptr();
  CUtensorMap x = maps.x, w = maps.w, w2 = maps.w2, xs = maps.xs, ws = maps.ws, y = maps.y;
  if (c.form == kFp4Side) {
    const int smem = side_smem(c.nt, c.splits, geglu, mx, c.stages);
    return launch_kernel(fn, dim3(c.clusters * c.splits), dim3(kSideThreads), static_cast<size_t>(smem), stream, pdl,
                         c.splits, x, w, xs, ws, p);
  }
  return launch_kernel(fn, dim3(2 * c.splits * c.clusters), dim3(kPairThreads), static_cast<size_t>(kPairSmem), stream,
                       pdl, 2 * c.splits, x, w, w2, xs, ws, y, p);
}

}  // namespace rfx

extern "C" int rfx_linear_fp4(const rfx_linear_fp4_desc* d, void* stream) {
  using namespace rfx;
  if (!d) return set_error(RFX_E_INVAL, "rfx_linear_fp4: null descriptor");
  LinearFp4Maps maps;
  const int rc = build_linear_fp4_maps(*d, &maps);
  if (rc) return rc;
  return launch_linear_fp4(*d, maps, static_cast<cudaStream_t>(stream), pdl_enabled());
}
