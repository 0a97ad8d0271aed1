// Linear layers in 8-bit integers: y = act(x_scale[t] * w_scale[o] * (x_q · w_qᵀ) + bias[o]).
//
// The integer products are summed exactly (tcgen05.mma kind::i8, s32
// accumulators in TMEM), so neither the order of the sum nor a split of K
// changes a result: the only roundings are the int -> fp32 conversion, the two
// scales, bias and activation in fp32, and one rounding to the output type.
//
// Three forms, whose results are the same bits: CTA-pair tiles of 256 tokens
// (tokens on the MMA's M side: a TMEM lane is a token, and a thread of the
// epilogue holds consecutive outputs of one row), tiles of 128 weight rows (the
// weights on the M side) for up to 128 tokens, and the integer units for up to
// 4.  The tiles' operands are K-major rows of 128 bytes per K step, staged by TMA
// with 128-byte swizzle; what lies past T, O or K is filled with zeros by the
// copy or not copied, and not stored.  For GeGLU half of a tile's weight rows
// are gate rows and half up rows of [Wgate; Wup].
#include "rfx_internal.h"
#include "tile_epilogue.cuh"

#include <algorithm>
#include <cmath>

namespace rfx {
namespace {

constexpr int kTileM = 128;
constexpr int kStepK = 128;  // int8 elements (bytes) of K per stage
constexpr int kSmemMax = 227 * 1024;
constexpr int kMaxRows = 1 << 30;  // of x and of w
constexpr int kMaxK = 65536;  // 65536 * 128 * 128 = 2^30: an s32 sum cannot overflow

struct I8Params {
  int T, O, K;
  int F;            // output columns: O, or O / 2 with GeGLU
  int k_steps;      // of 128
  int splits;       // parts of K: pairs per cluster, or warps per pair of rows
  int m_tiles;      // 256-token tiles
  int n_tile;       // weight rows per tile,
  int n_tail;       // of the tiles from column cols_a on
  int cols_a, units;
  int stages;
  const int8_t* x;
  long ldx;
  const int8_t* w;
  long ldw;
  const float* x_scale;
  const float* w_scale;
  const float* bias;
  void* y;
  long ldy;
  int* status;
};

__device__ __forceinline__ void st_dsmem_i4(uint32_t addr, const int (&v)[4]) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}

// ------------------------------------------------------- CTA-pair tiles ---
// A pair of CTAs computes 256 tokens x N weight rows (N a multiple of 32 up to
// 256) with cta_group::2 MMAs: each CTA stages its 128 tokens and half of the
// weight rows per K step, so a step moves 16 KB + 64 N bytes into each SM for
// 2 N clocks of MMA, and with N = 256 the L2 -> SM stream (64 B/clk) just keeps
// up.  With GeGLU the even CTA stages the gate
// rows and the odd one the up rows, and a thread of either finds both halves of
// its outputs in its own TMEM lane.
//
// splits == 1: persistent.  The pair walks the tiles, the two accumulators of
// 256 TMEM columns alternate, and a tile's epilogue (8 warps) runs under the
// next tile's MMAs.
// splits > 1: a cluster of `splits` pairs computes one tile, each pair a part
// of K; at the end each CTA pushes the s32 sums of the columns that another
// split owns into that CTA's (now idle) operand ring through DSMEM and adds
// what it receives to its own.
//
// Measured, T x O x K: 4096 x 4096 x 4096 48 us, 2.8 POP/s (85 % of twice the
// measured bf16 burst rate; 55 us, 89 % of twice the sustained one, in a loop under
// the power cap); 768 x 32768 x 2048 GeGLU 39 us (2.6 POP/s; this instance spills
// 32 bytes at its 168 registers); 768 x 2048 x 16384 24 us (2.1 POP/s, two
// splits).  With the MMAs left out the first takes 34 us and with the copies left
// out 39: both streams are near their limit, and they share the SM's shared
// memory.  Calls of one tile per pair spend about 7 us outside the product: set-up
// 1, the first copy 1.2 - 1.8, the last epilogue 2 - 3 and the pair's exit 0.8.
constexpr int kPairThreads = 320;
constexpr int kPairMaxStages = 10;
constexpr int kPairRing = 6 * 2 * kTileM * kStepK;     // operand ring: 6 stages of N = 256, more of a narrower N
constexpr int kPairOffVec = kPairRing;                 // [2][w_scale | bias][256]
constexpr int kPairOffOut = kPairOffVec + 2 * 2 * 256 * 4;  // output staging, 2 KB per epilogue warp
constexpr int kPairOffBars = kPairOffOut + 8 * 32 * 64;
constexpr int kPairSmem = kPairOffBars + 256 + 1024;
constexpr int kMaxSplits = 4;                          // clusters of at most 8 CTAs
static_assert(kPairSmem <= kSmemMax, "pair tiles fit in shared memory");
static_assert((kPairMaxStages * 2 + 4) * 8 + 4 <= 256, "barriers fit");

// 16 outputs of one token: scales and bias from shared memory.
template <int ACT>
__device__ __forceinline__ void finish16(const uint32_t (&acc)[16], const uint32_t (&up)[16], float sx,
                                         const float* ws, const float* bs, int half, float (&v)[16]) {
#pragma unroll
  for (int g = 0; g < 16; g += 4) {
    const float4 w = *reinterpret_cast<const float4*>(ws + g);
    const float4 b = *reinterpret_cast<const float4*>(bs + g);
    const float wv[4] = {w.x, w.y, w.z, w.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[g + j] = fmaf(static_cast<float>(static_cast<int>(acc[g + j])) * sx, wv[j], bv[j]);
    if (ACT == kActGeglu) {
      const float4 w2 = *reinterpret_cast<const float4*>(ws + half + g);
      const float4 b2 = *reinterpret_cast<const float4*>(bs + half + g);
      const float wu[4] = {w2.x, w2.y, w2.z, w2.w}, bu[4] = {b2.x, b2.y, b2.z, b2.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[g + j] = gelu_ex2(v[g + j]) * fmaf(static_cast<float>(static_cast<int>(up[g + j])) * sx, wu[j], bu[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[g + j] = activate<ACT>(v[g + j]);
    }
  }
}

template <int ACT, typename Tout>
__global__ void __launch_bounds__(kPairThreads, 1)
    linear_i8_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                          const __grid_constant__ CUtensorMap tmW2, const __grid_constant__ CUtensorMap tmY,
                          const I8Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr bool kGeglu = ACT == kActGeglu;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* vec = reinterpret_cast<float*>(smem + kPairOffVec);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kPairOffBars);
  uint64_t* empty = full + kPairMaxStages;
  uint64_t* acc_full = empty + kPairMaxStages;  // [2]
  uint64_t* acc_free = acc_full + 2;         // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_free + 2);
  const uint32_t crank = cluster_ctarank();
  const uint32_t rank = crank & 1u;  // in the pair
  const bool leader = rank == 0;
  const int split = static_cast<int>(crank >> 1);
  // Units, m_tiles to a column of tiles: first tiles of N = n_tile, then, from
  // column cols_a on, of N = n_tail, so that the last round of tiles is a narrow
  // one.  A walker keeps its place (tile row, column) and steps without dividing.
  const int ustep = gridDim.x / (2 * p.splits), unit0 = blockIdx.x / (2 * p.splits);
  struct Unit {
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
  auto unit_of = [&](const Walk& k) {
    const int w = kGeglu ? p.n_tile / 2 : p.n_tile, w2 = kGeglu ? p.n_tail / 2 : p.n_tail;
    Unit u;
    u.m = k.m;
    u.tail = k.n >= p.cols_a;
    u.N = u.tail ? p.n_tail : p.n_tile;
    u.o0 = u.tail ? p.cols_a * w + (k.n - p.cols_a) * w2 : k.n * w;
    return u;
  };
  const int stages = p.stages, stage = (kTileM + p.n_tile / 2) * kStepK;
  const int k0 = static_cast<int>(static_cast<long>(split) * p.k_steps / p.splits);
  const int nk = static_cast<int>(static_cast<long>(split + 1) * p.k_steps / p.splits) - k0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_free[i], 16);  // both CTAs' epilogue warps, on the even CTA's barrier
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
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
  constexpr int kGroup = 128 / static_cast<int>(sizeof(Tout));  // output columns of 128 bytes
  constexpr int kHalf = kGroup / 2;                              // of which a warp finishes half
  uint8_t* out_st = smem + kPairOffOut + (warp - 2) * 32 * 64;
  bool failed = false;
  int issued = 0;
  if (warp == 0) {
    // as in the MMA warp, the whole warp walks the steps and one lane issues
    bool ok = true;
    int s = 0;
    uint32_t phase = 0;
    const uint32_t full0 = mapa_shared(smem_u32(full), crank & ~1u);
    for (Walk k = first; k.un < p.units && ok; next(k)) {
      const Unit tile = unit_of(k);
      const int t0 = tile.m * 2 * kTileM + static_cast<int>(rank) * kTileM;
      const int wrow = kGeglu ? (rank ? p.F + tile.o0 : tile.o0) : tile.o0 + static_cast<int>(rank) * (tile.N / 2);
      const CUtensorMap* tw = tile.tail ? &tmW2 : &tmW;
      // both CTAs' copies count on the even CTA's barrier; a half without
      // tokens copies none (what its rows multiply is not stored)
      const bool has_x = t0 < p.T;
      const int x_rows = has_x && t0 + kTileM < p.T ? 2 * kTileM : kTileM;
      const uint32_t bytes = static_cast<uint32_t>(x_rows + tile.N) * kStepK;
      for (int i = 0; i < nk; ++i) {
        if (issued >= stages && !(ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], phase ^ 1, p.status, kDevTimeoutStageEmpty))))
          break;
        if (elect_one()) {
          uint8_t* st = smem + s * stage;
          if (leader) mbar_arrive_expect_tx(&full[s], bytes);
          if (has_x) tma_load_2d_pair(st, &tmX, full0 + 8u * s, (k0 + i) * kStepK, t0);
          tma_load_2d_pair(st + kTileM * kStepK, tw, full0 + 8u * s, (k0 + i) * kStepK, wrow);
        }
        __syncwarp();
        ++issued;
        if (++s == stages) {
          s = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (leader) {
      // the whole warp walks the steps and one elected lane issues: the loop's
      // values stay uniform, where a loop inside `if (lane == 0)` spends more
      // clocks on each instruction's operands than the MMA takes
      const uint64_t a0 = make_sdesc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t b0 = make_sdesc_sw128(smem_u32(smem + kTileM * kStepK), 16, 1024);
      bool ok = true;
      int s = 0, tl = 0;
      uint32_t phase = 0;
      for (Walk k = first; k.un < p.units && ok; next(k), ++tl) {
        const int buf = tl & 1;
        const uint32_t idesc = make_idesc_i8(2 * kTileM, k.n < p.cols_a ? p.n_tile : p.n_tail);
        if (tl >= 2 &&
            !(ok = __all_sync(0xffffffffu, mbar_wait(&acc_free[buf], ((tl >> 1) - 1) & 1, p.status, kDevTimeoutMmaDone))))
          break;
        tc_fence_after();
        const uint32_t acc = tmem + buf * 256;
        for (int i = 0; i < nk; ++i) {
          if (!(ok = __all_sync(0xffffffffu, mbar_wait(&full[s], phase, p.status, kDevTimeoutTmaFull)))) break;
          tc_fence_after();
          const uint64_t off = static_cast<uint64_t>((s * stage) >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kStepK / 32; ++kk)
              umma_i8_ss_pair(acc, a0 + off + kk * 2, b0 + off + kk * 2, idesc, (i > 0 || kk > 0) ? 1u : 0u);
            umma_commit_pair(smem_u32(&empty[s]));
            umma_commit_pair(mapa_shared(smem_u32(&empty[s]), crank | 1u));
            if (i == nk - 1) {
              umma_commit_pair(smem_u32(&acc_full[buf]));
              umma_commit_pair(mapa_shared(smem_u32(&acc_full[buf]), crank | 1u));
            }
          }
          __syncwarp();
          if (++s == stages) {
            s = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else {
    const int et = threadIdx.x - 64;  // 0..255
    const int quad = warp & 3;
    const int hw = (warp - 2) >> 2;  // which of the two warps of this TMEM quadrant
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t free_bar = mapa_shared(smem_u32(&acc_free[0]), crank & ~1u);
    int tl = 0;
    // a tile's scales and bias come asynchronously while the tile before it is
    // finished (a short K's products are there at once: the loads would be
    // waited for at every tile's start)
    float sx_next = 0.f;
    auto request = [&](const Unit& tile, int b) {
      if (et < tile.N) {
        const int nh = tile.N / 2;
        const int c = kGeglu ? (et < nh ? et : et - nh) : et;
        const bool in = tile.o0 + c < p.F;
        const int o = tile.o0 + c + (kGeglu && et >= nh ? p.F : 0);
        float* ws = vec + b * 512 + et;
        if (in)
          cp_async4(ws, p.w_scale + o);
        else
          *ws = 0.f;
        if (in && p.bias)
          cp_async4(ws + 256, p.bias + o);
        else
          ws[256] = 0.f;
      }
      cp_async_commit();
      const int t = tile.m * 2 * kTileM + static_cast<int>(rank) * kTileM + quad * 32 + lane;
      sx_next = t < p.T ? p.x_scale[t] : 0.f;
    };
    if (first.un < p.units) request(unit_of(first), 0);
    for (Walk k = first; k.un < p.units; next(k), ++tl) {
      const int buf = tl & 1;
      const Unit tile = unit_of(k);
      const int N = tile.N, nh = N / 2, oc = kGeglu ? nh : N;  // oc output columns
      const int tw = tile.m * 2 * kTileM + static_cast<int>(rank) * kTileM + quad * 32;  // the warp's first token
      const int o0 = tile.o0;
      const float* ws = vec + buf * 512;
      const float* bs = ws + 256;
      const float sx = sx_next;
      cp_async_wait_all();
      // every epilogue warp agrees before anyone leaves the loop
      if (!epi_agree(mbar_wait(&acc_full[buf], (tl >> 1) & 1, p.status, kDevTimeoutMmaDone))) {
        failed = true;
        break;
      }
      tc_fence_after();
      const uint32_t acc = tmem + buf * 256 + lane_base;
      if (p.splits > 1) break;  // one tile per cluster: summed below
      Walk ahead = k;
      next(ahead);
      if (ahead.un < p.units) request(unit_of(ahead), buf ^ 1);
      // groups of 128 output bytes, of which each warp of the quadrant finishes
      // and stores 64
#pragma unroll 1
      for (int g = hw * kHalf; g < oc; g += kGroup) {
        uint32_t w[16];
        uint32_t r[kHalf / 16][16], u[kHalf / 16][16];
#pragma unroll
        for (int q = 0; q < kHalf / 16; ++q) {
          if (g + 16 * q < oc) {
            tmem_ld16(acc + g + 16 * q, r[q]);
            if (kGeglu) tmem_ld16(acc + nh + g + 16 * q, u[q]);
          }
        }
        tmem_wait_ld();
        if (g + kGroup >= oc) {  // this warp's last read of the accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(free_bar + 8u * buf);  // (a releasing one: 1400 clocks a tile)
        }
#pragma unroll
        for (int q = 0; q < kHalf / 16; ++q) {
          if (g + 16 * q < oc) {
            float v[16];
            finish16<ACT>(r[q], u[q], sx, ws + g + 16 * q, bs + g + 16 * q, nh, v);
            pack16(v, w + q * 8, static_cast<const Tout*>(nullptr));
          }
        }
        store_part<Tout>(p, &tmY, out_st, w, tw, o0 + g, p.T - tw, min(min(kHalf, oc - g), p.F - o0 - g), tma_y, lane);
      }
      if (hw * kHalf >= oc && lane == 0) mbar_arrive_cluster_relaxed(free_bar + 8u * buf);  // a warp without columns
    }
  }
  if (p.splits > 1) {
    // Every CTA's products are summed and its ring is idle: each pushes the
    // groups of 128 output bytes that another split owns (group j: split
    // j % splits) to the CTA of the same token half there, as
    // [group][source][gate | up][4 columns][token], and adds what it receives
    // to its own.  s32 sums: any order is exact.
    const Unit tile = unit_of(first);
    const int nh = tile.N / 2, oc = kGeglu ? nh : tile.N;
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
      for (int j = hw; j < groups * (kGroup / 16); j += 2) {  // 16-column chunks
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
          for (int g = 0; g < 4; ++g) {
            const int v[4] = {static_cast<int>(r[4 * g]), static_cast<int>(r[4 * g + 1]), static_cast<int>(r[4 * g + 2]),
                              static_cast<int>(r[4 * g + 3])};
            st_dsmem_i4(dst + static_cast<uint32_t>(slot * kSlot + (q * 4 + g) * kTileM * 16), v);
          }
        }
      }
    }
    __syncwarp();
    cluster_sync();
    if (warp >= 2 && !failed) {
      const int tw = tile.m * 2 * kTileM + static_cast<int>(rank) * kTileM + quad * 32;
      const int o0 = tile.o0;
      const float sx = tw + lane < p.T ? p.x_scale[tw + lane] : 0.f;
#pragma unroll 1
      for (int lg = 0; lg * p.splits + split < groups; ++lg) {
        const int g0 = (lg * p.splits + split) * kGroup;
        uint32_t w[16];
#pragma unroll
        for (int qq = 0; qq < kHalf / 16; ++qq) {
          const int q = hw * (kHalf / 16) + qq;
          const int c = g0 + 16 * q;
          if (c < oc) {
            uint32_t r[kParts][16];
#pragma unroll
            for (int part = 0; part < kParts; ++part) tmem_ld16(acc + part * nh + c, r[part]);
            tmem_wait_ld();
#pragma unroll 1
            for (int src = 0; src < others; ++src) {
#pragma unroll
              for (int part = 0; part < kParts; ++part) {
                const int4* recv = reinterpret_cast<const int4*>(smem + ((lg * others + src) * kParts + part) * kSlot) +
                                   q * 4 * kTileM + rowt;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                  const int4 v = recv[g * kTileM];
                  r[part][4 * g] += static_cast<uint32_t>(v.x);
                  r[part][4 * g + 1] += static_cast<uint32_t>(v.y);
                  r[part][4 * g + 2] += static_cast<uint32_t>(v.z);
                  r[part][4 * g + 3] += static_cast<uint32_t>(v.w);
                }
              }
            }
            float v[16];
            finish16<ACT>(r[0], r[kParts - 1], sx, vec + c, vec + 256 + c, nh, v);
            pack16(v, w + qq * 8, static_cast<const Tout*>(nullptr));
          }
        }
        const int g = g0 + hw * kHalf;
        store_part<Tout>(p, &tmY, out_st, w, tw, o0 + g, p.T - tw, min(min(kHalf, oc - g), p.F - o0 - g), tma_y, lane);
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
// Few tokens leave most of a 256-token tile's TMEM lanes empty and its epilogue
// to one or two of a pair's eight quadrants.  Here 128 weight rows are the
// MMA's M (with GeGLU 64 gate rows and their 64 up rows) and the tokens, a
// multiple of 16 up to kSideTokens, its N: every lane of the accumulator holds
// outputs, lanes lie along a row of y, and the tokens are copied once per
// weight row tile at their own size.
//
// One CTA per tile and part of K; a cluster of `splits` CTAs computes a tile.
// A CTA gives the sums of 4 tokens x 128 rows (group g: CTA g % splits) to the
// CTA that finishes them, as [source][group][row][4], through DSMEM into memory
// of their own (not the ring: no CTA has to wait for another's products before
// it sends).  GeGLU goes the same way with one CTA, through its idle ring: a
// gate's lane and its up's differ.
//
// Bound by what an SM takes in, 16 KB of weights and T x 128 bytes of tokens per
// K step, about 75 GB/s of the former, and by 3 to 4 us around the product.
// Measured, T x O x K (captured; in brackets as pair tiles): 50 x 8192 x 1024 GeGLU
// 6.6 us (7.5), 50 x 1024 x 4096 5.5 (9.4), 16 x 2560 x 1024 3.3 (5.4), 50 x 32768 x
// 2048 GeGLU 14.8, 4.5 TB/s of weights (19.7), 16 x 2048 x 16384 10.0 (16.3).
constexpr int kSideTokens = 128;  // the registers of an SM allow three CTAs: 384 of its 512 TMEM columns
constexpr int kSideThreads = 320;
constexpr int kSideMaxSplits = 8;
constexpr int kSideMaxStages = 16;

int side_groups(int N, int splits) { return (N / 4 + splits - 1) / splits; }
int side_ring(int N, int splits, bool geglu, int stages) {
  const int ring = stages * (kTileM + N) * kStepK;
  return splits == 1 && geglu ? std::max(ring, N * kTileM * 4) : ring;
}
int side_smem(int N, int splits, bool geglu, int stages) {
  return side_ring(N, splits, geglu, stages) + (splits > 1 ? splits * side_groups(N, splits) * kTileM * 16 : 0) + N * 4 +
         (2 * stages + 2) * 8 + 1024;
}

template <int ACT, typename Tout>
__global__ void __launch_bounds__(kSideThreads, 3)
    linear_i8_side_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const I8Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr bool kGeglu = ACT == kActGeglu;
  constexpr int kRows = kGeglu ? kTileM / 2 : kTileM;  // output columns of a tile
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int N = p.n_tile, splits = p.splits, stages = p.stages;
  const int stage = (kTileM + N) * kStepK;
  const int shift = 31 - __clz(splits);            // splits is a power of 2
  const int mine = (N / 4 + splits - 1) >> shift;  // groups of 4 tokens per CTA, at most
  const bool joined = kGeglu || splits > 1;
  // one CTA's own sums go where its ring was
  const int ring = splits == 1 && kGeglu ? max(stages * stage, N * kTileM * 4) : stages * stage;
  uint8_t* red = splits == 1 ? smem : smem + ring;
  float* sx = reinterpret_cast<float*>(smem + ring + (splits > 1 ? splits * mine * kTileM * 16 : 0));
  uint64_t* full = reinterpret_cast<uint64_t*>(sx + N);
  uint64_t* empty = full + stages;
  uint64_t* acc_full = empty + stages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  const int rank = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int o0 = (static_cast<int>(blockIdx.x) >> shift) * kRows;
  const int k0 = static_cast<int>(static_cast<long>(rank) * p.k_steps / splits);
  const int nk = static_cast<int>(static_cast<long>(rank + 1) * p.k_steps / splits) - k0;
  const uint32_t cols = N <= 32 ? 32 : N <= 64 ? 64 : 128;

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(acc_full, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (splits > 1) cluster_arrive_release();  // waited for before the first store into a peer
  pdl_launch_dependents();
  pdl_wait();

  const int et = threadIdx.x - 64, quad = warp & 3, hw = (warp - 2) >> 2;
  const uint32_t acc = tmem + (static_cast<uint32_t>(quad * 32) << 16);
  const int rowt = quad * 32 + lane;
  float ws = 0.f, bs = 0.f, wu = 0.f, bu = 0.f;  // of the row that this thread finishes
  int o = 0;
  bool summed = false;
  int issued = 0;
  if (warp == 0) {
    bool ok = true;
    int s = 0;
    uint32_t phase = 0;
    for (int i = 0; i < nk; ++i) {
      if (issued >= stages && !(ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], phase ^ 1, p.status, kDevTimeoutStageEmpty))))
        break;
      if (elect_one()) {
        uint8_t* st = smem + s * stage;
        const int k = (k0 + i) * kStepK;
        mbar_arrive_expect_tx(&full[s], static_cast<uint32_t>((kTileM + p.T) * kStepK));
        tma_load_2d(st, &tmW, &full[s], k, o0);
        if (kGeglu) tma_load_2d(st + kRows * kStepK, &tmW, &full[s], k, p.F + o0);
        tma_load_2d(st + kTileM * kStepK, &tmX, &full[s], k, 0);
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
    const uint64_t b0 = make_sdesc_sw128(smem_u32(smem + kTileM * kStepK), 16, 1024);
    const uint32_t idesc = make_idesc_i8(kTileM, N);
    int s = 0;
    uint32_t phase = 0;
    for (int i = 0; i < nk; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full[s], phase, p.status, kDevTimeoutTmaFull))) break;
      tc_fence_after();
      const uint64_t off = static_cast<uint64_t>((s * stage) >> 4);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kStepK / 32; ++kk)
          umma_i8_ss(tmem, a0 + off + kk * 2, b0 + off + kk * 2, idesc, (i > 0 || kk > 0) ? 1u : 0u);
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
    if (et < N) sx[et] = et < p.T ? p.x_scale[et] : 0.f;
    o = o0 + (joined ? et % kRows : rowt);
    if (o < p.F) {
      ws = p.w_scale[o];
      if (p.bias) bs = p.bias[o];
      if (kGeglu) {
        wu = p.w_scale[p.F + o];
        if (p.bias) bu = p.bias[p.F + o];
      }
    }
    epi_agree(true);  // the scales are in shared memory
    summed = __all_sync(0xffffffffu, mbar_wait(acc_full, 0, p.status, kDevTimeoutMmaDone));
    tc_fence_after();
    if (!joined && summed) {
      for (int j = hw; j < N / 16; j += 2) {
        uint32_t r[16];
        tmem_ld16(acc + 16 * j, r);
        tmem_wait_ld();
        if (o < p.F) {
          Tout* y = static_cast<Tout*>(p.y) + 16l * j * p.ldy + o;
          float v[16];
#pragma unroll
          for (int q = 0; q < 16; ++q)
            v[q] = activate<ACT>(fmaf(static_cast<float>(static_cast<int>(r[q])) * sx[16 * j + q], ws, bs));
          // (the values first: behind its own branch each would wait for the one before it)
#pragma unroll
          for (int q = 0; q < 16; ++q, y += p.ldy)
            if (16 * j + q < p.T) put1(y, v[q]);
        }
      }
    }
  }
  if (joined) {
    __syncwarp();
    if (splits > 1) cluster_wait_acquire();
    if (warp >= 2 && summed) {
      for (int j = hw; j < N / 16; j += 2) {
        uint32_t r[16];
        tmem_ld16(acc + 16 * j, r);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int g = 4 * j + q;
          const int v[4] = {static_cast<int>(r[4 * q]), static_cast<int>(r[4 * q + 1]), static_cast<int>(r[4 * q + 2]),
                            static_cast<int>(r[4 * q + 3])};
          if (splits == 1) {
            reinterpret_cast<int4*>(red)[g * kTileM + rowt] = make_int4(v[0], v[1], v[2], v[3]);
          } else {
            const int owner = g & (splits - 1), slot = (rank * mine + (g >> shift)) * kTileM + rowt;
            st_dsmem_i4(mapa_shared(smem_u32(red), static_cast<uint32_t>(owner)) + static_cast<uint32_t>(slot) * 16u, v);
          }
        }
      }
    }
    if (splits > 1)
      cluster_sync();
    else
      __syncthreads();
    if (warp >= 2 && summed && o < p.F) {
      const int4* in = reinterpret_cast<const int4*>(red) + et % kRows;
      constexpr int kStep = 256 / kRows;  // groups that the warps take at a time
      constexpr int kAhead = kGeglu ? 1 : 2;  // of them per thread, values first and then their stores
      for (int it0 = et / kRows; it0 < mine && (it0 * splits + rank) * 4 < p.T; it0 += kAhead * kStep) {
        float v[kAhead][4];
#pragma unroll
        for (int h = 0; h < kAhead; ++h) {
          const int it = min(it0 + h * kStep, mine - 1), t = min((it * splits + rank) * 4, N - 4);
          int4 a = make_int4(0, 0, 0, 0), b = a;
          for (int src = 0; src < splits; ++src) {
            const int4 x = in[(src * mine + it) * kTileM];
            a = make_int4(a.x + x.x, a.y + x.y, a.z + x.z, a.w + x.w);
            if (kGeglu) {
              const int4 u = in[(src * mine + it) * kTileM + kRows];
              b = make_int4(b.x + u.x, b.y + u.y, b.z + u.z, b.w + u.w);
            }
          }
          const float4 s4 = *reinterpret_cast<const float4*>(sx + t);
          const int av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
          const float sv[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            v[h][q] = fmaf(static_cast<float>(av[q]) * sv[q], ws, bs);
            if (kGeglu)
              v[h][q] = gelu_ex2(v[h][q]) * fmaf(static_cast<float>(bv[q]) * sv[q], wu, bu);
            else
              v[h][q] = activate<ACT>(v[h][q]);
          }
        }
#pragma unroll
        for (int h = 0; h < kAhead; ++h) {
          const int it = it0 + h * kStep, t = (it * splits + rank) * 4;
          const int live = it < mine ? p.T - t : 0;
          Tout* y = static_cast<Tout*>(p.y) + t * p.ldy + o;
#pragma unroll
          for (int q = 0; q < 4; ++q, y += p.ldy)
            if (q < live) put1(y, v[h][q]);
        }
      }
    }
  }
  tc_fence_before();
  // a producer that stopped early waits (bounded) for its copies in flight
  if (warp == 0 && lane == 0)
    for (int i = (issued > stages ? issued - stages : 0); i < issued; ++i)
      mbar_wait(&full[i % stages], (i / stages) & 1, p.status, kDevTimeoutTmaFull);
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

// ------------------------------------------------------- few tokens ---
// Up to 4 tokens: the weights are read once, 16 bytes per lane and load, and
// multiplied on the integer units (4 products per instruction): no tiles, no
// shared-memory round trip, nothing to set up, so a single token's call costs
// little more than the memory's latency (O x K: 3.0 us for 2560 x 2048, 12.1 us or
// 5.5 TB/s for the 67 MB of a 32768 x 2048 GeGLU).  A warp takes two weight rows
// (GeGLU: a gate row and its up row) over a 1/kw part of K; x comes through L1.
constexpr int kFewTokens = 4;
constexpr long kFewSmall = 16 << 20;  // bytes of weights for 3 and 4 tokens
constexpr int kFewThreads = 256;

// (Not the read-only path: under programmatic launch this grid may start before
// the one that writes its operands has ended.)
__device__ __forceinline__ int4 ld_weights(const int8_t* p) {
  int4 v;
  asm volatile("ld.global.L1::no_allocate.v4.s32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ int dot16(const int4& a, const int4& b, int acc) {
  acc = __dp4a(a.x, b.x, acc);
  acc = __dp4a(a.y, b.y, acc);
  acc = __dp4a(a.z, b.z, acc);
  return __dp4a(a.w, b.w, acc);
}

template <int TT, int ACT, typename Tout>
__global__ void __launch_bounds__(kFewThreads) linear_i8_few_kernel(const I8Params p) {
  constexpr bool kGeglu = ACT == kActGeglu;
  constexpr int kUnroll = TT <= 2 ? 4 : 2;
  __shared__ int part[8][2 * TT];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kw = p.splits;                        // warps that share a pair of rows
  const int grp = (blockIdx.x * 8 + warp) / kw;   // pair of rows
  const int part_k = warp % kw;
  const int c0 = kGeglu ? grp : 2 * grp;          // output column
  const int r0 = c0, r1 = kGeglu ? p.F + grp : min(2 * grp + 1, p.O - 1);
  const bool live = c0 < p.F;
  int acc[2][TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) acc[0][t] = acc[1][t] = 0;
  if (live) {
    const int8_t* w0 = p.w + static_cast<long>(r0) * p.ldw;
    const int8_t* w1 = p.w + static_cast<long>(r1) * p.ldw;
    const int vecs = p.K / 16;
    const int v0 = static_cast<int>(static_cast<long>(part_k) * vecs / kw), v1 = static_cast<int>(static_cast<long>(part_k + 1) * vecs / kw);
    for (int v = v0 + lane; v < v1; v += 32 * kUnroll) {
      int4 a[kUnroll], b[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        a[i] = b[i] = make_int4(0, 0, 0, 0);
        if (v + 32 * i < v1) {
          a[i] = ld_weights(w0 + static_cast<long>(v + 32 * i) * 16);
          b[i] = ld_weights(w1 + static_cast<long>(v + 32 * i) * 16);
        }
      }
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        if (v + 32 * i < v1) {
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            if (TT > 1 && t >= p.T) break;
            const int4 x = reinterpret_cast<const int4*>(p.x + t * p.ldx)[v + 32 * i];
            acc[0][t] = dot16(a[i], x, acc[0][t]);
            acc[1][t] = dot16(b[i], x, acc[1][t]);
          }
        }
      }
    }
    // the last K % 16 elements, one per lane: nothing past a row's end is read
    const int k = vecs * 16 + lane;
    if (part_k == kw - 1 && k < p.K) {
      const int a = w0[k], b = w1[k];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        if (t < p.T) {
          const int x = p.x[t * p.ldx + k];
          acc[0][t] += a * x;
          acc[1][t] += b * x;
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TT; ++t) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int s = __reduce_add_sync(0xffffffffu, acc[r][t]);
      if (lane == 0) part[warp][2 * t + r] = s;
    }
  }
  if (kw > 1)
    __syncthreads();
  else
    __syncwarp();
  // the outputs of this warp's rows: the first warp of those that share them
  if (part_k == 0 && live && lane < (kGeglu ? TT : 2 * TT)) {
    const int t = kGeglu ? lane : lane >> 1, r = kGeglu ? 0 : lane & 1;
    const int o = c0 + r;
    if (t < p.T && o < p.F) {
      int s0 = 0, s1 = 0;
      for (int q = 0; q < kw; ++q) {
        s0 += part[warp + q][2 * t + r];
        if (kGeglu) s1 += part[warp + q][2 * t + 1];
      }
      const float sx = p.x_scale[t];
      float v = fmaf(static_cast<float>(s0) * sx, p.w_scale[o], p.bias ? p.bias[o] : 0.f);
      if (kGeglu)
        v = gelu_ex2(v) * fmaf(static_cast<float>(s1) * sx, p.w_scale[p.F + o], p.bias ? p.bias[p.F + o] : 0.f);
      else
        v = activate<ACT>(v);
      put1(static_cast<Tout*>(p.y) + t * p.ldy + o, v);
    }
  }
}

// ------------------------------------------------------------ host side ---
bool al(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int out_cols(const rfx_linear_i8_desc& d) { return d.epilogue == RFX_EPI_GEGLU ? d.O / 2 : d.O; }

template <int ACT>
const void* few_ptr(int out_dtype, int T) {
  if (out_dtype == kDtypeBF16) {
    if (T == 1) return reinterpret_cast<const void*>(linear_i8_few_kernel<1, ACT, __nv_bfloat16>);
    if (T == 2) return reinterpret_cast<const void*>(linear_i8_few_kernel<2, ACT, __nv_bfloat16>);
    return reinterpret_cast<const void*>(linear_i8_few_kernel<4, ACT, __nv_bfloat16>);
  }
  if (T == 1) return reinterpret_cast<const void*>(linear_i8_few_kernel<1, ACT, float>);
  if (T == 2) return reinterpret_cast<const void*>(linear_i8_few_kernel<2, ACT, float>);
  return reinterpret_cast<const void*>(linear_i8_few_kernel<4, ACT, float>);
}
template <int ACT>
const void* i8_ptr(int out_dtype, int form, int T) {
  if (form == kI8Few) return few_ptr<ACT>(out_dtype, T);
  if (form == kI8Side)
    return out_dtype == kDtypeBF16 ? reinterpret_cast<const void*>(linear_i8_side_kernel<ACT, __nv_bfloat16>)
                                   : reinterpret_cast<const void*>(linear_i8_side_kernel<ACT, float>);
  return out_dtype == kDtypeBF16 ? reinterpret_cast<const void*>(linear_i8_pair_kernel<ACT, __nv_bfloat16>)
                                 : reinterpret_cast<const void*>(linear_i8_pair_kernel<ACT, float>);
}
const void* i8_kernel(int epilogue, int out_dtype, int form, int T) {
  switch (epilogue) {
    case RFX_EPI_STORE: return i8_ptr<kActNone>(out_dtype, form, T);
    case RFX_EPI_SILU: return i8_ptr<kActSilu>(out_dtype, form, T);
    case RFX_EPI_GELU: return i8_ptr<kActGelu>(out_dtype, form, T);
    case RFX_EPI_GEGLU: return i8_ptr<kActGeglu>(out_dtype, form, T);
  }
  return nullptr;
}

// Tiles with the weights on the M side: the split of K and the CTAs meant to
// share an SM (fewer stages each) that finish soonest by this model, in us,
// fitted to measured times of seven projections at 8 to 128 tokens.  A K step
// takes an SM 0.215 + 0.00035 per token; the weights come at 6.2 TB/s at best; a
// ring that does not hold a CTA's whole part costs 0.5 and up to 1.1 per turn;
// joining a split 0.8 + 0.006 per token + 0.1 per part; a further round of CTAs
// 1.4 where each has the SM to itself, else 0.3; and a CTA that leaves room lets
// the next launch set up beside it.
void plan_side(const rfx_linear_i8_desc& d, int nsm, int k_steps, LinearI8Plan* c) {
  const bool geglu = d.epilogue == RFX_EPI_GEGLU;
  const void* fn = i8_kernel(d.epilogue, d.out_dtype, kI8Side, d.T);
  const int rows = geglu ? kTileM / 2 : kTileM;
  const int N = (d.T + 15) / 16 * 16;
  const long tiles = (out_cols(d) - 1) / rows + 1;
  const double step = 0.215 + 0.00035 * d.T, memory = static_cast<double>(d.O) * d.K / 6.2e6;
  double best = 0;
  for (int s = 1; s <= std::min(kSideMaxSplits, k_steps); s *= 2) {
    const int n = (k_steps + s - 1) / s;
    const long ctas = tiles * s;
    if (s > 1 && ctas > 2l * nsm) break;
    for (int share = 1; share <= 3; ++share) {
      const int room = share == 1 ? kSmemMax : 228 * 1024 / share - 1024;
      int stages = std::min(kSideMaxStages, n);
      while (stages > 1 && side_smem(N, s, geglu, stages) > room) --stages;
      if (side_smem(N, s, geglu, stages) > room || stages < std::min(n, 2)) continue;
      const long slots = s == 1 ? static_cast<long>(nsm) * share : static_cast<long>(max_active_clusters(fn, kSideThreads, kSmemMax, s)) * s * share;
      if (slots <= 0) continue;
      const long waves = (ctas + slots - 1) / slots;
      const double even = static_cast<double>(ctas) / nsm;
      const double per_sm = share == 1 ? std::max<double>(waves, std::ceil(even)) : waves == 1 ? std::ceil(even) : even;
      const double turns = static_cast<double>(n) / stages - 1.0;  // of the ring, after the first
      double cost = std::max({per_sm * n * step, waves * turns * 1.1, memory}) + (turns > 0 ? 0.5 + 0.3 * turns : 0.0);
      cost += (waves - 1) * (share == 1 ? 1.4 : 0.3) + (s > 1 ? 0.8 + 0.006 * d.T + 0.1 * s : 0.0);
      cost -= 0.15 * (share - 1);
      if (c->form == kI8Side && cost >= best) continue;
      best = cost;
      c->form = kI8Side;
      c->splits = s;
      c->stages = stages;
    }
  }
  c->nt = N;
  c->clusters = static_cast<int>(tiles);
}

// How a call is cut up.
//
// Up to 4 tokens go to the integer units, unless the layer is wide and short
// (16 output rows and more per column of K: a warp's part is then too small) or,
// with 3 or 4 tokens, large (the products bound them).  Measured there and with
// the weights on the M side, O x K: 1 token of 2560 x 1024 2.8 and 3.1 us, of 8000 x
// 1024 3.3 and 4.8, of 21953 x 256 5.8 and 3.8; 4 tokens of 8000 x 1024 4.7 and
// 4.8, of 2048 x 16384 12.3 and 10.1.
//
// The weights lie on the M side up to 128 tokens.  Measured there and as pair
// tiles, O x K: 50 tokens of 8192 x 1024 GeGLU 6.5 and 7.5 us, of 1024 x 4096 5.5 and
// 9.4, of 32768 x 2048 GeGLU 15.4 and 19.7; 96 tokens of 4304 x 1152 GELU 6.0 and 6.9;
// 128 of 20000 x 800 8.5 and 10.2, of 2560 x 1024 5.6 and 5.6, of 8192 x 1024 GeGLU
// 7.7 and 7.5.
//
// Pair tiles, above 128 tokens: the width N and the split of K that finish
// soonest by this model, whose figures are fitted to measured times of these
// projections at 16 to 4096 tokens.  A K step takes 150 ns + 0.45 ns per weight row while the
// copies into the SM bound it, 1.12 ns per weight row once the MMAs do, and
// 1.17 times that over several rounds of tiles, each at least its epilogue's
// 1.7 us + 10.5 ns per weight row (14.5 with GeGLU, 18.5 with an activation, 4
// more for fp32 and 16 more where output rows are off the 16-byte grid); the
// last epilogue is not hidden, and where K is split adding up costs 0.9 us + 0.4
// us per split.  (An epilogue's fixed part measures 0.5 us; counted as that, the
// model takes narrower tiles that are up to 18 % slower.  3200 x 21952 x 72: 73 us
// in tiles of 64 rows, 52 in tiles of 256.)
LinearI8Plan plan_i8(const rfx_linear_i8_desc& d, int nsm) {
  LinearI8Plan c{};
  const int div = d.epilogue == RFX_EPI_GEGLU ? 2 : 1;  // weight rows per output column
  const int F = out_cols(d);
  if (d.T <= kFewTokens && d.O <= 16l * d.K && (d.T <= 2 || static_cast<long>(d.O) * d.K <= kFewSmall)) {
    c.form = kI8Few;
    // warps per pair of rows: enough of them for 16 per SM, with at least one
    // 512-byte load per row each
    const int pairs = d.epilogue == RFX_EPI_GEGLU ? F : (F + 1) / 2;
    c.splits = 1;
    while (c.splits < 8 && static_cast<long>(pairs) * c.splits < 16l * nsm && d.K >= 1024 * c.splits) c.splits *= 2;
    c.clusters = static_cast<int>((static_cast<long>(pairs) * c.splits + 7) / 8);
    return c;
  }
  const int k_steps = (d.K + kStepK - 1) / kStepK;
  if (d.T <= kSideTokens) {
    plan_side(d, nsm, k_steps, &c);
    return c;
  }
  const int m = (d.T - 1) / (2 * kTileM) + 1;
  const int step = 32 * div;  // tiles of whole 64-byte pieces of output rows
  const void* fn = i8_kernel(d.epilogue, d.out_dtype, kI8Pair, d.T);
  auto tiles_of = [&](int cols, int nt) { return static_cast<int>((static_cast<long>(cols) * div + nt - 1) / nt); };
  const int esz = d.out_dtype == kDtypeBF16 ? 2 : 4;
  double row_ns = d.epilogue == RFX_EPI_STORE ? 10.5 : d.epilogue == RFX_EPI_GEGLU ? 14.5 : 18.5;
  if (esz == 4) row_ns += 4.0;
  if (!al(d.y, 16) || (d.ldy * esz) % 16 != 0) row_ns += 16.0 / div;
  auto sum_ns = [&](int nt, int s) { return (k_steps + s - 1) / s * std::max(150.0 + 0.45 * nt, 1.12 * nt); };
  auto tile_ns = [&](int nt, int rounds) { return rounds > 1 ? std::max(sum_ns(nt, 1), 1700.0 + row_ns * nt) : sum_ns(nt, 1); };
  double best = 0;
  for (int s = 1; s <= std::min(kMaxSplits, k_steps); ++s) {
    // clusters of 2s CTAs that are resident at once (GPCs hold whole clusters)
    int slots = max_active_clusters(fn, kPairThreads, kPairSmem, 2 * s);
    if (slots <= 0) {
      if (s > 1) break;
      slots = std::max(1, nsm / 2);
    }
    for (int nt = 64; nt <= 256; nt += step) {
      const int n = tiles_of(F, nt);
      const long tiles = static_cast<long>(m) * n;
      const long rounds = (tiles + slots - 1) / slots;
      if (s > 1 && rounds > 1) continue;
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
      // several rounds: every SM at work
      const double all = rounds > 1 ? 1.17 * tiles / slots * tile_ns(nt, 2) : 0.0;
      if (s > 1) {
        consider(sum_ns(nt, s) + 10.0 * nt + 900.0 + 400.0 * s, n, nt, 0);
        continue;
      }
      consider(std::max(rounds * tile_ns(nt, static_cast<int>(rounds)), all) + 10.0 * nt, n, nt, 0);
      if (rounds < 2) continue;
      // the full rounds at this width, the rest in narrower tiles
      const int n_a = static_cast<int>((rounds - 1) * slots / m);
      if (n_a < 1 || n_a >= n) continue;
      for (int nt2 = 64; nt2 < nt; nt2 += step) {
        const int n_b = tiles_of(F - n_a * (nt / div), nt2);
        const long ua = static_cast<long>(n_a) * m, ub = static_cast<long>(n_b) * m;
        // the tiles go round the slots: the busiest slot's time
        const double ta = tile_ns(nt, 2), tb = tile_ns(nt2, 2);
        const long qa = ua / slots, ra = ua % slots, first = slots - ra;  // `first` slots have one wide tile less
        double t;
        if (ub <= first) {
          t = std::max(qa * ta + tb, (qa + (ra ? 1 : 0)) * ta);
        } else {
          const long qb = (ub - first) / slots, rb = (ub - first) % slots;
          t = std::max(ra ? (qa + 1) * ta + (qb + (rb ? 1 : 0)) * tb : 0.0, qa * ta + (1 + qb + (rb > ra ? 1 : 0)) * tb);
        }
        // (a gain of a hundredth by this model is none by the clock)
        consider(1.01 * (std::max(t, 1.17 * (ua * ta + ub * tb) / slots) + 10.0 * nt2), n_a, nt2, n_b);
      }
    }
  }
  c.m_tiles = m;
  c.stages = std::min(kPairMaxStages, kPairRing / ((kTileM + c.nt / 2) * kStepK));
  return c;
}

}  // namespace

int validate_linear_i8(const rfx_linear_i8_desc& d) {
  if (d.T < 0 || d.T > kMaxRows || d.O < 1 || d.O > kMaxRows || d.K < 1 || d.K > kMaxK)
    return set_error(RFX_E_INVAL, "rfx_linear_i8: need 0<=T<=2^30, 1<=O<=2^30, 1<=K<=%d (T=%d O=%d K=%d)", kMaxK, d.T,
                     d.O, d.K);
  if (d.epilogue != RFX_EPI_STORE && d.epilogue != RFX_EPI_SILU && d.epilogue != RFX_EPI_GELU &&
      d.epilogue != RFX_EPI_GEGLU)
    return set_error(RFX_E_INVAL, "rfx_linear_i8: epilogue must be STORE, SILU, GELU or GEGLU");
  if (d.epilogue == RFX_EPI_GEGLU && d.O % 2)
    return set_error(RFX_E_INVAL, "rfx_linear_i8: GEGLU needs an even O (gate rows, then as many up rows)");
  if (d.out_dtype != kDtypeBF16 && d.out_dtype != kDtypeF32)
    return set_error(RFX_E_INVAL, "rfx_linear_i8: output dtype must be bf16 or f32");
  if (d.T == 0) return RFX_OK;
  if (!d.x || !d.w || !d.x_scale || !d.w_scale || !d.y)
    return set_error(RFX_E_INVAL, "rfx_linear_i8: null pointer");
  if (!al(d.x, 16) || !al(d.w, 16) || d.ldx < d.K || d.ldw < d.K || d.ldx % 16 || d.ldw % 16)
    return set_error(RFX_E_INVAL,
                     "rfx_linear_i8: int8 rows must begin on 16-byte boundaries (aligned x and w, ldx and ldw >= K and "
                     "multiples of 16)");
  if (d.ldy < out_cols(d) || !al(d.y, d.out_dtype == kDtypeBF16 ? 2 : 4) || !al(d.x_scale, 4) || !al(d.w_scale, 4) ||
      !al(d.bias, 4))
    return set_error(RFX_E_INVAL, "rfx_linear_i8: ldy below the output's columns, or a misaligned pointer");
  const long esz = d.out_dtype == kDtypeBF16 ? 2 : 4;
  const Rows y{d.y, d.T, d.ldy * esz, out_cols(d) * esz};
  if (rows_shared(y, {d.x, d.T, d.ldx, d.K}) || rows_shared(y, {d.w, d.O, d.ldw, d.K}) ||
      rows_shared(y, {d.x_scale, 1, 0, d.T * 4l}) || rows_shared(y, {d.w_scale, 1, 0, d.O * 4l}) ||
      rows_shared(y, {d.bias, 1, 0, d.O * 4l}))
    return set_error(RFX_E_INVAL, "rfx_linear_i8: y shares memory with an input");
  if ((static_cast<long>(d.T) / kTileM + 1) * (d.O / 32 + 1) > 0x7fffffffL / 8)
    return set_error(RFX_E_INVAL, "rfx_linear_i8: too many output tiles (T=%d O=%d)", d.T, d.O);
  return RFX_OK;
}

int build_linear_i8_maps(const rfx_linear_i8_desc& d, LinearI8Maps* maps) {
  int rc = validate_linear_i8(d);
  if (rc || d.T == 0) return rc;
  int nsm = 148;
  rfx_num_sms(&nsm);
  maps->plan = plan_i8(d, nsm);
  const LinearI8Plan& c = maps->plan;
  if (c.form == kI8Few) return RFX_OK;
  rc = make_tmap_2d(&maps->x, d.x, 1, d.K, d.T, d.ldx, kStepK, c.form == kI8Side ? d.T : kTileM, true);
  if (rc) return rc;
  if (c.form == kI8Side)
    return make_tmap_2d(&maps->w, d.w, 1, d.K, d.O, d.ldw, kStepK, d.epilogue == RFX_EPI_GEGLU ? kTileM / 2 : kTileM, true);
  rc = make_tmap_2d(&maps->w, d.w, 1, d.K, d.O, d.ldw, kStepK, c.nt / 2, true);
  if (rc) return rc;
  maps->w2 = maps->w;
  if (c.n_tiles2 > 0) {
    rc = make_tmap_2d(&maps->w2, d.w, 1, d.K, d.O, d.ldw, kStepK, c.nt2 / 2, true);
    if (rc) return rc;
  }
  const int esz = d.out_dtype == kDtypeBF16 ? 2 : 4;
  maps->y = maps->w;  // not used where y's rows are not 16-byte aligned
  if (al(d.y, 16) && (d.ldy * esz) % 16 == 0)
    rc = make_tmap_2d_swizzle(&maps->y, d.y, esz, out_cols(d), d.T, d.ldy * esz, 64 / esz, 32, 64);
  return rc;
}

int launch_linear_i8(const rfx_linear_i8_desc& d, const LinearI8Maps& maps, cudaStream_t stream, bool pdl) {
  if (d.T == 0) return RFX_OK;
  const LinearI8Plan& c = maps.plan;
  const void* fn = i8_kernel(d.epilogue, d.out_dtype, c.form, d.T);
  if (c.form != kI8Few) {
    const int rc = ensure_smem_attr(fn, kSmemMax);
    if (rc) return rc;
  }
  I8Params p{};
  p.T = d.T;
  p.O = d.O;
  p.K = d.K;
  p.F = out_cols(d);
  p.m_tiles = c.m_tiles;
  p.k_steps = (d.K + kStepK - 1) / kStepK;
  p.splits = c.splits;
  p.n_tile = c.nt;
  p.n_tail = c.nt2;
  p.cols_a = c.n_tiles;
  p.units = c.m_tiles * (c.n_tiles + c.n_tiles2);
  p.stages = c.stages;
  p.x = static_cast<const int8_t*>(d.x);
  p.ldx = d.ldx;
  p.w = static_cast<const int8_t*>(d.w);
  p.ldw = d.ldw;
  p.x_scale = d.x_scale;
  p.w_scale = d.w_scale;
  p.bias = d.bias;
  p.y = d.y;
  p.ldy = d.ldy;
  p.status = device_status_ptr();
  if (c.form == kI8Few) return launch_kernel(fn, dim3(c.clusters), dim3(kFewThreads), 0, stream, pdl, 1, p);
  CUtensorMap x = maps.x, w = maps.w, w2 = maps.w2, y = maps.y;
  if (c.form == kI8Side)
    return launch_kernel(fn, dim3(c.clusters * c.splits), dim3(kSideThreads),
                         static_cast<size_t>(side_smem(c.nt, c.splits, d.epilogue == RFX_EPI_GEGLU, c.stages)), stream, pdl,
                         c.splits, x, w, p);
  return launch_kernel(fn, dim3(2 * c.splits * c.clusters), dim3(kPairThreads), static_cast<size_t>(kPairSmem), stream,
                       pdl, 2 * c.splits, x, w, w2, y, p);
}

}  // namespace rfx

extern "C" int rfx_linear_i8(const rfx_linear_i8_desc* d, void* stream) {
  using namespace rfx;
  if (!d) return set_error(RFX_E_INVAL, "rfx_linear_i8: null descriptor");
  LinearI8Maps maps;
  const int rc = build_linear_i8_maps(*d, &maps);
  if (rc) return rc;
  return launch_linear_i8(*d, maps, static_cast<cudaStream_t>(stream), pdl_enabled());
}
