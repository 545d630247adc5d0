// The tensor-core products of the linear cross entropy: one persistent kernel
// with four epilogues.
//
//   kScore  z  = h w^T    -> per row and 128 columns (max, sum exp), target score
//   kDz     z  = h w^T    -> dz = c (exp(z - lse) - onehot), stored
//   kDh     dh = dz w     -> float32 partial sums, per split of the vocabulary
//   kDw     dw = dz^T h   -> the result, scaled and rounded once
//
// A cluster of two CTAs (two SMs of one TPC) makes 256 x 256 tiles with
// tcgen05.mma.cta_group::2: each CTA stages 128 rows of A and 128 of B by TMA,
// 32 KB for a contraction step of 64, so a tile reads half the shared memory
// and half the L2 bytes per product that two single-SM tiles would; those
// bytes, not the tensor pipe, would otherwise set the pace (a 128 x 256 tile
// needs 96 bytes a cycle from L2 per SM).  The accumulator (256 columns of
// TMEM in each CTA) is double-buffered: eight warps read one while the next
// tile is being multiplied.
//
// 16-bit dz of few rows that count (FEW_ROWS) is held as two planes, value and
// rounding error: with one row, or a few, the rounding of one dominant score's
// gradient is the whole gradient's error (1.8 times that of its own final
// rounding); over many rows it averages (1.0 to 1.4 times).  The second plane
// lies HALF rows below the first, in a part of dz's first tile of rows that so
// few leave unused; how many count is known on the device only.
//
// float32 operands come as three bfloat16 planes (x = hi + mid + lo exactly,
// each rounded to nearest, so mid is at most 2^-8 and lo 2^-17 of x's power of
// two) and the contraction runs over six of the nine plane pairs, smallest
// products first; what is left out, 2 mid lo + lo lo, is at most 2^-24 of a
// product and has either sign.  (Cut toward zero instead, the planes left out
// up to 2^-21, always of the product's sign: a bias.)
//
// Measured (bfloat16, one launch alone): 8192 x 32768 x 2048 scores 723 us (1520
// TFLOP/s), dz 749, dh 736, dw 732 us; tensor pipe about 80 % busy.  Bound by the
// tensor cores (by the power cap in a long run) from a width of about 512 on;
// below it by the exponentials of the scores' epilogue and by dz in HBM (8192 x
// 32768 x 64: scores 130 us, of which 60 the exponentials; dz 147, dh 96, dw 97,
// of which 82 each its 537 MB).  Taking the maximum off each score before the
// factor log2(e), instead of one fused step, costs 4 % of those 130 us.
#pragma once

#include "common.cuh"
#include "lm_embed.cuh"
#include "lm_xent.cuh"
#include "tc_common.cuh"

namespace theria {
namespace xent {

enum Epi { kScore = 0, kDz = 1, kDh = 2, kDw = 3 };

constexpr int BM = TILE_ROWS, BN = 256, BK = K_BLOCK;  // of a CTA pair
constexpr int HALF = 128;                   // rows of A and of B per CTA
constexpr int SUB = 128;                    // columns per score partial
static_assert(FEW_ROWS <= BK && BK <= HALF, "both planes of few rows in one tile");
constexpr int STAGES = 6;
constexpr int OPERAND = HALF * BK * 2;      // bytes of one operand's stage
constexpr int EPI_WARPS = 8;
constexpr int STAGE_OUT = 4096;             // a warp's stage of results: 32 rows of 128 bytes
constexpr int TC_THREADS = 128 + EPI_WARPS * 32;
constexpr uint32_t ACC_COLS = 256;
constexpr float LOG2E = 1.4426950408889634f;
constexpr uint32_t POLLS = 1u << 20;  // bound of one wait; a poll suspends the thread for a while

struct TcArgs {
  const int* n_live;
  int V, D;
  int c0, Cn;           // piece of the vocabulary (kDz, kDh, kDw): start, columns
  int plane_a, plane_b; // elements between planes of one row
  const Splits* plan;   // kDh; kDw where it is split (else NULL)
  int add;              // kDh: add to what the partials hold (a later piece)
  int rows;             // all rows; if every one counts, A (B for kDw) is h itself, unpacked
  int h_plain;          // ... where h can be read as it is
  const int* tgt;       // kScore, kDz
  float2* part;         // kScore: [row][sub_tiles]
  int sub_tiles;
  float* zt;
  const float4* row;    // kDz: see RowArgs
  int ld_dz;            // kDz: dz is [row][planes][ld_dz]
  int ld_acc;           // with a plan: [split][plan->acc_rows][ld_acc] partial sums
  void* out;            // kDw: [V][D], where it cannot be stored by TMA
  const float* post;    // kDw: the factor of the result
};

// Planes (of a, of b) of the i-th of six pairs, smallest products first.
__device__ __forceinline__ int pair_a(int i) { return (0x001102 >> (4 * i)) & 15; }
__device__ __forceinline__ int pair_b(int i) { return (0x010120 >> (4 * i)) & 15; }

// Arrives on a barrier of the pair.  What it orders is the reads of TMEM before
// it (tcgen05 fences); at cluster scope it would wait for this thread's global
// stores as well.
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// A warp's staged 32 x 128-byte tile to (x, y) of `map`, or added to it
// (float32); one bulk group of this thread.
__device__ __forceinline__ void store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];\n\t"
      "cp.async.bulk.commit_group;" ::"l"(reinterpret_cast<uint64_t>(map)),
      "r"(tc::smem_u32(src)), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void add_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile(
      "cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}],"
      " [%1];\n\t"
      "cp.async.bulk.commit_group;" ::"l"(reinterpret_cast<uint64_t>(map)),
      "r"(tc::smem_u32(src)), "r"(x), "r"(y)
      : "memory");
}
// Box at (x, y) of `map` into this CTA's shared memory; the bytes count on a
// barrier that may be the pair's other CTA's.
__device__ __forceinline__ void load_2d(void* dst, const CUtensorMap* map, uint32_t bar, int x,
                                        int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile"
      ".mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(tc::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on this barrier of both CTAs when all earlier products are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(tc::smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

struct TcSmem {
  static constexpr int oA = 0;
  static constexpr int oB = STAGES * OPERAND;
  static constexpr int oOut = 2 * STAGES * OPERAND;
  static constexpr int oBar = oOut + EPI_WARPS * STAGE_OUT;  // full, empty, acc_full, acc_empty
  static constexpr int kBars = 2 * STAGES + 4;
  static constexpr int oTmem = oBar + kBars * 8;
  static constexpr int oAbort = oTmem + 4;
  static constexpr int kBytes = oAbort + 4;
  static constexpr int kAlloc = kBytes + 1024;  // the base is aligned to 1024
  static_assert(kAlloc <= 232448, "shared memory of one CTA");
};

// What one cluster works on next.
struct Unit {
  int m0, n0;   // tile origin
  int kb0, kbs; // k blocks of each plane pair
  int split;
};

template <int EPI>
struct Sched {
  int mt, nt, kb, units, splits, split_kb, acc_rows;
  __device__ explicit Sched(const TcArgs& a) {
    const int live = *a.n_live;
    const int rows = (live + BM - 1) / BM > 0 ? (live + BM - 1) / BM : 1;
    splits = 1;
    acc_rows = 0;
    if (EPI == kScore || EPI == kDz) {
      mt = rows;
      nt = ((EPI == kScore ? a.V : a.Cn) + BN - 1) / BN;
      kb = (a.D + BK - 1) / BK;
    } else if (EPI == kDh) {
      mt = rows;
      nt = (a.D + BN - 1) / BN;
      kb = (a.Cn + BK - 1) / BK;
    } else {
      mt = (a.Cn + BM - 1) / BM;
      nt = (a.D + BN - 1) / BN;
      kb = live > 0 ? (live + BK - 1) / BK : 1;
    }
    split_kb = kb;
    if (EPI == kDh || (EPI == kDw && a.plan)) {
      split_kb = a.plan->split_kb;
      acc_rows = a.plan->acc_rows;
      splits = (kb + split_kb - 1) / split_kb;
    }
    units = mt * nt * splits;
  }
  // Tiles in groups of 8 rows of tiles, so that the clusters at work at one
  // time share both operands' tiles in L2.
  __device__ Unit at(int u) const {
    Unit r;
    r.split = u / (mt * nt);
    const int t = u - r.split * (mt * nt);
    const int g = t / (8 * nt), in = t - g * 8 * nt;
    const int gm = mt - g * 8 < 8 ? mt - g * 8 : 8;
    r.m0 = (g * 8 + in % gm) * BM;
    r.n0 = (in / gm) * BN;
    r.kb0 = r.split * split_kb;
    r.kbs = kb - r.kb0 < split_kb ? kb - r.kb0 : split_kb;
    return r;
  }
};

// 32 consecutive values of one row: into a 128-byte row of a warp's stage, as
// its 16-byte chunks c0 .. (128-byte swizzle).
template <typename O>
__device__ __forceinline__ void stage32(uint32_t row, int lane, const float (&v)[32], int c0) {
  if constexpr (sizeof(O) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      tc::st_shared_v4(row + ((i ^ (lane & 7)) << 4), __float_as_uint(v[4 * i]),
                       __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                       __float_as_uint(v[4 * i + 3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* e = v + 8 * i;
      tc::st_shared_v4(row + (((c0 + i) ^ (lane & 7)) << 4), tc::pack2<O>(e[0], e[1]),
                       tc::pack2<O>(e[2], e[3]), tc::pack2<O>(e[4], e[5]),
                       tc::pack2<O>(e[6], e[7]));
    }
  }
}

// x = hi + mid + lo, each the nearest 8 bits of what the ones before leave; hi
// is cut where the nearest would be infinite.
__device__ __forceinline__ void split3(float x, __nv_bfloat16 (&p)[3]) {
  p[0] = __float2bfloat16_rn(x);
  if (isinf(__bfloat162float(p[0]))) p[0] = __float2bfloat16_rz(x);
  const float r1 = isfinite(x) ? x - __bfloat162float(p[0]) : 0.f;
  p[1] = __float2bfloat16_rn(r1);
  p[2] = __float2bfloat16_rn(r1 - __bfloat162float(p[1]));
}

// k blocks that one accumulation in TMEM runs over where sums of chunks are
// added in registers.  The tensor core cuts each sum to the accumulator's
// precision instead of rounding it, which over a long contraction leaves a bias
// of about one unit in the last place per step: float32 results (4 blocks: dw
// over 2048 rows 2.6e-6 -> 4e-7), and the float32 loss of 16-bit operands wider
// than DEEP over few words (16 blocks; 100 words, width 4000: 1.3e-6 -> 3e-7).
// Over many words the scores' sums are larger and the same bias is less of them
// (131,072 words, width 4096: 4.8e-7), and the second read of the accumulators
// costs up to 8 % under the power cap: not where there are more tiles than
// DEEP_UNITS.  dz's scores of 16-bit operands go without: an error of a score is
// one of its p relative to p, and the target's p - 1 is not made from them.
constexpr int F32_CHUNK = 4, DEEP_CHUNK = 16, DEEP = 1024, DEEP_UNITS = 4 * CLUSTERS;

// T: the operands' type.  O: the type of the user's tensors (float32 with T =
// bfloat16 planes, else T).  CHUNKS: sums of chunks in registers.
template <typename T, typename O, int EPI, bool CHUNKS>
__global__ void __launch_bounds__(TC_THREADS, 1) __cluster_dims__(2, 1, 1)
tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
          const __grid_constant__ CUtensorMap map_h, const __grid_constant__ CUtensorMap map_o,
          const __grid_constant__ CUtensorMap map_p, const __grid_constant__ TcArgs args) {
  constexpr bool A_MN = EPI == kDw, B_MN = EPI == kDh || EPI == kDw;
  constexpr bool F32 = sizeof(O) == 4;
  using L = TcSmem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::oBar);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::oTmem);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::oAbort);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_rank();
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      tc::mbar_init(full + i, 1);
      tc::mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(acc_full + i, 1);
      tc::mbar_init(acc_empty + i, 2 * EPI_WARPS);
    }
    *abort = 0;
    tc::fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     tc::smem_u32(tmem_slot)),
                 "r"(2 * ACC_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::cluster_sync();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_launch();
  grid_wait();
  const Sched<EPI> sched(args);
  const bool few = !F32 && *args.n_live <= FEW_ROWS;  // two planes of dz
  const int pairs = F32 ? 6 : EPI >= kDh && few ? 2 : 1;
  // k blocks per accumulation
  constexpr int CHUNK_KB = F32 ? F32_CHUNK : DEEP_CHUNK;
  const auto chunk = [](const Unit& un) { return CHUNKS ? CHUNK_KB : un.kbs; };

  if (warp == 0 && lane == 0) {
    // ------------------------------------------------ loads, in both CTAs
    const bool plain = args.h_plain && *args.n_live == args.rows;
    const CUtensorMap* pa = EPI <= kDz && plain ? &map_h : &map_a;
    const CUtensorMap* pb = EPI == kDw && plain ? &map_h : &map_b;
    // no division and no mapping in the loop: with four loads a k block it sets
    // the pace (dw of 8192 x 32768 x 2048: 777 -> 720 us)
    const uint32_t bars = tc::map_rank(full, 0);
    uint32_t slot = 0, phase = 1, it = 0;
    bool ok = true;
    for (int u = cluster; ok && u < sched.units; u += clusters) {
      const Unit un = sched.at(u);
      const int m0 = un.m0 + rank * HALF, n0 = un.n0 + rank * HALF;
      for (int kc = 0; ok && kc < un.kbs; kc += chunk(un)) {
        const int k0 = un.kb0 + kc, k1 = k0 + min(chunk(un), un.kbs - kc);
        for (int pr = 0; ok && pr < pairs; ++pr) {
          // 16-bit: dz's second plane first, where it has one
          const int xa = F32 ? pair_a(pr) * args.plane_a : 0;
          const int ya = F32 ? 0 : (pairs - 1 - pr) * HALF;
          const int xb = F32 ? pair_b(pr) * args.plane_b : 0;
          for (int kb = k0; kb < k1; ++kb, ++it) {
            if (!tc::mbar_wait(empty + slot, phase, abort, POLLS)) {
              ok = false;
              break;
            }
            const int k = kb * BK;
            uint8_t* a = smem + L::oA + slot * OPERAND;
            uint8_t* b = smem + L::oB + slot * OPERAND;
            if (rank == 0) tc::mbar_expect_tx(full + slot, 4 * OPERAND);
            const uint32_t bar = bars + slot * 8;
            if constexpr (A_MN) {
              load_2d(a, pa, bar, xa + m0, ya + k);
              load_2d(a + OPERAND / 2, pa, bar, xa + m0 + 64, ya + k);
            } else {
              load_2d(a, pa, bar, xa + k, ya + m0);
            }
            if constexpr (B_MN) {
              const int y = (EPI == kDh ? args.c0 : 0) + k;
              load_2d(b, pb, bar, xb + n0, y);
              load_2d(b + OPERAND / 2, pb, bar, xb + n0 + 64, y);
            } else {
              load_2d(b, pb, bar, xb + k, (EPI == kDz ? args.c0 : 0) + n0);
            }
            if (++slot == STAGES) {
              slot = 0;
              phase ^= 1;
            }
          }
        }
      }
    }
    // every stage used is given back before the CTA may end
    for (int s = 0; ok && s < STAGES && s < (int)it; ++s) {
      const uint32_t last = it - 1 - s;
      ok = tc::mbar_wait(empty + last % STAGES, (last / STAGES) & 1, abort, POLLS);
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // --------------------------------------- products, in the leading CTA
    constexpr uint32_t id = tc::idesc_f16(BM, BN, tc::AbFmt<T>::v, A_MN, B_MN);
    constexpr uint32_t step_a = A_MN ? 2048 : 32, step_b = B_MN ? 2048 : 32;
    const uint64_t da = tc::sw128_desc(tc::smem_u32(smem + L::oA), A_MN ? OPERAND / 2 : 16, 1024);
    const uint64_t db = tc::sw128_desc(tc::smem_u32(smem + L::oB), B_MN ? OPERAND / 2 : 16, 1024);
    uint32_t slot = 0, phase = 0, n_acc = 0;
    bool ok = true;
    for (int u = cluster; ok && u < sched.units; u += clusters) {
      const Unit un = sched.at(u);
      for (int kc = 0; ok && kc < un.kbs; kc += chunk(un), ++n_acc) {
        const uint32_t buf = n_acc & 1;
        if (!tc::mbar_wait(acc_empty + buf, ((n_acc >> 1) & 1) ^ 1, abort, POLLS)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        const uint32_t d = tmem + buf * ACC_COLS;
        const int len = min(chunk(un), un.kbs - kc);
        for (int i = 0, n = pairs * len; i < n; ++i) {
          if (!tc::mbar_wait(full + slot, phase, abort, POLLS)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint64_t a = tc::desc_at(da, slot * OPERAND), b = tc::desc_at(db, slot * OPERAND);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma_pair(d, tc::desc_at(a, k * step_a), tc::desc_at(b, k * step_b), id,
                     (i > 0 || k > 0) ? 1u : 0u);
          commit_pair(empty + slot);
          if (++slot == STAGES) {
            slot = 0;
            phase ^= 1;
          }
        }
        if (ok) commit_pair(acc_full + buf);
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------- epilogue, in both CTAs
    const int quarter = warp & 3, side = (warp - 4) >> 2;  // TMEM lanes, column half
    const int live = *args.n_live;
    const uint32_t src = tmem + ((uint32_t)(quarter * 32) << 16) + side * SUB;
    uint8_t* out = smem + L::oOut + (warp - 4) * STAGE_OUT;
    const uint32_t out_row = tc::smem_u32(out) + lane * 128;
    const float post = EPI == kDw ? *args.post : 1.f;
    // The stage may be written again once the store before has read it.
    auto stage_free = [&] {
      if (lane == 0) tc::bulk_wait_read_all();
      __syncwarp();
    };
    auto stage_full = [&](int x, int y, const CUtensorMap* map) {
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (EPI == kDh && args.add) add_2d(map, out, x, y);
        else store_2d(map, out, x, y);
      }
    };
    // What a unit's row needs, fetched while the unit before is worked on: with
    // short contractions the latency would otherwise be a third of a unit.
    struct Row {
      Unit un;
      int t;
      float l, lo, rs, less;
    };
    auto fetch = [&](int u) {
      Row r;
      r.t = -1;
      r.l = r.lo = r.rs = r.less = 0.f;
      if (u >= sched.units) return r;
      r.un = sched.at(u);
      const int m = r.un.m0 + rank * HALF + quarter * 32 + lane;
      if (EPI <= kDz && m < live) {
        r.t = args.tgt[m] - (EPI == kDz ? args.c0 : 0);
        if (EPI == kDz) {
          const float4 s = args.row[m];
          r.l = s.x;
          r.lo = s.y;
          r.rs = s.z;
          r.less = s.w;
        }
      }
      return r;
    };
    uint32_t n_acc = 0;
    bool ok = true;
    Row next = fetch(cluster);
    for (int u = cluster; ok && u < sched.units; u += clusters) {
      const Unit un = next.un;
      const int t = next.t;
      const float l = next.l, lo = next.lo, rs = next.rs, less = next.less;
      const float base = l * LOG2E;
      const float rs_p = rs * tc::ex2(-fmaf(lo, LOG2E, fmaf(l, LOG2E, -base)));
      next = fetch(u + clusters);
      const int m_warp = un.m0 + rank * HALF + quarter * 32, m = m_warp + lane;
      const int n0 = un.n0 + side * SUB;
      float top = -INFINITY, sum = 0.f;

      // Rows past those that count: nothing of them is kept, but dz is zero up
      // to the end of a k block of dw's contraction over the rows.
      const bool idle = EPI == kDz ? m_warp >= (live > 0 ? (live + BK - 1) / BK * BK : BK)
                                   : EPI != kDw && m_warp >= live;

      // columns n .. n + 31 of this thread's row; c: their place in the half
      auto take = [&](float (&v)[32], int c) {
        const int n = n0 + c;
        if constexpr (EPI == kScore) {
          const int valid = args.V - n;
          if (valid <= 0) return;
          if (valid < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i >= valid) v[i] = -INFINITY;
          }
          if (t >= n && t < n + 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (n + i == t) args.zt[m] = v[i];
          }
          // four chains of three-input maxima, four sums in two pairs
          float top4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
          for (int i = 4; i < 28; i += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) top4[k] = tc::max3(top4[k], v[i + k], v[i + k + 4]);
#pragma unroll
          for (int k = 0; k < 4; ++k) top4[k] = fmaxf(top4[k], v[28 + k]);
          const float now = fmaxf(tc::max3(top4[0], top4[1], top4[2]), fmaxf(top4[3], top));
          // The difference first: the maximum's own term is exactly 1 then, and the
          // others' errors are relative to their distance, not to their size.
          const float ref = now == -INFINITY ? 0.f : now;
          float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float e0, e1, e2, e3;
            tc::add2(e0, e1, v[i], v[i + 1], -ref, -ref);
            tc::add2(e2, e3, v[i + 2], v[i + 3], -ref, -ref);
            tc::mul2(e0, e1, e0, e1, LOG2E, LOG2E);
            tc::mul2(e2, e3, e2, e3, LOG2E, LOG2E);
            tc::add2(s0, s1, s0, s1, tc::ex2(e0), tc::ex2(e1));
            tc::add2(s2, s3, s2, s3, tc::ex2(e2), tc::ex2(e3));
          }
          sum = fmaf(sum, tc::ex2((top - ref) * LOG2E), (s0 + s1) + (s2 + s3));
          top = now;
        } else if constexpr (EPI == kDz) {
          // Rows that do not count are zeros of h: their scores are 0, or NaN
          // beside a weight that is not finite; their dz is 0.
          if constexpr (F32) {
            // lse is l + lo; z - l is exact near the maximum
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = expf((v[i] - l) - lo) * rs;
          } else {
            // z log2(e) - base in one step, rounded once; what base leaves of lse
            // log2(e) is a factor of the row, in rs_p
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float e0, e1;
              tc::fma2(e0, e1, v[i], v[i + 1], LOG2E, LOG2E, -base, -base);
              tc::mul2(v[i], v[i + 1], tc::ex2(e0), tc::ex2(e1), rs_p, rs_p);
            }
          }
          if (t >= n && t < n + 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (n + i == t) v[i] = less;
          }
          const int valid = m < live ? args.Cn - n : 0;
          if (valid < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i >= valid) v[i] = 0.f;
          }
          if (F32 || few) {
            // 32 columns of each plane in turn, in rows of 64 bytes; |dz| <= |rs|, and
            // the nearest of the largest float32 numbers would be infinite
            const bool huge = F32 && fabsf(rs) > 1e38f;
#pragma unroll
            for (int pl = 0; pl < (F32 ? 3 : 2); ++pl) {
              uint32_t w[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float x, y;
                w[i] = tc::pack2<T>(v[2 * i], v[2 * i + 1]);
                if (F32 && huge && pl == 0) {
                  const __nv_bfloat162 q = __halves2bfloat162(__float2bfloat16_rz(v[2 * i]),
                                                              __float2bfloat16_rz(v[2 * i + 1]));
                  w[i] = *reinterpret_cast<const uint32_t*>(&q);
                }
                tc::unpack2<T>(w[i], x, y);
                v[2 * i] -= x;
                v[2 * i + 1] -= y;
              }
              stage_free();
#pragma unroll
              for (int i = 0; i < 4; ++i)
                tc::st_shared_v4(tc::smem_u32(out) + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4),
                                 w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
              if (F32) stage_full(pl * args.ld_dz + n, m_warp, &map_p);
              else stage_full(n, pl * HALF + m_warp, &map_p);
            }
          } else {
            if (c % 64 == 0) stage_free();
            stage32<T>(out_row, lane, v, c % 64 / 8);
            if (c % 64 == 32) stage_full(n - 32, m_warp, &map_o);
          }
        } else if (EPI == kDh || args.plan) {
          if (n >= args.ld_acc) return;
          stage_free();
          stage32<float>(out_row, lane, v, 0);
          stage_full(n, un.split * sched.acc_rows + m_warp, &map_o);
        } else if constexpr (EPI == kDw) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] *= post;
          if (args.out) {
            if (m < args.Cn) {
              O* dst = (O*)args.out + (int64_t)(args.c0 + m) * args.D + n;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (n + i < args.D) dst[i] = from_f32<O>(v[i]);
            }
            __syncwarp();  // the next columns' wait is warp-collective
          } else if constexpr (F32) {
            stage_free();
            stage32<float>(out_row, lane, v, 0);
            if (n < args.D && m_warp < args.Cn) stage_full(n, args.c0 + m_warp, &map_o);
          } else {
            if (c % 64 == 0) stage_free();
            stage32<O>(out_row, lane, v, c % 64 / 8);
            if (c % 64 == 32 && n - 32 < args.D && m_warp < args.Cn)
              stage_full(n - 32, args.c0 + m_warp, &map_o);
          }
        }
      };
      // the buffer is read: the leading CTA may multiply into it again
      auto give_back = [&](uint32_t buf) {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(tc::map_rank(acc_empty + buf, 0));
      };

      if constexpr (CHUNKS) {
        float acc[SUB / 32][32];
#pragma unroll
        for (int c = 0; c < SUB / 32; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[c][i] = 0.f;
        for (int kc = 0; kc < un.kbs; kc += CHUNK_KB, ++n_acc) {
          const uint32_t buf = n_acc & 1;
          ok = __all_sync(0xffffffffu,
                          tc::mbar_wait(acc_full + buf, (n_acc >> 1) & 1, abort, POLLS));
          if (!ok) break;
          tc::tc_fence_after();
#pragma unroll
          for (int c = 0; c < SUB / 32; ++c) {
            float v[32];
            tc::tmem_ld32(src + buf * ACC_COLS + c * 32, v);
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c][i] += v[i];
          }
          give_back(buf);
        }
        if (!ok) break;
        if (!idle) {
#pragma unroll
          for (int c = 0; c < SUB / 32; ++c) take(acc[c], c * 32);
        }
      } else {
        const uint32_t buf = n_acc & 1;
        ok = __all_sync(0xffffffffu,
                        tc::mbar_wait(acc_full + buf, (n_acc >> 1) & 1, abort, POLLS));
        if (!ok) break;
        ++n_acc;
        tc::tc_fence_after();
        if (idle) {
          give_back(buf);
        } else {
          // the next 32 columns are on their way while these are worked on
          uint32_t raw[2][32];
          tc::tmem_start32(src + buf * ACC_COLS, raw[0]);
#pragma unroll
          for (int c = 0; c < SUB / 32; ++c) {
            tc::tmem_wait32(raw[c & 1]);
            if (c + 1 < SUB / 32)
              tc::tmem_start32(src + buf * ACC_COLS + (c + 1) * 32, raw[(c + 1) & 1]);
            else
              give_back(buf);
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(raw[c & 1][i]);
            take(v, c * 32);
          }
        }
      }
      if (EPI == kScore && m < live && n0 < args.V)
        args.part[(int64_t)m * args.sub_tiles + n0 / SUB] = make_float2(top, sum);
    }
    if (lane == 0) tc::bulk_wait_all();
  }

  // Copies in flight after a wait that gave up land before the CTA ends.
  __syncwarp();
  __syncthreads();
  if (*abort) {
    for (int i = 0; i < 1000; ++i) __nanosleep(2000);
  }
  tc::tc_fence_before();
  tc::cluster_sync();
  tc::tc_fence_after();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(2 * ACC_COLS)
                 : "memory");
  }
}

// dst[m][plane][Kp] = the rows of src, packed: by `row_of` the n_live rows that
// count, then zeros up to a multiple of BM; without it all `rows`.  Zeros past D.
struct PackArgs {
  const void* src;
  void* dst;
  const int *row_of, *n_live;
  int64_t rows;
  int vec;    // src's rows can be read 16 bytes at a time
  int plain;  // where every row counts src is read as it is: nothing to do
};
// T: the operands' type; O float: three planes.
template <typename T, typename O>
__device__ __forceinline__ void pack_rows(const PackArgs& a, int64_t D, int64_t Kp, int64_t first,
                                          int64_t step) {
  const int64_t live = a.n_live ? *a.n_live : a.rows;
  if (a.plain && live == a.rows) return;
  const int64_t end = a.n_live ? (live > 0 ? (live + BM - 1) / BM * BM : BM) : a.rows;
  constexpr int planes = sizeof(O) == 4 ? 3 : 1;
  const int64_t units = Kp / 8;
  for (int64_t e = first; e < end * units; e += step) {
    const int64_t m = e / units, k = (e - m * units) * 8;
    const O* s = (const O*)a.src + (m < live ? (a.row_of ? a.row_of[m] : m) : 0) * D + k;
    __align__(16) O x[8];
    if (m < live && a.vec && k + 8 <= D) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(O) / 2; ++i)
        reinterpret_cast<uint4*>(x)[i] = reinterpret_cast<const uint4*>(s)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = m < live && k + i < D ? s[i] : from_f32<O>(0.f);
    }
    T* d = (T*)a.dst + m * planes * Kp + k;
    if constexpr (sizeof(O) == 4) {
      __nv_bfloat16 p[8][3];
#pragma unroll
      for (int i = 0; i < 8; ++i) split3(x[i], p[i]);
#pragma unroll
      for (int pl = 0; pl < 3; ++pl) {
        __align__(16) __nv_bfloat16 o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = p[i][pl];
        *reinterpret_cast<uint4*>(d + pl * Kp) = *reinterpret_cast<const uint4*>(o);
      }
    } else {
      *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(x);
    }
  }
}
// out[m] of each row that counts, for dz's epilogue: its lse, what that one's
// rounding left, its factor of dz, and dz of its target.
struct RowArgs {
  const float* lse;    // [3][N]: lse, what its rounding left, the row's loss
  const float* gloss;  // the rows' upstream gradients (NULL: 1) ...
  const float* most;   // ... in units of the largest
  float unit;
  float4* out;         // NULL: nothing to do (forward)
};
__device__ __forceinline__ void make_rows(const RowArgs& a, const int* row_of, int live, int64_t N,
                                          int first, int step) {
  const float most = a.gloss ? *a.most : 1.f;
  for (int m = first; m < live; m += step) {
    const int64_t i = row_of[m];
    const float rs = (a.gloss ? a.gloss[i] / most : 1.f) * a.unit;
    // p - 1 of a nearly certain token from its loss: p itself is rounded at 1
    a.out[m] = make_float4(a.lse[i], a.lse[N + i], rs, rs * expm1f(-a.lse[2 * N + i]));
  }
}
// h in the first `h_ctas` CTAs, w in the others (none where w is read as it is).
template <typename T, typename O>
__global__ void __launch_bounds__(256)
pack_kernel(const PackArgs h, const PackArgs w, const RowArgs rows, int h_ctas, int64_t D,
            int64_t Kp) {
  const int b = blockIdx.x;
  grid_launch();
  grid_wait();
  if (b < h_ctas && rows.out)
    make_rows(rows, h.row_of, *h.n_live, h.rows, b * 256 + threadIdx.x, h_ctas * 256);
  if (b < h_ctas)
    pack_rows<T, O>(h, D, Kp, (int64_t)b * 256 + threadIdx.x, (int64_t)h_ctas * 256);
  else
    pack_rows<T, O>(w, D, Kp, (int64_t)(b - h_ctas) * 256 + threadIdx.x,
                    (int64_t)(gridDim.x - h_ctas) * 256);
}

// out[i] = post * the sum of the splits' partials of row pos[i] (i itself
// without `pos`), or zeros, for dh and dw: the first `a_ctas` CTAs take a, the
// others b.  VEC values a thread.
struct SumArgs {
  const float* acc;
  const int* pos;
  const Splits* plan;
  void* out;
  int64_t rows;
};
template <typename O, int VEC>
__global__ void __launch_bounds__(256)
split_sum_kernel(const SumArgs a, const SumArgs b, int a_ctas, const float* post,
                 int ld_acc, int D) {
  const bool is_a = (int)blockIdx.x < a_ctas;
  const SumArgs& s = is_a ? a : b;
  const int64_t first = is_a ? blockIdx.x : blockIdx.x - a_ctas;
  const int64_t step = is_a ? a_ctas : (int)gridDim.x - a_ctas;
  grid_wait();
  const float f = *post;
  const int splits = s.plan->splits;
  const int64_t acc_rows = s.plan->acc_rows;
  const int units = D / VEC;
  for (int64_t i = first; i < s.rows; i += step) {
    const int64_t m = s.pos ? s.pos[i] : i;
    for (int u = threadIdx.x; u < units; u += 256) {
      float x[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = 0.f;
      if (m >= 0) {
#pragma unroll 4
        for (int k = 0; k < splits; ++k) {
          const float* p = s.acc + (k * acc_rows + m) * ld_acc + u * VEC;
          if constexpr (VEC == 1) {
            x[0] += p[0];
          } else {
#pragma unroll
            for (int q = 0; q < VEC / 4; ++q) {
              const float4 y = reinterpret_cast<const float4*>(p)[q];
              x[4 * q] += y.x;
              x[4 * q + 1] += y.y;
              x[4 * q + 2] += y.z;
              x[4 * q + 3] += y.w;
            }
          }
        }
      }
      if (m >= 0) {  // a row that does not count stays 0, also where f is not finite
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] *= f;
      }
      embed::store_vec<O, VEC>((O*)s.out + i * D + u * VEC, x);
    }
  }
}

}  // namespace xent
}  // namespace theria
