// Tensor-core (tcgen05) attention over packed sequences, backward: two kernels, each
// on a tile of 128 rows x1, x2 while it walks over tiles of rows y1, y2:
//     tc_dq:  x = (q, do), y = (k, v):  dq += ds k
//     tc_dkv: x = (k, v), y = (q, do):  dk += ds^T q, dv += p^T do
// with, per tile, s = x1 y1^T and dp = x2 y2^T, p = exp(scale s - lse) and
// ds = p (dp - z).  Seven products a pair of tiles instead of the five that one
// kernel for all three gradients needs; but then nothing is added atomically
// (the same bits every time), there is no float32 dq in HBM, and p and ds never
// leave the tensor memory: as 16-bit pairs they overwrite s and dp in place and are
// the A operands of the sums.
//
// The queries of the G heads that share a key head lie token by token in a
// tile of rows (as in the forward), so dk and dv sum over the group in TMEM.
//
//     warp 0       TMA producer; tc_dkv: also each tile's row terms
//     warps 1..    one thread each issues s, dp, the sum of ds y1, that of p y2
//     16 warps     p and ds, each 32 rows (a TMEM lane quarter) by 32 columns
// A hop from one of these to the next (a commit or an arrival, a wait that returns)
// takes 150 to 300 cycles, a wait that finds its barrier passed 200, a commit 100;
// with a few buffers the hops of the ring s -> p, ds -> sums -> s set the pace, not the
// products (bfloat16, 8192 tokens in two sequences, 16 heads on 4 of 128, not causal:
// dq 335 us of 160 us of products, dkv 466 to 490 of 320).  Hence one product a step and one
// thread a product (one issuing thread for all: dkv 640 us, two: 540), and, per side:
//
// tc_dq: tiles of 128 rows y, all 16 warps on one.  s, in one buffer, is free as soon
//   as the warps have read it, so the next tile's s is made while this one's p is; dp
//   has two, over which its ds goes.  An N = 128 product takes 64 cycles, two of N = 64
//   100 to 126.  (64 rows and two buffers of both: 386 us; three of dp, s early: 410.)
// tc_dkv: tiles of 64 rows y, two buffers of s and dp, 8 warps on the even tiles and 8
//   on the odd ones; p goes over s and ds over dp, so that p y2 is summed while ds is
//   still made.  The two sums take 256 columns at HD = 128, which leaves no room for
//   more.  (128 rows, one buffer: 549 us; s early, p and ds over dp: 710 and 774.)
//
// float16 (not bfloat16) has a short range: ds as it is would pass its largest number,
// or lose bits below its smallest normal one, with cotangents and values that are not of
// order 1 (4096 keys, cotangents of 1e-3: dq off by 5 times its final rounding, so by
// 1.2).  So ds is made times a power of two that takes the largest it can be to 2^15, by
// the norms of the cotangents and of v, and the results are divided by it: for dq each
// row's own, added to its term in the exponent; for dk and dv, whose sums run over rows,
// one for all rows that a CTA walks, taken into (dp - z) by the multiplication-and-
// addition that makes it.  Neither costs an instruction of the loop (2 x 4096 tokens, 16 / 4
// heads of 128: row terms 21 -> 28 us, dq 177 -> 181, dk, dv 249 -> 248 causal, 476 -> 497
// not; of 64: 11.6 -> 16.4, 137 -> 134, 196 -> 199).
//
// Rows behind the sequence's end in a tile of y belong to others and may be
// anything; p = 0 and ds = 0 would multiply them, so the producer warp sets them
// to zero.
#pragma once

#include "ragged_plan.cuh"
#include "ragged_tc_fwd.cuh"
#include "tc_common.cuh"

namespace theria {
namespace ragged {

__device__ __forceinline__ float2 ld_shared_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

constexpr int BX = 128;             // rows of x
constexpr int QY = 128, KY = 64;    // rows of y: of tc_dq (keys), of tc_dkv (packed queries)

// 32 columns of one of a kernel's sums, scaled and rounded, to row `to` of the result
// (columns c .. c + 31 of D, a multiple of 8).
template <typename T>
__device__ __forceinline__ void put_sums(const float (&v)[32], float mul, T* to, int c, int D) {
  const bool wide = wide_rows(to, D);  // (the same for every row)
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float* e = v + 16 * i;
    const int at = c + 16 * i;
    if (at >= D) continue;
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = tc::pack2<T>(e[2 * k] * mul, e[2 * k + 1] * mul);
    store16(to + at, w, wide, at + 8 < D);
  }
}

// ------------------------------------------------------------------ queries
template <int HD>
struct DqCfg {
  static constexpr int kCtl = 4, kWarps = 16, kThreads = 32 * (kCtl + kWarps);
  static constexpr int kX = BX * HD * 2, kY = QY * HD * 2;  // one operand's tile
  // Depths of the rings: k is in use from s to the sum of ds, a tile longer than v.
  static constexpr int R1 = HD == 128 ? 3 : 4, R2 = HD == 128 ? 2 : 4;
  static constexpr int oX1 = 0, oX2 = kX;
  static constexpr int oY1 = 2 * kX;              // [R1]
  static constexpr int oY2 = oY1 + R1 * kY;       // [R2]
  static constexpr int oBar = oY2 + R2 * kY;
  // x_full, edge, drain[3], s_full, s_read, dp_full[2], ds_full[2], done[2], y1_full[],
  // y1_empty[], y2_full[], y2_empty[]
  static constexpr int nBar = 13 + 2 * R1 + 2 * R2;
  static constexpr int oTmem = oBar + nBar * 8;
  static constexpr int oAbort = oTmem + 4;
  static constexpr int oFit = oAbort + 4;  // float16: each warp's largest norm_code
  static constexpr int kAlloc = oFit + 4 * (kThreads / 32) + 1024;  // slack to align the base
  static_assert(kAlloc <= 232448, "shared memory of a block");
};

template <typename T, int HD, bool CAUSAL>
__global__ void __launch_bounds__(DqCfg<HD>::kThreads, 1)
tc_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
             const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
             const float2* terms, const uint8_t* fits, T* __restrict__ dq, const int4* items,
             const int* count, const Problem pr) {
  using L = DqCfg<HD>;
  constexpr int R1 = L::R1, R2 = L::R2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oBar);
  uint64_t *x_full = bars, *edge = bars + 1, *drain = bars + 2;  // drain [3]
  uint64_t *s_full = bars + 5, *s_read = bars + 6;               // s made; s in registers
  // Of tile t at [t & 1], so that no phase can pass a waiting thread:
  uint64_t* dp_full = bars + 7;    // dp made
  uint64_t* ds_full = bars + 9;    // ds written
  uint64_t* done = bars + 11;      // and summed
  uint64_t *y1_full = bars + 13, *y1_empty = y1_full + R1;
  uint64_t *y2_full = y1_empty + R1, *y2_empty = y2_full + R2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::oTmem);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::oAbort);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_wait();
  const int hk = blockIdx.x % pr.Hkv, at = blockIdx.x / pr.Hkv;
  if (at >= *count) return;
  const int4 item = items[at];
  const int start = item.x, len = item.y, first = item.z, G = pr.G;
  const int xt = BX / G;  // tokens of a tile
  const int keys = CAUSAL ? min(first + xt, len) : len;
  const int n_iter = (keys + QY - 1) / QY;

  if (threadIdx.x == 0) {
    tc::mbar_init(x_full, 1);
    tc::mbar_init(edge, 1);
    for (int b = 0; b < 3; ++b) tc::mbar_init(drain + b, 1);
    tc::mbar_init(s_full, 1);
    tc::mbar_init(s_read, L::kWarps);  // a warp arrives once
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(dp_full + b, 1);
      tc::mbar_init(ds_full + b, L::kWarps);
      tc::mbar_init(done + b, 1);
    }
    for (int s = 0; s < R1; ++s) {
      tc::mbar_init(y1_full + s, 1);
      tc::mbar_init(y1_empty + s, 1);
    }
    for (int s = 0; s < R2; ++s) {
      tc::mbar_init(y2_full + s, 1);
      tc::mbar_init(y2_empty + s, 1);
    }
    *abort = 0;
    tc::fence_barrier_init();
  }
  if (warp == 1) tc::tmem_alloc(tmem_slot, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  // TMEM: s [0, 128), dp of tile t [128 + 128 (t & 1), +128), the sum [384, 384 + HD)
  const uint32_t tmem = *tmem_slot, t_a = tmem + 384;
  auto t_dp = [&](int t) { return tmem + 128 + (t & 1) * 128; };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tc::prefetch_tmap(&tm_k);
      tc::prefetch_tmap(&tm_v);
      tc::mbar_expect_tx(x_full, 2 * (HD / 64) * xt * G * 128);
      for (int cb = 0; cb < HD / 64; ++cb) {
        tma_load_rows(smem + L::oX1 + cb * BX * 128, &tm_q, x_full, cb * 64, start + first, hk);
        tma_load_rows(smem + L::oX2 + cb * BX * 128, &tm_do, x_full, cb * 64, start + first, hk);
      }
    }
    // k or v of tile t into its ring; k's last rows of the sequence by way of a barrier
    // of their own, with zeros behind the end (v is in dp alone, whose columns there
    // are masked)
    auto fetch = [&](int t, int which) {
      const int R = which ? R2 : R1, st = t % R;
      uint64_t* full = (which ? y2_full : y1_full) + st;
      uint64_t* empty = (which ? y2_empty : y1_empty) + st;
      uint8_t* y = smem + (which ? L::oY2 : L::oY1) + st * L::kY;
      const bool ends = (t + 1) * QY > len && which == 0;
      bool ok = true;
      if (lane == 0) {
        if (t >= R) ok = tc::mbar_wait(empty, ((t / R) - 1) & 1, abort);
        if (ok) {
          uint64_t* bar = ends ? edge : full;
          tc::mbar_expect_tx(bar, L::kY);
          for (int cb = 0; cb < HD / 64; ++cb)
            tc::tma_load_3d(y + cb * QY * 128, which ? &tm_v : &tm_k, bar, cb * 64,
                            start + t * QY, hk);
        }
      }
      if (!__shfl_sync(0xffffffffu, ok, 0)) return false;
      if (ends) {
        if (!__all_sync(0xffffffffu, tc::mbar_wait(edge, 0, abort))) {
          tc::mbar_wait_drain(edge, 0);
          return false;
        }
        zero_rows(y, QY, HD / 64, len - t * QY, QY, lane);
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(full);
      }
      return true;
    };
    int n1 = 0, n2 = 0;  // tiles fetched
    for (int t = 0; t < n_iter; ++t) {
      if (!fetch(t, 0)) break;
      n1 = t + 1;
      if (!fetch(t, 1)) break;
      n2 = t + 1;
    }
    // Every copy issued into this CTA's shared memory lands before it may exit.
    if (lane == 0) {
      tc::mbar_wait_drain(x_full, 0);
      for (int t = n1 > R1 ? n1 - R1 : 0; t < n1; ++t)
        tc::mbar_wait_drain(y1_full + t % R1, (t / R1) & 1);
      for (int t = n2 > R2 ? n2 - R2 : 0; t < n2; ++t)
        tc::mbar_wait_drain(y2_full + t % R2, (t / R2) & 1);
    }
  } else if (warp < L::kCtl) {
    // ------------------------------------------------------------ issuers
    if (lane == 0) {
      constexpr int ab = tc::AbFmt<T>::v;
      if (warp <= 2) {
        // s = q k^T (warp 1) or dp = do v^T (warp 2)
        constexpr uint32_t id_s = tc::idesc_f16(BX, QY, ab, 0, 0);
        const bool is_s = warp == 1;
        const uint64_t x = tc::sw128_desc(tc::smem_u32(smem + (is_s ? L::oX1 : L::oX2)), 16, 1024);
        const uint64_t y = tc::sw128_desc(tc::smem_u32(smem + (is_s ? L::oY1 : L::oY2)), 16, 1024);
        const int R = is_s ? R1 : R2;
        const bool ok = tc::mbar_wait(x_full, 0, abort);
        for (int t = 0; ok && t < n_iter; ++t) {
          const int st = t % R;
          // the columns are free; and with a summed tile its rows of k
          if (is_s) {
            if (t >= 1 && !tc::mbar_wait(s_read, (t - 1) & 1, abort)) break;
          } else if (t >= 2) {
            if (!tc::mbar_wait(done + (t & 1), ((t >> 1) - 1) & 1, abort)) break;
            tc::mbar_arrive(y1_empty + (t - 2) % R1);
          }
          if (!tc::mbar_wait((is_s ? y1_full : y2_full) + st, (t / R) & 1, abort)) break;
          tc::tc_fence_after();
          const uint32_t t_d = is_s ? tmem : t_dp(t);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            tc::mma_ss(t_d, tc::desc_at(x, (kk / 4) * (BX * 128) + (kk % 4) * 32),
                       tc::desc_at(y, st * L::kY + (kk / 4) * (QY * 128) + (kk % 4) * 32), id_s,
                       kk > 0 ? 1u : 0u);
          tc::mma_commit(is_s ? s_full : dp_full + (t & 1));
          if (!is_s) tc::mma_commit(y2_empty + st);
        }
      } else {
        // dq += ds k, the tile's keys as contraction
        constexpr uint32_t id_a = tc::idesc_f16(BX, HD, ab, 0, 1);
        const uint64_t y = tc::sw128_desc(tc::smem_u32(smem + L::oY1), QY * 128, 1024);
        for (int t = 0; t < n_iter; ++t) {
          if (!tc::mbar_wait(ds_full + (t & 1), (t >> 1) & 1, abort)) break;
          tc::tc_fence_after();
          // 16 keys: 8 TMEM columns of pairs, where the warp of those 32 columns put them
#pragma unroll
          for (int kk = 0; kk < QY / 16; ++kk)
            tc::mma_ts(t_a, t_dp(t) + (kk / 2) * 32 + (kk % 2) * 8,
                       tc::desc_at(y, (t % R1) * L::kY + kk * 2048), id_a,
                       t > 0 || kk > 0 ? 1u : 0u);
          tc::mma_commit(done + (t & 1));
        }
      }
      tc::mma_commit(drain + warp - 1);
      tc::mbar_wait_drain(drain + warp - 1, 0);
    }
  } else {
    // ------------------------------------------------------------ p and ds
    const int cg = (warp - L::kCtl) >> 2, quarter = warp & 3;  // columns [32 cg, +32)
    const int r = quarter * 32 + lane;  // TMEM lane: the row
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int tok = first + r / G;
    const bool live = tok < len && r < xt * G;
    const int64_t row = (int64_t)(start + tok) * pr.H + hk * G + r % G;
    float2 mine = live ? terms[row] : make_float2(-INFINITY, 0.f);  // {-lse log2 e, -z}
    float mul = pr.scale;
    if constexpr (std::is_same<T, __half>::value) {  // ds of the row times 2^e
      // the largest of the values that the tile's rows see
      uint32_t* largest = reinterpret_cast<uint32_t*>(smem + L::oFit);
      const uint8_t* values = fits + (int64_t)pr.T * pr.H + (int64_t)hk * pr.T + start;
      const uint32_t code = live ? fits[((int64_t)hk * pr.T + start + tok) * G + r % G] : 0u;
      const uint32_t of_mine = __reduce_max_sync(
          0xffffffffu, largest_of_mine(values, values + keys, threadIdx.x - 32 * L::kCtl,
                                       32 * L::kWarps));
      if (lane == 0) largest[warp - L::kCtl] = of_mine;
      tc::named_bar(1, 32 * L::kWarps);  // (before any wait that may give up)
      const int e = fit_power(
          code, __reduce_max_sync(0xffffffffu, lane < L::kWarps ? largest[lane] : 0u));
      mine.x += (float)e;
      mul *= pow2(-e);
    }
    const int warp_tok = first + quarter * 32 / G;  // the first token of the warp
    const int my_keys = CAUSAL ? min(len, tok + 1) : len;
    bool ok = true;
    // Waits are warp-uniform: the TMEM accesses that follow are warp-collective.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, abort));
    };
    // what the warp read from or wrote to TMEM is done: one arrival
    auto arrive = [&](uint64_t* bar) {
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(bar);
    };
    for (int t = 0; t < n_iter; ++t) {
      const int y0 = t * QY;
      const uint32_t t_d = t_dp(t) + cg * 32 + lane_off;
      if (!wait(s_full, t & 1)) { ok = false; break; }
      tc::tc_fence_after();
      float s[32];
      tc::tmem_ld32(tmem + cg * 32 + lane_off, s);
      arrive(s_read);
      // tiles on the diagonal and at the sequence's end need a mask; the test is the
      // same for a whole warp.  Valid: columns below `hi`.
      const bool masked = y0 + QY > len || (CAUSAL && y0 + QY - 1 > warp_tok);
      const int hi = my_keys - y0 - cg * 32;
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        tc::fma2(s[e], s[e + 1], s[e], s[e + 1], pr.scale_log2, pr.scale_log2, mine.x, mine.x);
        s[e] = tc::ex2(s[e]);
        s[e + 1] = tc::ex2(s[e + 1]);
      }
      if (!wait(dp_full + (t & 1), (t >> 1) & 1)) { ok = false; break; }
      tc::tc_fence_after();
      float dp[32];
      tc::tmem_ld32(t_d, dp);
      uint32_t pk[16];  // ds = p (dp - z) as 16-bit pairs
      auto make_ds = [&](auto mk) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float g0, g1;
          tc::add2(g0, g1, dp[e], dp[e + 1], mine.y, mine.y);
          tc::mul2(g0, g1, s[e], s[e + 1], g0, g1);
          if constexpr (decltype(mk)::value) {
            g0 = e < hi ? g0 : 0.f;
            g1 = e + 1 < hi ? g1 : 0.f;
          }
          pk[e / 2] = tc::pack2<T>(g0, g1);
        }
      };
      if (masked) make_ds(std::true_type{}); else make_ds(std::false_type{});
      tc::tmem_st16(t_d, pk);
      tc::tmem_wait_st();
      arrive(ds_full + (t & 1));
    }
    // ------------------------------------------------------------ results
    if (ok && wait(drain + 2, 0)) {
      tc::tc_fence_after();
      if (cg < HD / 32) {
        float v[32];
        tc::tmem_ld32(t_a + lane_off + cg * 32, v);
        if (live) put_sums<T>(v, mul, dq + row * pr.D, cg * 32, pr.D);
      }
    }
  }
  // ------------------------------------------------------------ teardown
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// --------------------------------------------------------------------- keys
template <int HD>
struct DkvCfg {
  static constexpr int kCtl = 5, kSet = 8;  // control warps; warps of one tile's p and ds
  static constexpr int kThreads = 32 * (kCtl + 2 * kSet);
  static constexpr int kX = BX * HD * 2, kY = KY * HD * 2;  // one operand's tile
  static constexpr int YST = HD == 128 ? 4 : 6;             // ring depth
  static constexpr int oX1 = 0, oX2 = kX;
  static constexpr int oY1 = 2 * kX;              // [YST]
  static constexpr int oY2 = oY1 + YST * kY;      // [YST]
  static constexpr int oTerm = oY2 + YST * kY;    // [YST][2][64] floats
  static constexpr int oBar = oTerm + YST * KY * 8;
  // x_full, x_tmem, edge, drain[4], and per buffer s_full, s_free, dp_full, dp_free,
  // p_full, ds_full; y_full[], y_empty[]
  static constexpr int nBar = 7 + 12 + 2 * YST;
  static constexpr int oTmem = oBar + nBar * 8;
  static constexpr int oAbort = oTmem + 4;
  static constexpr int oFit = oAbort + 4;  // float16: each warp's largest norm_codes
  static constexpr int kAlloc = oFit + 4 * (kThreads / 32) + 1024;
  static_assert(kAlloc <= 232448, "shared memory of a block");
};

// One split of a tile's queries.  part: NULL where there is one split (results rounded
// to T at once), else float32 [splits][2][T * Hkv][D].
template <typename T, int HD, bool CAUSAL>
__global__ void __launch_bounds__(DkvCfg<HD>::kThreads, 1)
tc_dkv_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
              const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
              const float2* terms, const uint8_t* fits, T* __restrict__ dk, T* __restrict__ dv,
              float* part, const int4* items, const int* count, int splits, const Problem pr) {
  using L = DkvCfg<HD>;
  constexpr int YST = L::YST;
  constexpr bool kXT = HD == 64;  // k and v in TMEM too, as the A operands of s and dp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oBar);
  uint64_t *x_full = bars, *x_tmem = bars + 1, *edge = bars + 2, *drain = bars + 3;  // drain [4]
  uint64_t *s_full = bars + 7, *dp_full = bars + 9;    // products done
  uint64_t *p_full = bars + 11, *ds_full = bars + 13;  // pairs written over them
  uint64_t *s_free = bars + 15, *dp_free = bars + 17;  // and summed
  uint64_t *y_full = bars + 19, *y_empty = y_full + YST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::oTmem);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::oAbort);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_wait();
  // a tile's splits side by side, so that the longest tiles' all start first
  const int hk = blockIdx.x % pr.Hkv, sp = blockIdx.x / pr.Hkv % splits;
  const int at = blockIdx.x / pr.Hkv / splits;
  if (at >= *count) return;
  const int4 item = items[at];
  const int start = item.x, len = item.y, first = item.z, G = pr.G;
  const int yt = KY / G, y_rows = yt * G;  // tokens, rows of a tile of queries
  // the queries' tokens from y_from on, and this split's share of their tiles
  const int y_from = CAUSAL ? first : 0;
  const int n_y = (len - y_from + yt - 1) / yt;
  const int t_at = (int)((int64_t)n_y * sp / splits);
  const int n_iter = (int)((int64_t)n_y * (sp + 1) / splits) - t_at;
  auto tok_of = [&](int t) { return y_from + (t_at + t) * yt; };  // tile t's first token

  if (threadIdx.x == 0) {
    tc::mbar_init(x_full, 1);
    tc::mbar_init(x_tmem, L::kSet);
    tc::mbar_init(edge, 1);
    for (int b = 0; b < 4; ++b) tc::mbar_init(drain + b, 1);
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(s_full + b, 1);
      tc::mbar_init(dp_full + b, 1);
      tc::mbar_init(p_full + b, L::kSet);  // a warp arrives once
      tc::mbar_init(ds_full + b, L::kSet);
      tc::mbar_init(s_free + b, 1);
      tc::mbar_init(dp_free + b, 1);
    }
    for (int s = 0; s < YST; ++s) {
      tc::mbar_init(y_full + s, 2);   // the tile and its row terms
      tc::mbar_init(y_empty + s, 2);  // both sums
    }
    *abort = 0;
    tc::fence_barrier_init();
  }
  if (warp == 1) tc::tmem_alloc(tmem_slot, 512);
  if (y_rows < KY)  // rows that no copy fills
    for (int s = warp; s < 2 * YST; s += L::kThreads / 32)
      zero_rows(smem + L::oY1 + s * L::kY, KY, HD / 64, y_rows, KY, lane);
  constexpr bool kFit = std::is_same<T, __half>::value;
  uint32_t* largest = reinterpret_cast<uint32_t*>(smem + L::oFit);
  if constexpr (kFit) {  // of the rows to walk, and of the values that their z may hold
    const uint8_t* rows = fits + ((int64_t)hk * pr.T + start) * G;
    const uint8_t* values = fits + (int64_t)pr.T * pr.H + (int64_t)hk * pr.T + start;
    const uint32_t a = __reduce_max_sync(
        0xffffffffu, largest_of_mine(rows + (int64_t)tok_of(0) * G,
                                     rows + (int64_t)min(tok_of(n_iter), len) * G,
                                     threadIdx.x, L::kThreads));
    const uint32_t b = __reduce_max_sync(
        0xffffffffu, largest_of_mine(values, values + len, threadIdx.x, L::kThreads));
    if (lane == 0) largest[warp] = a << 8 | b;
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  // ds is made times 2^fitted() (a whole warp calls it)
  auto fitted = [&] {
    const uint32_t w = lane < L::kThreads / 32 ? largest[lane] : 0u;
    return fit_power(__reduce_max_sync(0xffffffffu, w >> 8),
                     __reduce_max_sync(0xffffffffu, w & 255));
  };
  float up = 1.f;
  if constexpr (kFit) up = pow2(fitted());
  // TMEM: buffer b of s [128 b, +64), of dp [128 b + 64, +64); the sums from 256 on;
  // HD = 64: k and v from 384 on
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_a1 = tmem + 256, t_a2 = tmem + 256 + HD;
  const uint32_t t_x1 = tmem + 384, t_x2 = tmem + 384 + HD / 2;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (n_iter > 0) {
      if (lane == 0) {
        tc::prefetch_tmap(&tm_q);
        tc::prefetch_tmap(&tm_do);
        tc::mbar_expect_tx(x_full, 2 * L::kX);
        for (int cb = 0; cb < HD / 64; ++cb) {
          tc::tma_load_3d(smem + L::oX1 + cb * BX * 128, &tm_k, x_full, cb * 64, start + first, hk);
          tc::tma_load_3d(smem + L::oX2 + cb * BX * 128, &tm_v, x_full, cb * 64, start + first, hk);
        }
      }
      // {-lse log2 e, -z} of a tile's rows, loaded a tile ahead so that their
      // latency never delays a copy; rows past the end: p = exp2(-inf) = 0
      float2 rv[2];
      auto load_terms = [&](int t) {
        const int tok = tok_of(t);
        const int64_t base = (int64_t)(start + tok) * pr.H + hk * G;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int e = k * 32 + lane, g = e % G, dt = e / G;
          rv[k] = e < y_rows && tok + dt < len ? terms[base + (int64_t)dt * pr.H + g]
                                               : make_float2(-INFINITY, 0.f);
        }
      };
      load_terms(0);
      int issued = 0;
      for (int t = 0; t < n_iter; ++t) {
        const int st = t % YST, tok = tok_of(t);
        bool ok = true;
        if (lane == 0 && t >= YST) ok = tc::mbar_wait(y_empty + st, ((t / YST) - 1) & 1, abort);
        if (!__shfl_sync(0xffffffffu, ok, 0)) break;
        const bool ends = tok + yt > len;  // the last tile of the sequence, ragged
        uint64_t* full = ends ? edge : y_full + st;
        uint8_t *y1 = smem + L::oY1 + st * L::kY, *y2 = smem + L::oY2 + st * L::kY;
        if (lane == 0) {
          tc::mbar_expect_tx(full, 2 * (HD / 64) * y_rows * 128);
          for (int cb = 0; cb < HD / 64; ++cb) {
            tma_load_rows(y1 + cb * KY * 128, &tm_q, full, cb * 64, start + tok, hk);
            tma_load_rows(y2 + cb * KY * 128, &tm_do, full, cb * 64, start + tok, hk);
          }
        }
        float* rt = reinterpret_cast<float*>(smem + L::oTerm + st * KY * 8);
        rt[lane] = rv[0].x;
        rt[32 + lane] = rv[1].x;
        rt[KY + lane] = rv[0].y * up;
        rt[KY + 32 + lane] = rv[1].y * up;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(y_full + st);
        if (t + 1 < n_iter) load_terms(t + 1);
        if (ends) {
          if (!__all_sync(0xffffffffu, tc::mbar_wait(edge, 0, abort))) {
            tc::mbar_wait_drain(edge, 0);
            break;
          }
          zero_rows(y1, KY, HD / 64, (len - tok) * G, KY, lane);
          zero_rows(y2, KY, HD / 64, (len - tok) * G, KY, lane);
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(y_full + st);
        }
        issued = t + 1;
      }
      if (lane == 0) {
        tc::mbar_wait_drain(x_full, 0);
        for (int t = issued > YST ? issued - YST : 0; t < issued; ++t)
          tc::mbar_wait_drain(y_full + t % YST, (t / YST) & 1);
      }
    }
  } else if (warp < L::kCtl) {
    // ------------------------------------------------------------ issuers
    if (lane == 0 && n_iter > 0) {
      constexpr int ab = tc::AbFmt<T>::v;
      if (warp <= 2) {
        // s = k q^T (warp 1) or dp = v do^T (warp 2)
        constexpr uint32_t id_s = tc::idesc_f16(BX, KY, ab, 0, 0);
        const bool is_s = warp == 1;
        const uint64_t x = tc::sw128_desc(tc::smem_u32(smem + (is_s ? L::oX1 : L::oX2)), 16, 1024);
        const uint64_t y = tc::sw128_desc(tc::smem_u32(smem + (is_s ? L::oY1 : L::oY2)), 16, 1024);
        const uint32_t t_x = is_s ? t_x1 : t_x2, t_d = tmem + (is_s ? 0 : 64);
        uint64_t *full = is_s ? s_full : dp_full, *free_ = is_s ? s_free : dp_free;
        const bool ok = tc::mbar_wait(kXT ? x_tmem : x_full, 0, abort);
        for (int t = 0; ok && t < n_iter; ++t) {
          const int st = t % YST, b = t & 1;
          // the columns are free, and with a summed tile its rows
          if (t >= 2) {
            if (!tc::mbar_wait(free_ + b, ((t >> 1) - 1) & 1, abort)) break;
            tc::mbar_arrive(y_empty + (t - 2) % YST);
          }
          if (!tc::mbar_wait(y_full + st, (t / YST) & 1, abort)) break;
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint64_t yd =
                tc::desc_at(y, st * L::kY + (kk / 4) * (KY * 128) + (kk % 4) * 32);
            if constexpr (kXT)
              tc::mma_ts(t_d + b * 128, t_x + kk * 8, yd, id_s, kk > 0 ? 1u : 0u);
            else
              tc::mma_ss(t_d + b * 128, tc::desc_at(x, (kk / 4) * (BX * 128) + (kk % 4) * 32), yd,
                         id_s, kk > 0 ? 1u : 0u);
          }
          tc::mma_commit(full + b);
        }
      } else {
        // dk += ds^T q (warp 3) or dv += p^T do (warp 4), the tile's rows as contraction
        constexpr uint32_t id_a = tc::idesc_f16(BX, HD, ab, 0, 1);
        const bool is_ds = warp == 3;
        const uint64_t y =
            tc::sw128_desc(tc::smem_u32(smem + (is_ds ? L::oY1 : L::oY2)), KY * 128, 1024);
        const uint32_t t_d = is_ds ? t_a1 : t_a2, t_p = tmem + (is_ds ? 64 : 0);
        uint64_t *full = is_ds ? ds_full : p_full, *free_ = is_ds ? dp_free : s_free;
        for (int t = 0; t < n_iter; ++t) {
          const int st = t % YST, b = t & 1;
          if (!tc::mbar_wait(full + b, (t >> 1) & 1, abort)) break;
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < KY / 16; ++kk)
            // 16 columns of the tile: 8 TMEM columns of pairs, in the half of the
            // warps that wrote them
            tc::mma_ts(t_d, t_p + b * 128 + (kk / 2) * 32 + (kk % 2) * 8,
                       tc::desc_at(y, st * L::kY + kk * 2048), id_a, t > 0 || kk > 0 ? 1u : 0u);
          tc::mma_commit(free_ + b);
        }
      }
      tc::mma_commit(drain + warp - 1);
      tc::mbar_wait_drain(drain + warp - 1, 0);
    }
  } else {
    // ------------------------------------------------------------ p and ds
    const int set = (warp - L::kCtl) / L::kSet;                 // of even or of odd tiles
    const int grp = ((warp - L::kCtl) >> 2) & 1, quarter = warp & 3;  // columns [32 grp, +32)
    const int r = quarter * 32 + lane;  // TMEM lane: the key's row
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int tok = first + r;
    const bool live = tok < len;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, abort));
    };
    auto arrive = [&](uint64_t* bar) {
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(bar);
    };
    if (kXT && set == 0 && n_iter > 0) {
      // this row of k (group 0) or v (group 1) into TMEM: the 128-byte swizzled row of
      // 64 values is 32 pairs, one a column
      ok = wait(x_full, 0);
      if (ok) {
#pragma unroll
        for (int cb = 0; cb < HD / 64; ++cb) {
          const uint32_t row =
              tc::smem_u32(smem + (grp == 0 ? L::oX1 : L::oX2) + cb * BX * 128) + r * 128u;
          uint32_t w[32];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float4 x = tc::ld_shared_f4(row + (uint32_t)((c ^ (r & 7)) << 4));
            w[4 * c] = __float_as_uint(x.x);
            w[4 * c + 1] = __float_as_uint(x.y);
            w[4 * c + 2] = __float_as_uint(x.z);
            w[4 * c + 3] = __float_as_uint(x.w);
          }
          tc::tmem_st32u((grp == 0 ? t_x1 : t_x2) + cb * 32 + lane_off, w);
        }
        tc::tmem_wait_st();
        arrive(x_tmem);
      }
    }
    for (int t = set; ok && t < n_iter; t += 2) {
      const int b = set, st = t % YST, y0 = tok_of(t);
      const uint32_t t_s = tmem + b * 128 + grp * 32 + lane_off;
      if (!wait(y_full + st, (t / YST) & 1)) { ok = false; break; }  // the row terms
      if (!wait(s_full + b, (t >> 1) & 1)) { ok = false; break; }
      tc::tc_fence_after();
      // tiles on the diagonal need a mask.  Valid: columns from `lo` on.
      const bool masked = CAUSAL && y0 < first + BX;
      const int lo = (tok - y0) * G - grp * 32;
      // the row terms of this warp's columns: all -lse log2 e of a tile, then all -z
      const uint32_t lse_at = tc::smem_u32(smem + L::oTerm + st * KY * 8) + grp * 32 * 4;
      const uint32_t z_at = lse_at + KY * 4;
      float s[32];
      tc::tmem_ld32(t_s, s);
      // p = exp2(scale s - lse); rows past the end of y: exp2(-inf) = 0
      auto make_p = [&](auto mk) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 nl = ld_shared_f2(lse_at + e * 4);
          tc::fma2(s[e], s[e + 1], s[e], s[e + 1], pr.scale_log2, pr.scale_log2, nl.x, nl.y);
          s[e] = tc::ex2(s[e]);
          s[e + 1] = tc::ex2(s[e + 1]);
          if constexpr (decltype(mk)::value) {
            s[e] = e >= lo ? s[e] : 0.f;
            s[e + 1] = e + 1 >= lo ? s[e + 1] : 0.f;
          }
        }
      };
      if (masked) make_p(std::true_type{}); else make_p(std::false_type{});
      uint32_t pk[16];  // 16-bit pairs
#pragma unroll
      for (int i = 0; i < 16; ++i) pk[i] = tc::pack2<T>(s[2 * i], s[2 * i + 1]);
      tc::tmem_st16(t_s, pk);
      tc::tmem_wait_st();
      arrive(p_full + b);
      if (!wait(dp_full + b, (t >> 1) & 1)) { ok = false; break; }
      tc::tc_fence_after();
      float dp[32];
      tc::tmem_ld32(t_s + 64, dp);
      // ds = p (dp - z)
      auto make_ds = [&](auto mk) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 nz = ld_shared_f2(z_at + e * 4);
          float g0, g1;
          if constexpr (kFit) tc::fma2(g0, g1, dp[e], dp[e + 1], up, up, nz.x, nz.y);
          else tc::add2(g0, g1, dp[e], dp[e + 1], nz.x, nz.y);
          tc::mul2(g0, g1, s[e], s[e + 1], g0, g1);
          if constexpr (decltype(mk)::value) {
            g0 = e >= lo ? g0 : 0.f;
            g1 = e + 1 >= lo ? g1 : 0.f;
          }
          pk[e / 2] = tc::pack2<T>(g0, g1);
        }
      };
      if (masked) make_ds(std::true_type{}); else make_ds(std::false_type{});
      tc::tmem_st16(t_s + 64, pk);
      tc::tmem_wait_st();
      arrive(ds_full + b);
    }
    // ------------------------------------------------------------ results
    if (ok && n_iter > 0) {
      ok = wait(drain + 2, 0) && wait(drain + 3, 0);
      if (ok) tc::tc_fence_after();
    }
    if (ok) {
      float dk_mul = pr.scale;
      if constexpr (kFit) dk_mul *= pow2(-fitted());
      const int64_t row = (int64_t)(start + tok) * pr.Hkv + hk;
      const int64_t plane = (int64_t)pr.T * pr.Hkv * pr.D;
#pragma unroll 1
      for (int which = 0; which < 2; ++which) {
        const float mul = which == 0 ? dk_mul : 1.f;
        float* sums = part == nullptr ? nullptr
                                      : part + (2 * sp + which) * plane + row * pr.D;
#pragma unroll 1
        for (int c = grp + 2 * set; c < HD / 32; c += 4) {
          float v[32];
          __syncwarp();  // lanes without a row left the last trip early
          if (n_iter > 0) {
            tc::tmem_ld32((which == 0 ? t_a1 : t_a2) + lane_off + c * 32, v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.f;  // a split without a share
          }
          if (!live) continue;
          if (sums == nullptr) {
            put_sums<T>(v, mul, (which == 0 ? dk : dv) + row * pr.D, c * 32, pr.D);
            continue;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c * 32 + 4 * i < pr.D)
              reinterpret_cast<float4*>(sums + c * 32)[i] = make_float4(
                  v[4 * i] * mul, v[4 * i + 1] * mul, v[4 * i + 2] * mul, v[4 * i + 3] * mul);
        }
      }
    }
  }
  // ------------------------------------------------------------ teardown
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

}  // namespace ragged
}  // namespace theria
