// Tensor-core (tcgen05) attention over packed sequences, backward: one kernel
// for both sides.  A CTA stays on a tile of 128 rows x1, x2 and walks over tiles
// of 64 rows y1, y2:
//     queries: x = (q, do), y = (k, v):    dq += ds k
//     keys:    x = (k, v),  y = (q, do):   dk += ds^T q, dv += p^T do
// with, per tile, s = x1 y1^T and dp = x2 y2^T, p = exp(scale s - lse) and
// ds = p (dp - z).  Seven products a pair of tiles instead of the five that one
// kernel for all three gradients needs; but then nothing is added atomically
// (the same bits every time), there is no float32 dq in HBM, and p and ds never
// leave the tensor memory: they overwrite s and dp in place as 16-bit pairs and
// are the A operands of the sums.
//
// The queries of the G heads that share a key head lie token by token in a
// tile of rows (as in the forward), so dk and dv sum over the group in TMEM.
//
//     warp 0       TMA producer; keys: also each tile's row terms
//     warps 1..4   one thread each issues s, dp, the sum of ds y1, that of p y2
//     warps 5..20  p and ds: eight warps take the even tiles, eight the odd ones, each
//                  32 rows (a TMEM lane quarter) by 32 of the 64 columns
// A hop from one of these to the next (a commit or an arrival, a wait that returns)
// takes a few hundred cycles, and so does a wait that finds its barrier passed: with
// two buffers the hops of the ring s -> p -> sum -> s set the pace unless each product
// is its own step with its own barrier and its own waiting thread.  Measured at 8192
// tokens of two sequences, 16 heads of 128: one issuing thread for all products
// 2640 / 1170 us (both sides / queries), two (s and dp, the sums) 2260 / 1010.
// TMEM: buffer b at [128 b, +64) s and [128 b + 64, +64) dp; the sums at 256 and
// 256 + HD; where there is room (queries, or HD = 64) x1 and x2 as 16-bit pairs
// at [384, ...): A operands from TMEM leave shared memory, which otherwise sets
// the pace (128 bytes a cycle), to the B operands.
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

constexpr int BX = 128, BY = 64;
constexpr int B_SET = 256;  // threads that make one tile's p and ds
constexpr int B_CTL = 5;    // control warps
constexpr int B_THREADS = 32 * B_CTL + 2 * B_SET;

template <int HD>
struct BwdCfg {
  static constexpr int kX = BX * HD * 2, kY = BY * HD * 2;  // one operand's tile
  static constexpr int YST = HD == 128 ? 4 : 6;             // ring depth
  static constexpr int oX1 = 0, oX2 = kX;
  static constexpr int oY1 = 2 * kX;              // [YST]
  static constexpr int oY2 = oY1 + YST * kY;      // [YST]
  static constexpr int oTerm = oY2 + YST * kY;    // [YST][2][64] floats
  static constexpr int oBar = oTerm + YST * BY * 8;
  // x_full, x_tmem, edge, drain[4], and per buffer s_full, s_free, dp_full, dp_free,
  // p_full, ds_full; y_full[], y_empty[]
  static constexpr int nBar = 7 + 12 + 2 * YST;
  static constexpr int oTmem = oBar + nBar * 8;
  static constexpr int oAbort = oTmem + 4;
  static constexpr int kAlloc = oAbort + 4 + 1024;
};

template <typename T, int HD, bool KEYS, bool CAUSAL>
__global__ void __launch_bounds__(B_THREADS, 1)
tc_bwd_kernel(const __grid_constant__ CUtensorMap tm_x1, const __grid_constant__ CUtensorMap tm_x2,
              const __grid_constant__ CUtensorMap tm_y1, const __grid_constant__ CUtensorMap tm_y2,
              const float2* terms, T* __restrict__ out1, T* __restrict__ out2, float* part,
              const int4* items, const int* count, const Problem pr) {
  using L = BwdCfg<HD>;
  constexpr int YST = L::YST;
  constexpr bool kXT = !KEYS || HD == 64;  // x in TMEM
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oBar);
  uint64_t *x_full = bars, *x_tmem = bars + 1, *edge = bars + 2, *drain = bars + 3;  // drain [4]
  uint64_t *s_full = bars + 7, *dp_full = bars + 9;    // products done
  uint64_t *p_full = bars + 11, *ds_full = bars + 13;  // pairs written (keys; both)
  // s's columns free: keys, when p y2 is done; queries, when the warps have read s
  uint64_t *s_free = bars + 15, *dp_free = bars + 17;  // dp's: when ds y1 is done
  uint64_t *y_full = bars + 19, *y_empty = y_full + YST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::oTmem);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::oAbort);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_wait();
  const int hk = blockIdx.x % pr.Hkv, at = blockIdx.x / pr.Hkv;
  if (at >= *count) return;
  const int4 item = items[at];
  const int start = item.x, len = item.y, first = item.z, G = pr.G;
  const int xt = KEYS ? BX : BX / G;   // tokens of an x tile
  const int yt = KEYS ? BY / G : BY;   // ... of a y tile
  const int y_rows = KEYS ? yt * G : BY;
  // y tokens [y_from, y_to), and this split's share of their tiles
  const int y_from = KEYS && CAUSAL ? first : 0;
  const int y_to = !KEYS && CAUSAL ? min(first + xt, len) : len;
  const int n_y = (y_to - y_from + yt - 1) / yt;
  const int t_at = (int)((int64_t)n_y * blockIdx.y / gridDim.y);
  const int n_iter = (int)((int64_t)n_y * (blockIdx.y + 1) / gridDim.y) - t_at;
  auto tok_of = [&](int t) { return y_from + (t_at + t) * yt; };  // tile t's first token

  if (threadIdx.x == 0) {
    tc::mbar_init(x_full, 1);
    tc::mbar_init(x_tmem, B_SET / 32);
    tc::mbar_init(edge, 1);
    for (int b = 0; b < 4; ++b) tc::mbar_init(drain + b, 1);
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(s_full + b, 1);
      tc::mbar_init(dp_full + b, 1);
      tc::mbar_init(p_full + b, B_SET / 32);  // a warp arrives once
      tc::mbar_init(ds_full + b, B_SET / 32);
      tc::mbar_init(s_free + b, KEYS ? 1 : B_SET / 32);
      tc::mbar_init(dp_free + b, 1);
    }
    for (int s = 0; s < YST; ++s) {
      tc::mbar_init(y_full + s, KEYS ? 2 : 1);  // the tile (and its row terms)
      tc::mbar_init(y_empty + s, KEYS ? 2 : 1);  // the sums (s and dp read it before)
    }
    *abort = 0;
    tc::fence_barrier_init();
  }
  if (warp == 1) tc::tmem_alloc(tmem_slot, 512);
  if (KEYS && y_rows < BY)  // rows that no copy fills
    for (int s = warp; s < 2 * YST; s += B_THREADS / 32)
      zero_rows(smem + L::oY1 + s * L::kY, BY, HD / 64, y_rows, BY, lane);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_a1 = tmem + 256, t_a2 = tmem + 256 + HD;
  const uint32_t t_x1 = tmem + 384, t_x2 = tmem + 384 + HD / 2;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (n_iter > 0) {
      if (lane == 0) {
        tc::prefetch_tmap(&tm_y1);
        tc::prefetch_tmap(&tm_y2);
        tc::mbar_expect_tx(x_full, 2 * (HD / 64) * (KEYS ? BX : xt * G) * 128);
        for (int cb = 0; cb < HD / 64; ++cb) {
          uint8_t *x1 = smem + L::oX1 + cb * BX * 128, *x2 = smem + L::oX2 + cb * BX * 128;
          if constexpr (KEYS) {
            tc::tma_load_3d(x1, &tm_x1, x_full, cb * 64, start + first, hk);
            tc::tma_load_3d(x2, &tm_x2, x_full, cb * 64, start + first, hk);
          } else {
            tma_load_rows(x1, &tm_x1, x_full, cb * 64, start + first, hk);
            tma_load_rows(x2, &tm_x2, x_full, cb * 64, start + first, hk);
          }
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
      if (KEYS) load_terms(0);
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
            if constexpr (KEYS) {
              tma_load_rows(y1 + cb * BY * 128, &tm_y1, full, cb * 64, start + tok, hk);
              tma_load_rows(y2 + cb * BY * 128, &tm_y2, full, cb * 64, start + tok, hk);
            } else {
              tc::tma_load_3d(y1 + cb * BY * 128, &tm_y1, full, cb * 64, start + tok, hk);
              tc::tma_load_3d(y2 + cb * BY * 128, &tm_y2, full, cb * 64, start + tok, hk);
            }
          }
        }
        if (KEYS) {
          float* rt = reinterpret_cast<float*>(smem + L::oTerm + st * BY * 8);
          rt[lane] = rv[0].x;
          rt[32 + lane] = rv[1].x;
          rt[BY + lane] = rv[0].y;
          rt[BY + 32 + lane] = rv[1].y;
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(y_full + st);
          if (t + 1 < n_iter) load_terms(t + 1);
        }
        if (ends) {
          if (!__all_sync(0xffffffffu, tc::mbar_wait(edge, 0, abort))) {
            tc::mbar_wait_drain(edge, 0);
            break;
          }
          const int live = (len - tok) * (KEYS ? G : 1);
          zero_rows(y1, BY, HD / 64, live, BY, lane);
          if (KEYS) zero_rows(y2, BY, HD / 64, live, BY, lane);
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
  } else if (warp < B_CTL) {
    // ------------------------------------------------------------ issuers
    if (lane == 0 && n_iter > 0 && (KEYS || warp != 4)) {
      constexpr int ab = tc::AbFmt<T>::v;
      if (warp <= 2) {
        // s = x1 y1^T (warp 1) or dp = x2 y2^T (warp 2)
        constexpr uint32_t id_s = tc::idesc_f16(BX, BY, ab, 0, 0);
        const bool is_s = warp == 1;
        const uint64_t x = tc::sw128_desc(tc::smem_u32(smem + (is_s ? L::oX1 : L::oX2)), 16, 1024);
        const uint64_t y = tc::sw128_desc(tc::smem_u32(smem + (is_s ? L::oY1 : L::oY2)), 16, 1024);
        const uint32_t t_x = is_s ? t_x1 : t_x2, t_d = tmem + (is_s ? 0 : 64);
        uint64_t *full = is_s ? s_full : dp_full, *free_ = is_s ? s_free : dp_free;
        const bool ok = tc::mbar_wait(kXT ? x_tmem : x_full, 0, abort);
        for (int t = 0; ok && t < n_iter; ++t) {
          const int st = t % YST, b = t & 1;
          if (!tc::mbar_wait(y_full + st, (t / YST) & 1, abort)) break;
          if (t >= 2 && !tc::mbar_wait(free_ + b, ((t >> 1) - 1) & 1, abort)) break;
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint64_t yd =
                tc::desc_at(y, st * L::kY + (kk / 4) * (BY * 128) + (kk % 4) * 32);
            if constexpr (kXT)
              tc::mma_ts(t_d + b * 128, t_x + kk * 8, yd, id_s, kk > 0 ? 1u : 0u);
            else
              tc::mma_ss(t_d + b * 128, tc::desc_at(x, (kk / 4) * (BX * 128) + (kk % 4) * 32), yd,
                         id_s, kk > 0 ? 1u : 0u);
          }
          tc::mma_commit(full + b);
        }
      } else {
        // the sums of ds y1 (warp 3) or p y2 (warp 4), the tile's rows as contraction
        constexpr uint32_t id_a = tc::idesc_f16(BX, HD, ab, 0, 1);
        const bool is_ds = warp == 3;
        const uint64_t y =
            tc::sw128_desc(tc::smem_u32(smem + (is_ds ? L::oY1 : L::oY2)), BY * 128, 1024);
        const uint32_t t_d = is_ds ? t_a1 : t_a2, t_p = tmem + (is_ds ? 64 : 0);
        uint64_t* full = is_ds ? ds_full : p_full;
        for (int t = 0; t < n_iter; ++t) {
          const int st = t % YST, b = t & 1;
          if (!tc::mbar_wait(full + b, (t >> 1) & 1, abort)) break;
          tc::tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < BY / 16; ++kk)
            // 16 columns of the tile: 8 TMEM columns of pairs, in the half of the
            // warps that wrote them
            tc::mma_ts(t_d, t_p + b * 128 + (kk / 2) * 32 + (kk % 2) * 8,
                       tc::desc_at(y, st * L::kY + kk * 2048), id_a, t > 0 || kk > 0 ? 1u : 0u);
          if (is_ds) tc::mma_commit(dp_free + b);
          else tc::mma_commit(s_free + b);
          tc::mma_commit(y_empty + st);
        }
      }
      tc::mma_commit(drain + warp - 1);
      tc::mbar_wait_drain(drain + warp - 1, 0);
    }
  } else {
    // ------------------------------------------------------------ p and ds
    const int grp = ((warp - B_CTL) >> 2) & 1, quarter = warp & 3, set = (warp - B_CTL) >> 3;
    const int r = quarter * 32 + lane;  // TMEM lane: the row of x
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int tok = first + (KEYS ? r : r / G);      // its token
    const bool live = tok < len && (KEYS || r < xt * G);
    const float scale_log2 = pr.scale * kLog2e;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, abort));
    };
    if (kXT && set == 0 && n_iter > 0) {
      // this row of x1 (group 0) or x2 (group 1) into TMEM: the 128-byte
      // swizzled row of 64 values is 32 pairs, one a column
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
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(x_tmem);
      }
    }
    float2 mine = make_float2(-INFINITY, 0.f);  // queries: this row's terms
    if (!KEYS && live) mine = terms[(int64_t)(start + tok) * pr.H + hk * G + r % G];
    const int warp_tok = first + quarter * 32 / G;  // queries: the first token of the warp
    for (int t = set; ok && t < n_iter; t += 2) {
      const int b = set, st = t % YST, y0 = tok_of(t);
      const uint32_t t_s = tmem + b * 128 + grp * 32 + lane_off;
      if (KEYS && !wait(y_full + st, (t / YST) & 1)) { ok = false; break; }  // the terms
      if (!wait(s_full + b, (t >> 1) & 1)) { ok = false; break; }
      tc::tc_fence_after();
      // Tiles on the diagonal and (queries) at the sequence's end need a mask; the
      // test is the same for a whole warp.  Valid: columns from `lo` on (keys), or
      // below `hi` (queries).
      bool masked;
      int lo = 0, hi = 32;
      if constexpr (KEYS) {
        masked = CAUSAL && y0 < first + BX;
        lo = (tok - y0) * G - grp * 32;
      } else {
        masked = y0 + BY > len || (CAUSAL && y0 + BY - 1 > warp_tok);
        hi = (CAUSAL ? min(len, tok + 1) : len) - y0 - grp * 32;
      }
      // the row terms of this warp's columns: all -lse log2 e of a tile, then all -z
      const uint32_t lse_at = tc::smem_u32(smem + L::oTerm + st * BY * 8) + grp * 32 * 4;
      const uint32_t z_at = lse_at + BY * 4;
      float s[32];
      tc::tmem_ld32(t_s, s);
      if constexpr (!KEYS) {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(s_free + b);
      }
      auto on = [&](int e) { return KEYS ? e >= lo : e < hi; };
      // p = exp2(scale s - lse); rows past the end of y: exp2(-inf) = 0
      auto make_p = [&](auto mk) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float nl0 = mine.x, nl1 = mine.x;
          if constexpr (KEYS) {
            const float2 rr = ld_shared_f2(lse_at + e * 4);
            nl0 = rr.x;
            nl1 = rr.y;
          }
          tc::fma2(s[e], s[e + 1], s[e], s[e + 1], scale_log2, scale_log2, nl0, nl1);
          s[e] = tc::ex2(s[e]);
          s[e + 1] = tc::ex2(s[e + 1]);
          if constexpr (decltype(mk)::value) {
            s[e] = on(e) ? s[e] : 0.f;
            s[e + 1] = on(e + 1) ? s[e + 1] : 0.f;
          }
        }
      };
      if (masked) make_p(std::true_type{}); else make_p(std::false_type{});
      uint32_t pk[16];  // 16-bit pairs
      if constexpr (KEYS) {
#pragma unroll
        for (int i = 0; i < 16; ++i) pk[i] = tc::pack2<T>(s[2 * i], s[2 * i + 1]);
        tc::tmem_st16(t_s, pk);
        tc::tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full + b);
      }
      if (!wait(dp_full + b, (t >> 1) & 1)) { ok = false; break; }
      tc::tc_fence_after();
      float dp[32];
      tc::tmem_ld32(t_s + 64, dp);
      // ds = p (dp - z)
      auto make_ds = [&](auto mk) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float nz0 = mine.y, nz1 = mine.y, g0, g1;
          if constexpr (KEYS) {
            const float2 rr = ld_shared_f2(z_at + e * 4);
            nz0 = rr.x;
            nz1 = rr.y;
          }
          tc::add2(g0, g1, dp[e], dp[e + 1], nz0, nz1);
          tc::mul2(g0, g1, s[e], s[e + 1], g0, g1);
          if constexpr (decltype(mk)::value) {
            g0 = on(e) ? g0 : 0.f;
            g1 = on(e + 1) ? g1 : 0.f;
          }
          pk[e / 2] = tc::pack2<T>(g0, g1);
        }
      };
      if (masked) make_ds(std::true_type{}); else make_ds(std::false_type{});
      tc::tmem_st16(t_s + 64, pk);
      tc::tmem_wait_st();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(ds_full + b);
    }
    // ------------------------------------------------------------ results
    if (ok && n_iter > 0) {
      ok = wait(drain + 2, 0) && (!KEYS || wait(drain + 3, 0));  // the sums are complete
      if (ok) tc::tc_fence_after();
    }
    if (ok) {
      const int64_t row = KEYS ? (int64_t)(start + tok) * pr.Hkv + hk
                               : (int64_t)(start + tok) * pr.H + hk * G + r % G;
      const int64_t plane = (int64_t)pr.T * pr.Hkv * pr.D;
#pragma unroll 1
      for (int which = 0; which < (KEYS ? 2 : 1); ++which) {
        const float mul = which == 0 ? pr.scale : 1.f;
        T* out = which == 0 ? out1 : out2;
        float* sums = part == nullptr ? nullptr : part + (2 * blockIdx.y + which) * plane;
#pragma unroll 1
        for (int c = grp + 2 * set; c < HD / 32; c += 4) {
          float v[32];
          if (n_iter > 0) {
            tc::tmem_ld32((which == 0 ? t_a1 : t_a2) + lane_off + c * 32, v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.f;  // a split without a share
          }
          if (!live) continue;
          const int64_t to = row * pr.D + c * 32;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float* e = v + 8 * i;
            if (c * 32 + 8 * i >= pr.D) continue;  // D is a multiple of 8
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] *= mul;
            if (sums != nullptr) {
              float4* d4 = reinterpret_cast<float4*>(sums + to) + 2 * i;
              d4[0] = make_float4(e[0], e[1], e[2], e[3]);
              d4[1] = make_float4(e[4], e[5], e[6], e[7]);
            } else {
              reinterpret_cast<uint4*>(out + to)[i] =
                  make_uint4(tc::pack2<T>(e[0], e[1]), tc::pack2<T>(e[2], e[3]),
                             tc::pack2<T>(e[4], e[5]), tc::pack2<T>(e[6], e[7]));
            }
          }
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
