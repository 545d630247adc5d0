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
//     warp 1       issues s and dp into one of two buffers
//     warp 2       issues the sums
//     warps 3..10  p and ds, two groups on 32 of a tile's 64 columns each
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

constexpr int BX = 128, BY = 64;
constexpr int B_COMPUTE = 256, B_THREADS = 96 + B_COMPUTE;

template <int HD>
struct BwdCfg {
  static constexpr int kX = BX * HD * 2, kY = BY * HD * 2;  // one operand's tile
  static constexpr int YST = HD == 128 ? 4 : 6;             // ring depth
  static constexpr int oX1 = 0, oX2 = kX;
  static constexpr int oY1 = 2 * kX;              // [YST]
  static constexpr int oY2 = oY1 + YST * kY;      // [YST]
  static constexpr int oTerm = oY2 + YST * kY;    // [YST][64] float2
  static constexpr int oBar = oTerm + YST * BY * 8;
  // x_full, x_tmem, edge, drain[2], s_full[2], p_full[2], done[2], y_full[], y_empty[]
  static constexpr int nBar = 11 + 2 * YST;
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
  uint64_t *x_full = bars, *x_tmem = bars + 1, *edge = bars + 2, *drain = bars + 3;
  uint64_t *s_full = bars + 5, *p_full = bars + 7, *done = bars + 9;
  uint64_t *y_full = bars + 11, *y_empty = y_full + YST;
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
    tc::mbar_init(x_tmem, B_COMPUTE);
    tc::mbar_init(edge, 1);
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(drain + b, 1);
      tc::mbar_init(s_full + b, 1);
      tc::mbar_init(p_full + b, B_COMPUTE);
      tc::mbar_init(done + b, 1);
    }
    for (int s = 0; s < YST; ++s) {
      tc::mbar_init(y_full + s, KEYS ? 2 : 1);  // the tile (and its row terms)
      tc::mbar_init(y_empty + s, 1);
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
          float2* rt = reinterpret_cast<float2*>(smem + L::oTerm + st * BY * 8);
          rt[lane] = rv[0];
          rt[32 + lane] = rv[1];
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
  } else if (warp == 1 || warp == 2) {
    // ------------------------------------------------------------ issuers
    if (lane == 0 && n_iter > 0) {
      constexpr int ab = tc::AbFmt<T>::v;
      const uint32_t a_y1 = tc::smem_u32(smem + L::oY1), a_y2 = tc::smem_u32(smem + L::oY2);
      if (warp == 1) {
        constexpr uint32_t id_s = tc::idesc_f16(BX, BY, ab, 0, 0);
        const uint64_t x1 = tc::sw128_desc(tc::smem_u32(smem + L::oX1), 16, 1024);
        const uint64_t x2 = tc::sw128_desc(tc::smem_u32(smem + L::oX2), 16, 1024);
        const uint64_t y1 = tc::sw128_desc(a_y1, 16, 1024), y2 = tc::sw128_desc(a_y2, 16, 1024);
        bool ok = kXT ? tc::mbar_wait(x_tmem, 0, abort) : tc::mbar_wait(x_full, 0, abort);
        for (int t = 0; ok && t < n_iter; ++t) {
          const int st = t % YST, b = t & 1;
          if (!tc::mbar_wait(y_full + st, (t / YST) & 1, abort)) break;
          if (t >= 2 && !tc::mbar_wait(done + b, ((t >> 1) - 1) & 1, abort)) break;
          tc::tc_fence_after();
          const uint32_t t_s = tmem + b * 128;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t xo = (kk / 4) * (BX * 128) + (kk % 4) * 32;
            const uint32_t yo = st * L::kY + (kk / 4) * (BY * 128) + (kk % 4) * 32;
            if constexpr (kXT) {
              tc::mma_ts(t_s, t_x1 + kk * 8, tc::desc_at(y1, yo), id_s, kk > 0 ? 1u : 0u);
              tc::mma_ts(t_s + 64, t_x2 + kk * 8, tc::desc_at(y2, yo), id_s, kk > 0 ? 1u : 0u);
            } else {
              tc::mma_ss(t_s, tc::desc_at(x1, xo), tc::desc_at(y1, yo), id_s, kk > 0 ? 1u : 0u);
              tc::mma_ss(t_s + 64, tc::desc_at(x2, xo), tc::desc_at(y2, yo), id_s,
                         kk > 0 ? 1u : 0u);
            }
          }
          tc::mma_commit(s_full + b);
        }
      } else {
        constexpr uint32_t id_a = tc::idesc_f16(BX, HD, ab, 0, 1);
        const uint64_t y1 = tc::sw128_desc(a_y1, BY * 128, 1024);
        const uint64_t y2 = tc::sw128_desc(a_y2, BY * 128, 1024);
        for (int t = 0; t < n_iter; ++t) {
          const int st = t % YST, b = t & 1;
          if (!tc::mbar_wait(p_full + b, (t >> 1) & 1, abort)) break;
          tc::tc_fence_after();
          const uint32_t t_p = tmem + b * 128;
#pragma unroll
          for (int kk = 0; kk < BY / 16; ++kk) {
            // 16 columns of the tile: 8 TMEM columns of pairs, in the half of the
            // group that wrote them
            const uint32_t po = (kk / 2) * 32 + (kk % 2) * 8, yo = st * L::kY + kk * 2048;
            const uint32_t acc = t > 0 || kk > 0 ? 1u : 0u;
            tc::mma_ts(t_a1, t_p + 64 + po, tc::desc_at(y1, yo), id_a, acc);
            if constexpr (KEYS) tc::mma_ts(t_a2, t_p + po, tc::desc_at(y2, yo), id_a, acc);
          }
          tc::mma_commit(done + b);
          tc::mma_commit(y_empty + st);  // s and dp of the tile read it before
        }
      }
      tc::mma_commit(drain + warp - 1);
      tc::mbar_wait_drain(drain + warp - 1, 0);
    }
  } else {
    // ------------------------------------------------------------ p and ds
    const int grp = (warp - 3) >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;  // TMEM lane: the row of x
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int tok = first + (KEYS ? r : r / G);      // its token
    const bool live = tok < len && (KEYS || r < xt * G);
    const float scale_log2 = pr.scale * kLog2e;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, abort));
    };
    if (kXT && n_iter > 0) {
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
        tc::mbar_arrive(x_tmem);
      }
    }
    float2 mine = make_float2(-INFINITY, 0.f);  // queries: this row's terms
    if (!KEYS && live) mine = terms[(int64_t)(start + tok) * pr.H + hk * G + r % G];
    const int warp_tok = first + quarter * 32 / G;  // queries: the first token of the warp
    for (int t = 0; ok && t < n_iter; ++t) {
      const int b = t & 1, st = t % YST, y0 = tok_of(t);
      const uint32_t t_s = tmem + b * 128 + grp * 32 + lane_off;
      if (KEYS && !wait(y_full + st, (t / YST) & 1)) { ok = false; break; }  // the terms
      if (!wait(s_full + b, (t >> 1) & 1)) { ok = false; break; }
      tc::tc_fence_after();
      float s[32], dp[32];
      tc::tmem_ld32(t_s, s);
      tc::tmem_ld32(t_s + 64, dp);
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
      const uint32_t rows_at = tc::smem_u32(smem + L::oTerm + st * BY * 8) + grp * 32 * 8;
      auto make = [&](auto mk) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float nl0, nl1, nz0, nz1;
          if constexpr (KEYS) {
            const float4 rr = tc::ld_shared_f4(rows_at + e * 8);
            nl0 = rr.x; nz0 = rr.y; nl1 = rr.z; nz1 = rr.w;
          } else {
            nl0 = nl1 = mine.x;
            nz0 = nz1 = mine.y;
          }
          float x0, x1, g0, g1;
          tc::fma2(x0, x1, s[e], s[e + 1], scale_log2, scale_log2, nl0, nl1);
          float p0 = tc::ex2(x0), p1 = tc::ex2(x1);
          tc::add2(g0, g1, dp[e], dp[e + 1], nz0, nz1);
          tc::mul2(g0, g1, p0, p1, g0, g1);
          if constexpr (decltype(mk)::value) {
            const bool on0 = KEYS ? e >= lo : e < hi, on1 = KEYS ? e + 1 >= lo : e + 1 < hi;
            p0 = on0 ? p0 : 0.f;
            p1 = on1 ? p1 : 0.f;
            g0 = on0 ? g0 : 0.f;
            g1 = on1 ? g1 : 0.f;
          }
          s[e] = p0;
          s[e + 1] = p1;
          dp[e] = g0;
          dp[e + 1] = g1;
        }
      };
      if (masked) make(std::true_type{}); else make(std::false_type{});
      uint32_t pk[16];
      if constexpr (KEYS) {
#pragma unroll
        for (int i = 0; i < 16; ++i) pk[i] = tc::pack2<T>(s[2 * i], s[2 * i + 1]);
        tc::tmem_st16(t_s, pk);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) pk[i] = tc::pack2<T>(dp[2 * i], dp[2 * i + 1]);
      tc::tmem_st16(t_s + 64, pk);
      tc::tmem_wait_st();
      tc::tc_fence_before();
      tc::mbar_arrive(p_full + b);
    }
    // ------------------------------------------------------------ results
    if (ok && n_iter > 0) {
      const int tl = n_iter - 1;
      ok = wait(done + (tl & 1), (tl >> 1) & 1);
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
        for (int c = grp * (HD / 64); c < (grp + 1) * (HD / 64); ++c) {
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
