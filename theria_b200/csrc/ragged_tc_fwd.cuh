// Tensor-core (tcgen05) attention over packed sequences, forward: bf16/fp16,
// head widths up to 64 (HD = 64) or 128 (narrower heads are filled up with
// zeros by TMA, which costs products but no bytes).
//
// A CTA owns two tiles of up to 128 rows of one key head and sequence (rows:
// tokens x the G query heads that share the key head, token by token; a 4-D
// TMA box {64 values, G heads, 128 / G tokens} brings them in that order) and
// streams that sequence's keys in tiles of 128 through a 2-stage ring.  The
// tiles alternate on the tensor core, so that one's softmax runs while the
// other's products do:
//     warp 0       TMA producer
//     warp 1       issues S_t = Q_t K^T (HD = 128: and O_t += P_t V)
//     warp 2       HD = 64: issues O_t += P_t V
//     16 (HD = 128) or 8 softmax warps, by TMEM lane quarter, tile and, for
//     HD = 128, half of the key columns
// TMEM: S_t [128 t, +128), O_t [256 + t HD, +HD); P_t (16-bit pairs) over S_t's
// own columns, for HD = 64 in [384 + 64 t, +64).  Softmax in the log2 domain,
// O and the sum rescaled only when the maximum grows by more than 2^8.  These
// choices, and what was measured for them, are the dense forward's
// (sdpa_tc_fwd.cuh); what differs is where rows and keys come from and end.
// P is rounded to 16 bits, as the tensor core's operand, after its sum was taken.
//
// Keys behind the sequence's end belong to the next one and may be anything.
// Their scores are masked; their rows of V, which p = 0 would multiply, are set
// to zero in shared memory by the producer warp, once per CTA (NaN * 0 is NaN).
#pragma once

#include "pair_exchange.cuh"
#include "ragged_plan.cuh"
#include "tc_common.cuh"

namespace theria {
namespace ragged {

// 4-D tiled load of box {64, G, tokens, 1} at (x, 0, token, key head); x is 0 or 64.
__device__ __forceinline__ void tma_load_rows(void* dst, const CUtensorMap* map, uint64_t* bar,
                                              int x, int token, int hk) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(tc::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(tc::smem_u32(bar)), "r"(x), "r"(0), "r"(token),
      "r"(hk)
      : "memory");
}

// Zeros rows [from, to) of an operand of `rows` rows and `blocks` 64-wide blocks
// in shared memory, by one warp, visible to the tensor core.
__device__ __forceinline__ void zero_rows(uint8_t* tile, int rows, int blocks, int from, int to,
                                          int lane) {
  for (int cb = 0; cb < blocks; ++cb) {
    uint4* p = reinterpret_cast<uint4*>(tile + (cb * rows + from) * 128);
    for (int i = lane; i < (to - from) * 8; i += 32) p[i] = make_uint4(0, 0, 0, 0);
  }
  tc::fence_proxy_async_smem();
}

// 16 values as pairs to `to` (8 where only those lie within the row): a whole sector of
// 32 bytes at once where rows start on such boundaries (`wide`).  A thread has a row of
// its own, so two stores of 16 bytes are two half sectors each for 32 rows: the forward
// with o and what its rounding left, 8192 tokens, 16 heads of 128, 328 us, so 310
// (causal 181, 168).
__device__ __forceinline__ void store16(void* to, const uint32_t (&w)[8], bool wide, bool second) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]),
                 "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    static_cast<uint4*>(to)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    if (second) static_cast<uint4*>(to)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}
__device__ __forceinline__ bool wide_rows(const void* p, int D) {
  return D % 16 == 0 && (reinterpret_cast<uintptr_t>(p) & 31) == 0;
}

constexpr int FM = 128, FN = 128, FST = 2;  // rows of a tile, keys of a tile, ring depth
constexpr float kRescale = 8.f;             // log2 units

template <int HD>
struct FwdCfg {
  static constexpr int kHalves = HD == 64 ? 1 : 2;
  static constexpr int kCtl = HD == 64 ? 3 : 2;
  static constexpr int kThreads = 32 * (kCtl + 8 * kHalves);
  static constexpr int kQ = FM * HD * 2, kKV = FN * HD * 2;
  static constexpr int oQ = 0;
  static constexpr int oK = oQ + 2 * kQ;
  static constexpr int oV = oK + FST * kKV;
  static constexpr int oRed = oV + FST * kKV;  // the halves' row maxima and sums
  static constexpr int oBar = oRed + 2 * 2 * 2 * FM * 4;
  // q_full, edge, k_full[S], v_full[S], k_empty[S], v_empty[S], s_full[2], p_full[2],
  // o_done[2], s_read[2], pv_done[2], drain[2]
  static constexpr int nBar = 2 + 4 * FST + 12;
  static constexpr int oTmem = oBar + nBar * 8;
  static constexpr int oAbort = oTmem + 4;
  static constexpr int kAlloc = oAbort + 4 + 1024;  // slack to align the base to 1024
};

template <typename T, int HD, bool CAUSAL>
__global__ void __launch_bounds__(FwdCfg<HD>::kThreads, 1)
tc_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
              const __grid_constant__ CUtensorMap tm_v, T* __restrict__ out,
              T* __restrict__ rest, float* __restrict__ lse, const int4* items, const int* count,
              const Problem pr) {
  using L = FwdCfg<HD>;
  constexpr bool kSepP = HD == 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::oBar);
  uint64_t* q_full = bars;
  uint64_t* edge = bars + 1;       // the V tile at the sequence's end landed
  uint64_t* k_full = bars + 2;
  uint64_t* v_full = k_full + FST;
  uint64_t* k_empty = v_full + FST;
  uint64_t* v_empty = k_empty + FST;
  uint64_t* s_full = v_empty + FST;  // [2] per tile, as the following
  uint64_t* p_full = s_full + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* s_read = o_done + 2;   // HD = 64: S_t in registers
  uint64_t* pv_done = s_read + 2;  // HD = 64: P_t and O_t free
  uint64_t* drain = pv_done + 2;   // [2] per issuing warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::oTmem);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + L::oAbort);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_wait();
  const int hk = blockIdx.x % pr.Hkv, at = blockIdx.x / pr.Hkv;
  if (at >= *count) return;
  const int4 item = items[at];
  const int start = item.x, len = item.y, first = item.z, G = pr.G;
  const int tpt = FM / G;  // tokens of a tile
  // key tiles that tile t needs; 0: the tile has no rows
  auto tiles_of = [&](int t) {
    const int a = first + t * tpt;
    if (a >= len) return 0;
    return ((CAUSAL ? min(a + tpt, len) : len) + FN - 1) / FN;
  };
  const int n0 = tiles_of(0), n1 = tiles_of(1), n_tiles = max(n0, n1);

  if (threadIdx.x == 0) {
    tc::mbar_init(q_full, 1);
    tc::mbar_init(edge, 1);
    for (int s = 0; s < FST; ++s) {
      tc::mbar_init(k_full + s, 1);
      tc::mbar_init(v_full + s, 1);
      tc::mbar_init(k_empty + s, 1);
      tc::mbar_init(v_empty + s, 1);
    }
    for (int t = 0; t < 2; ++t) {
      tc::mbar_init(s_full + t, 1);
      tc::mbar_init(p_full + t, 4 * L::kHalves);  // a warp arrives once
      tc::mbar_init(o_done + t, 1);
      tc::mbar_init(s_read + t, 4 * L::kHalves);
      tc::mbar_init(pv_done + t, 1);
      tc::mbar_init(drain + t, 1);
    }
    *abort = 0;
    tc::fence_barrier_init();
  }
  if (warp == 1) tc::tmem_alloc(tmem_slot, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    // K and V stages are released separately: K_j once the S products of both
    // tiles are done, a step before V_j.
    const int edge_tile = len % FN ? len / FN : -1;  // its rows from len % FN on are others'
    if (lane == 0) {
      tc::prefetch_tmap(&tm_q);
      tc::prefetch_tmap(&tm_k);
      tc::prefetch_tmap(&tm_v);
      const int live = n1 > 0 ? 2 : 1;
      tc::mbar_expect_tx(q_full, live * (HD / 64) * tpt * G * 128);
      for (int t = 0; t < live; ++t)
        for (int cb = 0; cb < HD / 64; ++cb)
          tma_load_rows(smem + L::oQ + t * L::kQ + cb * FM * 128, &tm_q, q_full, cb * 64,
                        start + first + t * tpt, hk);
    }
    int k_issued = 0, v_issued = 0;
    for (int j = 0; j < n_tiles; ++j) {
      const int st = j % FST;
      bool ok = true;
      if (lane == 0 && j >= FST) ok = tc::mbar_wait(k_empty + st, ((j / FST) - 1) & 1, abort);
      if (!__shfl_sync(0xffffffffu, ok, 0)) break;
      if (lane == 0) {
        tc::mbar_expect_tx(k_full + st, L::kKV);
        for (int cb = 0; cb < HD / 64; ++cb)
          tc::tma_load_3d(smem + L::oK + st * L::kKV + cb * FN * 128, &tm_k, k_full + st, cb * 64,
                          start + j * FN, hk);
      }
      k_issued = j + 1;
      if (lane == 0 && j >= FST) ok = tc::mbar_wait(v_empty + st, ((j / FST) - 1) & 1, abort);
      if (!__shfl_sync(0xffffffffu, ok, 0)) break;
      uint64_t* full = j == edge_tile ? edge : v_full + st;
      uint8_t* v = smem + L::oV + st * L::kKV;
      if (lane == 0) {
        tc::mbar_expect_tx(full, L::kKV);
        for (int cb = 0; cb < HD / 64; ++cb)
          tc::tma_load_3d(v + cb * FN * 128, &tm_v, full, cb * 64, start + j * FN, hk);
      }
      if (j == edge_tile) {
        if (!__all_sync(0xffffffffu, tc::mbar_wait(edge, 0, abort))) {
          tc::mbar_wait_drain(edge, 0);
          break;
        }
        zero_rows(v, FN, HD / 64, len % FN, FN, lane);
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(v_full + st);
      }
      v_issued = j + 1;
    }
    // Every copy issued into this CTA's shared memory lands before it may exit
    // (bounded; returns at once on the normal path).
    if (lane == 0) {
      tc::mbar_wait_drain(q_full, 0);
      for (int j = k_issued > FST ? k_issued - FST : 0; j < k_issued; ++j)
        tc::mbar_wait_drain(k_full + j % FST, (j / FST) & 1);
      for (int j = v_issued > FST ? v_issued - FST : 0; j < v_issued; ++j)
        tc::mbar_wait_drain(v_full + j % FST, (j / FST) & 1);
    }
  } else if (kSepP && (warp == 1 || warp == 2)) {
    // ------------------------------------------------------------ issuers (HD = 64)
    if (lane == 0) {
      constexpr uint32_t id_s = tc::idesc_f16(FM, FN, tc::AbFmt<T>::v, 0, 0);
      constexpr uint32_t id_pv = tc::idesc_f16(FM, HD, tc::AbFmt<T>::v, 0, 1);
      bool ok = true;
      if (warp == 1) {
        const uint64_t dq0 = tc::sw128_desc(tc::smem_u32(smem + L::oQ), 16, 1024);
        const uint64_t dk0 = tc::sw128_desc(tc::smem_u32(smem + L::oK), 16, 1024);
        ok = tc::mbar_wait(q_full, 0, abort);
        for (int j = 0; ok && j < n_tiles; ++j) {
          const int st = j % FST;
          if (!tc::mbar_wait(k_full + st, (j / FST) & 1, abort)) break;
          const uint64_t dk = tc::desc_at(dk0, st * L::kKV);
          for (int t = 0; t < 2; ++t) {
            if (j >= (t ? n1 : n0)) continue;
            if (j >= 1 && !tc::mbar_wait(s_read + t, (j - 1) & 1, abort)) { ok = false; break; }
            tc::tc_fence_after();
            const uint64_t dq = tc::desc_at(dq0, t * L::kQ);
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              tc::mma_ss(tmem + t * 128, tc::desc_at(dq, kk * 32), tc::desc_at(dk, kk * 32), id_s,
                         kk > 0 ? 1u : 0u);
            tc::mma_commit(s_full + t);
          }
          if (!ok) break;
          tc::mma_commit(k_empty + st);
        }
      } else {
        const uint64_t dv0 = tc::sw128_desc(tc::smem_u32(smem + L::oV), FN * 128, 1024);
        for (int j = 0; ok && j < n_tiles; ++j) {
          const int st = j % FST;
          if (!tc::mbar_wait(v_full + st, (j / FST) & 1, abort)) break;
          const uint64_t dv = tc::desc_at(dv0, st * L::kKV);
          for (int t = 0; t < 2; ++t) {
            const int nt = t ? n1 : n0;
            if (j >= nt) continue;
            if (!tc::mbar_wait(p_full + t, j & 1, abort)) { ok = false; break; }
            tc::tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < FN / 16; ++kk)
              tc::mma_ts(tmem + 256 + t * HD, tmem + 384 + t * 64 + kk * 8,
                         tc::desc_at(dv, kk * 2048), id_pv, (j > 0 || kk > 0) ? 1u : 0u);
            tc::mma_commit(pv_done + t);
            if (j + 1 == nt) tc::mma_commit(o_done + t);
          }
          if (!ok) break;
          tc::mma_commit(v_empty + st);
        }
      }
      tc::mma_commit(drain + warp - 1);
      tc::mbar_wait_drain(drain + warp - 1, 0);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ issuer (HD = 128)
    if (lane == 0) {
      constexpr uint32_t id_s = tc::idesc_f16(FM, FN, tc::AbFmt<T>::v, 0, 0);
      constexpr uint32_t id_pv = tc::idesc_f16(FM, HD, tc::AbFmt<T>::v, 0, 1);
      const uint64_t dq0 = tc::sw128_desc(tc::smem_u32(smem + L::oQ), 16, 1024);
      const uint64_t dk0 = tc::sw128_desc(tc::smem_u32(smem + L::oK), 16, 1024);
      const uint64_t dv0 = tc::sw128_desc(tc::smem_u32(smem + L::oV), FN * 128, 1024);
      auto last_of = [&](int j) { return j < n1 ? 1 : 0; };  // the last tile to use K_j, V_j
      auto issue_s = [&](int t, int j) {
        const uint64_t dq = tc::desc_at(dq0, t * L::kQ);
        const uint64_t dk = tc::desc_at(dk0, (j % FST) * L::kKV);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          tc::mma_ss(tmem + t * 128, tc::desc_at(dq, (kk / 4) * (FM * 128) + (kk % 4) * 32),
                     tc::desc_at(dk, (kk / 4) * (FN * 128) + (kk % 4) * 32), id_s,
                     kk > 0 ? 1u : 0u);
        tc::mma_commit(s_full + t);
        if (t == last_of(j)) tc::mma_commit(k_empty + j % FST);
      };
      bool ok = tc::mbar_wait(q_full, 0, abort) && tc::mbar_wait(k_full, 0, abort);
      if (ok) {
        tc::tc_fence_after();
        issue_s(0, 0);
        if (n1 > 0) issue_s(1, 0);
      }
      for (int j = 0; ok && j < n_tiles; ++j) {
        const int st = j % FST;
        const uint64_t dv = tc::desc_at(dv0, st * L::kKV);
        // operand waits first: each costs this thread a few hundred cycles, which
        // must not sit between a softmax publishing P and the products that use it
        if (!tc::mbar_wait(v_full + st, (j / FST) & 1, abort)) break;
        if (j + 1 < n_tiles && !tc::mbar_wait(k_full + (j + 1) % FST, ((j + 1) / FST) & 1, abort))
          break;
        for (int t = 0; t < 2; ++t) {
          const int nt = t ? n1 : n0;
          if (j >= nt) continue;
          if (!tc::mbar_wait(p_full + t, j & 1, abort)) { ok = false; break; }
          tc::tc_fence_after();
          // P_t: keys 64.. start at the second half's S columns
#pragma unroll
          for (int kk = 0; kk < FN / 16; ++kk)
            tc::mma_ts(tmem + 256 + t * HD, tmem + t * 128 + (kk / 4) * 64 + (kk % 4) * 8,
                       tc::desc_at(dv, kk * 2048), id_pv, (j > 0 || kk > 0) ? 1u : 0u);
          if (j + 1 == nt) tc::mma_commit(o_done + t);
          if (t == last_of(j)) tc::mma_commit(v_empty + st);
          if (j + 1 < nt) issue_s(t, j + 1);
        }
      }
      tc::mma_commit(drain);
      tc::mbar_wait_drain(drain, 0);
    }
  } else {
    // ------------------------------------------------------------ softmax
    constexpr int kHalves = L::kHalves;
    constexpr int CW = FN / kHalves;      // key columns of a warp
    const int idx = warp - L::kCtl;
    const int t = idx / (4 * kHalves);
    const int h = kHalves == 2 ? (idx >> 2) & 1 : 0;
    const int quarter = warp & 3;         // TMEM lanes this warp may access
    const int r = quarter * 32 + lane;    // row within the tile
    const int tok0 = first + t * tpt;
    const uint32_t bar_id = 1 + t * 4 + quarter;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_s = tmem + t * 128 + h * CW + lane_off;
    constexpr int HO = HD / kHalves;      // O columns this warp rescales and stores
    const uint32_t t_o = tmem + 256 + t * HD + h * HO + lane_off;
    const uint32_t t_p = (kSepP ? tmem + 384 + t * 64 : tmem + t * 128 + h * 64) + lane_off;
    float* red = reinterpret_cast<float*>(smem + L::oRed);  // [2 parity][2 t][2 h][128]
    auto red_at = [&](int par, int hh) { return red + ((par * 2 + t) * 2 + hh) * FM + r; };
    auto meet = [&] { tc::named_bar(bar_id, 64); };  // the two halves' warps
    static_assert(kHalves == 1 || !kSepP, "two halves: no wait but s_full's ends the loop");
    // the keys of this row, and of the warp's first: tiles beyond those need the mask
    const int my_keys = CAUSAL ? min(len, tok0 + r / G + 1) : len;
    const int clean = CAUSAL ? min(len, tok0 + quarter * 32 / G + 1) : len;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    // Waits are warp-uniform: the TMEM accesses that follow are warp-collective.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, abort));
    };
    const int nt = t ? n1 : n0;
    for (int j = 0; j < nt; ++j) {
      if (!wait(s_full + t, j & 1)) {
        ok = false;
        if constexpr (kHalves == 2) {  // tell the other half
          float none;
          tc::pair_exchange(red_at(j & 1, h), red_at(j & 1, h ^ 1), false, 0.f, none, meet);
        }
        break;
      }
      tc::tc_fence_after();
      const int col0 = j * FN + h * CW;
      const bool masked = col0 + CW > clean;
      const int lim = my_keys - col0;  // valid columns < lim
      float v[CW];
      if constexpr (CW == 128) tc::tmem_ld128(t_s, v);
      else tc::tmem_ld64(t_s, v);  // for the row maximum only
      if constexpr (kSepP) {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(s_read + t);
      }
      float mp[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) mp[i] = -INFINITY;
      if (!masked) {
#pragma unroll
        for (int i = 0; i < CW; i += 2)
          mp[(i >> 1) & 7] = tc::max3(mp[(i >> 1) & 7], v[i], v[i + 1]);
      } else {
#pragma unroll
        for (int i = 0; i < CW; ++i) mp[i & 7] = fmaxf(mp[i & 7], i < lim ? v[i] : -INFINITY);
      }
      float mt = fmaxf(fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3])),
                       fmaxf(fmaxf(mp[4], mp[5]), fmaxf(mp[6], mp[7])));
      if constexpr (kHalves == 2) {
        float other;
        if (!tc::pair_exchange(red_at(j & 1, h), red_at(j & 1, h ^ 1), true, mt, other, meet)) {
          ok = false;
          break;
        }
        mt = fmaxf(mt, other);
      }
      mt *= pr.scale_log2;
      const float m_new = fmaxf(m, mt);
      float m_use = m;
      bool rescale = false;
      if (m == -INFINITY) {
        m_use = m_new;
      } else if (m_new - m > kRescale) {
        m_use = m_new;
        rescale = true;
      }
      if (__any_sync(0xffffffffu, rescale)) {
        // O_t holds PV_t(0..j-1), all complete: HD = 128, S_t(j) was issued after
        // them; HD = 64, the wait below
        if (kSepP && j >= 1) {
          if (!wait(pv_done + t, (j - 1) & 1)) { ok = false; break; }
          tc::tc_fence_after();
        }
        const float alpha = rescale ? tc::ex2(m - m_use) : 1.f;
        l *= alpha;
#pragma unroll 1
        for (int c = 0; c < HO / 32; ++c) {
          float o[32];
          tc::tmem_ld32(t_o + c * 32, o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= alpha;
          tc::tmem_st32(t_o + c * 32, o);
        }
      }
      m = m_use;
      const float m_sub = m_use == -INFINITY ? 0.f : m_use;
      float rs[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};  // partial row sums
      // P = exp2(s - m) as 16-bit pairs, summed before they are rounded, in four
      // chains of paired sums
      auto plain = [&](float s0, float s1, int c) {
        float x0, x1;
        tc::fma2(x0, x1, s0, s1, pr.scale_log2, pr.scale_log2, -m_sub, -m_sub);
        x0 = tc::ex2(x0);
        x1 = tc::ex2(x1);
        const int k = 2 * ((c >> 1) & 3);
        tc::add2(rs[k], rs[k + 1], rs[k], rs[k + 1], x0, x1);
        return tc::pack2<T>(x0, x1);
      };
      auto below = [&](float s0, float s1, int c) {  // columns from lim on are masked
        const float x0 = c < lim ? tc::ex2(fmaf(s0, pr.scale_log2, -m_sub)) : 0.f;
        const float x1 = c + 1 < lim ? tc::ex2(fmaf(s1, pr.scale_log2, -m_sub)) : 0.f;
        const int k = 2 * ((c >> 1) & 3);
        tc::add2(rs[k], rs[k + 1], rs[k], rs[k + 1], x0, x1);
        return tc::pack2<T>(x0, x1);
      };
      if constexpr (kHalves == 1) {
        uint32_t pk[CW / 2];
        if (!masked) {
#pragma unroll
          for (int i = 0; i < CW; i += 2) pk[i / 2] = plain(v[i], v[i + 1], i);
        } else {
#pragma unroll
          for (int i = 0; i < CW; i += 2) pk[i / 2] = below(v[i], v[i + 1], i);
        }
        if (j >= 1) {
          if (!wait(pv_done + t, (j - 1) & 1)) { ok = false; break; }
          tc::tc_fence_after();
        }
        tc::tmem_st64u(t_p, pk);
      } else {
        // S again from TMEM, in chunks whose P goes over columns already read
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x[32];
          tc::tmem_ld32(t_s + c * 32, x);
          uint32_t pk[16];
          if (!masked) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) pk[i / 2] = plain(x[i], x[i + 1], c * 32 + i);
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 2) pk[i / 2] = below(x[i], x[i + 1], c * 32 + i);
          }
          tc::tmem_st16(t_p + c * 16, pk);
        }
      }
      l += ((rs[0] + rs[1]) + (rs[2] + rs[3])) + ((rs[4] + rs[5]) + (rs[6] + rs[7]));
      tc::tmem_wait_st();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(p_full + t);
    }
    // ------------------------------------------------------------ epilogue
    if (nt > 0) {
      if constexpr (kHalves == 2) {
        // both halves or neither (the loop above ends for both with the same `ok`)
        if (ok) {
          *red_at(nt & 1, h) = l;
          meet();
          l += *red_at(nt & 1, h ^ 1);
        }
      }
      if (ok && wait(o_done + t, 0)) {
        tc::tc_fence_after();
        const float inv = 1.f / l;
        const bool wide = wide_rows(out, pr.D) && wide_rows(rest, pr.D);
        // (read again: kept over the loop, these would not fit in registers)
        const int4 it = items[blockIdx.x / pr.Hkv];
        const int per = FM / pr.G, tok = it.z + t * per + r / pr.G;
        const bool store = r < per * pr.G && tok < it.y;
        const int64_t row =
            (int64_t)(it.x + tok) * pr.H + (blockIdx.x % pr.Hkv) * pr.G + r % pr.G;
#pragma unroll
        for (int c = 0; c < HO / 32; ++c) {
          float v[32];
          __syncwarp();                    // lanes without a row left the last trip early
          tc::tmem_ld32(t_o + c * 32, v);  // warp-collective
          if (!store) continue;
          const int d = h * HO + c * 32;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float* e = v + 16 * i;
            const int at = d + 16 * i;
            if (at >= pr.D) continue;  // D is a multiple of 8
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              e[2 * k] *= inv;
              e[2 * k + 1] *= inv;
              w[k] = tc::pack2<T>(e[2 * k], e[2 * k + 1]);
            }
            store16(out + row * pr.D + at, w, wide, at + 8 < pr.D);
            if (rest == nullptr) continue;
            // what the rounding left
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              float r0, r1;
              tc::unpack2<T>(w[k], r0, r1);
              w[k] = tc::pack2<T>(e[2 * k] - r0, e[2 * k + 1] - r1);
            }
            store16(rest + row * pr.D + at, w, wide, at + 8 < pr.D);
          }
        }
        if (store && h == 0 && lse != nullptr) lse[row] = (m + log2f(l)) * kLn2;
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
