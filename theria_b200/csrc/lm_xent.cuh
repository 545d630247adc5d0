// Linear layer to the vocabulary fused with its softmax cross entropy.
//
//   z = h w^T,  lse_i = log sum_v exp z_iv,  loss_i = lse_i - z_{i, t_i}
//   dz_iv = c_i (exp(z_iv - lse_i) - [v == t_i]),  dh = dz w,  dw = dz^T h
//
// The scores z [N, V] are never stored: the forward makes them tile by tile
// and keeps each tile's row maximum and row sum of exponentials; the backward
// makes them again, a piece of the vocabulary at a time, as dz.  Rows whose
// target is ignored are left out from the start: the rows that count are
// numbered 0 .. n_live - 1 in order (`prep_kernel`) and only those are
// computed, so neither their scores nor what their hidden states hold (NaN
// included) reaches a result.
#pragma once

#include "common.cuh"

namespace theria {
namespace xent {

// The split of a contraction: parts of `split_kb` k blocks, `acc_rows` rows of
// float32 partial sums for each.
struct Splits {
  int split_kb, acc_rows, splits;
};
constexpr int CLUSTERS = 74, TILE_ROWS = 256, K_BLOCK = 64;
constexpr int FEW_ROWS = 64;  // that count: 16-bit dz in two planes
// splits * tiles, where there is more than one split: of dh (over a piece of the
// vocabulary) and of dw (over the rows that count, where it has few tiles)
constexpr int MAX_UNITS = 8 * CLUSTERS, MAX_UNITS_DW = 2 * CLUSTERS;

// What prep_kernel fills, and what it fills it from.
struct Prep {
  const void* target;
  int wide;
  int64_t ignore_index, N, V;
  int *pos, *row_of, *tgt, *n_live;  // see prep_kernel
  unsigned* done;                    // zeroed for join_kernel
  // forward: the rows that do not count get 0 here
  float *count, *loss, *lse;
  // backward: the upstream gradient; the largest row's factor (1 but for
  // float16) and the factor of the results
  const float *gloss, *mean_of;
  int per_row, half;
  float *most, *post;
  // how dh's and dw's contractions are split (see plan_splits); NULL: not
  Splits *plan_h, *plan_w;
  int kb, d_tiles, v_tiles, f32, ld_acc;
};

// float16 holds dz in units of 1 / 32768 of the largest row's factor, so that
// probabilities down to 2^-29 stay normal numbers.
constexpr float HALF_SCALE = 32768.f;

// pos[i] = the number of row i among the rows that count, or -1; row_of and
// tgt by that number; *n_live.  One CTA: each warp owns a run of rows, counts
// it, and after a scan over the warps numbers it; 8 loads of 32 rows are in
// flight at a time (8192 rows: 8.4 us, 9.1 with the backward's splits; a run per
// thread took 18.8).
constexpr int PREP_BATCH = 8;

// Splits a contraction of kb k blocks where whole 256 x 256 tiles (of `rows`
// rows, `tiles` in all) would leave clusters idle.  Cost in k blocks (0.28 us):
// the longest cluster's share with 8 for each unit's start and end, and the
// partials' traffic (written and read, at 6.5 TB/s).  All 1024 threads; the
// least cost wins, then the fewest splits.
__device__ __forceinline__ void plan_splits(Splits* out, int kb, int rows, int tiles, int most,
                                            int pairs, int ld_acc) {
  __shared__ float cost[32];
  __shared__ int which[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float best = INFINITY;
  int per = kb;
  const int s = threadIdx.x + 1;
  if (s == 1 || (s <= kb && (int64_t)s * tiles <= most)) {
    per = (kb + s - 1) / s;
    const int n = (kb + per - 1) / per;
    best = (float)((n * (int64_t)tiles + CLUSTERS - 1) / CLUSTERS) * (float)(per * pairs + 8) +
           (float)n * (float)rows * (float)ld_acc * (8.f / 6.5e12f / 0.28e-6f);
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float c = __shfl_xor_sync(0xffffffffu, best, o);
    const int p = __shfl_xor_sync(0xffffffffu, per, o);
    if (c < best || (c == best && p > per)) {
      best = c;
      per = p;
    }
  }
  if (lane == 0) {
    cost[warp] = best;
    which[warp] = per;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w)
      if (cost[w] < best) {
        best = cost[w];
        per = which[w];
      }
    *out = Splits{per, rows, (kb + per - 1) / per};
  }
  __syncthreads();
}

__global__ void __launch_bounds__(1024) prep_kernel(const Prep a) {
  grid_launch();
  __shared__ int part[32];
  __shared__ float peak[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t per = ((a.N + 31) / 32 + 31) / 32 * 32;  // rows of a warp
  const int64_t b = warp * per, e = b + per < a.N ? b + per : a.N;
  auto load = [&](int64_t i0, int64_t (&t)[PREP_BATCH]) {
#pragma unroll
    for (int k = 0; k < PREP_BATCH; ++k) {
      const int64_t i = i0 + k * 32 + lane;
      t[k] = i >= e ? a.ignore_index
             : a.wide ? static_cast<const int64_t*>(a.target)[i]
                      : (int64_t) static_cast<const int32_t*>(a.target)[i];
    }
  };
  auto live = [&](int64_t t) { return t != a.ignore_index && t >= 0 && t < a.V; };
  int mine = 0;
  float most = 0.f;
  for (int64_t i0 = b; i0 < e; i0 += PREP_BATCH * 32) {
    int64_t t[PREP_BATCH];
    load(i0, t);
#pragma unroll
    for (int k = 0; k < PREP_BATCH; ++k) {
      const bool is = live(t[k]);
      if (!is && t[k] != a.ignore_index) atomicExch(&g_device_error, THERIA_ERR_INVALID_ARG);
      mine += __popc(__ballot_sync(0xffffffffu, is));
      if (is && a.per_row && a.half) {
        const float g = fabsf(a.gloss[i0 + k * 32 + lane]);
        if (isfinite(g)) most = fmaxf(most, g);
      }
    }
  }
  if (a.per_row && a.half) most = warp_max(most);
  if (lane == 0) {
    part[warp] = mine;
    peak[warp] = most;
  }
  __syncthreads();
  int at = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 32; ++w) {
    at += w < warp ? part[w] : 0;
    total += part[w];
    most = fmaxf(most, peak[w]);
  }
  if (most == 0.f) most = 1.f;
  for (int64_t i0 = b; i0 < e; i0 += PREP_BATCH * 32) {
    int64_t t[PREP_BATCH];
    load(i0, t);
#pragma unroll
    for (int k = 0; k < PREP_BATCH; ++k) {
      const int64_t i = i0 + k * 32 + lane;
      const bool is = live(t[k]);
      const uint32_t all = __ballot_sync(0xffffffffu, is);
      const int to = at + __popc(all & ((1u << lane) - 1));
      at += __popc(all);
      if (i >= e) continue;
      a.pos[i] = is ? to : -1;
      if (is) {
        a.row_of[to] = (int)i;
        a.tgt[to] = (int)t[k];
      } else {
        if (a.loss) a.loss[i] = 0.f;
        if (a.lse) a.lse[i] = a.lse[a.N + i] = a.lse[2 * a.N + i] = 0.f;
      }
    }
  }
  const int live_tiles = total > 0 ? (total + TILE_ROWS - 1) / TILE_ROWS : 1;
  const int pairs = a.f32 ? 6 : total <= FEW_ROWS ? 2 : 1;  // of planes
  if (a.plan_h)
    plan_splits(a.plan_h, a.kb, live_tiles * TILE_ROWS, live_tiles * a.d_tiles, MAX_UNITS, pairs,
                a.ld_acc);
  if (a.plan_w)
    plan_splits(a.plan_w, total > 0 ? (total + K_BLOCK - 1) / K_BLOCK : 1, a.v_tiles * TILE_ROWS,
                a.v_tiles * a.d_tiles, MAX_UNITS_DW, pairs, a.ld_acc);
  if (threadIdx.x == 0) {
    *a.n_live = total;
    if (a.most) *a.most = most;
    if (a.done) *a.done = 0;
    if (a.count) *a.count = (float)total;
    if (a.post)
      // no row: zeros, whatever the upstream gradient is
      *a.post = (a.per_row    ? most
                 : total == 0 ? 0.f
                 : a.mean_of  ? a.gloss[0] / *a.mean_of
                              : a.gloss[0]) / (a.half ? HALF_SCALE : 1.f);
  }
}

// lse [3][N] and loss of each row that counts, from its tiles' (max, sum); a warp
// per row.  `out` not NULL: the CTA that ends last adds all N rows' losses in
// a fixed order (mean: over *count).
__global__ void __launch_bounds__(256)
join_kernel(const float2* part, const float* zt, const int* row_of, const int* n_live, int tiles,
            float* loss, float* lse, unsigned* done, float* out, int mean, int64_t N) {
  __shared__ float warps[8];
  __shared__ bool last;
  const int lane = threadIdx.x & 31;
  grid_wait();
  const int n = *n_live;
  for (int m = blockIdx.x * 8 + (threadIdx.x >> 5); m < n; m += gridDim.x * 8) {
    const float2* p = part + (int64_t)m * tiles;
    float top = -INFINITY, sum = 0.f;
    for (int j = lane; j < tiles; j += 32) top = fmaxf(top, p[j].x);
    top = warp_max(top);
    for (int j = lane; j < tiles; j += 32) sum += p[j].y * expf(p[j].x - top);
    sum = warp_sum(sum);
    if (lane == 0) {
      const int64_t i = row_of[m];
      // log(sum) is small beside top for a nearly certain token, and all of its
      // loss: it is never rounded to top's last place.  lse keeps what its own
      // rounding leaves (the error of a sum of two, Knuth's TwoSum).
      const float log_sum = logf(sum), l = top + log_sum, back = l - top;
      lse[i] = l;
      lse[N + i] = (top - (l - back)) + (log_sum - back);
      loss[i] = lse[2 * N + i] = log_sum + (top - zt[m]);
    }
  }
  if (out == nullptr) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(done, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  float s = 0.f;
  const volatile float* each = loss;
  for (int64_t i = threadIdx.x; i < N; i += 256) s += each[i];
  s = warp_sum(s);
  if (lane == 0) warps[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += warps[w];
    out[0] = mean ? s / (float)n : s;
  }
}

}  // namespace xent
}  // namespace theria
