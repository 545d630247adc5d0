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

// The split of dh's contraction over a piece of the vocabulary: parts of
// `split_kb` k blocks, `acc_rows` rows of float32 partial sums for each.
struct Splits {
  int split_kb, acc_rows, splits;
};
constexpr int CLUSTERS = 74, TILE_ROWS = 256;
constexpr int MAX_UNITS = 8 * CLUSTERS;  // split * tiles, where more than one split

// What prep_kernel fills, and what it fills it from.
struct Prep {
  const void* target;
  int wide;
  int64_t ignore_index, N, V;
  int *pos, *row_of, *tgt, *n_live;  // see prep_kernel
  unsigned* done;                    // zeroed for join_kernel
  // forward: the rows that do not count get 0 here
  float *count, *loss, *lse;
  // backward, by packed row: lse and the row's factor of dz, and the factor of
  // the results
  const float *gloss, *lse_in, *mean_of;
  int per_row, half;
  float *lse_p, *rowscale, *post;
  // the tensor cores' dh: how its contraction is split (see plan_splits)
  Splits* plan;
  int kb, d_tiles, pairs, ld_acc;
};

// float16 holds dz in units of 1 / 32768 of the largest row's factor, so that
// probabilities down to 2^-29 stay normal numbers.
constexpr float HALF_SCALE = 32768.f;

// pos[i] = the number of row i among the rows that count, or -1; row_of and
// tgt by that number; *n_live.  One CTA: each warp owns a run of rows, counts
// it, and after a scan over the warps numbers it; 8 loads of 32 rows are in
// flight at a time (8192 rows: 4.5 us, against 18.8 for a thread per run).
constexpr int PREP_BATCH = 8;

// Splits dh's contraction where whole 256 x 256 tiles of the rows that count
// would leave clusters idle.  Cost in k blocks (0.28 us): the longest cluster's
// share with 8 for each unit's start and end, and the partials' traffic (written
// and read, at 6.5 TB/s).  All 1024 threads; the least cost wins, then the
// fewest splits.
__device__ __forceinline__ void plan_splits(const Prep& a, int live) {
  __shared__ float cost[32];
  __shared__ int which[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = (live > 0 ? (live + TILE_ROWS - 1) / TILE_ROWS : 1) * TILE_ROWS;
  const int tiles = rows / TILE_ROWS * a.d_tiles;
  float best = INFINITY;
  int per = a.kb;
  const int s = threadIdx.x + 1;
  if (s == 1 || (s <= a.kb && (int64_t)s * tiles <= MAX_UNITS)) {
    per = (a.kb + s - 1) / s;
    const int n = (a.kb + per - 1) / per;
    best = (float)((n * (int64_t)tiles + CLUSTERS - 1) / CLUSTERS) * (float)(per * a.pairs + 8) +
           (float)n * (float)rows * (float)a.ld_acc * (8.f / 6.5e12f / 0.28e-6f);
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {  // the lower thread's on a tie
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
    *a.plan = Splits{per, rows, (a.kb + per - 1) / per};
  }
}

__global__ void __launch_bounds__(1024) prep_kernel(const Prep a) {
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
  const float unit = a.half ? HALF_SCALE : 1.f;
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
        if (a.lse_p) {
          a.lse_p[to] = a.lse_in[i];
          a.rowscale[to] = unit * (a.per_row ? a.gloss[i] / most : 1.f);
        }
      } else {
        if (a.loss) a.loss[i] = 0.f;
        if (a.lse) a.lse[i] = 0.f;
      }
    }
  }
  if (a.plan) plan_splits(a, total);
  if (threadIdx.x == 0) {
    *a.n_live = total;
    if (a.done) *a.done = 0;
    if (a.count) *a.count = (float)total;
    if (a.post)
      *a.post = (a.per_row ? most
                 : a.mean_of ? (total > 0 ? a.gloss[0] / *a.mean_of : 0.f)
                             : a.gloss[0]) / unit;
  }
}

// ------------------------------------------------------------- CUDA cores
// out(m, n) = sum_k a(m, k) b(n, k): 64 x 64 tiles, 16 x 16 threads of 4 x 4.
constexpr int TM = 64, TN = 64, TK = 16;

template <typename FA, typename FB>
__device__ __forceinline__ void tile_product(FA a, FB b, int64_t K, float (&acc)[4][4]) {
  __shared__ float sa[TK][TM + 4], sb[TK][TN + 4];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  for (int64_t k0 = 0; k0 < K; k0 += TK) {
#pragma unroll
    for (int i = 0; i < TM * TK / 256; ++i) {
      const int e = threadIdx.x + i * 256;
      a.load(sa, e, k0);
      b.load(sb, e, k0);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < TK; ++k) {
      float ra[4], rb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ra[i] = sa[k][ty * 4 + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) rb[j] = sb[k][tx * 4 + j];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(ra[i], rb[j], acc[i][j]);
    }
    __syncthreads();
  }
}

// Operands of tile_product.  Rows: element (r, k) of a matrix with k
// contiguous, rows through an index list (negative: zeros) or not; Cols: the r
// axis contiguous.
template <typename T>
struct Rows {
  const T* p;
  const int* list;
  int64_t r0, n, ld, K;
  __device__ void load(float (&s)[TK][TM + 4], int e, int64_t k0) const {
    const int k = e % TK, r = e / TK;
    const int64_t i = r0 + r, at = i < n ? (list ? list[i] : i) : -1;
    s[k][r] = at >= 0 && k0 + k < K ? to_f32(p[at * ld + k0 + k]) : 0.f;
  }
};
template <typename T>
struct Cols {
  const T* p;
  const int* list;  // of the k axis
  int64_t r0, n, ld, K;
  __device__ void load(float (&s)[TK][TM + 4], int e, int64_t k0) const {
    const int r = e % TM, k = e / TM;
    const int64_t i = r0 + r, kk = k0 + k;
    s[k][r] = i < n && kk < K ? to_f32(p[(list ? list[kk] : kk) * ld + i]) : 0.f;
  }
};

// part[m][tile] = (max, sum exp(z - max)) of the tile's columns; zt[m] the
// target's score.  Grid (vocabulary tiles, row tiles).
template <typename T>
__global__ void __launch_bounds__(256)
score_kernel(const T* __restrict__ h, const T* __restrict__ w, const int* __restrict__ row_of,
             const int* __restrict__ tgt, const int* __restrict__ n_live,
             float2* __restrict__ part, float* __restrict__ zt, int64_t V, int64_t D) {
  const int64_t n = *n_live, m0 = (int64_t)blockIdx.y * TM, v0 = (int64_t)blockIdx.x * TN;
  if (m0 >= n) return;
  float z[4][4];
  tile_product(Rows<T>{h, row_of, m0, n, D, D}, Rows<T>{w, nullptr, v0, V, D, D}, D, z);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty * 4 + i;
    const int t = m < n ? tgt[m] : -1;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t v = v0 + tx * 4 + j;
      if (v >= V) continue;
      top = fmaxf(top, z[i][j]);
      if (v == t) zt[m] = z[i][j];
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (v0 + tx * 4 + j < V) sum += expf(z[i][j] - top);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (tx == 0 && m < n) part[m * gridDim.x + blockIdx.x] = make_float2(top, sum);
  }
}

// lse and loss of each row that counts, from its tiles' (max, sum); a warp
// per row.  `out` not NULL: the CTA that ends last adds all N rows' losses in
// a fixed order (mean: over *count).
__global__ void __launch_bounds__(256)
join_kernel(const float2* __restrict__ part, const float* __restrict__ zt,
            const int* __restrict__ row_of, const int* __restrict__ n_live, int tiles,
            float* __restrict__ loss, float* __restrict__ lse, unsigned* __restrict__ done,
            float* __restrict__ out, int mean, int64_t N) {
  __shared__ float warps[8];
  __shared__ bool last;
  const int lane = threadIdx.x & 31;
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
      const float l = top + logf(sum);
      lse[i] = l;
      loss[i] = l - zt[m];
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

// dz[m][v], float32.
template <typename T>
__global__ void __launch_bounds__(256)
dz_kernel(const T* __restrict__ h, const T* __restrict__ w, const int* __restrict__ row_of,
          const int* __restrict__ tgt, const int* __restrict__ n_live,
          const float* __restrict__ lse, const float* __restrict__ rowscale,
          float* __restrict__ dz, int64_t V, int64_t D) {
  const int64_t n = *n_live, m0 = (int64_t)blockIdx.y * TM, v0 = (int64_t)blockIdx.x * TN;
  if (m0 >= n) return;
  float z[4][4];
  tile_product(Rows<T>{h, row_of, m0, n, D, D}, Rows<T>{w, nullptr, v0, V, D, D}, D, z);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty * 4 + i;
    if (m >= n) continue;
    const float l = lse[m], g = rowscale[m];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t v = v0 + tx * 4 + j;
      if (v < V) dz[m * V + v] = g * (expf(z[i][j] - l) - (v == tgt[m] ? 1.f : 0.f));
    }
  }
}

// dh[i][d] = sum_v dz[pos[i]][v] w[v][d]; zeros where row i does not count.
template <typename T>
__global__ void __launch_bounds__(256)
dh_kernel(const float* __restrict__ dz, const T* __restrict__ w, const int* __restrict__ pos,
          const float* __restrict__ post, T* __restrict__ dh, int64_t N, int64_t V, int64_t D) {
  const int64_t m0 = (int64_t)blockIdx.y * TM, d0 = (int64_t)blockIdx.x * TN;
  float o[4][4];
  tile_product(Rows<float>{dz, pos, m0, N, V, V}, Cols<T>{w, nullptr, d0, D, D, V}, V, o);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty * 4 + i, d = d0 + tx * 4 + j;
      if (m < N && d < D) dh[m * D + d] = from_f32<T>(pos[m] < 0 ? 0.f : *post * o[i][j]);
    }
}

// dw[v][d] = sum_m dz[m][v] h[m][d]
template <typename T>
__global__ void __launch_bounds__(256)
dw_kernel(const float* __restrict__ dz, const T* __restrict__ h, const int* __restrict__ row_of,
          const int* __restrict__ n_live, const float* __restrict__ post, T* __restrict__ dw,
          int64_t V, int64_t D) {
  const int64_t n = *n_live, r0 = (int64_t)blockIdx.y * TM, d0 = (int64_t)blockIdx.x * TN;
  float o[4][4];
  tile_product(Cols<float>{dz, nullptr, r0, V, V, n}, Cols<T>{h, row_of, d0, D, D, n}, n, o);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = r0 + ty * 4 + i, d = d0 + tx * 4 + j;
      if (r < V && d < D) dw[r * D + d] = from_f32<T>(*post * o[i][j]);
    }
}

}  // namespace xent
}  // namespace theria
