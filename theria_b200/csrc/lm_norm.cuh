// Layer norm over rows of any width, and its gradients.
//
//   xhat = (x - mean) * rstd,  rstd = (var + eps)^-1/2,  y = xhat * w + b
//   gx   = rstd * P(gy * w),   P(v) = v - mean(v) - xhat * mean(v * xhat)
//   gw   = sum_rows gy * xhat, gb = sum_rows gy
// and, for cotangents (u, a, c) of (gx, gw, gb), with g = gy * w and the row's
// sums <.,.>,
//   dgy = rstd * w * P(u) + a * xhat + c,   dw = sum_rows rstd * gy * P(u)
//   dx  = rstd * P(gy * a) - rstd^2 / D * (<P(u), g> * xhat
//                                          + P(<u, xhat> g + <g, xhat> u)).
// P is linear, so all of a row's sums in these are taken in one reduction.
//
// Both directions are bound by HBM: x read and y written once, then x and gy
// read and gx written once.  A row stays in registers between its load and
// its store (rows up to 256 threads x NV vectors); the variance is taken
// around the mean already known, so it loses nothing to cancellation.
// Statistics, sums and the weight gradients are float32; each result is
// rounded once.  The sums over rows go through per-CTA partials added by a
// second kernel in a fixed order: the same bits every time.
#pragma once

#include "common.cuh"
#include "lm_embed.cuh"  // load_vec / store_vec

namespace theria {
namespace norm {

using embed::load_vec;
using embed::store_vec;

constexpr int SUMS = 7;  // the most values one reduction carries

// NW warps (one, or the whole CTA) own a row; sums of NS values over it.
template <int NW, int NS>
__device__ __forceinline__ void row_sum(float (&s)[NS], float (*red)[SUMS]) {
#pragma unroll
  for (int i = 0; i < NS; ++i) s[i] = warp_sum(s[i]);
  if constexpr (NW > 1) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < NS; ++i) red[warp][i] = s[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      s[i] = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) s[i] += red[w][i];
    }
    __syncthreads();
  }
}

// One affine value (w, b may be of float32 or of x's type; NULL: `none`).
__device__ __forceinline__ float affine(const void* p, int dtype, int64_t i, float none) {
  return p ? load_any(p, i, dtype) : none;
}

// NW warps per row (1: each warp of the CTA has its own row; 8: the CTA has
// one), NV vectors of VEC values per thread.
template <typename T, int VEC, int NV, int NW>
__global__ void __launch_bounds__(256)
fwd_kernel(const T* __restrict__ x, const void* __restrict__ w, const void* __restrict__ b,
           int wdtype, T* __restrict__ y, float* __restrict__ stats, int64_t N, int D, float eps) {
  constexpr int G = NW * 32, ROWS = 256 / G;
  __shared__ float red[8][SUMS];
  const int g = threadIdx.x % G;
  for (int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / G; r < N;
       r += (int64_t)gridDim.x * ROWS) {
    float v[NV][VEC], s[1] = {0.f}, q[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + g) * VEC;
      if (c < D) {
        load_vec<T, VEC>(x + r * D + c, v[j]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) s[0] += v[j][k];
      }
    }
    row_sum<NW>(s, red);
    const float mean = s[0] / (float)D;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if ((j * G + g) * VEC < D) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          v[j][k] -= mean;
          q[0] = fmaf(v[j][k], v[j][k], q[0]);
          q[1] += v[j][k];
        }
      }
    row_sum<NW>(q, red);
    // what the rounding of a large mean left in the deviations
    const float left = q[1] / (float)D;
    const float rstd = rsqrtf(fmaxf(q[0] / (float)D - left * left, 0.f) + eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + g) * VEC;
      if (c < D) {
#pragma unroll
        for (int k = 0; k < VEC; ++k)
          v[j][k] = fmaf((v[j][k] - left) * rstd, affine(w, wdtype, c + k, 1.f),
                         affine(b, wdtype, c + k, 0.f));
        store_vec<T, VEC>(y + r * D + c, v[j]);
      }
    }
    if (stats && g == 0) {
      stats[r] = mean + left;
      stats[N + r] = rstd;
    }
  }
}

// This CTA's two column sums into part[cta][2][D] (row-per-warp shapes add the
// warps' through dynamic shared memory [8][2][D] first).
template <int NW, int NV, int VEC>
__device__ __forceinline__ void store_part(const float (&a)[NV][VEC], const float (&b)[NV][VEC],
                                           float* part, int D) {
  constexpr int G = NW * 32, ROWS = 256 / G;
  extern __shared__ float cols[];
  const int g = threadIdx.x % G;
  float* mine = part + (int64_t)blockIdx.x * 2 * D;
  float* row = NW > 1 ? mine : cols + (int64_t)(threadIdx.x / G) * 2 * D;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * G + g) * VEC;
    if (c < D)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        row[c + k] = a[j][k];
        row[D + c + k] = b[j][k];
      }
  }
  if constexpr (NW == 1) {
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * D; e += 256) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < ROWS; ++k) sum += cols[k * 2 * D + e];
      mine[e] = sum;
    }
  }
}

// part[cta][2][D]: this CTA's sums of gy * xhat and gy.
template <typename T, int VEC, int NV, int NW>
__global__ void __launch_bounds__(256)
bwd_kernel(const T* __restrict__ x, const void* __restrict__ w, int wdtype,
           const T* __restrict__ gy, const float* __restrict__ stats, T* __restrict__ gx,
           float* __restrict__ part, int64_t N, int D) {
  constexpr int G = NW * 32, ROWS = 256 / G;
  __shared__ float red[8][SUMS];
  const int g = threadIdx.x % G;
  float aw[NV][VEC], ab[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < VEC; ++k) aw[j][k] = ab[j][k] = 0.f;
  for (int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / G; r < N;
       r += (int64_t)gridDim.x * ROWS) {
    const float mean = stats[r], rstd = stats[N + r];
    float h[NV][VEC], u[NV][VEC], s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + g) * VEC;
      if (c < D) {
        load_vec<T, VEC>(x + r * D + c, h[j]);
        load_vec<T, VEC>(gy + r * D + c, u[j]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          h[j][k] = (h[j][k] - mean) * rstd;
          aw[j][k] = fmaf(u[j][k], h[j][k], aw[j][k]);
          ab[j][k] += u[j][k];
          u[j][k] *= affine(w, wdtype, c + k, 1.f);
          s[0] += u[j][k];
          s[1] = fmaf(u[j][k], h[j][k], s[1]);
        }
      }
    }
    if (gx == nullptr) continue;
    row_sum<NW>(s, red);
    s[0] /= (float)D;
    s[1] /= (float)D;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + g) * VEC;
      if (c < D) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) u[j][k] = rstd * (u[j][k] - s[0] - h[j][k] * s[1]);
        store_vec<T, VEC>(gx + r * D + c, u[j]);
      }
    }
  }
  if (part) store_part<NW, NV, VEC>(aw, ab, part, D);
}

// Rows too wide for the registers: three passes over the row (the second and
// third hit L2), one CTA per row.
template <typename T>
__global__ void __launch_bounds__(256)
fwd_wide_kernel(const T* __restrict__ x, const void* __restrict__ w, const void* __restrict__ b,
                int wdtype, T* __restrict__ y, float* __restrict__ stats, int64_t N, int64_t D,
                float eps) {
  __shared__ float red[8][SUMS];
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    const T* row = x + r * D;
    float s[1] = {0.f}, q[2] = {0.f, 0.f};
    for (int64_t c = threadIdx.x; c < D; c += 256) s[0] += to_f32(row[c]);
    row_sum<8>(s, red);
    const float mean = s[0] / (float)D;
    for (int64_t c = threadIdx.x; c < D; c += 256) {
      const float d = to_f32(row[c]) - mean;
      q[0] = fmaf(d, d, q[0]);
      q[1] += d;
    }
    row_sum<8>(q, red);
    const float left = q[1] / (float)D;
    const float rstd = rsqrtf(fmaxf(q[0] / (float)D - left * left, 0.f) + eps);
    for (int64_t c = threadIdx.x; c < D; c += 256)
      y[r * D + c] = from_f32<T>(fmaf((to_f32(row[c]) - mean - left) * rstd,
                                      affine(w, wdtype, c, 1.f), affine(b, wdtype, c, 0.f)));
    if (stats && threadIdx.x == 0) {
      stats[r] = mean + left;
      stats[N + r] = rstd;
    }
  }
}

// The same for the backward: the CTA's column sums live in its part of the
// workspace (zeroed here, each column kept by one thread).
template <typename T>
__global__ void __launch_bounds__(256)
bwd_wide_kernel(const T* __restrict__ x, const void* __restrict__ w, int wdtype,
                const T* __restrict__ gy, const float* __restrict__ stats, T* __restrict__ gx,
                float* __restrict__ part, int64_t N, int64_t D) {
  __shared__ float red[8][SUMS];
  float* mine = part ? part + (int64_t)blockIdx.x * 2 * D : nullptr;
  if (mine)
    for (int64_t c = threadIdx.x; c < D; c += 256) mine[c] = mine[D + c] = 0.f;
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    const float mean = stats[r], rstd = stats[N + r];
    float s[2] = {0.f, 0.f};
    for (int64_t c = threadIdx.x; c < D; c += 256) {
      const float h = (to_f32(x[r * D + c]) - mean) * rstd, u = to_f32(gy[r * D + c]);
      if (mine) {
        mine[c] = fmaf(u, h, mine[c]);
        mine[D + c] += u;
      }
      const float uw = u * affine(w, wdtype, c, 1.f);
      s[0] += uw;
      s[1] = fmaf(uw, h, s[1]);
    }
    if (gx == nullptr) continue;
    row_sum<8>(s, red);
    s[0] /= (float)D;
    s[1] /= (float)D;
    for (int64_t c = threadIdx.x; c < D; c += 256) {
      const float h = (to_f32(x[r * D + c]) - mean) * rstd;
      const float uw = to_f32(gy[r * D + c]) * affine(w, wdtype, c, 1.f);
      gx[r * D + c] = from_f32<T>(rstd * (uw - s[0] - h * s[1]));
    }
  }
}

// The seven sums of a row's second derivative.
struct Second {
  float mu, ux, mg, gx, mq, qx, k, invD, rstd;
  __device__ Second(const float (&s)[SUMS], int64_t D, float r) {
    // s: u, u xhat, g, g xhat, q, q xhat (q = gy a), u g
    invD = 1.f / (float)D;
    mu = s[0] * invD;
    ux = s[1];
    mg = s[2] * invD;
    gx = s[3];
    mq = s[4] * invD;
    qx = s[5] * invD;
    k = s[6] - mu * s[2] - ux * invD * gx;  // <P(u), g>
    rstd = r;
  }
  __device__ float pu(float u, float h) const { return u - mu - h * ux * invD; }
  __device__ float dx(float h, float u, float g, float q) const {
    const float pg = g - mg - h * gx * invD;
    return rstd * (q - mq - h * qx) -
           rstd * rstd * invD * (k * h + ux * pg + gx * pu(u, h));
  }
};
__device__ __forceinline__ void second_terms(float (&s)[SUMS], float h, float u, float g,
                                             float q) {
  s[0] += u;
  s[1] = fmaf(u, h, s[1]);
  s[2] += g;
  s[3] = fmaf(g, h, s[3]);
  s[4] += q;
  s[5] = fmaf(q, h, s[5]);
  s[6] = fmaf(u, g, s[6]);
}

// The backward's backward; u, a, c may be NULL (zero).  part[cta][2][D]: the
// CTA's sums for dw (the second half is unused, zero).
template <typename T, int VEC, int NV, int NW>
__global__ void __launch_bounds__(256)
bwd2_kernel(const T* __restrict__ x, const void* __restrict__ w, int wdtype,
            const T* __restrict__ gy, const float* __restrict__ stats, const T* __restrict__ u,
            const void* __restrict__ a, const void* __restrict__ c, T* __restrict__ dx,
            T* __restrict__ dgy, float* __restrict__ part, int64_t N, int D) {
  constexpr int G = NW * 32, ROWS = 256 / G;
  __shared__ float red[8][SUMS];
  const int lane = threadIdx.x % G;
  float aw[NV][VEC], none[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < VEC; ++k) aw[j][k] = none[j][k] = 0.f;
  for (int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / G; r < N;
       r += (int64_t)gridDim.x * ROWS) {
    const float mean = stats[r], rstd = stats[N + r];
    float h[NV][VEC], g[NV][VEC], v[NV][VEC], s[SUMS];
#pragma unroll
    for (int i = 0; i < SUMS; ++i) s[i] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int col = (j * G + lane) * VEC;
      if (col < D) {
        load_vec<T, VEC>(x + r * D + col, h[j]);
        load_vec<T, VEC>(gy + r * D + col, g[j]);
        if (u) {
          load_vec<T, VEC>(u + r * D + col, v[j]);
        } else {
#pragma unroll
          for (int k = 0; k < VEC; ++k) v[j][k] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          h[j][k] = (h[j][k] - mean) * rstd;
          second_terms(s, h[j][k], v[j][k], g[j][k] * affine(w, wdtype, col + k, 1.f),
                       g[j][k] * affine(a, wdtype, col + k, 0.f));
        }
      }
    }
    row_sum<NW>(s, red);
    const Second f(s, D, rstd);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int col = (j * G + lane) * VEC;
      if (col < D) {
        float o[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float wk = affine(w, wdtype, col + k, 1.f), ak = affine(a, wdtype, col + k, 0.f);
          const float pu = f.pu(v[j][k], h[j][k]);
          aw[j][k] = fmaf(rstd * g[j][k], pu, aw[j][k]);
          o[k] = rstd * wk * pu + ak * h[j][k] + affine(c, wdtype, col + k, 0.f);
          v[j][k] = f.dx(h[j][k], v[j][k], g[j][k] * wk, g[j][k] * ak);
        }
        store_vec<T, VEC>(dgy + r * D + col, o);
        store_vec<T, VEC>(dx + r * D + col, v[j]);
      }
    }
  }
  store_part<NW, NV, VEC>(aw, none, part, D);
}

template <typename T>
__global__ void __launch_bounds__(256)
bwd2_wide_kernel(const T* __restrict__ x, const void* __restrict__ w, int wdtype,
                 const T* __restrict__ gy, const float* __restrict__ stats,
                 const T* __restrict__ u, const void* __restrict__ a, const void* __restrict__ c,
                 T* __restrict__ dx, T* __restrict__ dgy, float* __restrict__ part, int64_t N,
                 int64_t D) {
  __shared__ float red[8][SUMS];
  float* mine = part + (int64_t)blockIdx.x * 2 * D;
  for (int64_t e = threadIdx.x; e < D; e += 256) mine[e] = mine[D + e] = 0.f;
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    const float mean = stats[r], rstd = stats[N + r];
    float s[SUMS];
#pragma unroll
    for (int i = 0; i < SUMS; ++i) s[i] = 0.f;
    for (int64_t e = threadIdx.x; e < D; e += 256) {
      const float h = (to_f32(x[r * D + e]) - mean) * rstd, g = to_f32(gy[r * D + e]);
      second_terms(s, h, u ? to_f32(u[r * D + e]) : 0.f, g * affine(w, wdtype, e, 1.f),
                   g * affine(a, wdtype, e, 0.f));
    }
    row_sum<8>(s, red);
    const Second f(s, D, rstd);
    for (int64_t e = threadIdx.x; e < D; e += 256) {
      const float h = (to_f32(x[r * D + e]) - mean) * rstd, g = to_f32(gy[r * D + e]);
      const float uu = u ? to_f32(u[r * D + e]) : 0.f, pu = f.pu(uu, h);
      const float wk = affine(w, wdtype, e, 1.f), ak = affine(a, wdtype, e, 0.f);
      mine[e] = fmaf(rstd * g, pu, mine[e]);
      dgy[r * D + e] = from_f32<T>(rstd * wk * pu + ak * h + affine(c, wdtype, e, 0.f));
      dx[r * D + e] = from_f32<T>(f.dx(h, uu, g * wk, g * ak));
    }
  }
}

// gw, gb from the partials: 32 of the 2 D columns per CTA, 32 warps over
// the partials, added in a fixed order.  gb == nullptr: the first D alone.
__global__ void __launch_bounds__(1024)
cols_kernel(const float* __restrict__ part, void* __restrict__ gw, void* __restrict__ gb,
            int wdtype, int ctas, int64_t D) {
  __shared__ float sum[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t e = (int64_t)blockIdx.x * 32 + lane;
  float v = 0.f;
  if (e < 2 * D)
    for (int k = warp; k < ctas; k += 32) v += part[(int64_t)k * 2 * D + e];
  sum[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && e < 2 * D) {
    v = 0.f;
#pragma unroll 8
    for (int k = 0; k < 32; ++k) v += sum[k][lane];
    if (e < D) store_any(gw, e, wdtype, v);
    else if (gb) store_any(gb, e - D, wdtype, v);
  }
}

}  // namespace norm
}  // namespace theria
