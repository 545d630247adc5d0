// Scaled token embedding and its gradient.
//
//   forward   y_i  = scale * W[id_i]                      (a gather of rows)
//   backward  dW_v = scale * sum_{i : id_i = v} g_i       (every row v of dW)
//
// The backward sorts the tokens by id with a stable radix sort, so that the
// rows that belong to one v are neighbours and in token order, and then every
// row of dW is one sum in a fixed order: no floating-point atomics, the same
// bits every time, float32 throughout with one rounding at the end.  Both
// directions are bound by HBM: the forward reads and writes n D values, the
// backward reads n D and writes V D (mostly zeros for a large vocabulary).
#pragma once

#include "common.cuh"

namespace theria {
namespace embed {

// id of token i, or -1 where it lies outside [0, V).
__device__ __forceinline__ int64_t token(const void* ids, int wide, int64_t i, int64_t V) {
  const int64_t t = wide ? static_cast<const int64_t*>(ids)[i]
                         : (int64_t) static_cast<const int32_t*>(ids)[i];
  return t >= 0 && t < V ? t : -1;
}

// A 16-byte vector of T, as floats.
template <typename T> struct Vec {
  static constexpr int n = 16 / sizeof(T);
};

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = to_f32(p[0]);
  } else {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(e[i]);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    p[0] = from_f32<T>(v[0]);
  } else {
    uint4 r;
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = r;
  }
}

// One warp per token row, lanes over its vectors.
constexpr int WARPS = 8;
template <typename T, int VEC>
__global__ void __launch_bounds__(WARPS * 32)
fwd_kernel(const void* __restrict__ ids, int wide, const T* __restrict__ w, T* __restrict__ out,
           int64_t n, int64_t V, int64_t D, float scale, int64_t zero_idx) {
  const int lane = threadIdx.x & 31;
  for (int64_t i = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5); i < n;
       i += (int64_t)gridDim.x * WARPS) {
    const int64_t t = token(ids, wide, i, V);
    if (t < 0 && lane == 0) atomicExch(&g_device_error, THERIA_ERR_INVALID_ARG);
    const bool zero = t < 0 || t == zero_idx;
    const T* src = w + (zero ? 0 : t) * D;
    T* dst = out + i * D;
    for (int64_t c = lane * VEC; c < D; c += 32 * VEC) {
      float v[VEC];
      if (zero) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = 0.f;
      } else {
        load_vec<T, VEC>(src + c, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] *= scale;
      }
      store_vec<T, VEC>(dst + c, v);
    }
  }
}

// ---------------------------------------------------------------- the sort
// Stable least-significant-digit radix sort of (key, token index), 8 bits a
// pass: keys are the ids, and V for a token without a row (outside the
// vocabulary, or the zero row), so those come last.  A tile of 2048 tokens
// per CTA; each warp owns 256 consecutive ones and ranks them 32 at a time.
constexpr int TILE = 2048, SORT_THREADS = 256, BINS = 256;

__device__ __forceinline__ uint32_t first_key(const void* ids, int wide, int64_t i, int64_t V,
                                              int64_t zero_idx) {
  const int64_t t = token(ids, wide, i, V);
  if (t < 0) atomicExch(&g_device_error, THERIA_ERR_INVALID_ARG);
  return (uint32_t)(t < 0 || t == zero_idx ? V : t);
}

// The digit counts of each tile, as hist[bin][tile].  keys == nullptr: the
// first pass, from the ids.
__global__ void __launch_bounds__(SORT_THREADS)
hist_kernel(const void* __restrict__ ids, int wide, const uint32_t* __restrict__ keys,
            uint32_t* __restrict__ hist, int64_t n, int64_t V, int64_t zero_idx, int shift) {
  __shared__ uint32_t bins[BINS];
  bins[threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * TILE;
  for (int k = threadIdx.x; k < TILE; k += SORT_THREADS) {
    const int64_t i = base + k;
    if (i >= n) break;
    const uint32_t key = keys ? keys[i] : first_key(ids, wide, i, V, zero_idx);
    atomicAdd(&bins[(key >> shift) & (BINS - 1)], 1u);
  }
  __syncthreads();
  hist[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = bins[threadIdx.x];
}

// Exclusive prefix sum of hist[0 .. m) in place, one CTA.
__global__ void __launch_bounds__(1024) scan_kernel(uint32_t* __restrict__ hist, int64_t m) {
  __shared__ uint32_t part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t per = (m + 1023) / 1024;
  const int64_t b = threadIdx.x * per, e = b + per < m ? b + per : m;
  uint32_t sum = 0;
  for (int64_t i = b; i < e; ++i) sum += hist[i];
  uint32_t run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) part[warp] = run;
  __syncthreads();
  if (warp == 0) {
    uint32_t p = part[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, p, o);
      if (lane >= o) p += up;
    }
    part[lane] = p;
  }
  __syncthreads();
  uint32_t at = run - sum + (warp ? part[warp - 1] : 0);
  for (int64_t i = b; i < e; ++i) {
    const uint32_t h = hist[i];
    hist[i] = at;
    at += h;
  }
}

__global__ void __launch_bounds__(SORT_THREADS)
scatter_kernel(const void* __restrict__ ids, int wide, const uint32_t* __restrict__ keys,
               const uint32_t* __restrict__ vals, const uint32_t* __restrict__ hist,
               uint32_t* __restrict__ keys_out, uint32_t* __restrict__ vals_out, int64_t n,
               int64_t V, int64_t zero_idx, int shift) {
  constexpr int W = SORT_THREADS / 32, ROUNDS = TILE / SORT_THREADS;
  __shared__ uint32_t count[W][BINS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int k = threadIdx.x; k < W * BINS; k += SORT_THREADS) (&count[0][0])[k] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * TILE + warp * (TILE / W) + lane;
  uint32_t key[ROUNDS], rank[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t i = base + r * 32;
    const bool in = i < n;
    key[r] = !in ? 0xffffffffu : keys ? keys[i] : first_key(ids, wide, i, V, zero_idx);
    const uint32_t d = (key[r] >> shift) & (BINS - 1);
    // lanes past the end form a group of their own
    const uint32_t peers = __match_any_sync(0xffffffffu, in ? d : BINS);
    const uint32_t before = __popc(peers & ((1u << lane) - 1));
    rank[r] = in ? count[warp][d] + before : 0;
    __syncwarp();
    if (in && before == 0) count[warp][d] += __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  {  // where each warp's tokens of a digit go
    uint32_t at = hist[(int64_t)threadIdx.x * gridDim.x + blockIdx.x];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint32_t c = count[w][threadIdx.x];
      count[w][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t i = base + r * 32;
    if (i >= n) continue;
    const uint32_t to = count[warp][(key[r] >> shift) & (BINS - 1)] + rank[r];
    keys_out[to] = key[r];
    vals_out[to] = vals ? vals[i] : (uint32_t)i;
  }
}

// start[v] = the first sorted position with a key >= v, for v = 0 .. V.
__global__ void starts_kernel(const uint32_t* __restrict__ keys, uint32_t* __restrict__ start,
                              int64_t n, int64_t V) {
  for (int64_t v = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; v <= V;
       v += (int64_t)gridDim.x * blockDim.x) {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (keys[mid] < (uint32_t)v) lo = mid + 1; else hi = mid;
    }
    start[v] = (uint32_t)lo;
  }
}

// -------------------------------------------------------------- the sums
// Tokens are counted in aligned chunks of CHUNK sorted positions.  A chunk
// whose tokens all have one id is summed on its own first (chunk_kernel,
// float32), so the row of a frequent token adds a few chunk sums and at most
// 2 * (CHUNK - 1) single rows.
constexpr int CHUNK = 32;

// A warp's work unit: COLS columns of one row.
template <typename T, int VEC>
__device__ __forceinline__ void add_rows(const T* __restrict__ gy, const uint32_t* __restrict__ vals,
                                         int64_t b, int64_t e, int64_t D, int64_t c,
                                         float (&acc)[VEC]) {
  for (; b + 4 <= e; b += 4) {
    float v[4][VEC];
#pragma unroll
    for (int j = 0; j < 4; ++j) load_vec<T, VEC>(gy + (int64_t)vals[b + j] * D + c, v[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += v[j][k];
  }
  for (; b < e; ++b) {
    float v[VEC];
    load_vec<T, VEC>(gy + (int64_t)vals[b] * D + c, v);
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] += v[k];
  }
}

// part[chunk][D] = the sum of the chunk's rows, for chunks of one id.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
chunk_kernel(const T* __restrict__ gy, const uint32_t* __restrict__ keys,
             const uint32_t* __restrict__ vals, float* __restrict__ part, int64_t chunks,
             int64_t V, int64_t D) {
  const int64_t units = (D + VEC - 1) / VEC;
  for (int64_t j = blockIdx.x; j < chunks; j += gridDim.x) {
    const int64_t b = j * CHUNK;
    const uint32_t key = keys[b];
    if (key != keys[b + CHUNK - 1] || key >= (uint32_t)V) continue;
    for (int64_t u = threadIdx.x; u < units; u += blockDim.x) {
      float acc[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
      add_rows<T, VEC>(gy, vals, b, b + CHUNK, D, u * VEC, acc);
#pragma unroll
      for (int k = 0; k < VEC; ++k) part[j * D + u * VEC + k] = acc[k];
    }
  }
}

// Every row of gw: zeros, or the sum of its tokens' rows.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
rows_kernel(const T* __restrict__ gy, const uint32_t* __restrict__ vals,
            const uint32_t* __restrict__ start, const float* __restrict__ part,
            T* __restrict__ gw, int64_t V, int64_t D, float scale) {
  const int64_t units = (D + VEC - 1) / VEC;
  for (int64_t v = blockIdx.x; v < V; v += gridDim.x) {
    const int64_t b = start[v], e = start[v + 1];
    // whole chunks inside [b, e)
    const int64_t cb = (b + CHUNK - 1) / CHUNK, ce = e / CHUNK;
    const bool whole = cb < ce;
    for (int64_t u = threadIdx.x; u < units; u += blockDim.x) {
      const int64_t c = u * VEC;
      float acc[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
      add_rows<T, VEC>(gy, vals, b, whole ? cb * CHUNK : e, D, c, acc);
      if (whole) {
        for (int64_t j = cb; j < ce; ++j)
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] += part[j * D + c + k];
        add_rows<T, VEC>(gy, vals, ce * CHUNK, e, D, c, acc);
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] *= scale;
      store_vec<T, VEC>(gw + v * D + c, acc);
    }
  }
}

}  // namespace embed
}  // namespace theria
