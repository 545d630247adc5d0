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
#include "tc_common.cuh"

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
// Stable least-significant-digit radix sort of (key, token index): keys are the
// ids, and V for a token without a row (outside the vocabulary, or the zero
// row), so those come last.  What follows needs the sorted tokens and, for each
// v, range[v] = (first position, one past the last), (0, 0) for no token.
//
// Up to 131,072 tokens one cluster does it all in one launch
// (cluster_sort_kernel); more tokens go through three launches a pass: a tile
// of 2048 tokens per CTA, each warp owning 256 consecutive ones, 8 bits a pass.
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

// range[] from the sorted keys (zeroed before).
__global__ void range_kernel(const uint32_t* __restrict__ keys, uint2* __restrict__ range,
                             int64_t n, int64_t V) {
  for (int64_t p = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; p < n;
       p += (int64_t)gridDim.x * blockDim.x) {
    const uint32_t k = keys[p];
    if (k >= (uint32_t)V) continue;
    if (p == 0 || keys[p - 1] != k) range[k].x = (uint32_t)p;
    if (p == n - 1 || keys[p + 1] != k) range[k].y = (uint32_t)p + 1;
  }
}

// The whole sort in one cluster of 1 or 8 CTAs of 1024 threads: R tokens a
// thread stay in registers while a pass ranks them, and go through the
// distributed shared memory of the cluster to their next place (8 bytes a
// token), 9 bits at most a pass.  A pass costs two cluster barriers instead of
// three launches: 65,536 tokens of a 131,072-word vocabulary 84 us before, in
// three passes of 8 bits.  R: a power of two.
constexpr int CS_THREADS = 1024, CS_BITS = 9, CS_BINS = 1 << CS_BITS, CS_CTAS = 8, CS_MOST = 16;
struct ClusterSmem {
  static constexpr int oCount = 0;                          // [32 warps][bins]
  static constexpr int oTotal = oCount + 32 * CS_BINS * 4;  // [bins], read by the other CTAs
  static constexpr int oBase = oTotal + CS_BINS * 4;
  static constexpr int oWarp = oBase + CS_BINS * 4;
  static constexpr int oBuf = oWarp + 128;                  // [1024 R] (key, index)
};
template <int R>
__global__ void __launch_bounds__(CS_THREADS)
cluster_sort_kernel(const void* __restrict__ ids, int wide, int ctas, int passes, int bits,
                    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ vals_out,
                    uint2* __restrict__ range, int n, int64_t V, int64_t zero_idx) {
  extern __shared__ __align__(16) uint8_t cs_mem[];
  using L = ClusterSmem;
  uint32_t(*count)[CS_BINS] = reinterpret_cast<uint32_t(*)[CS_BINS]>(cs_mem + L::oCount);
  uint32_t* total = reinterpret_cast<uint32_t*>(cs_mem + L::oTotal);
  uint32_t* base = reinterpret_cast<uint32_t*>(cs_mem + L::oBase);
  uint32_t* part = reinterpret_cast<uint32_t*>(cs_mem + L::oWarp);
  uint2* buf = reinterpret_cast<uint2*>(cs_mem + L::oBuf);
  constexpr int HELD = CS_THREADS * R;  // tokens of a CTA
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = tc::cluster_rank();
  const int local = warp * 32 * R + lane, first = (int)rank * HELD + local;
  for (int64_t v = (int64_t)rank * CS_THREADS + tid; v < V; v += (int64_t)ctas * CS_THREADS)
    range[v] = make_uint2(0, 0);
  uint32_t key[R], val[R], at[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = first + r * 32;
    key[r] = i < n ? first_key(ids, wide, i, V, zero_idx) : 0;
    val[r] = (uint32_t)i;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    const uint32_t mask = (1u << bits) - 1;
    for (int k = tid; k < 32 * CS_BINS; k += CS_THREADS) (&count[0][0])[k] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool in = first + r * 32 < n;
      const uint32_t d = (key[r] >> shift) & mask;
      const uint32_t peers = __match_any_sync(0xffffffffu, in ? d : CS_BINS);
      const uint32_t before = __popc(peers & ((1u << lane) - 1));
      at[r] = in ? count[warp][d] + before : 0;
      __syncwarp();
      if (in && before == 0) count[warp][d] += __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    if (tid < CS_BINS) {
      uint32_t sum = 0;
#pragma unroll
      for (int w = 0; w < 32; ++w) {
        const uint32_t c = count[w][tid];
        count[w][tid] = sum;
        sum += c;
      }
      total[tid] = sum;
    }
    tc::cluster_sync();  // every CTA's totals are there, every token in registers
    uint32_t all = 0, before = 0, run = 0;
    if (tid < CS_BINS) {
      for (int c = 0; c < ctas; ++c) {
        const uint32_t t = tc::ld_cluster(tc::map_rank(total + tid, c));
        all += t;
        before += c < (int)rank ? t : 0;
      }
      run = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += u;
      }
      if (lane == 31) part[warp] = run;
    }
    __syncthreads();
    if (tid < CS_BINS) {
      for (int w = 0; w < warp; ++w) before += part[w];
      base[tid] = before + run - all;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (first + r * 32 >= n) continue;
      const uint32_t d = (key[r] >> shift) & mask;
      const uint32_t to = base[d] + count[warp][d] + at[r];
      tc::st_cluster2(tc::map_rank(buf + to % HELD, to / HELD), key[r], val[r]);
    }
    tc::cluster_sync();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (first + r * 32 >= n) continue;
      const uint2 kv = buf[local + r * 32];
      key[r] = kv.x;
      val[r] = kv.y;
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int p = first + r * 32, l = local + r * 32;
    if (p >= n) continue;
    keys_out[p] = key[r];
    vals_out[p] = val[r];
    if (key[r] >= (uint32_t)V) continue;
    const bool starts =
        p == 0 || key[r] != (l > 0 ? buf[l - 1].x
                                   : tc::ld_cluster(tc::map_rank(buf + HELD - 1, rank - 1)));
    const bool ends = p == n - 1 || key[r] != (l < HELD - 1
                                                   ? buf[l + 1].x
                                                   : tc::ld_cluster(tc::map_rank(buf, rank + 1)));
    if (starts) range[key[r]].x = (uint32_t)p;
    if (ends) range[key[r]].y = (uint32_t)p + 1;
  }
  tc::cluster_sync();  // no CTA ends while another reads its tokens
}

// -------------------------------------------------------------- the sums
// Tokens are counted in aligned chunks of CHUNK sorted positions.  A chunk
// whose tokens all have one id is summed on its own first (chunk_kernel,
// float32), so the row of a frequent token adds a few chunk sums and at most
// 2 * (CHUNK - 1) single rows.
constexpr int CHUNK = 32;

// LEN consecutive values at p; `aligned`: as one 16-byte vector.
template <typename T, int LEN, bool ALIGNED>
__device__ __forceinline__ void load_run(const T* p, float (&v)[LEN]) {
  if constexpr (ALIGNED) {
    load_vec<T, LEN>(p, v);
  } else {
#pragma unroll
    for (int k = 0; k < LEN; ++k) v[k] = to_f32(p[k]);
  }
}

// acc += the rows of the tokens at sorted positions [b, e), columns c ..
template <typename T, int LEN, bool ALIGNED>
__device__ __forceinline__ void add_rows(const T* __restrict__ gy, const uint32_t* __restrict__ vals,
                                         int64_t b, int64_t e, int64_t D, int64_t c,
                                         float (&acc)[LEN]) {
  for (; b + 4 <= e; b += 4) {
    float v[4][LEN];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      load_run<T, LEN, ALIGNED>(gy + (int64_t)vals[b + j] * D + c, v[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < LEN; ++k) acc[k] += v[j][k];
  }
  for (; b < e; ++b) {
    float v[LEN];
    load_run<T, LEN, ALIGNED>(gy + (int64_t)vals[b] * D + c, v);
#pragma unroll
    for (int k = 0; k < LEN; ++k) acc[k] += v[k];
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
      add_rows<T, VEC, (VEC > 1)>(gy, vals, b, b + CHUNK, D, u * VEC, acc);
#pragma unroll
      for (int k = 0; k < VEC; ++k) part[j * D + u * VEC + k] = acc[k];
    }
  }
}

// LEN values of a row of gw (before `scale`): the tokens at [r.x, r.y).
template <typename T, int LEN, bool ALIGNED>
__device__ __forceinline__ void row_values(const T* __restrict__ gy,
                                           const uint32_t* __restrict__ vals,
                                           const float* __restrict__ part, uint2 r, int64_t D,
                                           int64_t c, float (&acc)[LEN]) {
#pragma unroll
  for (int k = 0; k < LEN; ++k) acc[k] = 0.f;
  // whole chunks inside [r.x, r.y)
  const int64_t cb = ((int64_t)r.x + CHUNK - 1) / CHUNK, ce = r.y / CHUNK;
  const bool whole = cb < ce;
  add_rows<T, LEN, ALIGNED>(gy, vals, r.x, whole ? cb * CHUNK : r.y, D, c, acc);
  if (whole) {
#pragma unroll 4
    for (int64_t j = cb; j < ce; ++j)
#pragma unroll
      for (int k = 0; k < LEN; ++k) acc[k] += part[j * D + c + k];
    add_rows<T, LEN, ALIGNED>(gy, vals, ce * CHUNK, r.y, D, c, acc);
  }
}

// gw as one run of V * D values, 16 bytes a thread: zeros, or the sums of the
// tokens' rows.  ROWS: every vector lies within a row (D a multiple of VEC) and
// gy's rows are vectors too; else a vector may reach into the rows after its
// first.  The large vocabulary's zeros set the pace: four vectors a thread are
// in flight, and odd widths are written as vectors all the same.
template <typename T, int VEC, bool ROWS>
__global__ void __launch_bounds__(256)
rows_kernel(const T* __restrict__ gy, const uint32_t* __restrict__ vals,
            const uint2* __restrict__ range, const float* __restrict__ part, T* __restrict__ gw,
            int64_t V, int64_t D, float scale) {
  constexpr int IN_FLIGHT = 4;
  const int64_t total = V * D, units = (total + VEC - 1) / VEC;
  const bool small = total < (1ll << 32);
  for (int64_t u0 = (int64_t)blockIdx.x * (256 * IN_FLIGHT) + threadIdx.x; u0 < units;
       u0 += (int64_t)gridDim.x * (256 * IN_FLIGHT)) {
    int64_t v[IN_FLIGHT];
    uint2 r[IN_FLIGHT];
#pragma unroll
    for (int i = 0; i < IN_FLIGHT; ++i) {
      const int64_t u = u0 + i * 256;
      v[i] = small ? (int64_t)((uint32_t)(u * VEC) / (uint32_t)D) : u * VEC / D;
      r[i] = u < units ? range[v[i]] : make_uint2(0, 0);
    }
#pragma unroll
    for (int i = 0; i < IN_FLIGHT; ++i) {
      const int64_t u = u0 + i * 256;
      if (u >= units) break;
      const int64_t c = u * VEC - v[i] * D;
      float acc[VEC];
      if (ROWS || c + VEC <= D) {
        if (r[i].x == r[i].y) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
        } else {
          row_values<T, VEC, ROWS && (VEC > 1)>(gy, vals, part, r[i], D, c, acc);
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] *= scale;
        }
        store_vec<T, VEC>(gw + u * VEC, acc);
      } else {  // the end of a row, and the start of the next ones
#pragma unroll 1
        for (int k = 0; k < VEC; ++k) {
          const int64_t e = u * VEC + k;
          if (e >= total) break;
          const int64_t row = e / D;
          const uint2 q = range[row];
          float one[1];
          row_values<T, 1, false>(gy, vals, part, q, D, e - row * D, one);
          gw[e] = from_f32<T>(one[0] * scale);
        }
      }
    }
  }
}

}  // namespace embed
}  // namespace theria
