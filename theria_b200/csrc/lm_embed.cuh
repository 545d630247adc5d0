// Scaled token embedding and its gradient.
//
//   forward   y_i  = scale * W[id_i]                      (a gather of rows)
//   backward  dW_v = scale * sum_{i : id_i = v} g_i       (every row v of dW)
//
// The backward sorts the tokens by id with a stable radix sort, so that the
// rows that belong to one v are neighbours and in token order, and then sums
// them in chunks of 32 sorted tokens: no floating-point atomics, the same bits
// every time, float32 throughout with one rounding at the end.  Both directions
// are bound by HBM: the forward reads and writes n D values, the backward
// reads n D and writes V D (mostly zeros for a large vocabulary, written while
// the tokens are being sorted).
//
// Measured, 65,536 tokens of 131,072 words (frequencies as 1 / rank), 2048
// columns of bfloat16: lookup 65 us; sort and zeros 85 us (537 MB, 6.3 TB/s),
// chunks 73 us (378 MB, 5.2 TB/s), joined runs 20 to 28 us.
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
// row), so those come last.
//
// Up to 65,536 tokens one cluster does it all in one launch
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

constexpr int CS_THREADS = 1024, CS_BITS = 9, CS_BINS = 1 << CS_BITS, CS_CTAS = 8, CS_MOST = 8;

// The lanes whose d (of `bits` bits) equals this lane's, among `in`: a ballot
// per bit.
__device__ __forceinline__ uint32_t peers_of(uint32_t d, int bits, uint32_t in) {
  uint32_t same = in;
#pragma unroll
  for (int b = 0; b < CS_BITS; ++b) {
    if (b >= bits) break;
    const bool one = (d >> b) & 1;
    const uint32_t v = __ballot_sync(0xffffffffu, one);
    same &= one ? v : ~v;
  }
  return same;
}

// The whole sort in the first cluster of 1 or 8 CTAs of 1024 threads: R tokens
// a thread stay in registers while a pass ranks them, and go through the
// distributed shared memory of the cluster to their next place (8 bytes a
// token), 9 bits at most a pass.  A pass costs two cluster barriers instead of
// three launches (65,536 tokens, vocabulary 131,072: 45 us, against 84 in three
// passes of three launches).  The other clusters meanwhile write the zeros of
// the gradient, which need no order.
struct ClusterSmem {
  static constexpr int oCount = 0;                          // [32 warps][bins]
  static constexpr int oTotal = oCount + 32 * CS_BINS * 4;  // [bins], read by the other CTAs
  static constexpr int oBase = oTotal + CS_BINS * 4;
  static constexpr int oOwn = oBase + CS_BINS * 4;
  static constexpr int oWarp = oOwn + CS_BINS * 4;
  static constexpr int oBuf = oWarp + 256;                  // 2 x [1024 R] (key, index)
};
template <int R>
__global__ void __launch_bounds__(CS_THREADS)
cluster_sort_kernel(const void* __restrict__ ids, int wide, int ctas, int passes, int bits,
                    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ vals_out, int n,
                    int64_t V, int64_t zero_idx, uint4* __restrict__ zeros, int64_t zeros_bytes) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if ((int)blockIdx.x >= ctas) {
    const int64_t n16 = zeros_bytes / 16, step = (int64_t)(gridDim.x - ctas) * CS_THREADS;
    int64_t i = (int64_t)(blockIdx.x - ctas) * CS_THREADS + tid;
    if (i < zeros_bytes % 16 / 2) reinterpret_cast<uint16_t*>(zeros + n16)[i] = 0;
#pragma unroll 4
    for (; i < n16; i += step) zeros[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  extern __shared__ __align__(16) uint8_t cs_mem[];
  using L = ClusterSmem;
  uint32_t(*count)[CS_BINS] = reinterpret_cast<uint32_t(*)[CS_BINS]>(cs_mem + L::oCount);
  uint32_t* total = reinterpret_cast<uint32_t*>(cs_mem + L::oTotal);
  uint32_t* base = reinterpret_cast<uint32_t*>(cs_mem + L::oBase);
  uint32_t* part = reinterpret_cast<uint32_t*>(cs_mem + L::oWarp);
  uint32_t* own = reinterpret_cast<uint32_t*>(cs_mem + L::oOwn);
  uint2* buf = reinterpret_cast<uint2*>(cs_mem + L::oBuf);
  uint2* mine = buf + CS_THREADS * R;  // this CTA's tokens by digit
  constexpr int HELD = CS_THREADS * R;  // tokens of a CTA
  const uint32_t rank = tc::cluster_rank();
  const int local = warp * 32 * R + lane, first = (int)rank * HELD + local;
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
      const uint32_t peers = peers_of(d, bits, __ballot_sync(0xffffffffu, in));
      const uint32_t before = __popc(peers & ((1u << lane) - 1));
      at[r] = in ? count[warp][d] + before : 0;
      __syncwarp();
      if (in && before == 0) count[warp][d] += __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    if (tid < CS_BINS) {
      uint32_t sum = 0, c[32];
#pragma unroll
      for (int w = 0; w < 32; ++w) c[w] = count[w][tid];
#pragma unroll
      for (int w = 0; w < 32; ++w) {
        count[w][tid] = sum;
        sum += c[w];
      }
      total[tid] = sum;
    }
    tc::cluster_sync();  // every CTA's totals are there, every token in registers
    // base[d]: where this CTA's tokens of digit d go; own[d]: their first place
    // among its own
    uint32_t all = 0, before = 0, run = 0, mine_d = 0, run_own = 0;
    if (tid < CS_BINS) {
      for (int c = 0; c < ctas; ++c) {
        const uint32_t t = tc::ld_cluster(tc::map_rank(total + tid, c));
        all += t;
        before += c < (int)rank ? t : 0;
      }
      run = all;
      run_own = mine_d = total[tid];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, run, o);
        const uint32_t v = __shfl_up_sync(0xffffffffu, run_own, o);
        if (lane >= o) {
          run += u;
          run_own += v;
        }
      }
      if (lane == 31) {
        part[warp] = run;
        part[32 + warp] = run_own;
      }
    }
    __syncthreads();
    if (tid < CS_BINS) {
      uint32_t own_before = 0;
      for (int w = 0; w < warp; ++w) {
        before += part[w];
        own_before += part[32 + w];
      }
      base[tid] = before + run - all;
      own[tid] = own_before + run_own - mine_d;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (first + r * 32 >= n) continue;
      const uint32_t d = (key[r] >> shift) & mask;
      mine[own[d] + count[warp][d] + at[r]] = make_uint2(key[r], val[r]);
    }
    __syncthreads();
    // neighbours of one digit go to neighbouring places: few segments a warp
    const int held = n - (int)rank * HELD < HELD ? n - (int)rank * HELD : HELD;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int j = r * CS_THREADS + tid;
      if (j >= held) break;
      const uint2 kv = mine[j];
      const uint32_t d = (kv.x >> shift) & mask, to = base[d] + (uint32_t)j - own[d];
      tc::st_cluster2(tc::map_rank(buf + to % HELD, to / HELD), kv.x, kv.y);
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
    const int p = first + r * 32;
    if (p >= n) continue;
    keys_out[p] = key[r];
    vals_out[p] = val[r];
  }
}

// -------------------------------------------------------------- the sums
// A group of `width` threads takes one chunk of CHUNK sorted tokens and one
// vector of columns a thread, and adds the tokens' rows in order.  A run of one
// id that lies within the chunk is a row of gw, written at once; one that
// reaches into a neighbouring chunk leaves its sum in part[chunk][0] (it
// starts the chunk) or [1], for join_kernel.  Every token's row is read once,
// and no chunk has more to do than another.
constexpr int CHUNK = 32;

// Grid (chunks / groups, column tiles).  VEC > 1: rows are whole 16-byte vectors.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
chunk_kernel(const T* __restrict__ gy, const uint32_t* __restrict__ keys,
             const uint32_t* __restrict__ vals, float* __restrict__ part, T* __restrict__ gw,
             int64_t n, int64_t V, int64_t D, float scale, int width) {
  constexpr int AT_ONCE = 8;  // loads on their way
  const int64_t chunk = (int64_t)blockIdx.x * (256 / width) + threadIdx.x / width;
  const int64_t c = ((int64_t)blockIdx.y * width + threadIdx.x % width) * VEC;
  const int64_t b = chunk * CHUNK, e = b + CHUNK < n ? b + CHUNK : n;
  if (b >= n || c >= D) return;
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
  uint32_t key = keys[b];
  // whether the run at hand came from the chunk before, and where it began
  bool from_before = b > 0 && keys[b - 1] == key, at_start = true;
  const uint32_t after = e < n ? keys[e] : 0xffffffffu;
  auto flush = [&](bool goes_on) {
    if (key < (uint32_t)V) {
      if (from_before || goes_on) {
        float* p = part + (chunk * 2 + (at_start ? 0 : 1)) * D + c;
#pragma unroll
        for (int k = 0; k < VEC; ++k) p[k] = acc[k];
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[k] *= scale;
        store_vec<T, VEC>(gw + (int64_t)key * D + c, acc);
      }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = 0.f;
    from_before = at_start = false;
  };
  for (int64_t p = b; p < e; p += AT_ONCE) {
    uint32_t ks[AT_ONCE], vs[AT_ONCE];
    float v[AT_ONCE][VEC];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int64_t q = p + j < e ? p + j : e - 1;  // past the end: read again, not added
      ks[j] = keys[q];
      vs[j] = vals[q];
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) load_vec<T, VEC>(gy + (int64_t)vs[j] * D + c, v[j]);
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      if (p + j >= e) break;
      if (ks[j] != key) {
        flush(false);
        key = ks[j];
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] += v[j][k];
    }
  }
  flush(after == key);
}

// Rows of runs over several chunks: the CTAs of the chunk in which a run begins
// add its parts in order, a vector of columns a thread; over more than 8 parts,
// the 8 warps take every eighth part of 32 vectors in turn, and their sums are
// added in order.  Grid (chunks, D / (256 VEC)): most CTAs find no such run (a
// CTA for every 32 columns of every chunk spent 139 us, mostly on leaving).
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
join_kernel(const uint32_t* __restrict__ keys, const float* __restrict__ part, T* __restrict__ gw,
            int64_t n, int64_t V, int64_t D, float scale) {
  __shared__ float sums[8][256 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t j = blockIdx.x, b = j * CHUNK, e = b + CHUNK;
  if (e >= n) return;
  const int64_t chunks = (n + CHUNK - 1) / CHUNK;
  const uint32_t key = keys[e - 1], after = keys[e], at_b = keys[b];
  const uint32_t before = b > 0 ? keys[b - 1] : 0xffffffffu;
  const int64_t ahead = j + 2 + lane;  // the next 32 chunks but one, at the same time
  const uint32_t probe = ahead < chunks ? keys[ahead * CHUNK] : 0xffffffffu;
  if (key >= (uint32_t)V || after != key) return;
  const bool whole = at_b == key;
  if (whole && before == key) return;  // began earlier
  // chunks that start within the run: [j + 1, lo)
  int64_t lo = j + 2 + __popc(__ballot_sync(0xffffffffu, probe == key)), hi = chunks;
  if (lo < j + 34) hi = lo;
  while (lo < hi) {  // a 32-ary search
    const int64_t step = (hi - lo + 31) / 32, p = lo + lane * step;
    const int in = __popc(__ballot_sync(0xffffffffu, p < hi && keys[p * CHUNK] == key));
    if (in == 0) break;
    hi = hi < lo + in * step ? hi : lo + in * step;
    lo += (in - 1) * step + 1;
  }
  const float* first = part + (j * 2 + (whole ? 0 : 1)) * D;
  if (lo - j <= 8) {
    const int64_t c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * VEC;
    if (c >= D) return;
    float s[VEC], v[7][VEC];
    load_vec<float, VEC>(first + c, s);
#pragma unroll
    for (int k = 0; k < 7; ++k)
      if (j + 1 + k < lo) load_vec<float, VEC>(part + (j + 1 + k) * 2 * D + c, v[k]);
#pragma unroll
    for (int k = 0; k < 7; ++k)
      if (j + 1 + k < lo) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[i] += v[k][i];
      }
#pragma unroll
    for (int i = 0; i < VEC; ++i) gw[(int64_t)key * D + c + i] = from_f32<T>(s[i] * scale);
    return;
  }
  // a warp's parts: of 8 x 32 vectors two at a time, of narrow rows' 32 eight
  const int64_t c0 = ((int64_t)blockIdx.y * 256 + lane) * VEC;
  auto share = [&](auto tiles, auto parts) {
    constexpr int TILES = decltype(tiles)::value, PARTS = decltype(parts)::value;
    float s[TILES][VEC];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[t][i] = 0.f;
    auto add = [&](const float* p) {
      float v[TILES][VEC];
#pragma unroll
      for (int t = 0; t < TILES; ++t)
        if (c0 + t * 32 * VEC < D) load_vec<float, VEC>(p + c0 + t * 32 * VEC, v[t]);
#pragma unroll
      for (int t = 0; t < TILES; ++t)
        if (c0 + t * 32 * VEC < D) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) s[t][i] += v[t][i];
        }
    };
    if (warp == 0) add(first);
#pragma unroll PARTS
    for (int64_t k = j + 1 + warp; k < lo; k += 8) add(part + k * 2 * D);
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sums[warp][(t * 32 + lane) * VEC + i] = s[t][i];
  };
  if (D <= 32 * VEC) share(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
  else share(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
  __syncthreads();
  for (int x = threadIdx.x; x < 256 * VEC; x += 256) {
    const int64_t c = (int64_t)blockIdx.y * 256 * VEC + x;
    if (c >= D) break;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += sums[w][x];
    gw[(int64_t)key * D + c] = from_f32<T>(sum * scale);
  }
}

}  // namespace embed
}  // namespace theria
