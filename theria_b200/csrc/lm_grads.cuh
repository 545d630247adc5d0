// The global norm of many tensors and their clipping by it, with the gradient.
//
//   norm = sqrt(sum of x^2 over all values of all tensors)
//   y    = c x,   c = min(1, max / norm)
//   back:  dx = a u + b x,  a = c,  b = -c (x . u) / norm^2 + dnorm / norm
//          (the first part of b only where the norm is over max)
//
// Memory bound: one launch reads every value for the sums, a second reads and
// writes it again.  The tensors come as a table in the kernel's parameters
// (nothing is copied to the device first, so a call can be captured), cut into
// chunks that the blocks of a fixed grid take in turn; each block leaves one
// float64 sum, and every block of the second launch adds those in one order.
// No atomics: the same inputs give the same bits.  The second launch starts
// with the chunks that the first read last, which L2 still holds.
//
// A thread multiplies and adds 8 values at a time in float32 and takes those
// sums to float64, which costs an eighth of the conversions (16 a cycle and SM:
// at one a value they would bound 16-bit tensors).  A thread that meets very large
// or very small values does its part of the chunk again in float64, so that norms
// of such gradients are right.  The second launch multiplies in float32, and in
// float64 where a factor is beyond float32's normal range.
#pragma once

#include <cfloat>

#include "common.cuh"
#include "lm_embed.cuh"

namespace theria {
namespace grads {

constexpr int THREADS = 256;
constexpr int CHUNK = 8192;    // values
constexpr int MOST = 256;      // tensors of one launch
constexpr int MOST_BLOCKS = 592;  // of the sums: 4 an SM, 2048 threads with 2 launches

struct Table {
  const void* x[MOST];
  const void* u[MOST];
  void* out[MOST];
  int64_t size[MOST];
  int first[MOST + 1];          // chunk at which each tensor starts
  unsigned char dtype[MOST];
  unsigned char vec[MOST];      // its pointers are 16-byte aligned
  int n;
  bool in_place;                // every out is its x
};

template <typename F>
__device__ __forceinline__ void by_type(int dtype, F f) {
  if (dtype == THERIA_F32) f(float{});
  else if (dtype == THERIA_F16) f(__half{});
  else f(__nv_bfloat16{});
}

// The tensor of a chunk.
__device__ __forceinline__ int tensor_of(const Table& t, int chunk) {
  int lo = 0, hi = t.n;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (t.first[m] <= chunk) lo = m; else hi = m;
  }
  return lo;
}

// Values whose products, or sums of a few, may leave float32's range.
__device__ __forceinline__ bool extreme(float big) {
  return big > 1e17f || (big < 1e-13f && big != 0.f);
}

// 8 values as they lie in memory, so that a thread can have several in flight.
template <typename T>
struct Eight {
  static constexpr int n = 8 * sizeof(T) / 16;
  uint4 r[n];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < n; ++i) r[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const T* e = reinterpret_cast<const T*>(r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(e[i]);
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    T* e = reinterpret_cast<T*>(r);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < n; ++i) reinterpret_cast<uint4*>(p)[i] = r[i];
  }
};
// A thread's eights of a whole chunk, and how many of them it has in flight (64 bytes).
constexpr int EIGHTS = CHUNK / (THREADS * 8);
template <typename T> constexpr int kFlight = 64 / (8 * (int)sizeof(T));

// The block's sum, in every thread.
__device__ __forceinline__ double block_sum(double x) {
  __shared__ double warps[THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = x;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) s += warps[w];
  return s;
}

// Calls f(T{}, p, n) for the chunk's values: tensor type, index of the tensor,
// first value and number of values.
template <typename F>
__device__ __forceinline__ void chunk_at(const Table& t, int chunk, F f) {
  const int i = tensor_of(t, chunk);
  const int64_t from = (int64_t)(chunk - t.first[i]) * CHUNK;
  const int n = (int)min((int64_t)CHUNK, t.size[i] - from);
  by_type(t.dtype[i], [&](auto e) { f(e, i, from, n); });
}

// part[block] = the block's share of sum x u (SAME: of sum x^2).
template <bool SAME>
__global__ void __launch_bounds__(THREADS, SAME ? 4 : 3)
dot_kernel(const __grid_constant__ Table t, double* part) {
  grid_launch();
  grid_wait();
  double acc = 0.0;
  for (int c = blockIdx.x; c < t.first[t.n]; c += gridDim.x)
    chunk_at(t, c, [&](auto e, int i, int64_t from, int n) {
      using T = decltype(e);
      const T* x = static_cast<const T*>(t.x[i]) + from;
      const T* u = static_cast<const T*>(SAME ? t.x[i] : t.u[i]) + from;
      bool odd = false;  // an eight of this thread is extreme
      double sum = 0.0;
      int at = 0;
      if (t.vec[i]) {
        constexpr int F = kFlight<T>;
#pragma unroll 1
        for (int j0 = 0; j0 < EIGHTS; j0 += F) {
          Eight<T> ra[F], rb[F];
#pragma unroll
          for (int j = 0; j < F; ++j) {
            const int k = ((j0 + j) * THREADS + threadIdx.x) * 8;
            if (k + 8 > n) continue;
            ra[j].load(x + k);
            if constexpr (!SAME) rb[j].load(u + k);
          }
#pragma unroll
          for (int j = 0; j < F; ++j) {
            if (((j0 + j) * THREADS + (int)threadIdx.x) * 8 + 8 > n) continue;
            float a[8], b[8], s = 0.f, ma = 0.f, mb = 0.f;
            ra[j].get(a);
            if constexpr (!SAME) rb[j].get(b);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              s = fmaf(a[e], SAME ? a[e] : b[e], s);
              ma = fmaxf(ma, fabsf(a[e]));
              if constexpr (!SAME) mb = fmaxf(mb, fabsf(b[e]));
            }
            odd |= extreme(ma) || (!SAME && extreme(mb));
            sum += (double)s;
          }
        }
        at = n / 8 * 8;
      }
      if (odd) {  // the thread's eights again, in float64
        sum = 0.0;
        for (int k0 = threadIdx.x * 8; k0 + 8 <= n; k0 += THREADS * 8)
          for (int k = k0; k < k0 + 8; ++k)
            sum = fma((double)to_f32<T>(x[k]), (double)to_f32<T>(u[k]), sum);
      }
      for (int k = at + threadIdx.x; k < n; k += THREADS)
        sum = fma((double)to_f32<T>(x[k]), (double)to_f32<T>(u[k]), sum);
      acc += sum;
    });
  acc = block_sum(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

__device__ __forceinline__ double all_parts(const double* part, int parts) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += THREADS) s += part[i];
  return block_sum(s);
}

// out = a x + b u (TWO false: a x)
template <bool TWO>
__device__ __forceinline__ void combine(const Table& t, float a, float b) {
  const int last = t.first[t.n] - 1;
  for (int c = blockIdx.x; c <= last; c += gridDim.x)
    chunk_at(t, last - c, [&](auto e, int i, int64_t from, int n) {
      using T = decltype(e);
      const T* x = static_cast<const T*>(t.x[i]) + from;
      const T* u = static_cast<const T*>(TWO ? t.u[i] : t.x[i]) + from;
      T* out = static_cast<T*>(t.out[i]) + from;
      int at = 0;
      if (t.vec[i]) {
        constexpr int F = kFlight<T>;
#pragma unroll 1
        for (int j0 = 0; j0 < EIGHTS; j0 += F) {
          Eight<T> rx[F], ru[F];
#pragma unroll
          for (int j = 0; j < F; ++j) {
            const int k = ((j0 + j) * THREADS + threadIdx.x) * 8;
            if (k + 8 > n) continue;
            rx[j].load(x + k);
            if constexpr (TWO) ru[j].load(u + k);
          }
#pragma unroll
          for (int j = 0; j < F; ++j) {
            const int k = ((j0 + j) * THREADS + threadIdx.x) * 8;
            if (k + 8 > n) continue;
            float v[8], w[8];
            rx[j].get(v);
            if constexpr (TWO) ru[j].get(w);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = TWO ? fmaf(a, v[e], b * w[e]) : a * v[e];
            rx[j].set(v);
            rx[j].store(out + k);
          }
        }
        at = n / 8 * 8;
      }
      for (int k = at + threadIdx.x; k < n; k += THREADS) {
        const float v = to_f32<T>(x[k]);
        out[k] = from_f32<T>(TWO ? fmaf(a, v, b * to_f32<T>(u[k])) : a * v);
      }
    });
}

// A factor that float32 has no normal number for: with norms near either end of
// float32's range c, and b more so, lie beyond it while a x + b u does not.
__device__ __forceinline__ bool beyond(double f) {
  const double m = fabs(f);
  return m != 0.0 && (m < (double)FLT_MIN || (m > (double)FLT_MAX && m < INFINITY));
}

// The same as combine, each value in float64: for factors beyond float32.
template <bool TWO>
__device__ __noinline__ void combine_wide(const Table& t, double a, double b) {
  const int last = t.first[t.n] - 1;
  for (int c = blockIdx.x; c <= last; c += gridDim.x)
    chunk_at(t, last - c, [&](auto e, int i, int64_t from, int n) {
      using T = decltype(e);
      const T* x = static_cast<const T*>(t.x[i]) + from;
      const T* u = static_cast<const T*>(TWO ? t.u[i] : t.x[i]) + from;
      T* out = static_cast<T*>(t.out[i]) + from;
      for (int k = threadIdx.x; k < n; k += THREADS) {
        double v = a * (double)to_f32<T>(x[k]);
        if (TWO) v = fma(b, (double)to_f32<T>(u[k]), v);
        out[k] = from_f32<T>((float)v);
      }
    });
}

// out = c x (out may be x; t.n == 0: the norm alone).  stats receives {norm, c}.
__global__ void __launch_bounds__(THREADS, 4)
clip_kernel(const __grid_constant__ Table t, const double* part, int parts, double most,
            float* norm, double* stats) {
  grid_wait();
  const double n = sqrt(all_parts(part, parts));
  const double c = n <= most ? 1.0 : most / n;  // NaN: every value becomes NaN
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (norm != nullptr) *norm = (float)n;
    if (stats != nullptr) {
      stats[0] = n;
      stats[1] = c;
    }
  }
  if (t.n == 0) return;
  if (c == 1.0 && t.in_place) return;  // in place, nothing to clip
  if (beyond(c)) combine_wide<false>(t, c, 0.0);
  else combine<false>(t, (float)c, 0.f);
}

// out = a u + b x (see above); u NULL: out = b x.  part: the sums of x u.
template <bool TWO>
__global__ void __launch_bounds__(THREADS, TWO ? 3 : 4)
clip_bwd_kernel(const __grid_constant__ Table t, const double* part, int parts,
                const double* stats, const float* gnorm) {
  grid_wait();
  const double n = stats[0], c = stats[1];
  double b = 0.0;
  if (gnorm != nullptr && n != 0.0) b = (double)*gnorm / n;
  if (parts > 0) {
    const double xu = all_parts(part, parts);
    if (c != 1.0) b -= c * xu / n / n;
  }
  // with u, the table has it first: combine's x is u, its u is x
  const double a = TWO ? c : b;
  // (|b x| <= |b| n, which may leave float32's range where the sum does not)
  if (beyond(a) || beyond(b) || beyond(b * n)) combine_wide<TWO>(t, a, b);
  else combine<TWO>(t, (float)a, (float)b);
}

}  // namespace grads
}  // namespace theria
