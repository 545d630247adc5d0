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
// at one a value they would bound 16-bit tensors).  Where eight products
// overflow or come near the smallest float32, they are done again in float64, so
// that norms of very large and very small gradients are right.
#pragma once

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

// sum of a[i] * b[i]
template <int N>
__device__ __forceinline__ double dot(const float (&a)[N], const float (&b)[N]) {
  float s = 0.f, big = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s = fmaf(a[i], b[i], s);
    big = fmaxf(big, fabsf(a[i] * b[i]));
  }
  if (big > 1e-28f && big < 1e37f) return (double)s;
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (a[i] != 0.f && b[i] != 0.f) d = fma((double)a[i], (double)b[i], d);
  return d;
}

template <typename T, int VEC>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += VEC) {
    float w[VEC];
    embed::load_vec<T, VEC>(p + i, w);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[i + k] = w[k];
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += VEC) {
    float w[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) w[k] = v[i + k];
    embed::store_vec<T, VEC>(p + i, w);
  }
}

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

// part[block] = the block's share of sum x u (u NULL: of sum x^2).
__global__ void __launch_bounds__(THREADS)
dot_kernel(const __grid_constant__ Table t, double* part) {
  grid_launch();
  grid_wait();
  double acc = 0.0;
  for (int c = blockIdx.x; c < t.first[t.n]; c += gridDim.x)
    chunk_at(t, c, [&](auto e, int i, int64_t from, int n) {
      using T = decltype(e);
      const T* x = static_cast<const T*>(t.x[i]) + from;
      const T* u = static_cast<const T*>(t.u[i] ? t.u[i] : t.x[i]) + from;
      const bool same = x == u;
      int at = 0;
      if (t.vec[i]) {
        constexpr int VEC = embed::Vec<T>::n;
#pragma unroll 4
        for (int k = threadIdx.x * 8; k + 8 <= n; k += THREADS * 8) {
          float a[8], b[8];
          load8<T, VEC>(x + k, a);
          if (same) {
            acc += dot<8>(a, a);
          } else {
            load8<T, VEC>(u + k, b);
            acc += dot<8>(a, b);
          }
        }
        at = n / 8 * 8;
      }
      for (int k = at + threadIdx.x; k < n; k += THREADS) {
        const float a[1] = {to_f32<T>(x[k])}, b[1] = {to_f32<T>(u[k])};
        acc += dot<1>(a, b);
      }
    });
  acc = block_sum(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

__device__ __forceinline__ double all_parts(const double* part, int parts) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += THREADS) s += part[i];
  return block_sum(s);
}

// out = a x + b u, from the values a, b (u NULL: a x)
__device__ __forceinline__ void combine(const Table& t, float a, float b) {
  const int last = t.first[t.n] - 1;
  for (int c = blockIdx.x; c <= last; c += gridDim.x)
    chunk_at(t, last - c, [&](auto e, int i, int64_t from, int n) {
      using T = decltype(e);
      const T* x = static_cast<const T*>(t.x[i]) + from;
      const T* u = t.u[i] ? static_cast<const T*>(t.u[i]) + from : nullptr;
      T* out = static_cast<T*>(t.out[i]) + from;
      int at = 0;
      if (t.vec[i]) {
        constexpr int VEC = embed::Vec<T>::n;
#pragma unroll 4
        for (int k = threadIdx.x * 8; k + 8 <= n; k += THREADS * 8) {
          float v[8], w[8];
          load8<T, VEC>(x + k, v);
          if (u != nullptr) load8<T, VEC>(u + k, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = u != nullptr ? fmaf(a, v[j], b * w[j]) : a * v[j];
          store8<T, VEC>(out + k, v);
        }
        at = n / 8 * 8;
      }
      for (int k = at + threadIdx.x; k < n; k += THREADS) {
        const float v = to_f32<T>(x[k]);
        out[k] = from_f32<T>(u != nullptr ? fmaf(a, v, b * to_f32<T>(u[k])) : a * v);
      }
    });
}

// out = c x (out may be x; t.n == 0: the norm alone).  stats receives {norm, c}.
__global__ void __launch_bounds__(THREADS)
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
  if (c == 1.0 && t.out[0] == t.x[0]) return;  // in place, nothing to clip
  combine(t, (float)c, 0.f);
}

// out = a u + b x (see above); u NULL: out = b x.  part: the sums of x u.
__global__ void __launch_bounds__(THREADS)
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
  combine(t, parts > 0 ? (float)c : (float)b, (float)b);
}

}  // namespace grads
}  // namespace theria
