// Rotary positions.  The pair m of a head at position t turns by the angle
// t * w_m: (a, b) -> amplitude * (a cos - b sin, b cos + a sin); the gradient
// turns back.  Pairs lie side by side (interleaved) or half the rotated part
// apart; values behind the rotated part pass through.
//
// Memory bound: each value is read and written once, queries and keys in one
// launch.  A block takes a few tokens; their angles are shared by all heads, so
// cos and sin go to shared memory first.  The angle is reduced in float64: t *
// w in float32 would be off by t * w * 2^-24, 0.06 at position 10^6.  As whole
// turns less their nearest integer it is exact to 2^-52 t w / 2 pi turns, and the
// remaining half turn at most is float32's to compute (sincospi, 1 to 2 units), as are
// the products with the amplitude and the pair.
//
// A thread stays on one column of 16 bytes of the heads and has the loads of four
// rows (token, head) in flight.  With the halves apart it moves 16 bytes of each half
// where a half is a whole number of such vectors, else 16 bytes of the output whose
// partners it reads one by one (from the cache: a neighbour has just loaded them).
#pragma once

#include "common.cuh"
#include "tc_common.cuh"

namespace theria {
namespace rotary {

constexpr int THREADS = 256;
constexpr int MOST_TOKENS = 16;  // of a block

enum Layout { kHalves = 0, kHalvesAnywhere = 1, kInterleaved = 2 };

struct Side {  // queries or keys
  const void* x;
  void* y;
  int64_t xb, xt, xh, yb, yt, yh;  // strides of batch, token, head in elements
};

struct Args {
  Side s[2];
  int heads[2];
  int T, D, pairs;       // tokens of a batch, values of a head, rotated pairs
  int64_t n;             // tokens in all
  const void* positions; // [n_positions], token i's at i % n_positions; or NULL
  int64_t n_positions;
  const void* offsets;   // [S + 1]: positions count from each sequence's start; or NULL
  int S, wide;
  const double* freq;    // [pairs]
  float amplitude;
  int back, tokens;      // the angle negated; tokens of a block
  uint64_t magic;        // 2^32 / heads + 1: row / heads as a product's high half
};

__device__ __forceinline__ int64_t int_at(const void* p, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int*>(p)[i];
}

// Token i's position; 0 for a token of no sequence.
__device__ __forceinline__ int64_t position_of(const Args& a, int64_t i) {
  if (a.positions != nullptr) return int_at(a.positions, a.wide, i % a.n_positions);
  i %= a.T;
  if (a.offsets == nullptr) return i;
  if (i < int_at(a.offsets, a.wide, 0) || i >= int_at(a.offsets, a.wide, a.S)) return 0;
  int lo = 0, hi = a.S;  // offsets[lo] <= i < offsets[hi]
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (int_at(a.offsets, a.wide, m) <= i) lo = m; else hi = m;
  }
  return i - int_at(a.offsets, a.wide, lo);
}

// VEC values as they lie in memory, and as floats.
template <typename T, int VEC>
struct Raw {
  uint4 r;
  __device__ __forceinline__ void load(const T* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = r; }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (VEC == 4) v[i] = __uint_as_float(w[i]);
      else tc::unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void set(const float (&v)[VEC]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (VEC == 4) w[i] = __float_as_uint(v[i]);
      else w[i] = tc::pack2<T>(v[2 * i], v[2 * i + 1]);
    }
    r = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <typename T>
struct Raw<T, 1> {
  T r;
  __device__ __forceinline__ void load(const T* p) { r = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = r; }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = to_f32<T>(r); }
  __device__ __forceinline__ void set(const float (&v)[1]) { r = from_f32<T>(v[0]); }
};

// N floats of shared memory, 16 bytes at a time where N is a multiple of 4 and
// they start on such a boundary.
template <int N>
__device__ __forceinline__ void load_floats(const float* p, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 q = *reinterpret_cast<const float4*>(p + i);
      v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 q = *reinterpret_cast<const float2*>(p + i);
      v[i] = q.x; v[i + 1] = q.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = p[i];
  }
}

template <typename T, int VEC, int LAYOUT>
__global__ void __launch_bounds__(THREADS, 4) rotary_kernel(const Args a) {
  // [tokens][2][padded pairs]: all cos * amplitude of a token, then all sin
  extern __shared__ float4 turn4[];
  float* turn = reinterpret_cast<float*>(turn4);
  const int padded = (a.pairs + 3) & ~3;
  __shared__ double at_pos[MOST_TOKENS];
  __shared__ int64_t base[MOST_TOKENS][4];  // where the token's q, yq, k, yk start
  constexpr int LOADS = LAYOUT == kHalves ? 2 : 4;  // heads in flight
  using R = Raw<T, VEC>;
  const int64_t first = (int64_t)blockIdx.x * a.tokens;
  const int tokens = (int)min((int64_t)a.tokens, a.n - first);
  if ((int)threadIdx.x < tokens) {
    const int64_t tok = first + threadIdx.x, b = tok / a.T, at = tok - b * a.T;
    at_pos[threadIdx.x] = (double)position_of(a, tok);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      base[threadIdx.x][2 * i] = b * a.s[i].xb + at * a.s[i].xt;
      base[threadIdx.x][2 * i + 1] = b * a.s[i].yb + at * a.s[i].yt;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tokens * a.pairs; i += THREADS) {
    const int t = i / a.pairs, m = i - t * a.pairs;
    const double turns = at_pos[t] * a.freq[m] * 0.15915494309189533577;
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    turn[2 * t * padded + m] = c * a.amplitude;
    turn[(2 * t + 1) * padded + m] = (a.back ? -s : s) * a.amplitude;
  }
  __syncthreads();
  const int halves = LAYOUT == kHalves ? a.pairs / VEC : 0;  // columns of both halves at once
  const int columns = a.D / VEC - halves;                   // of a head
  const unsigned heads = a.heads[0] + a.heads[1], all = tokens * heads;
  // threads over the columns of a head, then over the rows (token, head)
  const int wide = min(columns, THREADS), step = THREADS / wide;
  const int row0 = threadIdx.x / wide;
  if (row0 >= step) return;
  for (int u = threadIdx.x % wide; u < columns; u += wide) {
    const bool both = LAYOUT == kHalves && u < halves;
    const int d0 = (LAYOUT == kHalves && !both ? u + halves : u) * VEC;
    const bool turns = LAYOUT == kHalves ? both : d0 < 2 * a.pairs;
    for (unsigned rb = row0; rb < all; rb += LOADS * step) {
      const T* x[LOADS];
      T* y[LOADS];
      R p[LOADS], q[LAYOUT == kHalves ? LOADS : 1];
      int cs_at[LOADS];
#pragma unroll
      for (int k = 0; k < LOADS; ++k) {
        const unsigned r = rb + k * step;
        if (r >= all) continue;
        const unsigned t = (unsigned)((r * a.magic) >> 32);
        int h = r - t * heads;
        const int i = h >= a.heads[0];
        if (i) h -= a.heads[0];
        x[k] = static_cast<const T*>(a.s[i].x) + base[t][2 * i] + h * a.s[i].xh + d0;
        y[k] = static_cast<T*>(a.s[i].y) + base[t][2 * i + 1] + h * a.s[i].yh + d0;
        cs_at[k] = 2 * t * padded;
        p[k].load(x[k]);
        if constexpr (LAYOUT == kHalves)
          if (both) q[k].load(x[k] + a.pairs);
      }
#pragma unroll
      for (int k = 0; k < LOADS; ++k) {
        if (rb + k * step >= all) continue;
        const float *cs = turn + cs_at[k], *sn = cs + padded;
        if (turns) {
          float v[VEC];
          p[k].get(v);
          if constexpr (LAYOUT == kHalves) {
            float g[VEC], c[VEC], n[VEC], r[VEC];
            q[k].get(g);
            load_floats(cs + d0, c);
            load_floats(sn + d0, n);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              r[e] = v[e] * c[e] - g[e] * n[e];
              g[e] = g[e] * c[e] + v[e] * n[e];
            }
            p[k].set(r);
            q[k].set(g);
            q[k].store(y[k] + a.pairs);
          } else if constexpr (LAYOUT == kInterleaved && VEC > 1) {
            // a vector holds whole pairs; the last may go past the rotated ones (the
            // floats read there are not used)
            float c[VEC / 2], n[VEC / 2];
            load_floats(cs + d0 / 2, c);
            load_floats(sn + d0 / 2, n);
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
              const float f = v[e], g = v[e + 1];
              const bool on = d0 + e < 2 * a.pairs;
              v[e] = on ? f * c[e / 2] - g * n[e / 2] : f;
              v[e + 1] = on ? g * c[e / 2] + f * n[e / 2] : g;
            }
            p[k].set(v);
          } else {
            // the first of a pair gets a cos - b sin, the second b cos + a sin
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
              const int d = d0 + e;
              if (d >= 2 * a.pairs) continue;
              const bool second = LAYOUT == kInterleaved ? d & 1 : d >= a.pairs;
              const int far = LAYOUT == kInterleaved ? 1 : a.pairs;
              const int m = LAYOUT == kInterleaved ? d >> 1 : second ? d - a.pairs : d;
              const float other = to_f32<T>(x[k][second ? e - far : e + far]);
              v[e] = v[e] * cs[m] + (second ? other * sn[m] : -(other * sn[m]));
            }
            p[k].set(v);
          }
        }
        p[k].store(y[k]);
      }
    }
  }
}

}  // namespace rotary
}  // namespace theria
