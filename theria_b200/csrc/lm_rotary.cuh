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
// remaining half turn at most is float32's to compute (sincospi, 1 to 2 units).
//
// With the halves apart a thread moves 16 bytes of each half where a half is a
// whole number of such vectors, else 16 bytes of the output whose partners it
// reads one by one (from the cache: a neighbour has just loaded them).
#pragma once

#include "common.cuh"
#include "lm_embed.cuh"

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

template <typename T, int VEC, int LAYOUT>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const Args a) {
  extern __shared__ float2 turn[];  // [tokens][pairs] {cos, sin} * amplitude
  const int64_t first = (int64_t)blockIdx.x * a.tokens;
  const int tokens = (int)min((int64_t)a.tokens, a.n - first);
  for (int i = threadIdx.x; i < tokens * a.pairs; i += THREADS) {
    const int t = i / a.pairs, m = i % a.pairs;
    const double turns = (double)position_of(a, first + t) * a.freq[m] * 0.15915494309189533577;
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    turn[i] = make_float2(c * a.amplitude, (a.back ? -s : s) * a.amplitude);
  }
  __syncthreads();
  const int halves = LAYOUT == kHalves ? a.pairs / VEC : 0;  // units of both halves at once
  const unsigned units = a.D / VEC - halves;                // a head's
  const unsigned heads = a.heads[0] + a.heads[1];
  const unsigned all = (unsigned)tokens * heads * units;
  for (unsigned i = threadIdx.x; i < all; i += THREADS) {
    const unsigned th = i / units, u = i - th * units;
    const unsigned t = th / heads;
    int h = th - t * heads;
    const int side = h >= a.heads[0];
    if (side) h -= a.heads[0];
    const Side& sd = a.s[side];
    const int64_t tok = first + t, b = tok / a.T, at = tok - b * a.T;
    const T* x = static_cast<const T*>(sd.x) + b * sd.xb + at * sd.xt + h * sd.xh;
    T* y = static_cast<T*>(sd.y) + b * sd.yb + at * sd.yt + h * sd.yh;
    const float2* cs = turn + t * a.pairs;
    if constexpr (LAYOUT == kHalves) {
      if ((int)u < halves) {
        const int m = u * VEC;
        float p[VEC], q[VEC];
        embed::load_vec<T, VEC>(x + m, p);
        embed::load_vec<T, VEC>(x + a.pairs + m, q);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float2 w = cs[m + e];
          const float f = p[e], g = q[e];
          p[e] = f * w.x - g * w.y;
          q[e] = g * w.x + f * w.y;
        }
        embed::store_vec<T, VEC>(y + m, p);
        embed::store_vec<T, VEC>(y + a.pairs + m, q);
      } else {
        const int d = (u + halves) * VEC;
        float p[VEC];
        embed::load_vec<T, VEC>(x + d, p);
        embed::store_vec<T, VEC>(y + d, p);
      }
    } else {
      const int d0 = u * VEC;
      float p[VEC], r[VEC];
      embed::load_vec<T, VEC>(x + d0, p);
#pragma unroll
      for (int e = 0; e < VEC; ++e) r[e] = p[e];
      if (d0 < 2 * a.pairs) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int d = d0 + e;
          if (d >= 2 * a.pairs) continue;
          // the first of a pair gets a cos - b sin, the second b cos + a sin
          bool second;
          float other;
          int m;
          if constexpr (LAYOUT == kInterleaved) {
            second = d & 1;
            m = d >> 1;
            other = VEC > 1 ? p[e ^ (VEC > 1)] : to_f32<T>(x[d ^ 1]);
          } else {
            second = d >= a.pairs;
            m = second ? d - a.pairs : d;
            other = to_f32<T>(x[second ? m : d + a.pairs]);
          }
          const float2 w = cs[m];
          r[e] = p[e] * w.x + (second ? other * w.y : -(other * w.y));
        }
      }
      embed::store_vec<T, VEC>(y + d0, r);
    }
  }
}

}  // namespace rotary
}  // namespace theria
