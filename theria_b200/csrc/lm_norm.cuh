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
// The mean is kept as two floats, itself and what its rounding left (`left`):
// with a mean far above the deviations half a unit of the one float would shift
// every xhat of the row.
//
// Both directions are bound by HBM: x read and y written once, then x and gy
// read and gx written once.  A row stays in registers between its load and
// its store; the variance is taken around the mean already known, so it loses
// nothing to cancellation.  Statistics, sums and the weight gradients are
// float32; each result is rounded once.  The sums over rows go through per-CTA
// partials added by a second kernel in a fixed order: the same bits every time.
//
// Measured: 16384 x 4096 bfloat16 forward 54 us (5.0 TB/s), backward 78 us (5.1
// TB/s) and 3 us for the column sums, second derivative 243 us (2.8 TB/s);
// float32 83 us (6.5 TB/s), 128 (6.3) and 305 (4.4).  By its counters no unit is
// full in either 16-bit direction: the forward issues in 67 % of its cycles (19
// instructions a value), and its warps, 46 % of the most an SM holds, mostly wait
// for loads; the backward issues in 62 % (25 instructions a value), uses 45 % of
// the shared-memory pipe and 57 % of DRAM.  For each of its instructions 2.6 warps
// stand ready but not chosen and 1.7 wait for the arithmetic pipe: work in bursts,
// between the barriers of a batch's rows.  Rows that are no 16-byte vectors go
// value by value: 32768 x 1111 float16 104, 132 and 460 us.
#pragma once

#include "common.cuh"
#include "lm_embed.cuh"  // load_vec / store_vec
#include "tc_common.cuh"

namespace theria {
namespace norm {

using embed::load_vec;
using embed::store_vec;

constexpr int SUMS = 7;  // the most values one reduction carries

// NW warps own a row (one of several in the CTA for NW == 1, else the whole
// CTA); sums of NS values over it.  `red` alternates between two halves from
// call to call, so one barrier per call is enough.
template <int NW, int NS>
__device__ __forceinline__ void row_sum(float (&s)[NS], float (*red)[32][SUMS], int& turn) {
#pragma unroll
  for (int i = 0; i < NS; ++i) s[i] = warp_sum(s[i]);
  if constexpr (NW > 1) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float (*r)[SUMS] = red[turn];
    turn ^= 1;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < NS; ++i) r[warp][i] = s[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if constexpr (NW >= 8) {
        s[i] = warp_sum(lane < NW ? r[lane][i] : 0.f);
      } else {
        s[i] = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) s[i] += r[w][i];
      }
    }
  }
}

// VEC affine values from column c (float32 where f32, else x's type; NULL:
// `none`).  VEC > 1: p is 16-byte aligned there.
template <typename T, int VEC>
__device__ __forceinline__ void affine_vec(const void* p, bool f32, int64_t c, float none,
                                           float (&v)[VEC]) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = none;
  } else if (sizeof(T) == 4 || !f32) {
    load_vec<T, VEC>(static_cast<const T*>(p) + c, v);
  } else if constexpr (VEC == 8) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + c);
    const float4 a = q[0], b = q[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = static_cast<const float*>(p)[c + k];
  }
}
// Vector arithmetic two values to an instruction (issue slots, not HBM, set the
// pace of 16-bit rows otherwise: 20 instructions a value without).
struct Pair {
  float a = 0.f, b = 0.f;
  __device__ __forceinline__ float total() const { return a + b; }
};
template <int VEC>
__device__ __forceinline__ void vsum(Pair& p, const float (&v)[VEC]) {  // p += sum v
  if constexpr (VEC == 1) {
    p.a += v[0];
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 2) tc::add2(p.a, p.b, p.a, p.b, v[k], v[k + 1]);
  }
}
template <int VEC>  // p += sum u v
__device__ __forceinline__ void vdot(Pair& p, const float (&u)[VEC], const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    p.a = fmaf(u[0], v[0], p.a);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 2)
      tc::fma2(p.a, p.b, u[k], u[k + 1], v[k], v[k + 1], p.a, p.b);
  }
}
template <int VEC>  // d = a b + c
__device__ __forceinline__ void vfma(float (&d)[VEC], const float (&a)[VEC],
                                     const float (&b)[VEC], const float (&c)[VEC]) {
  if constexpr (VEC == 1) {
    d[0] = fmaf(a[0], b[0], c[0]);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 2)
      tc::fma2(d[k], d[k + 1], a[k], a[k + 1], b[k], b[k + 1], c[k], c[k + 1]);
  }
}
template <int VEC>  // d = a m + s
__device__ __forceinline__ void vscale(float (&d)[VEC], const float (&a)[VEC], float m, float s) {
  if constexpr (VEC == 1) {
    d[0] = fmaf(a[0], m, s);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 2) tc::fma2(d[k], d[k + 1], a[k], a[k + 1], m, m, s, s);
  }
}
template <int VEC>  // d += a m
__device__ __forceinline__ void vaxpy(float (&d)[VEC], const float (&a)[VEC], float m) {
  if constexpr (VEC == 1) {
    d[0] = fmaf(a[0], m, d[0]);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 2)
      tc::fma2(d[k], d[k + 1], a[k], a[k + 1], m, m, d[k], d[k + 1]);
  }
}
template <int VEC>  // d += a
__device__ __forceinline__ void vadd(float (&d)[VEC], const float (&a)[VEC]) {
  if constexpr (VEC == 1) {
    d[0] += a[0];
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 2) tc::add2(d[k], d[k + 1], d[k], d[k + 1], a[k], a[k + 1]);
  }
}
template <int VEC>  // d += s
__device__ __forceinline__ void vshift(float (&d)[VEC], float s) {
  if constexpr (VEC == 1) {
    d[0] += s;
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 2) tc::add2(d[k], d[k + 1], d[k], d[k + 1], s, s);
  }
}
template <int VEC>  // d *= a
__device__ __forceinline__ void vmul(float (&d)[VEC], const float (&a)[VEC]) {
  if constexpr (VEC == 1) {
    d[0] *= a[0];
  } else {
#pragma unroll
    for (int k = 0; k < VEC; k += 2) tc::mul2(d[k], d[k + 1], d[k], d[k + 1], a[k], a[k + 1]);
  }
}

// A row's statistics, 16 bytes: the mean rounded, the reciprocal standard
// deviation, what the mean's rounding left, and 0.  xhat = (x - mean) rstd + off,
// where the difference is exact for a mean far above the deviations.
struct Stats {
  float mean, rstd, off;
  __device__ __forceinline__ explicit Stats(const float* p) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    mean = v.x;
    rstd = v.y;
    off = -v.z * v.y;
  }
  __device__ __forceinline__ float xhat(float x) const { return fmaf(x - mean, rstd, off); }
};
// Stores row r's, where `own`; the mean comes as `mean` + `left`.  One predicated
// store whose address is made here: as an expression it becomes a pointer carried
// through the rows' loop, two registers that the row needs (65536 x 1024 bfloat16
// 58 us, this way 54).
__device__ __forceinline__ void store_stats(float* stats, int64_t r, bool own, float mean,
                                            float left, float rstd) {
  const float m = mean + left, rest = (mean - m) + left;
  asm volatile(
      "{\n\t.reg .pred q;\n\t.reg .b64 a;\n\t"
      "setp.ne.s32 q, %0, 0;\n\t"
      "shl.b64 a, %1, 4;\n\t"
      "add.s64 a, a, %2;\n\t"
      "@q st.global.v4.f32 [a], {%3, %4, %5, %6};\n\t}" ::"r"((int)own),
      "l"(r), "l"(stats), "f"(m), "f"(rstd), "f"(rest), "f"(0.f)
      : "memory");
}

// One affine value, for the kernels of wide rows.
__device__ __forceinline__ float affine(const void* p, int dtype, int64_t i, float none) {
  return p ? load_any(p, i, dtype) : none;
}

// Threads and rows of a CTA whose rows belong to NW warps.
template <int NW> struct Block {
  static constexpr int threads = NW == 1 ? 256 : NW * 32;
  static constexpr int G = NW * 32;        // threads of a row
  static constexpr int rows = threads / G; // rows at a time
  // CTAs an SM, for 128 registers a thread at most
  static constexpr int least = threads < 512 ? 512 / threads : 1;
};

// Sums of M values (a power of two) over NW warps.  Each step of the butterfly
// halves the values a lane keeps, so M sums cost little more than one.
template <int NW, int M>
__device__ __forceinline__ void batch_sum(float (&s)[M], float (*red)[32][8], int& turn) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int LANES = 32 / M;  // lanes that end with the same value
  float t[M];
#pragma unroll
  for (int i = 0; i < M; ++i) t[i] = s[i];
#pragma unroll
  for (int m = M, o = 16; o > 0; m >>= 1, o >>= 1) {
    if (m > 1) {
#pragma unroll
      for (int i = 0; i < m / 2; ++i) {
        const bool upper = lane & o;
        const float give = upper ? t[i] : t[i + m / 2], keep = upper ? t[i + m / 2] : t[i];
        t[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
    } else {
      t[0] += __shfl_xor_sync(0xffffffffu, t[0], o);
    }
  }
  if constexpr (NW > 1) {
    float (*r)[8] = red[turn];
    turn ^= 1;
    if (lane % LANES == 0) r[warp][lane / LANES] = t[0];
    __syncthreads();
    t[0] = 0.f;
#pragma unroll
    for (int w = 0; w < (NW + LANES - 1) / LANES; ++w)
      if (w * LANES + lane % LANES < NW) t[0] += r[w * LANES + lane % LANES][lane / LANES];
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) t[0] += __shfl_xor_sync(0xffffffffu, t[0], o);
  }
#pragma unroll
  for (int i = 0; i < M; ++i) s[i] = __shfl_sync(0xffffffffu, t[0], i * LANES);
}

// NW warps per row, R rows at a time, NV vectors of VEC values of each per
// thread; the rows go through the reductions together and share the affine
// values.  1024 threads an SM (64 registers), so that as many rows as possible
// are on their way.
template <typename T, int VEC, int NV, int NW, int R>
__global__ void __launch_bounds__(Block<NW>::threads, 1024 / Block<NW>::threads)
fwd_kernel(const T* __restrict__ x, const void* __restrict__ w, const void* __restrict__ b,
           int wf32, T* __restrict__ y, float* __restrict__ stats, int64_t N, int D, float eps) {
  constexpr int G = Block<NW>::G, ROWS = Block<NW>::rows * R;
  __shared__ float red[2][32][8];
  int turn = 0;
  const int g = threadIdx.x % G;
  const float inv = 1.f / (float)D;
  for (int64_t r0 = (int64_t)blockIdx.x * ROWS + threadIdx.x / G * R; r0 < N;
       r0 += (int64_t)gridDim.x * ROWS) {
    float v[R][NV][VEC];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * G + g) * VEC;
        // past the last row: the last one again, not stored
        if (c < D) load_vec<T, VEC>(x + (r0 + i < N ? r0 + i : N - 1) * D + c, v[i][j]);
      }
    float s[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      Pair sum;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if ((j * G + g) * VEC < D) vsum(sum, v[i][j]);
      s[i] = sum.total();
    }
    batch_sum<NW>(s, red, turn);
    float q[2 * R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      Pair dev, sq;
      s[i] *= inv;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if ((j * G + g) * VEC < D) {
          vshift(v[i][j], -s[i]);
          vdot(sq, v[i][j], v[i][j]);
          vsum(dev, v[i][j]);
        }
      q[2 * i] = sq.total();
      q[2 * i + 1] = dev.total();
    }
    batch_sum<NW>(q, red, turn);
    float rstd[R], off[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      // what the rounding of a large mean left in the deviations
      const float left = q[2 * i + 1] * inv;
      rstd[i] = rsqrtf(fmaxf(q[2 * i] * inv - left * left, 0.f) + eps);
      off[i] = -left * rstd[i];
      store_stats(stats, r0 + i, stats && g == 0 && r0 + i < N, s[i], left, rstd[i]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + g) * VEC;
      if (c < D) {
        float wv[VEC], bv[VEC];
        affine_vec<T, VEC>(w, wf32, c, 1.f, wv);
        affine_vec<T, VEC>(b, wf32, c, 0.f, bv);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          vscale(v[i][j], v[i][j], rstd[i], off[i]);
          vfma(v[i][j], v[i][j], wv, bv);
          if (r0 + i < N) store_vec<T, VEC>(y + (r0 + i) * D + c, v[i][j]);
        }
      }
    }
  }
}

// This CTA's two column sums into part[cta][2][D] (row-per-warp shapes add the
// warps' through dynamic shared memory [8][2][D] first).
template <int NW, int NV, int VEC>
__device__ __forceinline__ void store_part(const float (&a)[NV][VEC], const float (&b)[NV][VEC],
                                           float* part, int D) {
  constexpr int G = Block<NW>::G, ROWS = Block<NW>::rows;
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

// One row of the backward in registers: x in h and gy in u become xhat and gx;
// the column sums aw, ab take the row in.
template <typename T, int VEC, int NV, int NW>
__device__ __forceinline__ void bwd_row(float (&h)[NV][VEC], float (&u)[NV][VEC],
                                        float (&aw)[NV][VEC], float (&ab)[NV][VEC],
                                        const void* w, int wf32, const Stats& st, int D,
                                        float inv, float (*red)[32][SUMS], int& turn) {
  constexpr int G = Block<NW>::G;
  const int g = threadIdx.x % G;
  Pair p, q;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * G + g) * VEC;
    if (c < D) {
      float wv[VEC];
      affine_vec<T, VEC>(w, wf32, c, 1.f, wv);
      vshift(h[j], -st.mean);
      vscale(h[j], h[j], st.rstd, st.off);
      vfma(aw[j], u[j], h[j], aw[j]);
      vadd(ab[j], u[j]);
      vmul(u[j], wv);
      vsum(p, u[j]);
      vdot(q, u[j], h[j]);
    }
  }
  float s[2] = {p.total(), q.total()};
  row_sum<NW>(s, red, turn);
  // the means first: where they cancel u, they do so before rstd enlarges it
  const float c0 = -s[0] * inv, c1 = -s[1] * inv;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if ((j * G + g) * VEC < D) {
      vshift(u[j], c0);
      vaxpy(u[j], h[j], c1);
      vscale(u[j], u[j], st.rstd, 0.f);
    }
  }
}

// part[cta][2][D]: this CTA's sums of gy * xhat and gy.  Persistent CTAs, rows
// read by each thread (rows that are not whole 16-byte vectors).
template <typename T, int VEC, int NV, int NW>
__global__ void __launch_bounds__(Block<NW>::threads)
bwd_kernel(const T* __restrict__ x, const void* __restrict__ w, int wf32,
           const T* __restrict__ gy, const float* __restrict__ stats, T* __restrict__ gx,
           float* __restrict__ part, int64_t N, int D) {
  constexpr int G = Block<NW>::G, ROWS = Block<NW>::rows;
  __shared__ float red[2][32][SUMS];
  int turn = 0;
  const int g = threadIdx.x % G;
  const float inv = 1.f / (float)D;
  float aw[NV][VEC], ab[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < VEC; ++k) aw[j][k] = ab[j][k] = 0.f;
  for (int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / G; r < N;
       r += (int64_t)gridDim.x * ROWS) {
    float h[NV][VEC], u[NV][VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + g) * VEC;
      if (c < D) {
        load_vec<T, VEC>(x + r * D + c, h[j]);
        load_vec<T, VEC>(gy + r * D + c, u[j]);
      }
    }
    bwd_row<T, VEC, NV, NW>(h, u, aw, ab, w, wf32, Stats(stats + 4 * r), D, inv, red, turn);
    if (gx) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * G + g) * VEC;
        if (c < D) store_vec<T, VEC>(gx + r * D + c, u[j]);
      }
    }
  }
  if (part) store_part<NW, NV, VEC>(aw, ab, part, D);
}

// Blocks of consecutive rows, of x, of gy and of the statistics, in a ring of
// shared-memory stages filled by bulk copies.  A wait that gives up sets the device error
// word, and the kernel goes on with what the stage holds.
constexpr int MAX_STAGES = 4;
struct Ring {
  uint64_t* full;
  volatile int* abort;
  uint8_t* mem;
  const uint8_t *x, *gy, *stats;
  int rows, stages, stage = 0;
  uint32_t phase = 0;
  int64_t N, row_bytes, blocks;
  __device__ Ring(uint64_t* f, volatile int* a, uint8_t* m, const void* x_, const void* gy_,
                  const float* stats_, int rows_, int stages_, int64_t n, int64_t rb)
      : full(f), abort(a), mem(m), x((const uint8_t*)x_), gy((const uint8_t*)gy_),
        stats((const uint8_t*)stats_), rows(rows_), stages(stages_), N(n), row_bytes(rb),
        blocks((n + rows_ - 1) / rows_) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < MAX_STAGES; ++i) tc::mbar_init(full + i, 1);
      *abort = 0;
      tc::fence_barrier_init();
      for (int i = 0; i < stages; ++i) fetch(blockIdx.x + (int64_t)i * gridDim.x, i);
    }
    __syncthreads();
  }
  __device__ uint8_t* at(int s) const { return mem + (int64_t)s * rows * (2 * row_bytes + 16); }
  // block b into stage s, by one thread
  __device__ void fetch(int64_t b, int s) {
    if (b >= blocks) return;
    const int64_t r0 = b * rows;
    const int n = (int)(N - r0 < rows ? N - r0 : rows);
    const uint32_t bytes = (uint32_t)(n * row_bytes);
    tc::mbar_expect_tx(full + s, 2 * bytes + 16 * n);
    tc::bulk_load(at(s), x + r0 * row_bytes, bytes, full + s);
    tc::bulk_load(at(s) + rows * row_bytes, gy + r0 * row_bytes, bytes, full + s);
    tc::bulk_load(at(s) + 2 * rows * row_bytes, stats + r0 * 16, 16 * n, full + s);
  }
  __device__ void wait() { tc::mbar_wait(full + stage, phase, abort); }
  __device__ void next() {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
  // copies in flight after a wait that gave up land before the CTA ends
  __device__ void end() {
    if (*abort)
      for (int i = 0; i < 1000; ++i) __nanosleep(2000);
    __syncthreads();
  }
};

// bwd_kernel for rows of whole 16-byte vectors.  A batch of R rows per group of
// NW warps goes through the reduction together: one barrier and one butterfly
// for 2 R sums.  The rows are read from their stage twice (for the sums, and
// for gx) instead of being held in registers, which the column sums need.
template <typename T, int VEC, int NV, int NW, int R>
__global__ void __launch_bounds__(Block<NW>::threads)
bwd_batch_kernel(const T* __restrict__ x, const void* __restrict__ w, int wf32,
                 const T* __restrict__ gy, const float* __restrict__ stats, T* __restrict__ gx,
                 float* __restrict__ part, int64_t N, int D, int stages) {
  constexpr int G = Block<NW>::G, ROWS = Block<NW>::rows * R;
  extern __shared__ __align__(16) uint8_t ring_mem[];  // afterwards store_part's
  __shared__ float red[2][32][8];
  __shared__ __align__(8) uint64_t full[MAX_STAGES];
  __shared__ volatile int abort;
  int turn = 0;
  const int g = threadIdx.x % G, q = threadIdx.x / G;
  const float inv = 1.f / (float)D;
  Ring ring(full, &abort, ring_mem, x, gy, stats, ROWS, stages, N, (int64_t)D * sizeof(T));
  float wr[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if ((j * G + g) * VEC < D) affine_vec<T, VEC>(w, wf32, (j * G + g) * VEC, 1.f, wr[j]);
  float aw[NV][VEC], ab[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < VEC; ++k) aw[j][k] = ab[j][k] = 0.f;
  int before = -1;  // the stage of the batch before, read by every thread at the next barrier
  for (int64_t blk = blockIdx.x; blk < ring.blocks; blk += gridDim.x) {
    ring.wait();
    const T* sx = reinterpret_cast<const T*>(ring.at(ring.stage)) + q * R * D;
    const T* sg = sx + ROWS * D;
    const int64_t r0 = blk * ROWS + q * R;
    const float* row_stats =
        reinterpret_cast<const float*>(sx - q * R * D + 2 * ROWS * D) + 4 * q * R;
    float s[2 * R];
    Pair su[R], sh[R];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * G + g) * VEC;
      if (c >= D) continue;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (r0 + i >= N) continue;
        float h[VEC], u[VEC];
        load_vec<T, VEC>(sx + i * D + c, h);
        load_vec<T, VEC>(sg + i * D + c, u);
        const Stats st(row_stats + 4 * i);
        vshift(h, -st.mean);
        vscale(h, h, st.rstd, st.off);
        vfma(aw[j], u, h, aw[j]);
        vadd(ab[j], u);
        vmul(u, wr[j]);
        vsum(su[i], u);
        vdot(sh[i], u, h);
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      s[2 * i] = su[i].total();
      s[2 * i + 1] = sh[i].total();
    }
    batch_sum<NW>(s, red, turn);
    if (NW == 1) __syncthreads();
    if (threadIdx.x == 0 && before >= 0)
      ring.fetch(blk + (int64_t)(stages - 1) * gridDim.x, before);
    before = ring.stage;
    if (gx) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * G + g) * VEC;
        if (c >= D) continue;
#pragma unroll
        for (int i = 0; i < R; ++i) {
          if (r0 + i >= N) continue;
          float h[VEC], u[VEC];
          load_vec<T, VEC>(sx + i * D + c, h);
          load_vec<T, VEC>(sg + i * D + c, u);
          const Stats st(row_stats + 4 * i);
          vshift(h, -st.mean);
          // the means first: where they cancel u, they do so before rstd
          // enlarges it
          vmul(u, wr[j]);
          vshift(u, -fmaf(st.off, s[2 * i + 1], s[2 * i]) * inv);
          vaxpy(u, h, -s[2 * i + 1] * inv * st.rstd);
          vscale(u, u, st.rstd, 0.f);
          store_vec<T, VEC>(gx + (r0 + i) * D + c, u);
        }
      }
    }
    ring.next();
  }
  ring.end();
  if (part) store_part<NW, NV, VEC>(aw, ab, part, D);
}

// Rows too wide for the registers: three passes over the row (the second and
// third hit L2), one CTA per row.
template <typename T>
__global__ void __launch_bounds__(256)
fwd_wide_kernel(const T* __restrict__ x, const void* __restrict__ w, const void* __restrict__ b,
                int wdtype, T* __restrict__ y, float* __restrict__ stats, int64_t N, int64_t D,
                float eps) {
  __shared__ float red[2][32][SUMS];
  int turn = 0;
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    const T* row = x + r * D;
    float s[1] = {0.f}, q[2] = {0.f, 0.f};
    for (int64_t c = threadIdx.x; c < D; c += 256) s[0] += to_f32(row[c]);
    row_sum<8>(s, red, turn);
    const float mean = s[0] / (float)D;
    for (int64_t c = threadIdx.x; c < D; c += 256) {
      const float d = to_f32(row[c]) - mean;
      q[0] = fmaf(d, d, q[0]);
      q[1] += d;
    }
    row_sum<8>(q, red, turn);
    const float left = q[1] / (float)D;
    const float rstd = rsqrtf(fmaxf(q[0] / (float)D - left * left, 0.f) + eps);
    for (int64_t c = threadIdx.x; c < D; c += 256)
      y[r * D + c] = from_f32<T>(fmaf((to_f32(row[c]) - mean - left) * rstd,
                                      affine(w, wdtype, c, 1.f), affine(b, wdtype, c, 0.f)));
    store_stats(stats, r, stats && threadIdx.x == 0, mean, left, rstd);
  }
}

// The same for the backward: the CTA's column sums live in its part of the
// workspace (zeroed here, each column kept by one thread).
template <typename T>
__global__ void __launch_bounds__(256)
bwd_wide_kernel(const T* __restrict__ x, const void* __restrict__ w, int wdtype,
                const T* __restrict__ gy, const float* __restrict__ stats, T* __restrict__ gx,
                float* __restrict__ part, int64_t N, int64_t D) {
  __shared__ float red[2][32][SUMS];
  int turn = 0;
  float* mine = part ? part + (int64_t)blockIdx.x * 2 * D : nullptr;
  if (mine)
    for (int64_t c = threadIdx.x; c < D; c += 256) mine[c] = mine[D + c] = 0.f;
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    const Stats st(stats + 4 * r);
    float s[2] = {0.f, 0.f};
    for (int64_t c = threadIdx.x; c < D; c += 256) {
      const float h = st.xhat(to_f32(x[r * D + c])), u = to_f32(gy[r * D + c]);
      if (mine) {
        mine[c] = fmaf(u, h, mine[c]);
        mine[D + c] += u;
      }
      const float uw = u * affine(w, wdtype, c, 1.f);
      s[0] += uw;
      s[1] = fmaf(uw, h, s[1]);
    }
    if (gx == nullptr) continue;
    row_sum<8>(s, red, turn);
    s[0] /= (float)D;
    s[1] /= (float)D;
    for (int64_t c = threadIdx.x; c < D; c += 256) {
      const float h = st.xhat(to_f32(x[r * D + c]));
      const float uw = to_f32(gy[r * D + c]) * affine(w, wdtype, c, 1.f);
      gx[r * D + c] = from_f32<T>(st.rstd * (uw - s[0] - h * s[1]));
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
__global__ void __launch_bounds__(Block<NW>::threads, Block<NW>::least)
bwd2_kernel(const T* __restrict__ x, const void* __restrict__ w, int wf32,
            const T* __restrict__ gy, const float* __restrict__ stats, const T* __restrict__ u,
            const void* __restrict__ a, const void* __restrict__ c, T* __restrict__ dx,
            T* __restrict__ dgy, float* __restrict__ part, int64_t N, int D) {
  constexpr int G = Block<NW>::G, ROWS = Block<NW>::rows;
  __shared__ float red[2][32][SUMS];
  int turn = 0;
  const int lane = threadIdx.x % G;
  float aw[NV][VEC], none[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < VEC; ++k) aw[j][k] = none[j][k] = 0.f;
  for (int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / G; r < N;
       r += (int64_t)gridDim.x * ROWS) {
    const Stats st(stats + 4 * r);
    const float rstd = st.rstd;
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
        float wv[VEC], av[VEC];
        affine_vec<T, VEC>(w, wf32, col, 1.f, wv);
        affine_vec<T, VEC>(a, wf32, col, 0.f, av);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          h[j][k] = st.xhat(h[j][k]);
          second_terms(s, h[j][k], v[j][k], g[j][k] * wv[k], g[j][k] * av[k]);
        }
      }
    }
    row_sum<NW>(s, red, turn);
    const Second f(s, D, rstd);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int col = (j * G + lane) * VEC;
      if (col < D) {
        float o[VEC], wv[VEC], av[VEC], cv[VEC];
        affine_vec<T, VEC>(w, wf32, col, 1.f, wv);
        affine_vec<T, VEC>(a, wf32, col, 0.f, av);
        affine_vec<T, VEC>(c, wf32, col, 0.f, cv);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float pu = f.pu(v[j][k], h[j][k]);
          aw[j][k] = fmaf(rstd * g[j][k], pu, aw[j][k]);
          o[k] = rstd * wv[k] * pu + av[k] * h[j][k] + cv[k];
          v[j][k] = f.dx(h[j][k], v[j][k], g[j][k] * wv[k], g[j][k] * av[k]);
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
  __shared__ float red[2][32][SUMS];
  int turn = 0;
  float* mine = part + (int64_t)blockIdx.x * 2 * D;
  for (int64_t e = threadIdx.x; e < D; e += 256) mine[e] = mine[D + e] = 0.f;
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    const Stats st(stats + 4 * r);
    const float rstd = st.rstd;
    float s[SUMS];
#pragma unroll
    for (int i = 0; i < SUMS; ++i) s[i] = 0.f;
    for (int64_t e = threadIdx.x; e < D; e += 256) {
      const float h = st.xhat(to_f32(x[r * D + e])), g = to_f32(gy[r * D + e]);
      second_terms(s, h, u ? to_f32(u[r * D + e]) : 0.f, g * affine(w, wdtype, e, 1.f),
                   g * affine(a, wdtype, e, 0.f));
    }
    row_sum<8>(s, red, turn);
    const Second f(s, D, rstd);
    for (int64_t e = threadIdx.x; e < D; e += 256) {
      const float h = st.xhat(to_f32(x[r * D + e])), g = to_f32(gy[r * D + e]);
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
