// Attention over packed sequences on the CUDA cores: float32 (always in
// float32), and 16-bit tensors that the tensor-core kernels cannot take
// (more than 64 query heads a key head, or rows off 16-byte boundaries).
//
// A block is 16 warps on one tile of rows: in the forward four groups of 4 warps on
// 32 rows, in the backward two of 8 on 64, each group taking every fourth (second)
// tile of 64 (32) columns; their sums are put together at the end.  One block fills
// an SM, the longest row of tiles takes a quarter (half) of the time, and the groups'
// loads, softmax and barriers hide behind one another's products.  (One group a block
// and two or three blocks an SM, which the hardware put on few SMs: 2395 tokens, 5
// heads of 72, forward 148 us, queries 410, keys 254; blocks of one group alone on
// their SM 188, 208, 301.)
//
// In a group a thread holds rows 4 ty + i and columns tx + 16 j of the tile's scores
// and, of the sums over its columns, the same 4 rows of DT / 16 values.  Operands lie
// in shared memory as float32 rows of DT + 4 values: a step of 4 along a row is one
// 16-byte load, free of bank conflicts down the columns' 16 rows.  float32 rows come
// by cp.async: in the forward K's while the softmax and V's sum run and V's while the
// next scores do, in the backward into a second buffer.
//
// The backward is one kernel for both sides.  Its tile stays on 64 rows x1, x2
// and walks over tiles of 32 y1, y2:
//     queries: x = (q, do), y = (k, v):  dq += ds k
//     keys:    x = (k, v), y = (q, do):  dk += ds^T q, dv += p^T do
// so no sum is shared between blocks and nothing is added atomically.
#pragma once

#include "ragged_plan.cuh"
#include "tc_common.cuh"

namespace theria {
namespace ragged {

constexpr int FR = 32, FC = 64;    // rows and columns of a forward tile
constexpr int SR = 64, SC = 32;    // ... of a backward tile
constexpr int FWD_THREADS = FR * 4, BWD_THREADS = SR * 4;  // ... of a group

template <int DT>
struct SimtSmem {
  static constexpr int kRow = DT + 4;            // floats of an operand's row
  // groups of a forward, of a backward block; narrow heads take one, whose tiles are done
  // sooner where sequences are short or many, later where they are few and long (4 heads
  // of 16; forward, dq, dk and dv, us, with one group and with four and two: 25 x 64: 6, 8,
  // 8 and 9, 13, 12; 200 x 64: 17, 21, 29 and 49, 34, 37; 8192: 388, 933, 854 and 397, 736,
  // 965; 2 x 2048: 81, 239, 196 and 67, 107, 140.  The kernels do not know the lengths.)
  static constexpr int FG = DT <= 32 ? 1 : 4, SG = DT <= 32 ? 1 : 2;
  // a group's k, v (wide heads: tiles of half the columns), scores; a block's q
  static constexpr int kFC = DT <= 64 ? FC : FC / 2;
  static constexpr int kFwdGroup = 2 * kFC * kRow + FR * (kFC + 4);
  static constexpr int kFwd = (FR * kRow + FG * kFwdGroup) * 4;
  // a group's two of y1, y2, scores, two of terms; a block's x1, x2, terms
  static constexpr int kBwdGroup = 4 * SC * kRow + SR * (SC + 4) + 4 * SC;
  static constexpr int kBwd = (2 * SR * kRow + 2 * SR + SG * kBwdGroup) * 4;
  static_assert(kFwd <= 232448 && kBwd <= 232448, "shared memory of a block");
  // a forward group's sums go over its buffers at the end
  static_assert(FR * kRow + 2 * FR <= kFwdGroup, "room for a group's sums");
};

__device__ __forceinline__ void async16(float* dst, const float* src, bool on) {
  // on false: 16 bytes of zeros, src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::smem_u32(dst)), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
// All but the newest `left` groups have landed (for this thread's copies).
template <int left>
__device__ __forceinline__ void async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(left) : "memory");
}

// 16 bytes (VEC > 1) or one value, as floats.
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = to_f32<T>(*p);
  } else {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32<T>(e[i]);
  }
}

// N rows of a tensor into shared memory as float32, zero beyond row `n` and
// column D.  row_at(r): the element where row r starts.  ASYNC (float32, whole
// rows of 16 bytes on such boundaries): by cp.async, else at once.
template <typename T, int DT, int N, int THREADS, bool ASYNC, typename F>
__device__ __forceinline__ void load_tile(float* dst, const T* src, int n, int D, int tid,
                                          F row_at) {
  if constexpr (ASYNC) {
    constexpr int CH = DT / 4;
#pragma unroll
    for (int i0 = 0; i0 < N * CH; i0 += THREADS) {
      const int i = i0 + tid, r = i / CH, d = (i % CH) * 4;
      if (N * CH % THREADS != 0 && i >= N * CH) continue;
      const bool on = r < n && d < D;
      async16(dst + r * SimtSmem<DT>::kRow + d, on ? src + row_at(r) + d : src, on);
    }
  } else {
    for (int i = tid; i < N * DT; i += THREADS) {
      const int r = i / DT, d = i % DT;
      dst[r * SimtSmem<DT>::kRow + d] = r < n && d < D ? to_f32<T>(src[row_at(r) + d]) : 0.f;
    }
  }
}

// s[i][j] = x[4 ty + i] . y[tx + 16 j]
template <int DT, int J>
__device__ __forceinline__ void tile_scores(float (&s)[4][J], const float* x, const float* y,
                                            int ty) {
  constexpr int K = SimtSmem<DT>::kRow;
  const int tx = threadIdx.x & 15;
  // even and odd values of the rows apart, two at a time (narrow rows, whose few
  // steps leave the pairs' sums to weigh: each value in turn, 7.5 against 8.7 us for dq
  // of 25 sequences of 64, 4 heads of 16)
  float s2[4][J];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) s[i][j] = s2[i][j] = 0.f;
#pragma unroll 4
  for (int d = 0; d < DT; d += 4) {
    float4 a[4], b[J];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(x + (4 * ty + i) * K + d);
#pragma unroll
    for (int j = 0; j < J; ++j) b[j] = *reinterpret_cast<const float4*>(y + (tx + 16 * j) * K + d);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if constexpr (DT >= 64) {
          tc::fma2(s[i][j], s2[i][j], a[i].x, a[i].y, b[j].x, b[j].y, s[i][j], s2[i][j]);
          tc::fma2(s[i][j], s2[i][j], a[i].z, a[i].w, b[j].z, b[j].w, s[i][j], s2[i][j]);
        } else {
          s[i][j] = fmaf(a[i].x, b[j].x, s[i][j]);
          s[i][j] = fmaf(a[i].y, b[j].y, s[i][j]);
          s[i][j] = fmaf(a[i].z, b[j].z, s[i][j]);
          s[i][j] = fmaf(a[i].w, b[j].w, s[i][j]);
        }
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j)
      if constexpr (DT >= 64) s[i][j] += s2[i][j];
}

// The columns of DT that a thread sums: DT / 16 of them, in runs of up to 4.
template <int DT>
struct Cols {
  static constexpr int n = DT / 16;
  static constexpr int run = n % 4 == 0 ? 4 : n % 2 == 0 ? 2 : 1;
  __device__ static int at(int c) {  // column of the thread's value c
    return (c / run) * (16 * run) + (threadIdx.x & 15) * run + c % run;
  }
};

// acc[i][c] += sum over the tile's columns e of p[4 ty + i][e] * y[e][column c]
template <int DT, int C>
__device__ __forceinline__ void tile_sums(float (&acc)[4][DT / 16], const float* p,
                                          const float* y, int ty) {
  constexpr int K = SimtSmem<DT>::kRow, KS = C + 4, RUN = Cols<DT>::run;
#pragma unroll 2
  for (int e = 0; e < C; e += 4) {
    float4 a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(p + (4 * ty + i) * KS + e);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float* row = y + (e + u) * K;
#pragma unroll
      for (int c = 0; c < DT / 16; c += RUN) {
        float b[RUN];
        if constexpr (RUN == 4) {
          const float4 t = *reinterpret_cast<const float4*>(row + Cols<DT>::at(c));
          b[0] = t.x; b[1] = t.y; b[2] = t.z; b[3] = t.w;
        } else if constexpr (RUN == 2) {
          const float2 t = *reinterpret_cast<const float2*>(row + Cols<DT>::at(c));
          b[0] = t.x; b[1] = t.y;
        } else {
          b[0] = row[Cols<DT>::at(c)];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float pi = u == 0 ? a[i].x : u == 1 ? a[i].y : u == 2 ? a[i].z : a[i].w;
          if constexpr (DT < 64) {
#pragma unroll
            for (int x = 0; x < RUN; ++x) acc[i][c + x] = fmaf(pi, b[x], acc[i][c + x]);
          } else {
#pragma unroll
            for (int x = 0; x < RUN; x += 2)
              tc::fma2(acc[i][c + x], acc[i][c + x + 1], pi, pi, b[x], b[x + 1], acc[i][c + x],
                       acc[i][c + x + 1]);
          }
        }
      }
    }
  }
}

template <int J>
__device__ __forceinline__ void put_scores(float* p, const float (&s)[4][J], int ty) {
  const int tx = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) p[(4 * ty + i) * (16 * J + 4) + tx + 16 * j] = s[i][j];
}

template <typename T, int DT, bool ASYNC>
__global__ void __launch_bounds__(SimtSmem<DT>::FG * FWD_THREADS)
simt_fwd_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                T* __restrict__ o, T* __restrict__ rest, float* __restrict__ lse,
                const int4* items, const int* count, Problem pr) {
  using L = SimtSmem<DT>;
  extern __shared__ float4 smem4[];
  constexpr int C = L::kFC, FG = L::FG;
  const int g = threadIdx.x / FWD_THREADS, tid = threadIdx.x % FWD_THREADS;
  float* xs = reinterpret_cast<float*>(smem4);
  float* mine = xs + FR * L::kRow + g * L::kFwdGroup;  // the group's
  float *ks = mine, *vs = ks + C * L::kRow, *ps = vs + C * L::kRow;
  auto sync = [&] { tc::named_bar(1 + g, FWD_THREADS); };
  grid_wait();
  const int tile = blockIdx.x / pr.Hkv, hk = blockIdx.x % pr.Hkv;
  if (tile >= *count) return;
  const int4 it = items[tile];
  const int G = pr.G, len = it.y, first = it.z;
  const int rows = (int)min((int64_t)len * G - first, (int64_t)FR);
  const int ty = tid >> 4, tx = tid & 15;
  auto load_k = [&](int j0) {
    load_tile<T, DT, C, FWD_THREADS, ASYNC>(ks, k, len - j0, pr.D, tid, [&](int r) {
      return (int64_t)(it.x + j0 + r) * pr.k_t + hk * pr.k_h;
    });
  };
  auto load_v = [&](int j0) {
    load_tile<T, DT, C, FWD_THREADS, ASYNC>(vs, v, len - j0, pr.D, tid, [&](int r) {
      return (int64_t)(it.x + j0 + r) * pr.v_t + hk * pr.v_h;
    });
  };
  load_tile<T, DT, FR, FG * FWD_THREADS, ASYNC>(xs, q, rows, pr.D, threadIdx.x, [&](int r) {
    const int p = first + r, t = p / G;
    return (int64_t)(it.x + t) * pr.q_t + (int64_t)(hk * G + p - t * G) * pr.q_h;
  });
  async_commit();
  const int last = (first + rows - 1) / G;  // the last row's token
  const int keys = pr.causal ? last + 1 : len;
  const float c = pr.scale_log2;
  float m[4], l[4], acc[4][DT / 16];
  int lim[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    lim[i] = pr.causal ? min((first + 4 * ty + i) / G + 1, len) : len;
#pragma unroll
    for (int x = 0; x < DT / 16; ++x) acc[i][x] = 0.f;
  }
  async_wait<0>();
  __syncthreads();  // q
  if (g * C < keys) load_k(g * C);
  async_commit();
  if (g * C < keys) load_v(g * C);
  async_commit();
  for (int j0 = g * C; j0 < keys; j0 += FG * C) {
    const bool more = j0 + FG * C < keys;
    async_wait<1>();
    sync();
    float s[4][C / 16];
    tile_scores<DT>(s, xs, ks, ty);
    sync();
    if (more) load_k(j0 + FG * C);
    async_commit();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mt = -INFINITY;
#pragma unroll
      for (int j = 0; j < C / 16; ++j) {
        s[i][j] = j0 + tx + 16 * j < lim[i] ? s[i][j] * c : -INFINITY;
        mt = fmaxf(mt, s[i][j]);
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, x));
      const float mn = fmaxf(m[i], mt), sub = mn == -INFINITY ? 0.f : mn;
      const float alpha = tc::ex2(m[i] - sub);
      m[i] = mn;
      float rs = 0.f;
#pragma unroll
      for (int j = 0; j < C / 16; ++j) {
        s[i][j] = tc::ex2(s[i][j] - sub);
        rs += s[i][j];
      }
      l[i] = l[i] * alpha + rs;
#pragma unroll
      for (int x = 0; x < DT / 16; ++x) acc[i][x] *= alpha;
    }
    put_scores(ps, s, ty);
    async_wait<1>();
    sync();
    tile_sums<DT, C>(acc, ps, vs, ty);
    sync();
    if (more) load_v(j0 + FG * C);
    async_commit();
  }
  async_wait<0>();
  // the groups' sums together, in their order: each goes over the group's buffers
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
  if (g > 0) {
    sync();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * ty + i;
#pragma unroll
      for (int x = 0; x < DT / 16; ++x) mine[r * L::kRow + Cols<DT>::at(x)] = acc[i][x];
      if (tx == 0) {
        mine[FR * L::kRow + r] = m[i];
        mine[FR * L::kRow + FR + r] = l[i];
      }
    }
  }
  __syncthreads();
  if (g > 0) return;
#pragma unroll 1
  for (int o_ = 1; o_ < FG; ++o_) {
    const float* theirs = mine + o_ * L::kFwdGroup;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * ty + i;
      const float m2 = theirs[FR * L::kRow + r], l2 = theirs[FR * L::kRow + FR + r];
      const float mn = fmaxf(m[i], m2), sub = mn == -INFINITY ? 0.f : mn;
      const float a1 = tc::ex2(m[i] - sub), a2 = tc::ex2(m2 - sub);
      m[i] = mn;
      l[i] = l[i] * a1 + l2 * a2;
#pragma unroll
      for (int x = 0; x < DT / 16; ++x)
        acc[i][x] = acc[i][x] * a1 + theirs[r * L::kRow + Cols<DT>::at(x)] * a2;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float sum = l[i];
    const int r = 4 * ty + i;
    if (r >= rows) continue;
    const int p = first + r;
    const int64_t row = (int64_t)(it.x + p / G) * pr.H + hk * G + p % G;
    const float inv = 1.f / sum;
#pragma unroll
    for (int x = 0; x < DT / 16; ++x) {
      const int d = Cols<DT>::at(x);
      if (d >= pr.D) continue;
      const T value = from_f32<T>(acc[i][x] * inv);
      o[row * pr.D + d] = value;
      if (rest != nullptr) rest[row * pr.D + d] = from_f32<T>(acc[i][x] * inv - to_f32<T>(value));
    }
    if (lse != nullptr && tx == 0) lse[row] = (m[i] + log2f(sum)) * kLn2;
  }
}

// terms[row] = {-lse * log2(e), -rowsum(do * (o + rest))} for every row [T, H], rest
// (may be NULL) being what o's rounding left: LANES neighbouring lanes a row, each on
// VEC of its values at a time.  Rows of no sequence get whatever their memory holds: no
// tile reads them.
// float16 (fits may be NULL): norm_code of do's rows [Hkv, T, G], and behind them of v's
// rows [Hkv, T] (see ragged_tc_bwd.cuh).
template <typename T, int VEC, int LANES>
__global__ void __launch_bounds__(256)
terms_kernel(const T* __restrict__ o, const T* __restrict__ rest, const T* __restrict__ dout,
             const float* __restrict__ lse,
             float2* __restrict__ terms, const T* __restrict__ v, uint8_t* __restrict__ fits,
             int64_t rows, const Problem pr) {
  const int D = pr.D;
  grid_launch();
  grid_wait();
  const int lane = threadIdx.x % LANES;
  const int64_t step = (int64_t)gridDim.x * (256 / LANES);
  const int64_t r0 = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  constexpr bool kFit = std::is_same<T, __half>::value;
  const int64_t all = kFit && fits != nullptr ? rows + (int64_t)pr.T * pr.Hkv : rows;
  for (int64_t base = 0; base < all; base += step) {  // the same trips for every lane
    const int64_t r = base + r0;
    float z = 0.f, squares = 0.f;
    if (r < rows) {
      for (int d = lane * VEC; d < D; d += LANES * VEC) {
        float a[VEC], b[VEC];
        load_vec<T, VEC>(o + r * D + d, a);
        load_vec<T, VEC>(dout + r * D + d, b);
        if (rest != nullptr) {
          float c[VEC];
          load_vec<T, VEC>(rest + r * D + d, c);
#pragma unroll
          for (int i = 0; i < VEC; ++i) a[i] += c[i];
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) z = fmaf(a[i], b[i], z);
        if constexpr (kFit)
#pragma unroll
          for (int i = 0; i < VEC; ++i) squares = fmaf(b[i], b[i], squares);
      }
    } else if (kFit && r < all) {
      const unsigned vr = (unsigned)(r - rows), t = pr.by_Hkv.quotient(vr), hk = vr - t * pr.Hkv;
      for (int d = lane * VEC; d < D; d += LANES * VEC) {
        float b[VEC];
        load_vec<T, VEC>(v + t * pr.v_t + hk * pr.v_h + d, b);
#pragma unroll
        for (int i = 0; i < VEC; ++i) squares = fmaf(b[i], b[i], squares);
      }
    }
#pragma unroll
    for (int x = LANES / 2; x > 0; x >>= 1) z += __shfl_xor_sync(0xffffffffu, z, x);
    if (r < rows && lane == 0) terms[r] = make_float2(-lse[r] * kLog2e, -z);
    if constexpr (kFit) {
      if (fits == nullptr) continue;
#pragma unroll
      for (int x = LANES / 2; x > 0; x >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, x);
      if (r >= all || lane != 0) continue;
      if (r < rows) {
        const unsigned t = pr.by_H.quotient((unsigned)r), h = (unsigned)r - t * pr.H;
        const unsigned hk = pr.by_G.quotient(h);
        fits[((int64_t)hk * pr.T + t) * pr.G + (h - hk * pr.G)] = norm_code(squares);
      } else {
        const unsigned vr = (unsigned)(r - rows), t = pr.by_Hkv.quotient(vr);
        fits[rows + (int64_t)(vr - t * pr.Hkv) * pr.T + t] = norm_code(squares);
      }
    }
  }
}

// One split of a backward tile (see above).  part: NULL where there is one split
// (results rounded to T at once), else float32 [splits][2][T * Hkv][D], for queries
// [splits][T * H][D].
template <typename T, int DT, bool KEYS, bool ASYNC>
__global__ void __launch_bounds__(SimtSmem<DT>::SG * BWD_THREADS)
simt_bwd_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                const T* __restrict__ dout, const float2* terms, T* __restrict__ out1,
                T* __restrict__ out2, float* part, const int4* items, const int* count,
                int splits, Problem pr) {
  using L = SimtSmem<DT>;
  constexpr int SG = L::SG;
  extern __shared__ float4 smem4[];
  const int g = threadIdx.x / BWD_THREADS, tid = threadIdx.x % BWD_THREADS;
  float* x1 = reinterpret_cast<float*>(smem4);
  float* x2 = x1 + SR * L::kRow;
  float2* tx_ = reinterpret_cast<float2*>(x2 + SR * L::kRow);  // queries: x's terms [SR]
  float* mine = reinterpret_cast<float*>(tx_ + SR) + g * L::kBwdGroup;  // the group's
  float* ps = mine + 4 * SC * L::kRow;                         // y1, y2 of even, odd tiles first
  float2* ts = reinterpret_cast<float2*>(ps + SR * (SC + 4));  // keys: [2][SC]
  auto sync = [&] { tc::named_bar(1 + g, BWD_THREADS); };
  grid_wait();
  // a tile's splits side by side, so that the longest tiles' all start first
  const int hk = blockIdx.x % pr.Hkv, sp = blockIdx.x / pr.Hkv % splits;
  const int tile = blockIdx.x / pr.Hkv / splits;
  if (tile >= *count) return;
  const int4 it = items[tile];
  const int G = pr.G, len = it.y, first = it.z;
  const int ty = tid >> 4, tx = tid & 15;
  const int64_t q_rows = (int64_t)len * G;
  const int rows = (int)min((int64_t)SR, (KEYS ? len : q_rows) - first);
  auto q_at = [&](int p, int64_t st, int64_t sh) {
    const int t = p / G;
    return (it.x + t) * st + (int64_t)(hk * G + p - t * G) * sh;
  };
  // (the numbers of rows and threads are types: integral_constant)
  auto load_q = [&](auto rows_, auto threads_, int id, float* a, float* b, float2* tm, int p0,
                    int n) {
    constexpr int N = decltype(rows_)::value, TH = decltype(threads_)::value;
    load_tile<T, DT, N, TH, ASYNC>(
        a, q, n, pr.D, id, [&](int r) { return q_at(p0 + r, pr.q_t, pr.q_h); });
    load_tile<T, DT, N, TH, ASYNC>(
        b, dout, n, pr.D, id, [&](int r) { return q_at(p0 + r, (int64_t)pr.H * pr.D, pr.D); });
    if (id < N) tm[id] = id < n ? terms[q_at(p0 + id, pr.H, 1)] : make_float2(-INFINITY, 0.f);
  };
  auto load_k = [&](auto rows_, auto threads_, int id, float* a, float* b, int j0, int n) {
    constexpr int N = decltype(rows_)::value, TH = decltype(threads_)::value;
    load_tile<T, DT, N, TH, ASYNC>(a, k, n, pr.D, id, [&](int r) {
      return (int64_t)(it.x + j0 + r) * pr.k_t + hk * pr.k_h;
    });
    load_tile<T, DT, N, TH, ASYNC>(b, v, n, pr.D, id, [&](int r) {
      return (int64_t)(it.x + j0 + r) * pr.v_t + hk * pr.v_h;
    });
  };
  using XRows = std::integral_constant<int, SR>;
  using YRows = std::integral_constant<int, SC>;
  using All = std::integral_constant<int, SG * BWD_THREADS>;
  using Group = std::integral_constant<int, BWD_THREADS>;
  if (KEYS) load_k(XRows{}, All{}, threadIdx.x, x1, x2, first, rows);
  else load_q(XRows{}, All{}, threadIdx.x, x1, x2, tx_, first, rows);
  async_commit();
  // the tiles of y, and this split's share of them
  int64_t y_from = 0, y_to = KEYS ? q_rows : len;
  if (pr.causal && KEYS) y_from = (int64_t)first * G;
  if (pr.causal && !KEYS) y_to = (first + rows - 1) / G + 1;
  const int n_y = (int)((y_to - y_from + SC - 1) / SC);
  const int t0 = (int)((int64_t)n_y * sp / splits);
  const int t1 = (int)((int64_t)n_y * (sp + 1) / splits);
  const float c = pr.scale_log2;
  float a1[4][DT / 16], a2[KEYS ? 4 : 1][DT / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int x = 0; x < DT / 16; ++x) {
      a1[i][x] = 0.f;
      if (KEYS) a2[KEYS ? i : 0][x] = 0.f;
    }
  auto load_y = [&](int t) {
    const int64_t e0 = y_from + (int64_t)t * SC;
    const int n = (int)min((int64_t)SC, (KEYS ? q_rows : len) - e0);
    const int b = ((t - t0) / SG) & 1;
    float* y1 = mine + b * 2 * SC * L::kRow;
    if (KEYS)
      load_q(YRows{}, Group{}, tid, y1, y1 + SC * L::kRow, ts + b * SC, (int)e0, n);
    else
      load_k(YRows{}, Group{}, tid, y1, y1 + SC * L::kRow, (int)e0, n);
  };
  if (t0 + g < t1) load_y(t0 + g);
  async_commit();
  async_wait<1>();
  __syncthreads();  // x
  for (int t = t0 + g; t < t1; t += SG) {
    const int64_t e0 = y_from + (int64_t)t * SC;
    const int b = ((t - t0) / SG) & 1;
    const float *y1 = mine + b * 2 * SC * L::kRow, *y2 = y1 + SC * L::kRow;
    const float2* tq = KEYS ? ts + b * SC : tx_;
    if (t + SG < t1) load_y(t + SG);
    async_commit();
    async_wait<1>();
    sync();
    float s[4][SC / 16], dp[4][SC / 16];
    tile_scores<DT>(s, x1, y1, ty);
    tile_scores<DT>(dp, x2, y2, ty);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < SC / 16; ++j) {
        const int r = 4 * ty + i, e = tx + 16 * j;
        const float2 tm = tq[KEYS ? e : r];
        // key <= query token: key * G <= query row
        const int64_t qr = KEYS ? e0 + e : (int64_t)first + r;
        const int64_t key = KEYS ? (int64_t)first + r : e0 + e;
        const bool on = key < len && qr < q_rows && (!pr.causal || key * G <= qr);
        const float p = on ? tc::ex2(fmaf(s[i][j], c, tm.x)) : 0.f;
        s[i][j] = p;
        dp[i][j] = on ? p * (dp[i][j] + tm.y) : 0.f;
      }
    if constexpr (KEYS) {
      put_scores(ps, s, ty);
      sync();
      tile_sums<DT, SC>(a2, ps, y2, ty);
      sync();
    }
    put_scores(ps, dp, ty);
    sync();
    tile_sums<DT, SC>(a1, ps, y1, ty);
    sync();
  }
  async_wait<0>();
  if constexpr (SG > 1) {
    // the second group's sums are added to the first's, by way of x1's and x2's place
    float* theirs = x1;
    __syncthreads();
    if (g == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < DT / 16; ++x) {
          const int at = (4 * ty + i) * L::kRow + Cols<DT>::at(x);
          theirs[at] = a1[i][x];
          if constexpr (KEYS) theirs[SR * L::kRow + at] = a2[i][x];
        }
    }
    __syncthreads();
    if (g == 1) return;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int x = 0; x < DT / 16; ++x) {
        const int at = (4 * ty + i) * L::kRow + Cols<DT>::at(x);
        a1[i][x] += theirs[at];
        if constexpr (KEYS) a2[i][x] += theirs[SR * L::kRow + at];
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * ty + i;
    if (r >= rows) continue;
    const int64_t row = KEYS ? (int64_t)(it.x + first + r) * pr.Hkv + hk : q_at(first + r, pr.H, 1);
#pragma unroll
    for (int x = 0; x < DT / 16; ++x) {
      const int d = Cols<DT>::at(x);
      if (d >= pr.D) continue;
      if (part == nullptr) {
        out1[row * pr.D + d] = from_f32<T>(a1[i][x] * pr.scale);
        if constexpr (KEYS) out2[row * pr.D + d] = from_f32<T>(a2[i][x]);
      } else {
        const int64_t plane = (int64_t)pr.T * (KEYS ? pr.Hkv : pr.H) * pr.D;
        float* to = part + (KEYS ? 2 : 1) * plane * sp + row * pr.D + d;
        to[0] = a1[i][x] * pr.scale;
        if constexpr (KEYS) to[plane] = a2[i][x];
      }
    }
  }
}

// A gradient (two, b not NULL: dk and dv) of `heads` heads from the splits' float32
// sums, added in the splits' order.
template <typename T>
__global__ void __launch_bounds__(256)
join_kernel(const float* part, int splits, const int* count, const void* offsets, int wide,
            T* __restrict__ a, T* __restrict__ b, int heads, Problem pr) {
  grid_wait();
  if (*count == 0) return;
  const int64_t row = (int64_t)heads * pr.D, plane = row * pr.T, step = b ? 2 * plane : plane;
  const int64_t lo = offset_at(offsets, wide, 0) * row, hi = offset_at(offsets, wide, pr.S) * row;
  // (the rows of no sequence are zeroed with the others)
  for (int64_t i = lo + (int64_t)blockIdx.x * 256 + threadIdx.x; i < hi;
       i += (int64_t)gridDim.x * 256) {
    float x = 0.f, y = 0.f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      x += part[step * s + i];
      if (b) y += part[step * s + plane + i];
    }
    a[i] = from_f32<T>(x);
    if (b) b[i] = from_f32<T>(y);
  }
}

}  // namespace ragged
}  // namespace theria
