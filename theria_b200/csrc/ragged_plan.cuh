// Packed sequences: the problem's description, the lists of tiles that the
// attention kernels work through, and the rows that belong to no sequence.
//
// Rows of a key head: the G query heads that share it are packed token by
// token, row = token * G + g, so that one tile of rows reads each key tile
// once for the whole group, and a short sequence fills a tile G times better.
// The number of tiles depends on the offsets, which only the device knows: a
// kernel of a few CTAs writes the list of them, and the attention kernels are
// launched for the largest number that T and S allow; a CTA past the list's
// end returns at once.  The list runs from the tiles with the most keys to
// those with the fewest (a counting sort), which evens out the end of a causal
// or ragged launch; the order of equals is left to chance and changes no
// result, since no tile shares a sum with another.
#pragma once

#include "common.cuh"

namespace theria {
namespace ragged {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

// Division of numbers below 2^31 by a constant, as a product's high half: with 2^(l - 1) <
// d <= 2^l, m = 2^(31 + l) / d + 1 has m d - 2^(31 + l) in (0, 2^l], so the quotient is exact.
struct Divisor {
  uint32_t m;  // 0: by 1
  int shift;
  __device__ __forceinline__ unsigned quotient(unsigned n) const {
    return m ? __umulhi(n, m) >> shift : n;
  }
};
inline Divisor divisor(int d) {
  if (d <= 1) return Divisor{0, 0};
  int l = 1;
  while ((1 << l) < d) ++l;
  return Divisor{(uint32_t)((1ull << (31 + l)) / (unsigned)d + 1), l - 1};
}

struct Problem {
  int T, S, H, Hkv, G, D;
  Divisor by_H, by_Hkv, by_G;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;  // strides in elements
  float scale, scale_log2;  // the scores' factor; and times log2(e)
  int causal;
};

// One list: sequence s of n tokens has ceil(n * per / step) tiles, tile i
// starting at first = i * step (in tokens * per).  `by_key`: tiles of keys,
// which all later queries visit; else tiles of queries, which visit all
// earlier keys (with a causal mask).
struct List {
  int4* items;   // {start, n, first, 0}; NULL: no list
  int* count;    // the number of items
  int* base;     // [S] scratch
  int per, step, by_key;
};

// Rows of a tensor that belong to no sequence are set to zero.
struct Blank {
  void* p[3];
  int64_t row_bytes[3];  // any number
};

// A bound on the 2-norm of a row of float16 values, as a byte that grows with it: from the
// sum of its squares, 50 + e with the norm below 2^(e + 1), e from -24 (float16's smallest
// number) to 19 (128 of its largest); 0 for zeros, and for a row that is not finite, whose
// gradients are not either: it leaves the others theirs.
__device__ __forceinline__ uint8_t norm_code(float squares) {
  const int e = (int)(__float_as_uint(squares) >> 23 & 255);
  return squares == 0.f || e == 255 ? 0 : (uint8_t)(((e - 127) >> 1) + 50);
}
// The power of two that ds = p (dp - z) is multiplied by: with cotangents' norms below
// 2^(e + 1), values' below 2^(f + 1), |dp - z| is below 2^(e + f + 3), so |ds| then
// below 2^15 (p <= 1).
__device__ __forceinline__ int fit_power(unsigned cotangents, unsigned values) {
  return cotangents == 0 || values == 0 ? 0 : 112 - (int)cotangents - (int)values;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// The largest of the bytes [from, to), of those that thread `id` of `threads` (32 and more,
// which all call it) looks at: whole vectors, and the ends by bytes, none outside.
__device__ __forceinline__ uint32_t largest_of_mine(const uint8_t* from, const uint8_t* to,
                                                    unsigned id, unsigned threads) {
  const uintptr_t first = (reinterpret_cast<uintptr_t>(from) + 15) & ~uintptr_t(15);
  const uintptr_t last = reinterpret_cast<uintptr_t>(to) & ~uintptr_t(15);
  uint32_t most = 0;
  if (first < last) {
    const uint4* end = reinterpret_cast<const uint4*>(last);
    for (const uint4* p = reinterpret_cast<const uint4*>(first) + id; p < end;
         p += threads) {
      const uint4 w = *p;
      most = __vmaxu4(most, __vmaxu4(__vmaxu4(w.x, w.y), __vmaxu4(w.z, w.w)));
    }
    most = __vmaxu4(most, most >> 16);
    most = max(most & 255, most >> 8 & 255);
    const uint8_t* head = from + id;
    const uint8_t* tail = reinterpret_cast<const uint8_t*>(last) + id;
    if (head < reinterpret_cast<const uint8_t*>(first)) most = max(most, (uint32_t)*head);
    if (tail < to) most = max(most, (uint32_t)*tail);
  } else {  // fewer than 32
    const uint8_t* p = from + id;
    if (p < to) most = *p;
  }
  return most;
}

constexpr int kPlanThreads = 1024;
constexpr int kBuckets = 1024;   // of 128 keys: 131072 keys and more share one

__device__ __forceinline__ int64_t offset_at(const void* o, int wide, int i) {
  return wide ? static_cast<const int64_t*>(o)[i] : static_cast<const int*>(o)[i];
}

// Inclusive sum over the block (kPlanThreads threads), in thread order.
__device__ __forceinline__ int block_scan(int x, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  return x + (warp ? warp_sums[warp - 1] : 0);
}

__device__ __forceinline__ int tiles_of(int64_t n, const List& l) {
  return (int)((n * l.per + l.step - 1) / l.step);
}

// Zeros from `b` to `e` (even addresses), by thread `at` of `all`.
__device__ __forceinline__ void zero_bytes(char* b, char* e, int64_t at, int64_t all) {
  char* mid = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(b) + 15) & ~uintptr_t(15));
  if (mid > e) mid = e;
  const int64_t quads = (e - mid) / 16;
  for (char* p = b + 2 * at; p < mid; p += 2 * all) *reinterpret_cast<uint16_t*>(p) = 0;
  for (int64_t i = at; i < quads; i += all)
    reinterpret_cast<uint4*>(mid)[i] = make_uint4(0, 0, 0, 0);
  for (char* p = mid + 16 * quads + 2 * at; p < e; p += 2 * all)
    *reinterpret_cast<uint16_t*>(p) = 0;
}

// Blocks 0 and 1 write lists a and b; the others zero the rows of `blank` that
// lie outside the sequences.  With bad offsets the lists are empty and every
// row is outside.
__global__ void __launch_bounds__(kPlanThreads)
plan_kernel(const void* offsets, int wide, int S, int T, int causal, List a, List b,
            Blank blank) {
  __shared__ int warp_sums[32], hist[kBuckets], total;
  grid_launch();
  grid_wait();
  const int tid = threadIdx.x;
  bool bad = false;
  for (int i = tid; i < S; i += kPlanThreads)
    bad |= offset_at(offsets, wide, i) > offset_at(offsets, wide, i + 1);
  const int64_t lo = offset_at(offsets, wide, 0), hi = offset_at(offsets, wide, S);
  bad |= lo < 0 || hi > T;
  bad = __syncthreads_or(bad);
  if (blockIdx.x >= 2) {
    const int64_t before = bad ? T : lo, after = bad ? T : hi;
    const int64_t at = (int64_t)(blockIdx.x - 2) * kPlanThreads + tid;
    const int64_t all = (int64_t)(gridDim.x - 2) * kPlanThreads;
    for (int k = 0; k < 3; ++k) {
      if (blank.p[k] == nullptr) continue;
      char* p = static_cast<char*>(blank.p[k]);
      const int64_t rb = blank.row_bytes[k];
      zero_bytes(p, p + before * rb, at, all);
      zero_bytes(p + after * rb, p + T * rb, at, all);
    }
    return;
  }
  const List l = blockIdx.x == 0 ? a : b;
  if (l.items == nullptr) return;
  if (bad) {
    if (tid == 0) {
      *l.count = 0;
      atomicExch(&g_device_error, THERIA_ERR_INVALID_ARG);
    }
    return;
  }
  // where each sequence's tiles start
  if (tid == 0) total = 0;
  for (int i = tid; i < kBuckets; i += kPlanThreads) hist[i] = 0;
  __syncthreads();
  for (int s0 = 0; s0 < S; s0 += kPlanThreads) {
    const int s = s0 + tid;
    const int mine =
        s < S ? tiles_of(offset_at(offsets, wide, s + 1) - offset_at(offsets, wide, s), l) : 0;
    const int upto = block_scan(mine, warp_sums);
    const int old = total;
    if (s < S) l.base[s] = old + upto - mine;
    __syncthreads();
    if (tid == kPlanThreads - 1) total = old + upto;
    __syncthreads();
  }
  const int n_items = total;
  auto item = [&](int i, int& cost) {
    int s = 0, e = S;  // base[s] <= i < base[e], base[S] taken as n_items
    while (e - s > 1) {
      const int m = (s + e) >> 1;
      if (l.base[m] <= i) s = m; else e = m;
    }
    const int start = (int)offset_at(offsets, wide, s);
    const int n = (int)offset_at(offsets, wide, s + 1) - start;
    const int first = (i - l.base[s]) * l.step;
    cost = n;
    if (causal) cost = l.by_key ? n - first : min(n, (first + l.step - 1) / l.per + 1);
    cost = kBuckets - 1 - min(kBuckets - 1, cost / 128);
    return make_int4(start, n, first, 0);
  };
  for (int i = tid; i < n_items; i += kPlanThreads) {
    int cost;
    item(i, cost);
    atomicAdd(hist + cost, 1);
  }
  __syncthreads();
  const int h = hist[tid];
  const int upto = block_scan(h, warp_sums);
  hist[tid] = upto - h;
  __syncthreads();
  for (int i = tid; i < n_items; i += kPlanThreads) {
    int cost;
    const int4 it = item(i, cost);
    l.items[atomicAdd(hist + cost, 1)] = it;
  }
  if (tid == 0) *l.count = n_items;
}

static_assert(kBuckets == kPlanThreads, "one bucket a thread");

}  // namespace ragged
}  // namespace theria
