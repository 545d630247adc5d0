// The language-model operators of include/theria_lm.h: argument checks,
// workspace carving and kernel selection.
#include <algorithm>

#include "common.cuh"
#include "lm_embed.cuh"
#include "lm_norm.cuh"
#include "lm_xent.cuh"
#include "lm_xent_tc.cuh"
#include "tc_host.cuh"
#include "../../include/theria_lm.h"

namespace theria {

// This translation unit's copy of the device error word, for
// theria_get_device_error / theria_clear_device_error.
int lm_read_device_error(int* out, cudaStream_t st) {
  return cudaMemcpyFromSymbolAsync(out, g_device_error, sizeof(int), 0, cudaMemcpyDeviceToHost,
                                   st) == cudaSuccess
             ? THERIA_OK
             : THERIA_ERR_LAUNCH;
}
int lm_clear_device_error(cudaStream_t st) {
  static const int zero = 0;
  return cudaMemcpyToSymbolAsync(g_device_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice,
                                 st) == cudaSuccess
             ? THERIA_OK
             : THERIA_ERR_LAUNCH;
}

namespace {

constexpr int kSMs = 148;

bool lm_dtype(int dt) { return dt == THERIA_F32 || dt == THERIA_F16 || dt == THERIA_BF16; }
int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether rows of D elements at these addresses can be moved 16 bytes at a time.
bool vec_rows(int64_t D, int dtype, std::initializer_list<const void*> ptrs) {
  if (D * elem_size(dtype) % 16 != 0) return false;
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) & 15u) return false;
  return true;
}

// Calls f(T{}) for the element type of `dtype`.
template <typename F>
int by_type(int dtype, F f) {
  if (dtype == THERIA_F32) return f(float{});
  if (dtype == THERIA_F16) return f(__half{});
  return f(__nv_bfloat16{});
}

// A workspace handed out piece by piece, 256-byte aligned.
struct Carver {
  char* base;
  int64_t used = 0;
  template <typename T>
  T* take(int64_t count) {
    T* p = reinterpret_cast<T*>(base + used);
    used += up(count * (int64_t)sizeof(T), 256);
    return p;
  }
};

// ------------------------------------------------------------ embedding
struct EmbedWs {
  uint32_t *keys[2], *vals[2], *hist;
  float* part;
  int64_t bytes;
};
constexpr int64_t kClusterSort = (int64_t)embed::CS_CTAS * embed::CS_THREADS * embed::CS_MOST;
EmbedWs embed_ws(void* base, int64_t n, int64_t V, int64_t D) {
  Carver c{(char*)base};
  EmbedWs w;
  for (int k = 0; k < (n <= kClusterSort ? 1 : 2); ++k) {
    w.keys[k] = c.take<uint32_t>(n);
    w.vals[k] = c.take<uint32_t>(n);
  }
  w.hist = n <= kClusterSort ? nullptr : c.take<uint32_t>(cdiv(n, embed::TILE) * embed::BINS);
  w.part = c.take<float>(cdiv(n, embed::CHUNK) * 2 * D);
  w.bytes = c.used;
  return w;
}

// The sort of up to kClusterSort tokens, one CTA up to 4 tokens a thread, else a
// cluster of 8, while further clusters zero gw (16-byte aligned).
int embed_cluster_sort(const void* ids, int wide, const EmbedWs& ws, int64_t n, int64_t V,
                       int64_t zero_idx, int bits, void* gw, int64_t gw_bytes, cudaStream_t st) {
  using L = embed::ClusterSmem;
  const int ctas = n <= 4 * embed::CS_THREADS ? 1 : embed::CS_CTAS;
  const int64_t each = cdiv(n, (int64_t)ctas * embed::CS_THREADS);
  const int passes = (int)cdiv(bits, embed::CS_BITS), digit = (int)cdiv(bits, passes);
  auto launch = [&](auto rc) -> int {
    constexpr int R = decltype(rc)::value;
    auto kern = embed::cluster_sort_kernel<R>;
    const int smem = L::oBuf + 2 * embed::CS_THREADS * R * 8;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
        cudaSuccess)
      return THERIA_ERR_LAUNCH;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    // 16 KB of zeros a CTA at least; no more clusters than run at one time
    // beside the sort's (14 of 8: two fit a GPC)
    const int64_t fill =
        std::min<int64_t>(cdiv(gw_bytes, (16 << 10) * ctas), ctas > 1 ? 14 : kSMs - 1);
    cfg.gridDim = dim3((unsigned)(ctas + ctas * std::max<int64_t>(fill, 1)));
    cfg.blockDim = dim3(embed::CS_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kern, ids, wide, ctas, passes, digit, ws.keys[0], ws.vals[0],
                       (int)n, V, zero_idx, (uint4*)gw, gw_bytes);
    return launch_status();
  };
  if (each <= 1) return launch(std::integral_constant<int, 1>{});
  if (each <= 2) return launch(std::integral_constant<int, 2>{});
  if (each <= 4) return launch(std::integral_constant<int, 4>{});
  return launch(std::integral_constant<int, embed::CS_MOST>{});
}

int embed_check(int64_t n, int64_t V, int64_t D, int dtype) {
  if (n < 0 || V <= 0 || D <= 0 || !lm_dtype(dtype)) return THERIA_ERR_INVALID_ARG;
  if (n >= (1ll << 30) || V >= (1ll << 31) - 1 || D > 32 * 65535ll) return THERIA_ERR_UNSUPPORTED;
  return THERIA_OK;
}

}  // namespace
}  // namespace theria

using namespace theria;

extern "C" {

int theria_embed_fwd(const void* ids, int wide, const void* w, void* out, int64_t n, int64_t V,
                     int64_t D, int dtype, float scale, int64_t zero_idx, void* stream) {
  if (int e = embed_check(n, V, D, dtype)) return e;
  if (n == 0) return THERIA_OK;
  if (!ids || !w || !out) return THERIA_ERR_INVALID_ARG;
  const bool vec = vec_rows(D, dtype, {w, out});
  const unsigned grid = (unsigned)std::min<int64_t>(cdiv(n, embed::WARPS), kSMs * 64);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int VEC = embed::Vec<T>::n;
    auto kern = vec ? embed::fwd_kernel<T, VEC> : embed::fwd_kernel<T, 1>;
    kern<<<grid, embed::WARPS * 32, 0, (cudaStream_t)stream>>>(ids, wide, (const T*)w, (T*)out, n,
                                                               V, D, scale, zero_idx);
    return launch_status();
  });
}

int64_t theria_embed_bwd_workspace_bytes(int64_t n, int64_t V, int64_t D) {
  return n <= 0 || V <= 0 || D <= 0 ? 0 : embed_ws(nullptr, n, V, D).bytes;
}

int theria_embed_bwd(const void* ids, int wide, const void* gy, void* gw, void* workspace,
                     int64_t workspace_bytes, int64_t n, int64_t V, int64_t D, int dtype,
                     float scale, int64_t zero_idx, void* stream) {
  if (int e = embed_check(n, V, D, dtype)) return e;
  cudaStream_t st = (cudaStream_t)stream;
  if (!gw) return THERIA_ERR_INVALID_ARG;
  if (n == 0)
    return cudaMemsetAsync(gw, 0, V * D * elem_size(dtype), st) == cudaSuccess
               ? THERIA_OK
               : THERIA_ERR_LAUNCH;
  if (!ids || !gy) return THERIA_ERR_INVALID_ARG;
  if (!workspace || workspace_bytes < theria_embed_bwd_workspace_bytes(n, V, D))
    return THERIA_ERR_WORKSPACE;
  const EmbedWs ws = embed_ws(workspace, n, V, D);
  int bits = 1;  // keys are 0 .. V
  while ((V >> bits) != 0) ++bits;
  const uint32_t *keys = nullptr, *vals = nullptr;
  const int64_t gw_bytes = V * D * elem_size(dtype);
  const bool fill = n <= kClusterSort && tc::aligned16(gw);
  if (!fill && cudaMemsetAsync(gw, 0, gw_bytes, st) != cudaSuccess) return THERIA_ERR_LAUNCH;
  if (n <= kClusterSort) {
    if (int e = embed_cluster_sort(ids, wide, ws, n, V, zero_idx, bits, gw, fill ? gw_bytes : 0,
                                   st))
      return e;
    keys = ws.keys[0];
    vals = ws.vals[0];
  } else {
    const unsigned tiles = (unsigned)cdiv(n, embed::TILE);
    int to = 0;
    for (int shift = 0; shift < bits; shift += 8, to ^= 1) {
      embed::hist_kernel<<<tiles, embed::SORT_THREADS, 0, st>>>(ids, wide, keys, ws.hist, n, V,
                                                                zero_idx, shift);
      if (int e = launch_status()) return e;
      embed::scan_kernel<<<1, 1024, 0, st>>>(ws.hist, (int64_t)tiles * embed::BINS);
      if (int e = launch_status()) return e;
      embed::scatter_kernel<<<tiles, embed::SORT_THREADS, 0, st>>>(
          ids, wide, keys, vals, ws.hist, ws.keys[to], ws.vals[to], n, V, zero_idx, shift);
      if (int e = launch_status()) return e;
      keys = ws.keys[to];
      vals = ws.vals[to];
    }
  }
  const bool vec = vec_rows(D, dtype, {gy, gw});
  const int64_t chunks = cdiv(n, embed::CHUNK);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int VEC = embed::Vec<T>::n;
    const int64_t units = cdiv(D, vec ? VEC : 1);
    int width = 1;  // threads of a chunk: a power of two
    while (width < 256 && width < units) width *= 2;
    auto kern = vec ? embed::chunk_kernel<T, VEC> : embed::chunk_kernel<T, 1>;
    kern<<<dim3((unsigned)cdiv(chunks, 256 / width), (unsigned)cdiv(units, width)), 256, 0, st>>>(
        (const T*)gy, keys, vals, ws.part, (T*)gw, n, V, D, scale, width);
    if (int e = launch_status()) return e;
    if (chunks < 2) return (int)THERIA_OK;
    auto join = D % 4 == 0 ? embed::join_kernel<T, 4> : embed::join_kernel<T, 1>;
    join<<<dim3((unsigned)(chunks - 1), (unsigned)cdiv(D, D % 4 == 0 ? 1024 : 256)), 256, 0, st>>>(
        keys, ws.part, (T*)gw, n, V, D, scale);
    return launch_status();
  });
}

}  // extern "C"

// ------------------------------------------------------------ layer norm
namespace theria {
namespace {

int norm_check(int64_t N, int64_t D, int dtype, int wdtype) {
  if (N < 0 || D <= 0 || !lm_dtype(dtype)) return THERIA_ERR_INVALID_ARG;
  if (wdtype != dtype && wdtype != THERIA_F32) return THERIA_ERR_INVALID_ARG;
  if (D >= (1ll << 31)) return THERIA_ERR_UNSUPPORTED;
  return THERIA_OK;
}

// Calls f(NV, NW) (integral constants) for rows of `units` vectors of VEC
// values: the fewest warps per row that hold it in MOST values a thread (one
// warp needs no barrier), and the fewest vectors a thread among MOST / VEC and
// its half (a quarter and an eighth for one warp); false where even 32 warps
// do not hold it.
template <int VEC, int MOST, int NW, typename F>
bool norm_vectors(int64_t units, F f) {
  constexpr int NV = MOST / VEC;
  constexpr int64_t G = 32 * NW;
  using W = std::integral_constant<int, NW>;
  if (units > G * NV) return false;
  if constexpr (NW == 1 && NV >= 8)
    if (units <= G * (NV / 8)) return f(std::integral_constant<int, NV / 8>{}, W{}), true;
  if constexpr (NW == 1 && NV >= 4)
    if (units <= G * (NV / 4)) return f(std::integral_constant<int, NV / 4>{}, W{}), true;
  if constexpr (NV >= 2)
    if (units <= G * (NV / 2)) return f(std::integral_constant<int, NV / 2>{}, W{}), true;
  return f(std::integral_constant<int, NV>{}, W{}), true;
}
template <int VEC, int MOST, typename F>
bool norm_shape(int64_t D, F f) {
  const int64_t units = cdiv(D, VEC);
  return norm_vectors<VEC, MOST, 1>(units, f) || norm_vectors<VEC, MOST, 4>(units, f) ||
         norm_vectors<VEC, MOST, 8>(units, f) || norm_vectors<VEC, MOST, 16>(units, f) ||
         norm_vectors<VEC, MOST, 32>(units, f);
}
// Values a thread: more of them share the cost of a row's reduction (forward,
// 16384 x 4096 bfloat16: 32 values 58 us, 16 values 76, 8 values 108); the
// backward holds column sums besides, and takes 16 only for rows too wide for 8.
constexpr int kNormFwd = 32, kNormBwd = 8, kNormBwdWide = 16;

// CTAs of the backward: what its column sums are split over.
constexpr int64_t kMaxGrid = (1ll << 31) - 1;
int64_t norm_ctas(int64_t N) { return std::min<int64_t>(N, kSMs * 4); }
// What of them runs at one time: with more, some SMs would take another whole
// share of the rows (32768 x 1111 float16, three CTAs an SM instead of the four
// asked for: second derivative 868 us, with their number 484).
template <typename K>
int64_t norm_wave(K kern, int threads, size_t smem, int64_t N) {
  int per_sm = 1;
  cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem);
  return std::min<int64_t>(norm_ctas(N), kSMs * std::max(per_sm, 1));
}

}  // namespace
}  // namespace theria

extern "C" {

int theria_norm_fwd(const void* x, const void* w, const void* b, int wdtype, void* y,
                    float* stats, int64_t N, int64_t D, int dtype, float eps, void* stream) {
  if (int e = norm_check(N, D, dtype, wdtype)) return e;
  if (N == 0) return THERIA_OK;
  if (!x || !y || !tc::aligned16(stats)) return THERIA_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const bool vec = vec_rows(D, dtype, {x, y, w, b});
  const int wf32 = wdtype == THERIA_F32;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto vecn) {
      constexpr int VEC = decltype(vecn)::value;
      auto run = [&](auto nv, auto nw, auto rc) {
        constexpr int NV = decltype(nv)::value, NW = decltype(nw)::value, R = decltype(rc)::value;
        using B = norm::Block<NW>;
        norm::fwd_kernel<T, VEC, NV, NW, R>
            <<<(unsigned)std::min<int64_t>(cdiv(N, B::rows * R), NW == 1 ? kSMs * 32 : kMaxGrid),
               B::threads, 0, st>>>((const T*)x, w, b, wf32, (T*)y, stats, N, (int)D, eps);
      };
      auto four = [&](auto nv, auto nw) { run(nv, nw, std::integral_constant<int, 4>{}); };
      auto two = [&](auto nv, auto nw) { run(nv, nw, std::integral_constant<int, 2>{}); };
      auto one = [&](auto nv, auto nw) { run(nv, nw, std::integral_constant<int, 1>{}); };
      // a warp takes as many rows at a time as make kNormFwd values a lane
      const int64_t units = cdiv(D, VEC);
      return norm_vectors<VEC, kNormFwd / 4, 1>(units, four) ||
             norm_vectors<VEC, kNormFwd / 2, 1>(units, two) || norm_shape<VEC, kNormFwd>(D, one);
    };
    const bool done = vec ? launch(std::integral_constant<int, embed::Vec<T>::n>{})
                          : launch(std::integral_constant<int, 1>{});
    if (!done)
      norm::fwd_wide_kernel<T><<<(unsigned)std::min<int64_t>(N, kSMs * 8), 256, 0, st>>>(
          (const T*)x, w, b, wdtype, (T*)y, stats, N, D, eps);
    return launch_status();
  });
}

int64_t theria_norm_bwd_workspace_bytes(int64_t N, int64_t D) {
  return N <= 0 || D <= 0 ? 0 : norm_ctas(N) * 2 * D * (int64_t)sizeof(float);
}

int theria_norm_bwd(const void* x, const void* w, int wdtype, const void* gy,
                    const float* stats, void* gx, void* gw, void* gb, void* workspace,
                    int64_t workspace_bytes, int64_t N, int64_t D, int dtype, void* stream) {
  if (int e = norm_check(N, D, dtype, wdtype)) return e;
  if ((gw == nullptr) != (gb == nullptr)) return THERIA_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  if (N == 0) {
    if (gw) {
      cudaMemsetAsync(gw, 0, D * elem_size(wdtype), st);
      cudaMemsetAsync(gb, 0, D * elem_size(wdtype), st);
    }
    return THERIA_OK;
  }
  if (!x || !gy || !stats || !tc::aligned16(stats)) return THERIA_ERR_INVALID_ARG;
  if (!gx && !gw) return THERIA_OK;
  if (gw && (!workspace || workspace_bytes < theria_norm_bwd_workspace_bytes(N, D)))
    return THERIA_ERR_WORKSPACE;
  const bool vec = vec_rows(D, dtype, {x, gy, gx, w});
  const int wf32 = wdtype == THERIA_F32;
  float* part = gw ? (float*)workspace : nullptr;
  int ctas = 0;
  int e = by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto vecn) {
      constexpr int VEC = decltype(vecn)::value;
      auto run = [&](auto nv, auto nw) {
        constexpr int NV = decltype(nv)::value, NW = decltype(nw)::value;
        using B = norm::Block<NW>;
        // the partial sums of a CTA's eight rows at a time
        const int64_t sums = NW == 1 && part ? 8 * 2 * D * (int64_t)sizeof(float) : 0;
        if constexpr (VEC > 1) {
          const int64_t row = 2 * D * (int64_t)sizeof(T);  // of x and gy
          if (2 * (row + 16) <= 201 << 10) {  // and the row's statistics
            // Rows of a batch: 4 for a warp of its own and where they make a
            // stage of at most 16 KB (65536 x 1024 bfloat16: 73 us, with 2 rows
            // 80, with one 97), 2 up to 32 KB (16384 x 4096 bfloat16: 78 us,
            // with one 94, with 4 106), else 1.
            auto batch = [&](auto rc) {
              constexpr int R = decltype(rc)::value;
              auto kern = norm::bwd_batch_kernel<T, VEC, NV, NW, R>;
              const int64_t rows = B::rows * R, stage = rows * row;
              // float32 rows need more bytes on their way (16384 x 4096: 128 KB
              // 128 us, 96 KB 140), 16-bit rows a second CTA (78 us, 82)
              const int64_t ring = (sizeof(T) == 4 ? 128 : 96) << 10;
              const int stages = (int)std::clamp<int64_t>(ring / stage, 2, norm::MAX_STAGES);
              const int64_t smem = std::max(sums, (stage + 16 * rows) * stages);
              if (smem > 40 << 10)  // with the kernel's static part, above the default limit
                cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
              ctas = (int)std::min(cdiv(N, rows), norm_wave(kern, B::threads, smem, N));
              kern<<<(unsigned)ctas, B::threads, smem, st>>>((const T*)x, w, wf32, (const T*)gy,
                                                             stats, (T*)gx, part, N, (int)D,
                                                             stages);
            };
            if constexpr (NW == 1) batch(std::integral_constant<int, 4>{});
            else if (4 * row <= 16 << 10) batch(std::integral_constant<int, 4>{});
            else if (2 * row <= 32 << 10) batch(std::integral_constant<int, 2>{});
            else batch(std::integral_constant<int, 1>{});
            return;
          }
        }
        auto kern = norm::bwd_kernel<T, VEC, NV, NW>;
        ctas = (int)std::min(cdiv(N, B::rows), norm_wave(kern, B::threads, sums, N));
        kern<<<(unsigned)ctas, B::threads, sums, st>>>(
            (const T*)x, w, wf32, (const T*)gy, stats, (T*)gx, part, N, (int)D);
      };
      if (norm_shape<VEC, kNormBwd>(D, run)) return true;
      // wider rows need all 32 warps
      constexpr int NV = kNormBwdWide / VEC;
      if (cdiv(D, VEC) > 32 * 32 * NV) return false;
      run(std::integral_constant<int, NV>{}, std::integral_constant<int, 32>{});
      return true;
    };
    const bool done = vec ? launch(std::integral_constant<int, embed::Vec<T>::n>{})
                          : launch(std::integral_constant<int, 1>{});
    if (!done) {
      ctas = (int)norm_ctas(N);
      norm::bwd_wide_kernel<T><<<(unsigned)ctas, 256, 0, st>>>(
          (const T*)x, w, wdtype, (const T*)gy, stats, (T*)gx, part, N, D);
    }
    return launch_status();
  });
  if (e || !gw) return e;
  norm::cols_kernel<<<(unsigned)cdiv(2 * D, 32), 1024, 0, st>>>(part, gw, gb, wdtype, ctas, D);
  return launch_status();
}

int theria_norm_bwd2(const void* x, const void* w, int wdtype, const void* gy,
                     const float* stats, const void* u, const void* a, const void* c, void* dx,
                     void* dw, void* dgy, void* workspace, int64_t workspace_bytes, int64_t N,
                     int64_t D, int dtype, void* stream) {
  if (int e = norm_check(N, D, dtype, wdtype)) return e;
  cudaStream_t st = (cudaStream_t)stream;
  if (N == 0) {
    if (dw) cudaMemsetAsync(dw, 0, D * elem_size(wdtype), st);
    return THERIA_OK;
  }
  if (!x || !gy || !stats || !dx || !dgy || (dw && !w) || !tc::aligned16(stats))
    return THERIA_ERR_INVALID_ARG;
  if (!workspace || workspace_bytes < theria_norm_bwd_workspace_bytes(N, D))
    return THERIA_ERR_WORKSPACE;
  const bool vec = vec_rows(D, dtype, {x, gy, u, dx, dgy, w, a, c});
  const int wf32 = wdtype == THERIA_F32;
  float* part = (float*)workspace;
  int ctas = 0;
  int e = by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto vecn) {
      constexpr int VEC = decltype(vecn)::value;
      return norm_shape<VEC, kNormBwdWide>(D, [&](auto nv, auto nw) {
        constexpr int NV = decltype(nv)::value, NW = decltype(nw)::value;
        using B = norm::Block<NW>;
        auto kern = norm::bwd2_kernel<T, VEC, NV, NW>;
        const size_t smem = NW == 1 ? 8 * 2 * D * sizeof(float) : 0;
        if (smem > 48 * 1024)
          cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        ctas = (int)std::min(cdiv(N, B::rows), norm_wave(kern, B::threads, smem, N));
        kern<<<(unsigned)ctas, B::threads, smem, st>>>((const T*)x, w, wf32, (const T*)gy, stats,
                                                (const T*)u, a, c, (T*)dx, (T*)dgy, part, N,
                                                (int)D);
      });
    };
    const bool done = vec ? launch(std::integral_constant<int, embed::Vec<T>::n>{})
                          : launch(std::integral_constant<int, 1>{});
    if (!done) {
      ctas = (int)norm_ctas(N);
      norm::bwd2_wide_kernel<T><<<(unsigned)ctas, 256, 0, st>>>(
          (const T*)x, w, wdtype, (const T*)gy, stats, (const T*)u, a, c, (T*)dx, (T*)dgy, part,
          N, D);
    }
    return launch_status();
  });
  if (e || !dw) return e;
  norm::cols_kernel<<<(unsigned)cdiv(D, 32), 1024, 0, st>>>(part, dw, nullptr, wdtype, ctas, D);
  return launch_status();
}

}  // extern "C"

// --------------------------------------------------- linear cross entropy
namespace theria {
namespace {

int xent_check(int64_t N, int64_t V, int64_t D, int dtype, int reduction) {
  if (N < 0 || V <= 0 || D <= 0 || !lm_dtype(dtype)) return THERIA_ERR_INVALID_ARG;
  if (reduction < THERIA_LOSS_NONE || reduction > THERIA_LOSS_MEAN) return THERIA_ERR_INVALID_ARG;
  if (N >= (1ll << 30) || V >= (1ll << 30) || D >= (1ll << 27))
    return THERIA_ERR_UNSUPPORTED;
  return THERIA_OK;
}

struct XentRows {  // filled by prep_kernel
  int *pos, *row_of, *tgt, *n_live;
  unsigned* done;
  float4* row;  // backward, by packed row (see RowArgs)
  float *post, *most;
  xent::Splits *plan_h, *plan_w;
};
XentRows xent_rows(Carver& c, int64_t N) {
  XentRows r;
  r.pos = c.take<int>(N);
  r.row_of = c.take<int>(N);
  r.tgt = c.take<int>(N);
  r.row = c.take<float4>(N);
  r.n_live = c.take<int>(64);  // and what else is one value
  r.done = (unsigned*)r.n_live + 1;
  r.post = (float*)r.n_live + 2;
  r.most = r.post + 1;
  r.plan_h = (xent::Splits*)(r.n_live + 4);
  r.plan_w = r.plan_h + 1;
  return r;
}
xent::Prep xent_prep(const XentRows& r, const void* target, int wide, int64_t ignore_index,
                     int64_t N, int64_t V) {
  xent::Prep p{};
  p.target = target;
  p.wide = wide;
  p.ignore_index = ignore_index;
  p.N = N;
  p.V = V;
  p.pos = r.pos;
  p.row_of = r.row_of;
  p.tgt = r.tgt;
  p.n_live = r.n_live;
  p.done = r.done;
  return p;
}
// Where the forward's loss goes: each row's, and their sum or mean (NULL: no).
struct LossOut {
  float *each, *lse, *out;
  int mean;
};
int xent_join(const XentRows& r, const float2* part, const float* zt, int tiles,
              const LossOut& o, int64_t N, cudaStream_t st) {
  return launch_chained(xent::join_kernel, dim3((unsigned)std::min<int64_t>(cdiv(N, 8), kSMs * 8)),
                        dim3(256), 0, st, part, zt, r.row_of, r.n_live, tiles, o.each, o.lse,
                        r.done, o.out, o.mean, N);
}
constexpr int kClusters = xent::CLUSTERS;
static_assert(kClusters == kSMs / 2 && xent::BM == xent::TILE_ROWS, "dh's split");

struct XentSizes {
  int64_t Mp, Kp;          // packed rows, elements of a packed row (one plane)
  int planes;              // of a value, dz's as well
  bool pack_w;             // w needs a packed copy
  int64_t piece;           // of the vocabulary, backward
  int64_t ld_acc, acc_rows;  // dh's partial sums: at most these rows
  // dw is split over the rows that count (and made by partial sums) where it has
  // no more tiles than half the clusters; its partial sums' rows
  bool split_w;
  int64_t acc_rows_w;
};
XentSizes xent_sizes(int64_t N, int64_t V, int64_t D, int dtype) {
  XentSizes z;
  z.Mp = up(N, xent::BM);
  z.Kp = up(D, xent::BK);
  z.planes = dtype == THERIA_F32 ? 3 : 1;
  z.pack_w = z.planes > 1 || D % 8 != 0;
  // dz of a piece within 512 MB
  const int64_t fit = (512ll << 20) / (z.Mp * 2 * z.planes) / xent::BN * xent::BN;
  z.piece = std::min(up(V, xent::BN), std::max<int64_t>(xent::BN, fit));
  z.ld_acc = up(D, 32);
  z.acc_rows = std::max(z.Mp, std::min(xent::MAX_UNITS / cdiv(D, xent::BN) * xent::BM,
                                       cdiv(z.piece, xent::BK) * z.Mp));
  const int64_t vt = cdiv(V, xent::BM), dt = cdiv(D, xent::BN);
  z.split_w = vt * dt * 2 <= kClusters && z.piece >= V;
  z.acc_rows_w = std::max(vt, std::min(xent::MAX_UNITS_DW / dt, cdiv(N, xent::BK) * vt)) * xent::BM;
  return z;
}

struct XentFwdWs {
  XentRows rows;
  void *hp, *wp;
  float2* part;
  float *zt, *each;
  int64_t bytes;
};
XentFwdWs xent_fwd_ws(void* base, int64_t N, int64_t V, int64_t D, const XentSizes& z) {
  Carver c{(char*)base};
  XentFwdWs w;
  w.rows = xent_rows(c, N);
  w.hp = c.take<uint16_t>(z.Mp * z.Kp * z.planes);
  w.wp = z.pack_w ? c.take<uint16_t>(V * z.Kp * z.planes) : nullptr;
  w.part = c.take<float2>(z.Mp * cdiv(V, xent::SUB));
  w.zt = c.take<float>(z.Mp);
  w.each = c.take<float>(N);
  w.bytes = c.used;
  return w;
}
struct XentBwdWs {
  XentRows rows;
  void *hp, *wp, *dz;
  float *acc, *acc_w;
  int64_t bytes;
};
XentBwdWs xent_bwd_ws(void* base, int64_t N, int64_t V, int64_t D, const XentSizes& z) {
  Carver c{(char*)base};
  XentBwdWs w;
  w.rows = xent_rows(c, N);
  w.hp = c.take<uint16_t>(z.Mp * z.Kp * z.planes);
  w.wp = z.pack_w ? c.take<uint16_t>(V * z.Kp * z.planes) : nullptr;
  w.dz = c.take<uint16_t>(z.Mp * z.piece * z.planes);
  w.acc = c.take<float>(z.acc_rows * z.ld_acc);
  w.acc_w = z.split_w ? c.take<float>(z.acc_rows_w * z.ld_acc) : nullptr;
  w.bytes = c.used;
  return w;
}

// 2-D map of rows [rows][inner] of `dtype`, `inner` apart, box {bytes / size,
// box_rows}, swizzled by `bytes` (128 or 64).
bool map_2d(CUtensorMap* map, const void* base, int dtype, int64_t inner, int64_t rows,
            int box_rows, int bytes = 128) {
  tc::EncodeTiledFn fn = tc::encode_fn();
  if (fn == nullptr) return false;
  const int64_t size = elem_size(dtype);
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(inner * size)};
  cuuint32_t box[2] = {(cuuint32_t)(bytes / size), (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map,
            dtype == THERIA_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
            : dtype == THERIA_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                  : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, typename O, int EPI, bool CHUNKS = sizeof(O) == 4>
int tc_launch(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& h,
              const CUtensorMap& o, const CUtensorMap& p, const xent::TcArgs& args, int64_t units,
              cudaStream_t st) {
  auto kern = xent::tc_kernel<T, O, EPI, CHUNKS>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           xent::TcSmem::kAlloc) != cudaSuccess)
    return THERIA_ERR_LAUNCH;
  const unsigned grid = 2 * (unsigned)std::min<int64_t>(units, kClusters);
  return launch_chained(kern, dim3(grid), dim3(xent::TC_THREADS), xent::TcSmem::kAlloc, st, a, b, h,
                        o, p, args);
}

// T: the operands' type; O: the tensors'.
template <typename T, typename O>
struct Tc {
  static constexpr int op = std::is_same<T, __half>::value ? THERIA_F16 : THERIA_BF16;

  // h can be read by TMA as it is (where every row counts)
  static bool plain(const void* h, int64_t D, const XentSizes& z) {
    return z.planes == 1 && D % 8 == 0 && tc::aligned16(h);
  }
  // h (the rows that count) and, where it is not read as it is, w; and `rows`
  static int pack(const void* h, const void* w, const XentRows& r, const xent::RowArgs& rows,
                  void* hp, void* wp, const XentSizes& z, int64_t N, int64_t V, int64_t D,
                  cudaStream_t st) {
    const int dtype = std::is_same<O, float>::value ? THERIA_F32 : op;
    const int64_t units = z.Kp / 8;
    auto ctas = [&](int64_t rows) {
      return (int)std::min<int64_t>(cdiv(rows * units, 256), kSMs * 16);
    };
    const xent::PackArgs ph{h, hp, r.row_of, r.n_live, N, vec_rows(D, dtype, {h}), plain(h, D, z)};
    const xent::PackArgs pw{w, wp, nullptr, nullptr, V, vec_rows(D, dtype, {w}), 0};
    const int h_ctas = ctas(z.Mp), w_ctas = z.pack_w ? ctas(V) : 0;
    return launch_chained(xent::pack_kernel<T, O>, dim3(h_ctas + w_ctas), dim3(256), 0, st, ph, pw,
                          rows, h_ctas, D, z.Kp);
  }
  // dh and dw from their partial sums (either may have no rows)
  static int sum(const xent::SumArgs& a, const xent::SumArgs& b, const float* post,
                 const XentSizes& z, int64_t D, cudaStream_t st) {
    constexpr int VEC = embed::Vec<O>::n;
    const int dtype = std::is_same<O, float>::value ? THERIA_F32 : op;
    auto kern = vec_rows(D, dtype, {a.out, b.out}) ? xent::split_sum_kernel<O, VEC>
                                                   : xent::split_sum_kernel<O, 1>;
    const int a_ctas = (int)std::min<int64_t>(a.rows, kSMs * 16);
    const int b_ctas = (int)std::min<int64_t>(b.rows, kSMs * 16);
    if (a_ctas + b_ctas == 0) return THERIA_OK;
    return launch_chained(kern, dim3(a_ctas + b_ctas), dim3(256), 0, st, a, b, a_ctas, post,
                          (int)z.ld_acc, (int)D);
  }
  static xent::TcArgs common(const void* h, const XentRows& r, const XentSizes& z, int64_t N,
                             int64_t V, int64_t D) {
    xent::TcArgs a{};
    a.n_live = r.n_live;
    a.V = (int)V;
    a.D = (int)D;
    a.plane_a = a.plane_b = (int)z.Kp;
    a.tgt = r.tgt;
    a.rows = (int)N;
    a.h_plain = plain(h, D, z);
    return a;
  }

  static int fwd(const void* h, const void* w, const XentFwdWs& ws, const XentSizes& z,
                 const LossOut& out, int64_t N, int64_t V, int64_t D, cudaStream_t st) {
    xent::TcArgs a = common(h, ws.rows, z, N, V, D);
    if (int e = pack(h, w, ws.rows, {}, ws.hp, ws.wp, z, N, V, D, st)) return e;
    const int64_t row = z.Kp * z.planes;
    CUtensorMap ma, mb, mh;
    if (!map_2d(&ma, ws.hp, op, row, z.Mp, xent::HALF) ||
        !map_2d(&mb, z.pack_w ? ws.wp : w, op, z.pack_w ? row : D, V, xent::HALF))
      return THERIA_ERR_LAUNCH;
    mh = ma;
    if (a.h_plain && !map_2d(&mh, h, op, D, N, xent::HALF)) return THERIA_ERR_LAUNCH;
    a.part = ws.part;
    a.sub_tiles = (int)cdiv(V, xent::SUB);
    a.zt = ws.zt;
    const int64_t units = z.Mp / xent::BM * cdiv(V, xent::BN);
    if (int e = D > xent::DEEP && units <= xent::DEEP_UNITS
                    ? tc_launch<T, O, xent::kScore, true>(ma, mb, mh, ma, ma, a, units, st)
                    : tc_launch<T, O, xent::kScore>(ma, mb, mh, ma, ma, a, units, st))
      return e;
    return xent_join(ws.rows, ws.part, ws.zt, a.sub_tiles, out, N, st);
  }

  // gloss: the rows' upstream gradients; NULL where there is one for all
  static int bwd(const void* h, const void* w, const float* lse, const float* gloss,
                 const XentBwdWs& ws, const XentSizes& z, void* dh, void* dw, int64_t N,
                 int64_t V, int64_t D, int dtype, cudaStream_t st) {
    const XentRows& r = ws.rows;
    const xent::TcArgs base = common(h, r, z, N, V, D);
    const xent::RowArgs rows{lse, gloss, r.most, op == THERIA_F16 ? xent::HALF_SCALE : 1.f, r.row};
    if (int e = pack(h, w, r, rows, ws.hp, ws.wp, z, N, V, D, st)) return e;
    const int64_t row = z.Kp * z.planes, zrow = z.piece * z.planes;
    const void* wsrc = z.pack_w ? ws.wp : w;
    const int64_t wrow = z.pack_w ? row : D;
    const bool dw_tma = dw && (z.split_w || vec_rows(D, dtype, {dw}));
    // contraction along the row (k) or across rows (m); outputs (o)
    CUtensorMap hk, hm, hk1, hm1, wk, wm, zk, zm, zo, zp, ho, wo;
    if (!map_2d(&hk, ws.hp, op, row, z.Mp, xent::HALF) ||
        !map_2d(&hm, ws.hp, op, row, z.Mp, xent::BK) ||
        !map_2d(&wk, wsrc, op, wrow, V, xent::HALF) ||
        !map_2d(&wm, wsrc, op, wrow, V, xent::BK) ||
        !map_2d(&zk, ws.dz, op, zrow, z.Mp, xent::HALF) ||
        !map_2d(&zm, ws.dz, op, zrow, z.Mp, xent::BK) ||
        !map_2d(&zo, ws.dz, op, zrow, z.Mp, 32) || !map_2d(&zp, ws.dz, op, zrow, z.Mp, 32, 64) ||
        !map_2d(&ho, ws.acc, THERIA_F32, z.ld_acc, z.acc_rows, 32))
      return THERIA_ERR_LAUNCH;
    hk1 = hk;
    hm1 = hm;
    wo = zo;
    if (base.h_plain && (!map_2d(&hk1, h, op, D, N, xent::HALF) ||
                         !map_2d(&hm1, h, op, D, N, xent::BK)))
      return THERIA_ERR_LAUNCH;
    if (dw_tma && !(z.split_w
                        ? map_2d(&wo, ws.acc_w, THERIA_F32, z.ld_acc, z.acc_rows_w, 32)
                        : map_2d(&wo, dw, dtype, D, V, 32)))
      return THERIA_ERR_LAUNCH;
    const int64_t mt = z.Mp / xent::BM, dt = cdiv(D, xent::BN);
    for (int64_t c0 = 0; c0 < V; c0 += z.piece) {
      const int64_t C = std::min(z.piece, V - c0), ct = cdiv(C, xent::BN);
      xent::TcArgs a = base;
      a.c0 = (int)c0;
      a.Cn = (int)C;
      a.row = r.row;
      a.ld_dz = (int)z.piece;
      a.plan = r.plan_h;
      a.ld_acc = (int)z.ld_acc;
      a.out = dw_tma ? nullptr : dw;
      a.post = r.post;
      a.add = c0 > 0;
      if (int e = tc_launch<T, O, xent::kDz>(hk, wk, hk1, zo, zp, a, mt * ct, st)) return e;
      a.plane_a = (int)z.piece;
      if (dh)
        if (int e = tc_launch<T, O, xent::kDh>(zk, wm, zk, ho, ho, a,
                                                std::max<int64_t>(mt * dt, kClusters), st))
          return e;
      if (!dw) continue;
      a.plan = z.split_w ? r.plan_w : nullptr;
      if (int e = tc_launch<T, O, xent::kDw>(
              zm, hm, hm1, wo, wo, a, z.split_w ? kClusters : ct * dt, st))
        return e;
    }
    return sum({ws.acc, r.pos, r.plan_h, dh, dh ? N : 0},
               {ws.acc_w, nullptr, r.plan_w, dw, dw && z.split_w ? V : 0}, r.post, z, D, st);
  }
};

// Whether the tensor-core kernels can read w: 16 bytes at a time, where they
// do not pack it first.
bool w_readable(const void* w, int64_t D, int dtype) {
  return dtype == THERIA_F32 || D % 8 != 0 || tc::aligned16(w);
}

}  // namespace
}  // namespace theria

extern "C" {

int64_t theria_xent_fwd_workspace_bytes(int64_t N, int64_t V, int64_t D, int dtype) {
  if (N <= 0 || V <= 0 || D <= 0) return 0;
  return xent_fwd_ws(nullptr, N, V, D, xent_sizes(N, V, D, dtype)).bytes;
}
int64_t theria_xent_bwd_workspace_bytes(int64_t N, int64_t V, int64_t D, int dtype) {
  if (N <= 0 || V <= 0 || D <= 0) return 0;
  return xent_bwd_ws(nullptr, N, V, D, xent_sizes(N, V, D, dtype)).bytes;
}

int theria_xent_fwd(const void* h, const void* w, const void* target, int wide,
                    int64_t ignore_index, int reduction, float* loss, float* lse, float* count,
                    void* workspace, int64_t workspace_bytes, int64_t N, int64_t V, int64_t D,
                    int dtype, void* stream) {
  if (int e = xent_check(N, V, D, dtype, reduction)) return e;
  if (!count || (!loss && (N > 0 || reduction != THERIA_LOSS_NONE)) || (!lse && N > 0))
    return THERIA_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  if (N > 0 && (!h || !w || !target)) return THERIA_ERR_INVALID_ARG;
  if (N > 0 && (!workspace || workspace_bytes < theria_xent_fwd_workspace_bytes(N, V, D, dtype)))
    return THERIA_ERR_WORKSPACE;
  if (N == 0) {
    // the sum of no rows, and their mean
    if (cudaMemsetAsync(count, 0, sizeof(float), st) != cudaSuccess) return THERIA_ERR_LAUNCH;
    if (reduction == THERIA_LOSS_NONE) return THERIA_OK;
    return cudaMemsetAsync(loss, reduction == THERIA_LOSS_MEAN ? 0xff : 0, sizeof(float), st) ==
                   cudaSuccess  // all bits set: NaN
               ? THERIA_OK
               : THERIA_ERR_LAUNCH;
  }
  if (!w_readable(w, D, dtype)) return THERIA_ERR_INVALID_ARG;
  const XentSizes z = xent_sizes(N, V, D, dtype);
  const XentFwdWs ws = xent_fwd_ws(workspace, N, V, D, z);
  const LossOut out{reduction == THERIA_LOSS_NONE ? loss : ws.each, lse,
                    reduction == THERIA_LOSS_NONE ? nullptr : loss,
                    reduction == THERIA_LOSS_MEAN};
  xent::Prep p = xent_prep(ws.rows, target, wide, ignore_index, N, V);
  p.count = count;
  p.loss = out.each;
  p.lse = lse;
  xent::prep_kernel<<<1, 1024, 0, st>>>(p);
  if (int e = launch_status()) return e;
  return dtype == THERIA_F32   ? Tc<__nv_bfloat16, float>::fwd(h, w, ws, z, out, N, V, D, st)
         : dtype == THERIA_F16 ? Tc<__half, __half>::fwd(h, w, ws, z, out, N, V, D, st)
                               : Tc<__nv_bfloat16, __nv_bfloat16>::fwd(h, w, ws, z, out, N, V, D,
                                                                       st);
}

int theria_xent_bwd(const void* h, const void* w, const void* target, int wide,
                    int64_t ignore_index, int reduction, const float* gloss, const float* lse,
                    const float* count, void* dh, void* dw, void* workspace,
                    int64_t workspace_bytes, int64_t N, int64_t V, int64_t D, int dtype,
                    void* stream) {
  if (int e = xent_check(N, V, D, dtype, reduction)) return e;
  cudaStream_t st = (cudaStream_t)stream;
  if (N == 0) {
    if (dw && cudaMemsetAsync(dw, 0, V * D * elem_size(dtype), st) != cudaSuccess)
      return THERIA_ERR_LAUNCH;
    return THERIA_OK;
  }
  if (!h || !w || !target || !gloss || !lse || !count) return THERIA_ERR_INVALID_ARG;
  if (!dh && !dw) return THERIA_OK;
  if (!workspace || workspace_bytes < theria_xent_bwd_workspace_bytes(N, V, D, dtype))
    return THERIA_ERR_WORKSPACE;
  if (!w_readable(w, D, dtype)) return THERIA_ERR_INVALID_ARG;
  const XentSizes z = xent_sizes(N, V, D, dtype);
  const XentBwdWs ws = xent_bwd_ws(workspace, N, V, D, z);
  const XentRows& r = ws.rows;
  xent::Prep p = xent_prep(r, target, wide, ignore_index, N, V);
  p.gloss = gloss;
  p.mean_of = reduction == THERIA_LOSS_MEAN ? count : nullptr;
  p.per_row = reduction == THERIA_LOSS_NONE;
  p.half = dtype == THERIA_F16;
  p.most = r.most;
  p.post = r.post;
  p.plan_h = dh ? r.plan_h : nullptr;
  p.plan_w = dw && z.split_w ? r.plan_w : nullptr;
  p.kb = (int)cdiv(std::min(z.piece, V), xent::BK);
  p.d_tiles = (int)cdiv(D, xent::BN);
  p.v_tiles = (int)cdiv(V, xent::BM);
  p.f32 = dtype == THERIA_F32;
  p.ld_acc = (int)z.ld_acc;
  xent::prep_kernel<<<1, 1024, 0, st>>>(p);
  if (int e = launch_status()) return e;
  auto run = [&](auto tc) {
    return decltype(tc)::bwd(h, w, lse, p.per_row ? gloss : nullptr, ws, z, dh, dw, N, V, D, dtype,
                             st);
  };
  return dtype == THERIA_F32   ? run(Tc<__nv_bfloat16, float>{})
         : dtype == THERIA_F16 ? run(Tc<__half, __half>{})
                               : run(Tc<__nv_bfloat16, __nv_bfloat16>{});
}

}  // extern "C"
