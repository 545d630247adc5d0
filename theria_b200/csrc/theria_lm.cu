// The language-model operators of include/theria_lm.h: argument checks,
// workspace carving and kernel selection.
#include <algorithm>

#include "common.cuh"
#include "lm_embed.cuh"
#include "lm_norm.cuh"
#include "lm_xent.cuh"
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
  uint32_t *keys[2], *vals[2], *hist, *start;
  float* part;
  int64_t bytes;
};
EmbedWs embed_ws(void* base, int64_t n, int64_t V, int64_t D) {
  Carver c{(char*)base};
  EmbedWs w;
  for (int k = 0; k < 2; ++k) {
    w.keys[k] = c.take<uint32_t>(n);
    w.vals[k] = c.take<uint32_t>(n);
  }
  w.hist = c.take<uint32_t>(cdiv(n, embed::TILE) * embed::BINS);
  w.start = c.take<uint32_t>(V + 1);
  w.part = c.take<float>(n / embed::CHUNK * D);
  w.bytes = c.used;
  return w;
}

int embed_check(int64_t n, int64_t V, int64_t D, int dtype) {
  if (n < 0 || V <= 0 || D <= 0 || !lm_dtype(dtype)) return THERIA_ERR_INVALID_ARG;
  if (n >= (1ll << 30) || V >= (1ll << 31) - 1) return THERIA_ERR_UNSUPPORTED;
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
  const unsigned tiles = (unsigned)cdiv(n, embed::TILE);
  int bits = 1;  // keys are 0 .. V
  while ((V >> bits) != 0) ++bits;
  const uint32_t *keys = nullptr, *vals = nullptr;
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
  embed::starts_kernel<<<(unsigned)std::min<int64_t>(cdiv(V + 1, 256), kSMs * 8), 256, 0, st>>>(
      keys, ws.start, n, V);
  if (int e = launch_status()) return e;
  const bool vec = vec_rows(D, dtype, {gy, gw});
  const int64_t chunks = n / embed::CHUNK;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int VEC = embed::Vec<T>::n;
    if (chunks > 0) {
      auto kern = vec ? embed::chunk_kernel<T, VEC> : embed::chunk_kernel<T, 1>;
      kern<<<(unsigned)std::min<int64_t>(chunks, kSMs * 16), 256, 0, st>>>(
          (const T*)gy, keys, vals, ws.part, chunks, V, D);
      if (int e = launch_status()) return e;
    }
    auto kern = vec ? embed::rows_kernel<T, VEC> : embed::rows_kernel<T, 1>;
    kern<<<(unsigned)std::min<int64_t>(V, kSMs * 32), 256, 0, st>>>(
        (const T*)gy, vals, ws.start, ws.part, (T*)gw, V, D, scale);
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
// values: a warp per row where a lane holds up to 8 values' worth of vectors,
// else a CTA of 8 warps per row; false where the row does not fit the
// registers (32 values a thread).
template <int VEC, typename F>
bool norm_shape(int64_t D, F f) {
  const int64_t units = cdiv(D, VEC);
  constexpr int A = VEC == 1 ? 4 : 1, B = VEC == 1 ? 16 : VEC == 4 ? 4 : 2,
                C = 32 / VEC;  // vectors per thread
  if (units <= 32 * A) f(std::integral_constant<int, A>{}, std::integral_constant<int, 1>{});
  else if (units <= 32 * B) f(std::integral_constant<int, B>{}, std::integral_constant<int, 1>{});
  else if (units <= 256 * A) f(std::integral_constant<int, A>{}, std::integral_constant<int, 8>{});
  else if (units <= 256 * C) f(std::integral_constant<int, C>{}, std::integral_constant<int, 8>{});
  else return false;
  return true;
}

int64_t norm_ctas(int64_t N) { return std::min<int64_t>(N, kSMs * 2); }

}  // namespace
}  // namespace theria

extern "C" {

int theria_norm_fwd(const void* x, const void* w, const void* b, int wdtype, void* y,
                    float* stats, int64_t N, int64_t D, int dtype, float eps, void* stream) {
  if (int e = norm_check(N, D, dtype, wdtype)) return e;
  if (N == 0) return THERIA_OK;
  if (!x || !y) return THERIA_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const bool vec = vec_rows(D, dtype, {x, y});
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto vecn) {
      constexpr int VEC = decltype(vecn)::value;
      return norm_shape<VEC>(D, [&](auto nv, auto nw) {
        constexpr int NV = decltype(nv)::value, NW = decltype(nw)::value;
        const int64_t rows = 8 / NW;
        norm::fwd_kernel<T, VEC, NV, NW>
            <<<(unsigned)std::min<int64_t>(cdiv(N, rows), kSMs * 32), 256, 0, st>>>(
                (const T*)x, w, b, wdtype, (T*)y, stats, N, (int)D, eps);
      });
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
  if (!x || !gy || !stats) return THERIA_ERR_INVALID_ARG;
  if (!gx && !gw) return THERIA_OK;
  if (gw && (!workspace || workspace_bytes < theria_norm_bwd_workspace_bytes(N, D)))
    return THERIA_ERR_WORKSPACE;
  const bool vec = vec_rows(D, dtype, {x, gy, gx});
  float* part = gw ? (float*)workspace : nullptr;
  int ctas = 0;
  int e = by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto vecn) {
      constexpr int VEC = decltype(vecn)::value;
      return norm_shape<VEC>(D, [&](auto nv, auto nw) {
        constexpr int NV = decltype(nv)::value, NW = decltype(nw)::value;
        const int64_t rows = 8 / NW;
        ctas = (int)std::min<int64_t>(cdiv(N, rows), norm_ctas(N));
        auto kern = norm::bwd_kernel<T, VEC, NV, NW>;
        const size_t smem = NW == 1 && part ? 8 * 2 * D * sizeof(float) : 0;
        if (smem > 48 * 1024)
          cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        kern<<<(unsigned)ctas, 256, smem, st>>>((const T*)x, w, wdtype, (const T*)gy, stats,
                                                (T*)gx, part, N, (int)D);
      });
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
  if (!x || !gy || !stats || !dx || !dgy || (dw && !w)) return THERIA_ERR_INVALID_ARG;
  if (!workspace || workspace_bytes < theria_norm_bwd_workspace_bytes(N, D))
    return THERIA_ERR_WORKSPACE;
  const bool vec = vec_rows(D, dtype, {x, gy, u, dx, dgy});
  float* part = (float*)workspace;
  int ctas = 0;
  int e = by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto vecn) {
      constexpr int VEC = decltype(vecn)::value;
      return norm_shape<VEC>(D, [&](auto nv, auto nw) {
        constexpr int NV = decltype(nv)::value, NW = decltype(nw)::value;
        ctas = (int)std::min<int64_t>(cdiv(N, 8 / NW), norm_ctas(N));
        auto kern = norm::bwd2_kernel<T, VEC, NV, NW>;
        const size_t smem = NW == 1 ? 8 * 2 * D * sizeof(float) : 0;
        if (smem > 48 * 1024)
          cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        kern<<<(unsigned)ctas, 256, smem, st>>>((const T*)x, w, wdtype, (const T*)gy, stats,
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
  if (N > 65535ll * xent::TM || V > 65535ll * xent::TN || D >= (1ll << 31))
    return THERIA_ERR_UNSUPPORTED;
  return THERIA_OK;
}

struct XentRows {  // filled by prep_kernel
  int *pos, *row_of, *tgt, *n_live;
};
XentRows xent_rows(Carver& c, int64_t N) {
  XentRows r;
  r.pos = c.take<int>(N);
  r.row_of = c.take<int>(N);
  r.tgt = c.take<int>(N);
  r.n_live = c.take<int>(1);
  return r;
}
struct XentFwdWs {
  XentRows rows;
  float2* part;
  float *zt, *each;
  int64_t bytes;
};
XentFwdWs xent_fwd_ws(void* base, int64_t N, int64_t V) {
  Carver c{(char*)base};
  XentFwdWs w;
  w.rows = xent_rows(c, N);
  w.part = c.take<float2>(N * cdiv(V, xent::TN));
  w.zt = c.take<float>(N);
  w.each = c.take<float>(N);
  w.bytes = c.used;
  return w;
}
struct XentBwdWs {
  XentRows rows;
  float *dz, *acc;
  int64_t piece, bytes;
};
XentBwdWs xent_bwd_ws(void* base, int64_t N, int64_t V, int64_t D) {
  Carver c{(char*)base};
  XentBwdWs w;
  w.rows = xent_rows(c, N);
  w.piece = std::min<int64_t>(up(V, xent::TN),
                              std::max<int64_t>(xent::TN, up((64ll << 20) / N, xent::TN)));
  w.dz = c.take<float>(N * w.piece);
  w.acc = c.take<float>(N * D);
  w.bytes = c.used;
  return w;
}

}  // namespace
}  // namespace theria

extern "C" {

int64_t theria_xent_fwd_workspace_bytes(int64_t N, int64_t V, int64_t D, int dtype) {
  return N <= 0 || V <= 0 || D <= 0 ? 0 : xent_fwd_ws(nullptr, N, V).bytes;
}
int64_t theria_xent_bwd_workspace_bytes(int64_t N, int64_t V, int64_t D, int dtype) {
  return N <= 0 || V <= 0 || D <= 0 ? 0 : xent_bwd_ws(nullptr, N, V, D).bytes;
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
  const XentFwdWs ws = xent_fwd_ws(workspace, N > 0 ? N : 1, V);
  float* each = reduction == THERIA_LOSS_NONE ? loss : ws.each;
  if (N == 0) {
    cudaMemsetAsync(count, 0, sizeof(float), st);
    if (reduction == THERIA_LOSS_NONE) return THERIA_OK;
  } else {
    const int tiles = (int)cdiv(V, xent::TN);
    xent::prep_kernel<<<1, 1024, 0, st>>>(target, wide, ignore_index, N, V, ws.rows.pos,
                                          ws.rows.row_of, ws.rows.tgt, ws.rows.n_live, count, each,
                                          lse);
    if (int e = launch_status()) return e;
    int e = by_type(dtype, [&](auto t) {
      using T = decltype(t);
      xent::score_kernel<T><<<dim3((unsigned)tiles, (unsigned)cdiv(N, xent::TM)), 256, 0, st>>>(
          (const T*)h, (const T*)w, ws.rows.row_of, ws.rows.tgt, ws.rows.n_live, ws.part, ws.zt, V,
          D);
      return launch_status();
    });
    if (e) return e;
    xent::join_kernel<<<(unsigned)std::min<int64_t>(cdiv(N, 8), kSMs * 8), 256, 0, st>>>(
        ws.part, ws.zt, ws.rows.row_of, ws.rows.n_live, tiles, each, lse);
    if (int e2 = launch_status()) return e2;
    if (reduction == THERIA_LOSS_NONE) return THERIA_OK;
  }
  xent::total_kernel<<<1, 1024, 0, st>>>(each, N, count, reduction == THERIA_LOSS_MEAN, loss);
  return launch_status();
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
  const XentBwdWs ws = xent_bwd_ws(workspace, N, V, D);
  const XentRows& r = ws.rows;
  xent::prep_kernel<<<1, 1024, 0, st>>>(target, wide, ignore_index, N, V, r.pos, r.row_of, r.tgt,
                                        r.n_live, nullptr, nullptr, nullptr);
  if (int e = launch_status()) return e;
  const unsigned mt = (unsigned)cdiv(N, xent::TM), dt = (unsigned)cdiv(D, xent::TN);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    for (int64_t c0 = 0; c0 < V; c0 += ws.piece) {
      const int64_t C = std::min(ws.piece, V - c0);
      const unsigned ct = (unsigned)cdiv(C, xent::TN);
      xent::dz_kernel<T><<<dim3(ct, mt), 256, 0, st>>>(
          (const T*)h, (const T*)w, r.row_of, r.tgt, r.n_live, lse, gloss,
          reduction == THERIA_LOSS_NONE, reduction == THERIA_LOSS_MEAN ? count : nullptr, ws.dz,
          c0, C, V, D);
      if (int e = launch_status()) return e;
      if (dh) {
        xent::dh_kernel<T><<<dim3(dt, mt), 256, 0, st>>>(ws.dz, (const T*)w, r.n_live, ws.acc, c0,
                                                         C, C, D, c0 == 0);
        if (int e = launch_status()) return e;
      }
      if (dw) {
        xent::dw_kernel<T><<<dim3(dt, ct), 256, 0, st>>>(ws.dz, (const T*)h, r.row_of, r.n_live,
                                                         (T*)dw, c0, C, C, D);
        if (int e = launch_status()) return e;
      }
    }
    if (dh) {
      xent::dh_finish_kernel<T><<<(unsigned)std::min<int64_t>(cdiv(N * D, 256), kSMs * 16), 256, 0,
                                  st>>>(ws.acc, r.pos, (T*)dh, N, D);
      return launch_status();
    }
    return THERIA_OK;
  });
}

}  // extern "C"
