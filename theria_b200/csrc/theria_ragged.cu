// The attention over packed sequences of include/theria_ragged.h: argument
// checks, workspace carving and kernel selection.
#include <algorithm>

#include "common.cuh"
#include "ragged_plan.cuh"
#include "ragged_simt.cuh"
#include "ragged_tc_bwd.cuh"
#include "ragged_tc_fwd.cuh"
#include "tc_host.cuh"
#include "../../include/theria_ragged.h"

namespace theria {

// This translation unit's copy of the device error word, for
// theria_get_device_error / theria_clear_device_error.
int ragged_read_device_error(int* out, cudaStream_t st) {
  return cudaMemcpyFromSymbolAsync(out, g_device_error, sizeof(int), 0, cudaMemcpyDeviceToHost,
                                   st) == cudaSuccess
             ? THERIA_OK
             : THERIA_ERR_LAUNCH;
}
int ragged_clear_device_error(cudaStream_t st) {
  static const int zero = 0;
  return cudaMemcpyToSymbolAsync(g_device_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice,
                                 st) == cudaSuccess
             ? THERIA_OK
             : THERIA_ERR_LAUNCH;
}

namespace ragged {
namespace {

constexpr int kSMs = 148;
constexpr int kBlankBlocks = 32;  // CTAs that zero the rows of no sequence

int64_t up(int64_t x) { return (x + 255) / 256 * 256; }
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Carver {
  char* base;
  int64_t used = 0;
  template <typename T>
  T* take(int64_t count) {
    T* p = reinterpret_cast<T*>(base + used);
    used += up(count * (int64_t)sizeof(T));
    return p;
  }
};

// The most tiles of `step` rows that T tokens of `per` rows in S sequences make.
int64_t most_items(int64_t T, int64_t S, int64_t per, int64_t step) {
  return T * per / step + std::min(S, T);
}
List take_list(Carver& c, const Problem& p, int per, int step, int by_key) {
  List l{};
  l.per = per;
  l.step = step;
  l.by_key = by_key;
  l.items = c.take<int4>(most_items(p.T, p.S, per, step));
  l.count = c.take<int>(1);
  l.base = c.take<int>(p.S);
  return l;
}

int check(const Problem& p, int64_t T, int64_t S, int64_t H, int64_t Hkv, int64_t D, int dtype) {
  if (T < 0 || S < 0 || H <= 0 || Hkv <= 0 || D <= 0 || H % Hkv) return THERIA_ERR_INVALID_ARG;
  // (the maximum of the scores is taken before the factor)
  if (!(p.scale > 0.f) || !(p.scale_log2 < INFINITY)) return THERIA_ERR_INVALID_ARG;
  if (dtype != THERIA_F32 && dtype != THERIA_F16 && dtype != THERIA_BF16)
    return THERIA_ERR_INVALID_ARG;
  if (D > THERIA_MAX_HEAD_DIM || T >= (1ll << 30) || S >= (1ll << 30) || H >= 65536 ||
      T * H >= (1ll << 31))
    return THERIA_ERR_UNSUPPORTED;
  return THERIA_OK;
}

Problem problem(const int64_t* st, int64_t T, int64_t S, int64_t H, int64_t Hkv, int64_t D,
                float scale, int causal) {
  Problem p{};
  p.T = (int)T;
  p.S = (int)S;
  p.H = (int)H;
  p.Hkv = (int)Hkv;
  p.G = Hkv > 0 ? (int)(H / Hkv) : 0;
  p.D = (int)D;
  p.by_H = divisor(p.H);
  p.by_Hkv = divisor(p.Hkv);
  p.by_G = divisor(p.G);
  if (st != nullptr) {
    p.q_t = st[0];
    p.q_h = st[1];
    p.k_t = st[2];
    p.k_h = st[3];
    p.v_t = st[4];
    p.v_h = st[5];
    // strides that no address uses: as if contiguous, so that they rule no kernel out
    if (T == 1) {
      p.q_t = H * D;
      p.k_t = p.v_t = Hkv * D;
    }
    if (H == 1) p.q_h = D;
    if (Hkv == 1) p.k_h = p.v_h = D;
  }
  p.scale = scale;
  p.scale_log2 = scale * kLog2e;
  p.causal = causal != 0;
  return p;
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == THERIA_F32) return f(float{});
  if (dtype == THERIA_F16) return f(__half{});
  return f(__nv_bfloat16{});
}
// Calls f(DT, ASYNC): the kernels' width, and whether rows come by cp.async.
template <typename T, typename F>
int by_width(int D, bool async, F f) {
  using No = std::false_type;
  auto go = [&](auto w) {
    if constexpr (std::is_same<T, float>::value)
      if (async) return f(w, std::true_type{});
    return f(w, No{});
  };
  if constexpr (std::is_same<T, float>::value) {
    if (D <= 16) return go(std::integral_constant<int, 16>{});
    if (D <= 32) return go(std::integral_constant<int, 32>{});
  }
  if (D <= 64) return go(std::integral_constant<int, 64>{});
  if constexpr (std::is_same<T, float>::value)
    if (D <= 96) return go(std::integral_constant<int, 96>{});
  return go(std::integral_constant<int, 128>{});
}
// Whether the rows are whole 16-byte vectors on such boundaries.
bool whole_rows(int dtype, const Problem& p, std::initializer_list<const void*> ptrs) {
  const int64_t vec = 16 / elem_size(dtype);
  bool ok = p.D % vec == 0;
  for (const void* x : ptrs) ok = ok && tc::aligned16(x);
  for (int64_t s : {p.q_t, p.q_h, p.k_t, p.k_h, p.v_t, p.v_h}) ok = ok && s % vec == 0;
  return ok;
}

int run_plan(const void* offsets, int wide, const Problem& p, const List& a, const List& b,
             const Blank& blank, cudaStream_t st) {
  plan_kernel<<<2 + kBlankBlocks, kPlanThreads, 0, st>>>(offsets, wide, p.S, p.T, p.causal, a, b,
                                                         blank);
  return launch_status();
}

// Parts that the walk of a tile is split into, of `tiles` in an even batch: until they
// would fill the GPU `waves` times, and no more than 32.
int parts_of(int64_t tiles, int waves) {
  const int64_t parts = waves * kSMs / std::max<int64_t>(1, tiles);
  return (int)std::min<int64_t>(32, std::max<int64_t>(1, parts));
}
// dk, dv on the tensor cores: two waves (their tiles are few where the keys have few
// heads).  On the CUDA cores, whose tiles take longer, three, for dq too (2395 tokens, 5
// heads of 72 on one: dq 137 us and 6 to join, unsplit 229, the longest tile's own time).
int tc_splits(const Problem& p) { return parts_of(cdiv(p.T, BX) * p.Hkv, 2); }
int simt_splits(const Problem& p) { return parts_of(cdiv(p.T, SR) * p.Hkv, 3); }
int simt_q_splits(const Problem& p) {
  return parts_of(cdiv((int64_t)p.T * p.G, SR) * p.Hkv, 3);
}

// Lists have room for the CUDA-core kernels' tiles of 32 or 64 packed rows; the
// tensor-core kernels' are larger, hence fewer (128 / G, rounded down, is at
// least 64 / G).
void retile(List& l, int per, int step) {
  l.per = per;
  l.step = step;
}

struct FwdWs {
  List list;
  int64_t bytes;
};
FwdWs fwd_ws(void* base, const Problem& p) {
  Carver c{(char*)base};
  FwdWs w{};
  w.list = take_list(c, p, p.G, FR, 0);
  w.bytes = c.used;
  return w;
}

struct BwdWs {
  List lq, lk;
  float2* terms;
  uint8_t* fits;  // [Hkv, T, G] and [Hkv, T], float16 on the tensor cores
  float* part;  // room for the larger tiles' splits
  int64_t bytes;
};
BwdWs bwd_ws(void* base, const Problem& p) {
  Carver c{(char*)base};
  BwdWs w{};
  w.lq = take_list(c, p, p.G, SR, 0);
  w.lk = take_list(c, p, 1, SR, 1);
  w.terms = c.take<float2>((int64_t)p.T * p.H);
  w.fits = c.take<uint8_t>((int64_t)p.T * (p.H + p.Hkv));
  const int ks = std::max(tc_splits(p), simt_splits(p)), qs = simt_q_splits(p);
  const int64_t k_row = 2ll * p.Hkv * p.D, q_row = (int64_t)p.H * p.D;
  const int64_t part = std::max(ks > 1 ? ks * k_row : 0, qs > 1 ? qs * q_row : 0) * p.T;
  w.part = part > 0 ? c.take<float>(part) : nullptr;
  w.bytes = c.used;
  return w;
}

// Blocks: the key heads of a tile side by side.
bool grid_fits(const Problem& p) {
  return (most_items(p.T, p.S, p.G, FR) + 1) * p.Hkv < (1ll << 31);
}
unsigned blocks(const Problem& p, int per, int step) {
  return (unsigned)(std::max<int64_t>(1, most_items(p.T, p.S, per, step)) * p.Hkv);
}

template <typename T>
int simt_fwd(const void* q, const void* k, const void* v, void* o, void* rest, float* lse,
             const FwdWs& ws, const Problem& p, cudaStream_t st) {
  return by_width<T>(p.D, whole_rows(THERIA_F32, p, {q, k, v}), [&](auto w, auto async) {
    constexpr int DT = decltype(w)::value;
    auto kern = simt_fwd_kernel<T, DT, decltype(async)::value>;
    constexpr int smem = SimtSmem<DT>::kFwd;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
        cudaSuccess)
      return (int)THERIA_ERR_LAUNCH;
    return launch_chained(kern, dim3(blocks(p, p.G, FR)), dim3(SimtSmem<DT>::FG * FWD_THREADS),
                          smem, st, (const T*)q, (const T*)k, (const T*)v, (T*)o, (T*)rest, lse,
                          (const int4*)ws.list.items, (const int*)ws.list.count, p);
  });
}

template <typename T>
int run_join(const BwdWs& ws, int splits, const int* count, const void* offsets, int wide, void* a,
             void* b, int heads, const Problem& p, cudaStream_t st) {
  return launch_chained(join_kernel<T>, dim3(kSMs * 4), dim3(256), 0, st, (const float*)ws.part,
                        splits, count, offsets, wide, (T*)a, (T*)b, heads, p);
}

template <typename T>
int simt_bwd(const void* q, const void* k, const void* v, const void* dout, void* dq, void* dk,
             void* dv, const BwdWs& ws, const void* offsets, int wide, const Problem& p,
             cudaStream_t st) {
  return by_width<T>(p.D, whole_rows(THERIA_F32, p, {q, k, v, dout}), [&](auto w, auto async) {
    constexpr int DT = decltype(w)::value;
    constexpr bool ASYNC = decltype(async)::value;
    constexpr int smem = SimtSmem<DT>::kBwd;
    auto run = [&](auto kern, const List& l, int splits, void* o1, void* o2, float* part) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
          cudaSuccess)
        return (int)THERIA_ERR_LAUNCH;
      return launch_chained(kern, dim3(blocks(p, l.per, SR) * (unsigned)splits),
                            dim3(SimtSmem<DT>::SG * BWD_THREADS), smem, st, (const T*)q,
                            (const T*)k, (const T*)v, (const T*)dout, (const float2*)ws.terms,
                            (T*)o1, (T*)o2, part, (const int4*)l.items,
                            (const int*)l.count, splits, p);
    };
    if (dq != nullptr) {
      const int splits = simt_q_splits(p);
      if (int e = run(simt_bwd_kernel<T, DT, false, ASYNC>, ws.lq, splits, dq, nullptr,
                      splits > 1 ? ws.part : nullptr))
        return e;
      if (splits > 1)
        if (int e = run_join<T>(ws, splits, ws.lq.count, offsets, wide, dq, nullptr, p.H, p, st))
          return e;
    }
    if (dk == nullptr) return (int)THERIA_OK;
    const int splits = simt_splits(p);
    if (int e = run(simt_bwd_kernel<T, DT, true, ASYNC>, ws.lk, splits, dk, dv,
                    splits > 1 ? ws.part : nullptr))
      return e;
    return splits > 1 ? run_join<T>(ws, splits, ws.lk.count, offsets, wide, dk, dv, p.Hkv, p, st)
                      : (int)THERIA_OK;
  });
}

// ------------------------------------------------------ tensor-core launches
// Rows of 16 bytes on 16-byte boundaries, and a group that a tile of 64 rows
// holds.  Whatever the size, the CUDA-core kernels take longer (bf16; forward, dq, dk
// and dv, us, tensor cores first): one token, 8 / 2 heads of 64: 8, 6, 7 against 10, 9, 10;
// 25 x 64, 4 heads of 16: 8, 6, 16 against 24, 39, 38; 300 x 20, 8 / 2 heads of 64: 32, 25,
// 67 against 130, 108, 138; 2 x 2048, 16 / 4 heads of 64: 47, 45, 62 against 761, 954, 1749.
bool use_tc(int dtype, const Problem& p, std::initializer_list<const void*> ptrs) {
  if (dtype == THERIA_F32 || p.G > KY || tc::encode_fn() == nullptr) return false;
  if (!whole_rows(dtype, p, ptrs)) return false;
  for (int64_t s : {p.q_t, p.q_h, p.k_t, p.k_h, p.v_t, p.v_h})
    if (s <= 0 || s >= (1ll << 38)) return false;
  return true;
}

bool encode(CUtensorMap* m, const void* base, int dtype, int rank, const cuuint64_t* dims,
            const cuuint64_t* strides, const cuuint32_t* box) {
  const cuuint32_t one[4] = {1, 1, 1, 1};
  return tc::encode_fn()(m,
                         dtype == THERIA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                              : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         rank, const_cast<void*>(base), dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Keys or values [T, Hkv, D]: box {64 values, `rows` tokens, 1 head}.
bool key_map(CUtensorMap* m, const void* base, int dtype, const Problem& p, int64_t st, int64_t sh,
             int rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)p.D, (cuuint64_t)p.T, (cuuint64_t)p.Hkv};
  const cuuint64_t strides[2] = {(cuuint64_t)(2 * st), (cuuint64_t)(2 * sh)};
  const cuuint32_t box[3] = {64, (cuuint32_t)rows, 1};
  return encode(m, base, dtype, 3, dims, strides, box);
}
// Queries (or their gradients) [T, Hkv, G, D]: box {64 values, G heads, `tokens`, 1}.
bool row_map(CUtensorMap* m, const void* base, int dtype, const Problem& p, int64_t st, int64_t sh,
             int tokens) {
  const cuuint64_t dims[4] = {(cuuint64_t)p.D, (cuuint64_t)p.G, (cuuint64_t)p.T,
                              (cuuint64_t)p.Hkv};
  const cuuint64_t strides[3] = {(cuuint64_t)(2 * sh), (cuuint64_t)(2 * st),
                                 (cuuint64_t)(2 * sh * p.G)};
  const cuuint32_t box[4] = {64, (cuuint32_t)p.G, (cuuint32_t)tokens, 1};
  return encode(m, base, dtype, 4, dims, strides, box);
}

template <typename T, int HD, bool CAUSAL>
int tc_fwd(const void* q, const void* k, const void* v, void* o, void* rest, float* lse,
           const FwdWs& ws, int dtype, const Problem& p, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  if (!row_map(&mq, q, dtype, p, p.q_t, p.q_h, FM / p.G) ||
      !key_map(&mk, k, dtype, p, p.k_t, p.k_h, FN) || !key_map(&mv, v, dtype, p, p.v_t, p.v_h, FN))
    return THERIA_ERR_UNSUPPORTED;
  auto kern = tc_fwd_kernel<T, HD, CAUSAL>;
  constexpr int smem = FwdCfg<HD>::kAlloc;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return THERIA_ERR_LAUNCH;
  return launch_chained(kern, dim3(blocks(p, ws.list.per, ws.list.step)),
                        dim3(FwdCfg<HD>::kThreads), smem, st, mq, mk, mv, (T*)o, (T*)rest, lse,
                        (const int4*)ws.list.items, (const int*)ws.list.count, p);
}

template <typename T, int HD, bool CAUSAL>
int tc_bwd(const void* q, const void* k, const void* v, const void* dout, void* dq, void* dk,
           void* dv, const BwdWs& ws, const void* offsets, int wide, int dtype, const Problem& p,
           cudaStream_t st) {
  const int64_t o_t = (int64_t)p.H * p.D, o_h = p.D;
  auto prepare = [&](auto kern, int smem) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) ==
           cudaSuccess;
  };
  CUtensorMap mq, mo, mk, mv;
  if (dq != nullptr) {
    using Cfg = DqCfg<HD>;
    auto kern = tc_dq_kernel<T, HD, CAUSAL>;
    if (!row_map(&mq, q, dtype, p, p.q_t, p.q_h, BX / p.G) ||
        !row_map(&mo, dout, dtype, p, o_t, o_h, BX / p.G) ||
        !key_map(&mk, k, dtype, p, p.k_t, p.k_h, QY) ||
        !key_map(&mv, v, dtype, p, p.v_t, p.v_h, QY))
      return THERIA_ERR_UNSUPPORTED;
    if (!prepare(kern, Cfg::kAlloc)) return THERIA_ERR_LAUNCH;
    if (int e = launch_chained(kern, dim3(blocks(p, ws.lq.per, ws.lq.step)), dim3(Cfg::kThreads),
                               Cfg::kAlloc, st, mq, mo, mk, mv, (const float2*)ws.terms,
                               (const uint8_t*)ws.fits, (T*)dq,
                               (const int4*)ws.lq.items, (const int*)ws.lq.count, p))
      return e;
  }
  if (dk == nullptr) return THERIA_OK;
  using Cfg = DkvCfg<HD>;
  auto kern = tc_dkv_kernel<T, HD, CAUSAL>;
  if (!row_map(&mq, q, dtype, p, p.q_t, p.q_h, KY / p.G) ||
      !row_map(&mo, dout, dtype, p, o_t, o_h, KY / p.G) ||
      !key_map(&mk, k, dtype, p, p.k_t, p.k_h, BX) || !key_map(&mv, v, dtype, p, p.v_t, p.v_h, BX))
    return THERIA_ERR_UNSUPPORTED;
  if (!prepare(kern, Cfg::kAlloc)) return THERIA_ERR_LAUNCH;
  const int splits = tc_splits(p);
  if (int e = launch_chained(kern, dim3(blocks(p, ws.lk.per, ws.lk.step) * (unsigned)splits),
                             dim3(Cfg::kThreads), Cfg::kAlloc, st, mk, mv, mq, mo,
                             (const float2*)ws.terms, (const uint8_t*)ws.fits, (T*)dk, (T*)dv,
                             splits > 1 ? ws.part : nullptr, (const int4*)ws.lk.items,
                             (const int*)ws.lk.count, splits, p))
    return e;
  return splits > 1 ? run_join<T>(ws, splits, ws.lk.count, offsets, wide, dk, dv, p.Hkv, p, st)
                    : THERIA_OK;
}

// Calls f(HD, CAUSAL) as integral constants.
template <typename F>
int by_tile(const Problem& p, F f) {
  using W64 = std::integral_constant<int, 64>;
  using W128 = std::integral_constant<int, 128>;
  if (p.D <= 64)
    return p.causal ? f(W64{}, std::true_type{}) : f(W64{}, std::false_type{});
  return p.causal ? f(W128{}, std::true_type{}) : f(W128{}, std::false_type{});
}

template <typename T>
int run_terms(const void* o, const void* rest, const void* dout, const void* v,
              const float* lse, const BwdWs& ws, bool on_tc, const Problem& p, cudaStream_t st) {
  const int64_t rows = (int64_t)p.T * p.H;
  uint8_t* fits = on_tc && std::is_same<T, __half>::value ? ws.fits : nullptr;
  constexpr int VEC = 16 / sizeof(T);
  const bool vec = p.D % VEC == 0 && tc::aligned16(o) && tc::aligned16(rest) && tc::aligned16(dout);
  const int64_t units = vec ? p.D / VEC : p.D;  // a row's
  auto run = [&](auto kern, int lanes) {
    const int64_t need = cdiv(rows + (fits ? (int64_t)p.T * p.Hkv : 0), 256 / lanes);
    return launch_chained(kern, dim3((unsigned)std::min<int64_t>(need, kSMs * 32)), dim3(256), 0,
                          st, (const T*)o, (const T*)rest, (const T*)dout, lse, ws.terms,
                          (const T*)v, fits, rows, p);
  };
  if (!vec) return run(terms_kernel<T, 1, 32>, 32);
  if (units <= 4) return run(terms_kernel<T, VEC, 4>, 4);
  if (units <= 8) return run(terms_kernel<T, VEC, 8>, 8);
  return run(terms_kernel<T, VEC, 16>, 16);
}

}  // namespace
}  // namespace ragged
}  // namespace theria

using namespace theria;
using namespace theria::ragged;

extern "C" {

int64_t theria_ragged_fwd_workspace_bytes(int64_t T, int64_t S, int64_t H, int64_t Hkv) {
  const Problem p = problem(nullptr, T, S, H, Hkv, 1, 1.f, 0);
  if (check(p, T, S, H, Hkv, 1, THERIA_F32) != THERIA_OK) return 0;
  return fwd_ws(nullptr, p).bytes;
}

int theria_ragged_fwd(const void* q, const void* k, const void* v, const int64_t* strides,
                      const void* offsets, int wide, void* o, void* o_rest, float* lse,
                      void* workspace,
                      int64_t workspace_bytes, int64_t T, int64_t S, int64_t H, int64_t Hkv,
                      int64_t D, int dtype, float scale, int causal, void* stream) {
  const Problem p = problem(strides, T, S, H, Hkv, D, scale, causal);
  if (int e = check(p, T, S, H, Hkv, D, dtype)) return e;
  if (T == 0) return THERIA_OK;
  if (!q || !k || !v || !strides || !offsets || !o) return THERIA_ERR_INVALID_ARG;
  if (!workspace || workspace_bytes < theria_ragged_fwd_workspace_bytes(T, S, H, Hkv))
    return THERIA_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  FwdWs ws = fwd_ws(workspace, p);
  if (!grid_fits(p)) return THERIA_ERR_UNSUPPORTED;
  const bool on_tc = use_tc(dtype, p, {q, k, v, o, o_rest});
  if (on_tc) retile(ws.list, 1, 2 * (FM / p.G));
  Blank blank{};
  blank.p[0] = o;
  blank.row_bytes[0] = H * D * elem_size(dtype);
  if (int e = run_plan(offsets, wide, p, ws.list, List{}, blank, st)) return e;
  return by_type(dtype, [&](auto t) -> int {
    using E = decltype(t);
    if constexpr (!std::is_same<E, float>::value)
      if (on_tc)
        return by_tile(p, [&](auto hd, auto causal_) {
          return tc_fwd<E, decltype(hd)::value, decltype(causal_)::value>(
              q, k, v, o, o_rest, lse, ws, dtype, p, st);
        });
    return simt_fwd<E>(q, k, v, o, o_rest, lse, ws, p, st);
  });
}

int64_t theria_ragged_bwd_workspace_bytes(int64_t T, int64_t S, int64_t H, int64_t Hkv,
                                          int64_t D) {
  const Problem p = problem(nullptr, T, S, H, Hkv, D, 1.f, 0);
  if (check(p, T, S, H, Hkv, D, THERIA_F32) != THERIA_OK) return 0;
  return bwd_ws(nullptr, p).bytes;
}

int theria_ragged_bwd(const void* q, const void* k, const void* v, const int64_t* strides,
                      const void* offsets, int wide, const void* o, const void* o_rest,
                      const void* dout, const float* lse, void* dq, void* dk, void* dv,
                      void* workspace, int64_t workspace_bytes, int64_t T, int64_t S, int64_t H,
                      int64_t Hkv, int64_t D, int dtype, float scale, int causal, void* stream) {
  const Problem p = problem(strides, T, S, H, Hkv, D, scale, causal);
  if (int e = check(p, T, S, H, Hkv, D, dtype)) return e;
  if ((dk == nullptr) != (dv == nullptr)) return THERIA_ERR_INVALID_ARG;
  if (T == 0 || (dq == nullptr && dk == nullptr)) return THERIA_OK;
  if (!q || !k || !v || !strides || !offsets || !o || !dout || !lse)
    return THERIA_ERR_INVALID_ARG;
  if (!workspace || workspace_bytes < theria_ragged_bwd_workspace_bytes(T, S, H, Hkv, D))
    return THERIA_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  BwdWs ws = bwd_ws(workspace, p);
  if (!grid_fits(p)) return THERIA_ERR_UNSUPPORTED;
  const bool on_tc = use_tc(dtype, p, {q, k, v, dout, dq, dk, dv});
  if (on_tc) {
    retile(ws.lq, 1, BX / p.G);
    retile(ws.lk, 1, BX);
  }
  Blank blank{};
  blank.p[0] = dq;
  blank.p[1] = dk;
  blank.p[2] = dv;
  blank.row_bytes[0] = H * D * elem_size(dtype);
  blank.row_bytes[1] = blank.row_bytes[2] = Hkv * D * elem_size(dtype);
  if (int e = run_plan(offsets, wide, p, dq ? ws.lq : List{}, dk ? ws.lk : List{}, blank, st))
    return e;
  return by_type(dtype, [&](auto t) -> int {
    using E = decltype(t);
    if (int e = run_terms<E>(o, o_rest, dout, v, lse, ws, on_tc, p, st)) return e;
    if constexpr (!std::is_same<E, float>::value)
      if (on_tc)
        return by_tile(p, [&](auto hd, auto causal_) {
          return tc_bwd<E, decltype(hd)::value, decltype(causal_)::value>(
              q, k, v, dout, dq, dk, dv, ws, offsets, wide, dtype, p, st);
        });
    return simt_bwd<E>(q, k, v, dout, dq, dk, dv, ws, offsets, wide, p, st);
  });
}

}  // extern "C"
