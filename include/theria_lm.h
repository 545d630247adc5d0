/*
 * theria_lm.h -- C ABI of the language-model operators around the attention
 * (libtheria_sm100.so): the scaled token embedding, the layer norm of any
 * width, and the linear layer to the vocabulary fused with its softmax cross
 * entropy, each with its gradient.
 *
 * Raw device pointers to contiguous row-major tensors, int64 sizes, dtype
 * codes THERIA_F32 / THERIA_F16 / THERIA_BF16 (theria_sdpa.h), cudaStream_t
 * as void*.  Stream-ordered, no allocation, no host synchronisation; each
 * call returns a THERIA_* status.  Sums and softmax statistics are float32
 * whatever the element type, results are rounded once, and no result depends
 * on the order in which thread blocks run.
 *
 * Token ids and targets are int64 (`wide` != 0) or int32.  One outside the
 * vocabulary cannot be refused by the host: it counts as a row of zeros (as
 * an ignored row in the loss), and THERIA_ERR_INVALID_ARG is left in the
 * device error word (theria_get_device_error).
 *
 * The reference library has no such operators; its decoder example composes
 * them from torch modules (examples/minimal_decoder_transformer.py:82-263).
 */
#ifndef THERIA_LM_H
#define THERIA_LM_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------- embedding
 * out[i] = scale * w[ids[i]] for ids [n], w [V, D], out [n, D]; a row whose
 * id is `zero_idx` (negative: none) is zero. */
int theria_embed_fwd(const void* ids, int wide, const void* w, void* out, int64_t n, int64_t V,
                     int64_t D, int dtype, float scale, int64_t zero_idx, void* stream);

/* gw[v] = scale * sum over i with ids[i] == v of gy[i], summed in the order
 * of i; rows of no token, and the row `zero_idx`, are zero.  The tokens are
 * sorted by id in a workspace of theria_embed_bwd_workspace_bytes(n, V, D)
 * bytes.  n < 2^30, V < 2^31 - 1, D <= 2^21 - 32 (both directions). */
int64_t theria_embed_bwd_workspace_bytes(int64_t n, int64_t V, int64_t D);
int theria_embed_bwd(const void* ids, int wide, const void* gy, void* gw, void* workspace,
                     int64_t workspace_bytes, int64_t n, int64_t V, int64_t D, int dtype,
                     float scale, int64_t zero_idx, void* stream);

/* ------------------------------------------------------------ layer norm
 * y = (x - mean) * rstd * w + b over rows of D values, rstd = (var +
 * eps)^-1/2; x, y [N, D] of `dtype`; w, b [D] of `wdtype` (`dtype` or
 * THERIA_F32), either may be NULL.  stats (may be NULL; 16-byte
 * aligned) receives [N, 4] float32: the row's mean, its reciprocal standard
 * deviation, what the mean's rounding to float32 left, and 0. */
int theria_norm_fwd(const void* x, const void* w, const void* b, int wdtype, void* y,
                    float* stats, int64_t N, int64_t D, int dtype, float eps, void* stream);

/* gx = rstd * P(gy * w), gw = sum_rows gy * xhat, gb = sum_rows gy, with
 * P(v) = v - mean(v) - xhat * mean(v * xhat).  gx, or gw and gb together,
 * may be NULL (not wanted). */
int64_t theria_norm_bwd_workspace_bytes(int64_t N, int64_t D);
int theria_norm_bwd(const void* x, const void* w, int wdtype, const void* gy,
                    const float* stats, void* gx, void* gw, void* gb, void* workspace,
                    int64_t workspace_bytes, int64_t N, int64_t D, int dtype, void* stream);

/* The backward's backward, for cotangents u of gx [N, D] (`dtype`), a of gw
 * and c of gb [D] (`wdtype`), each may be NULL (zero): dx, dgy [N, D], and
 * dw [D] (NULL: not wanted, and where w is).  Workspace as the backward's. */
int theria_norm_bwd2(const void* x, const void* w, int wdtype, const void* gy,
                     const float* stats, const void* u, const void* a, const void* c, void* dx,
                     void* dw, void* dgy, void* workspace, int64_t workspace_bytes, int64_t N,
                     int64_t D, int dtype, void* stream);

/* --------------------------------------------------- linear cross entropy
 * z = h w^T for h [N, D], w [V, D]; lse[i] = log sum_v exp z[i, v];
 * loss[i] = lse[i] - z[i, target[i]], 0 where target[i] == ignore_index.
 * The scores z are made in tiles and never stored.  A 16-bit w with D a
 * multiple of 8 has to start on a 16-byte boundary (else
 * THERIA_ERR_INVALID_ARG).  N, V < 2^30, D < 2^27.
 *   reduction THERIA_LOSS_NONE: loss [N]; _SUM, _MEAN: loss [1], the mean
 *   over the rows that count (NaN if there is none).
 * lse [3, N] and count [1] (the rows that count, float32) are what the backward
 * needs: the lse of each row, what its rounding to float32 left, and the row's
 * loss (of which the gradient of a nearly certain token, p - 1, is made); rows
 * that do not count leave 0. */
#define THERIA_LOSS_NONE 0
#define THERIA_LOSS_SUM 1
#define THERIA_LOSS_MEAN 2

int64_t theria_xent_fwd_workspace_bytes(int64_t N, int64_t V, int64_t D, int dtype);
int theria_xent_fwd(const void* h, const void* w, const void* target, int wide,
                    int64_t ignore_index, int reduction, float* loss, float* lse, float* count,
                    void* workspace, int64_t workspace_bytes, int64_t N, int64_t V, int64_t D,
                    int dtype, void* stream);

/* For the upstream gradient gloss (float32, [N] for THERIA_LOSS_NONE, else
 * [1]): dz[i, v] = c[i] (exp(z[i, v] - lse[i]) - [v == target[i]]) with c[i] =
 * gloss[i], gloss[0] or gloss[0] / count[0]; dh = dz w, dw = dz^T h.  dz is
 * made again in pieces of the vocabulary, held in the workspace.  dh or dw
 * may be NULL. */
int64_t theria_xent_bwd_workspace_bytes(int64_t N, int64_t V, int64_t D, int dtype);
int theria_xent_bwd(const void* h, const void* w, const void* target, int wide,
                    int64_t ignore_index, int reduction, const float* gloss, const float* lse,
                    const float* count, void* dh, void* dw, void* workspace,
                    int64_t workspace_bytes, int64_t N, int64_t V, int64_t D, int dtype,
                    void* stream);

#ifdef __cplusplus
}
#endif

#endif /* THERIA_LM_H */
