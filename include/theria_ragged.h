/*
 * theria_ragged.h -- C ABI of the attention over packed sequences of different
 * lengths with grouped heads (libtheria_sm100.so).
 *
 * T tokens in one row hold S sequences one after the other: sequence s is the
 * tokens offsets[s] .. offsets[s+1] - 1 (int64 if `wide`, else int32; device
 * memory, S + 1 values), and may be empty.  Each token attends within its own
 * sequence, causally (to itself and the tokens before it) or to all of it:
 *
 *   o[i, h] = sum_j p_ij v[j, h / G],  p_i. = softmax over j of
 *             scale * q[i, h] . k[j, h / G],       G = H / Hkv
 *
 * q, o, dout, dq [T, H, D]; k, v, dk, dv [T, Hkv, D]; lse [T, H] float32, the
 * row logsumexp of the scaled scores.  o, dout and the gradients are
 * contiguous; q, k, v lie at strides[6] elements (host memory): between the
 * tokens and between the heads of q, of k, of v, with a head's D values side
 * by side.  Tokens before offsets[0] or from offsets[S] on belong to no
 * sequence: their o and gradients are zero (lse: not written), and nothing
 * that they, or another sequence, hold reaches a result.
 *
 * (T > 0:) offsets that decrease or leave 0 .. T cannot be refused by the host: every
 * result is then zero, and THERIA_ERR_INVALID_ARG is left in the device error
 * word (theria_get_device_error).
 *
 * Softmax statistics and sums are float32, and results are rounded once.  In
 * float16 and bfloat16 the probabilities p (forward and backward) and ds = p
 * (dp - z) (backward) are besides rounded to that type, as operands of the tensor
 * cores: o is off by 1.2 to 1.3 times its final rounding, dq, dk, dv by 1.4.
 * float16's short range: p loses bits below 2^-14; ds is made times a power of two
 * by the norms of dout's and v's rows, so that their sizes do not matter.  float32
 * uses the hardware's approximate 2^x, and float32 throughout.  No
 * result depends on the order in which thread blocks run.  Stream-ordered, no
 * allocation, no host synchronisation; each call returns a THERIA_* status.
 * scale > 0.  D <= THERIA_MAX_HEAD_DIM; T, S < 2^30, T * H < 2^31, H and Hkv < 65536.
 * With T == 0 nothing is launched, and the offsets are not looked at.
 *
 * The reference library has no such operator: its attention takes one head
 * count and one length (theria/attention/triton_qk.py:307-369).
 */
#ifndef THERIA_RAGGED_H
#define THERIA_RAGGED_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* o_rest [T, H, D] receives what o's rounding to its type left, for the backward's row
 * term dout . o, which cancels against other terms; it and lse may be NULL. */
int64_t theria_ragged_fwd_workspace_bytes(int64_t T, int64_t S, int64_t H, int64_t Hkv);
int theria_ragged_fwd(const void* q, const void* k, const void* v, const int64_t* strides,
                      const void* offsets, int wide, void* o, void* o_rest, float* lse,
                      void* workspace,
                      int64_t workspace_bytes, int64_t T, int64_t S, int64_t H, int64_t Hkv,
                      int64_t D, int dtype, float scale, int causal, void* stream);

/* dq, dk, dv of <o, dout>; dq, or dk and dv together, may be NULL, as may o_rest. */
int64_t theria_ragged_bwd_workspace_bytes(int64_t T, int64_t S, int64_t H, int64_t Hkv,
                                          int64_t D);
int theria_ragged_bwd(const void* q, const void* k, const void* v, const int64_t* strides,
                      const void* offsets, int wide, const void* o, const void* o_rest,
                      const void* dout, const float* lse, void* dq, void* dk, void* dv,
                      void* workspace, int64_t workspace_bytes, int64_t T, int64_t S, int64_t H,
                      int64_t Hkv, int64_t D, int dtype, float scale, int causal, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* THERIA_RAGGED_H */
