"""Attention over packed sequences of different lengths, with grouped heads.

``sdpa_ragged(q, k, v, offsets)``: q [T, H, D], k, v [T, Hkv, D] hold the
tokens of all sequences one after the other, sequence s being the rows
``offsets[s]`` to ``offsets[s + 1] - 1`` (offsets int32 or int64, on the
device; sequences may be empty).  Each query head h reads key head h // (H /
Hkv).  Nothing is padded and nothing is copied to the host: the kernels read
the offsets (``include/theria_ragged.h``).

Differentiable once, in q, k and v: a second derivative, and forward mode,
raise (the dense operators of this package have both).  The gradients use no
floating-point atomics, so the same inputs give the same bits.

The reference library has no such operator; its fused attention takes one head
count and one length (``theria/attention/triton_qk.py:307-369``).
"""

from __future__ import annotations

import ctypes
import math

import torch

from theria_b200 import _lib
from theria_b200.attention.ops import MAX_HEAD_DIM, default_scale
from theria_b200.lm import _DTYPES, _call, _check, _check_ids, _no_tangents, _ptr, _workspace

_opaque = torch.compiler.disable
_WHAT = "theria sdpa_ragged"
_Strides = ctypes.c_int64 * 6


def _check_args(q, k, v, offsets):
    device, dtype, shape, kv = q.device, q.dtype, tuple(q.shape), tuple(k.shape)
    _check(_WHAT, "q", q)
    _check(_WHAT, "k", k, device)
    _check(_WHAT, "v", v, device)
    if len(shape) != 3 or 0 in shape[1:]:
        raise AssertionError("q must have shape (T,H,D)")
    T, H, D = shape
    if len(kv) != 3 or kv[0] != T or kv[2] != D or kv[1] == 0 or H % kv[1]:
        raise AssertionError("k must have shape (T,Hkv,D) with Hkv a divisor of H")
    if tuple(v.shape) != kv:
        raise AssertionError("v must have shape (T,Hkv,D) as k")
    if k.dtype != dtype or v.dtype != dtype:
        raise AssertionError("q, k, v must share one dtype")
    if D > MAX_HEAD_DIM:
        raise AssertionError(f"theria_b200 supports D<={MAX_HEAD_DIM}")
    _check_ids(_WHAT, "offsets", offsets, device)
    if offsets.ndim != 1 or offsets.shape[0] == 0:
        raise AssertionError("offsets must have shape (S+1,)")


def _kernel_layout(t):
    """t itself where its heads lie as the kernels read them, else a copy: the
    values of a head side by side and, for the 16-bit tensor-core kernels, every
    row on a 16-byte boundary."""
    a, b, c = t.stride()
    if c != 1 or (a <= 0 and t.shape[0] > 1) or (b <= 0 and t.shape[1] > 1):
        return t.contiguous()
    if t.element_size() == 2 and (a % 8 or b % 8 or t.data_ptr() % 16):
        t = t.contiguous()
        return t if t.data_ptr() % 16 == 0 else t.clone()
    return t


def _strides(q, k, v):
    (a, b, _), (c, d, _), (e, f, _) = q.stride(), k.stride(), v.stride()
    return _Strides(a, b, c, d, e, f)


def _forward(q, k, v, offsets, causal, scale, grad):
    """o and, for the backward, the rows' logsumexp and what o's rounding left."""
    T, H, D = q.shape
    Hkv, S = k.shape[1], offsets.shape[0] - 1
    o = torch.empty(T, H, D, dtype=q.dtype, device=q.device)
    lse = torch.empty(T, H, dtype=torch.float32, device=q.device) if grad else None
    rest = torch.empty_like(o) if grad and q.element_size() == 2 else None
    ws, size = _workspace("theria_ragged_fwd_workspace_bytes", q.device, T, S, H, Hkv)
    _call("theria_ragged_fwd", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(),
          _strides(q, k, v), offsets.data_ptr(), int(offsets.dtype == torch.int64), o.data_ptr(),
          _ptr(rest), _ptr(lse), ws.data_ptr(), size, T, S, H, Hkv, D,
          _DTYPES[q.dtype], scale, causal)
    return o, rest, lse


def _backward(q, k, v, offsets, o, rest, lse, dout, causal, scale, need):
    T, H, D = q.shape
    Hkv, S = k.shape[1], offsets.shape[0] - 1
    dout = dout.contiguous()
    if dout.data_ptr() % 16:
        dout = dout.clone()
    dq = torch.empty(T, H, D, dtype=q.dtype, device=q.device) if need[0] else None
    dk = dv = None
    if need[1] or need[2]:
        dk, dv = (torch.empty(T, Hkv, D, dtype=q.dtype, device=q.device) for _ in range(2))
    ws, size = _workspace("theria_ragged_bwd_workspace_bytes", q.device, T, S, H, Hkv, D)
    _call("theria_ragged_bwd", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(),
          _strides(q, k, v), offsets.data_ptr(), int(offsets.dtype == torch.int64), o.data_ptr(),
          _ptr(rest), dout.data_ptr(), lse.data_ptr(), _ptr(dq), _ptr(dk), _ptr(dv),
          ws.data_ptr(), size, T, S, H, Hkv, D, _DTYPES[q.dtype], scale, causal)
    return dq, dk if need[1] else None, dv if need[2] else None


class _RaggedBackward(torch.autograd.Function):
    """(q, k, v, dout) -> (dq, dk, dv); a second derivative is refused."""

    @staticmethod
    def forward(ctx, q, k, v, dout, saved):
        offsets, o, rest, lse, *more = saved
        return _backward(q, k, v, offsets, o, rest, lse, dout, *more)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("theria sdpa_ragged is differentiable once: its gradients have no "
                           "second derivative here")


class _Ragged(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, causal, scale):
        o, rest, lse = _forward(q, k, v, offsets, causal, scale, True)
        ctx.save_for_backward(q, k, v, offsets, o, rest, lse)
        ctx.rest = causal, scale
        return o

    @staticmethod
    def backward(ctx, dout):
        _no_tangents(_WHAT, dout)
        q, k, v, offsets, o, rest, lse = ctx.saved_tensors
        causal, scale = ctx.rest
        need = ctx.needs_input_grad[:3]
        if torch.is_grad_enabled():
            grads = _RaggedBackward.apply(q, k, v, dout,
                                          (offsets, o, rest, lse, causal, scale, need))
        else:
            grads = _backward(q, k, v, offsets, o, rest, lse, dout, causal, scale, need)
        return (*grads, None, None, None)


@_opaque
def sdpa_ragged(q, k, v, offsets, causal=True, scale=None):
    """softmax(scale q k^T) v within each packed sequence (see the module).

    q [T, H, D]; k, v [T, Hkv, D], Hkv a divisor of H; float32, float16 or
    bfloat16, D <= 128; any strides (heads split out of a fused projection are
    read in place).  Returns o [T, H, D].  Rows of no sequence (before
    ``offsets[0]``, from ``offsets[-1]`` on) get zeros, and may hold anything,
    NaN included: no sequence is affected by what lies outside it.

    Offsets that decrease or leave 0..T are found on the device: o and the
    gradients are then zero, and ``theria_b200.check_device_error()`` raises
    (not with T = 0, where nothing is launched).

    Sums and softmax statistics are float32.  With 16-bit tensors the
    probabilities, and in the backward their gradients, are also rounded to 16
    bits as operands of the tensor cores: o is off by 1.2 to 1.3 times its own
    rounding, the gradients by 1.4.  A token that holds NaN or infinity may reach
    earlier tokens of its own sequence.
    """
    _check_args(q, k, v, offsets)
    _no_tangents(_WHAT, q, k, v)
    D = q.shape[2]
    scale = default_scale(q) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise AssertionError(f"scale must be positive and finite, got {scale}")
    causal = int(bool(causal))
    if q.element_size() == 2 and D % 8:
        # zero columns up to a whole number of 16-byte rows change no score and
        # add zero columns to o
        q, k, v = (torch.nn.functional.pad(t, (0, -D % 8)) for t in (q, k, v))
    q, k, v, offsets = _kernel_layout(q), _kernel_layout(k), _kernel_layout(v), offsets.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        o = _Ragged.apply(q, k, v, offsets, causal, scale)
    else:
        o = _forward(q, k, v, offsets, causal, scale, False)[0]
    return o if q.shape[2] == D else o[..., :D]


__all__ = ["sdpa_ragged"]
