"""Language-model operators around the attention: what stands before, between
and after the blocks of a pre-LN decoder.

    embedding(ids, weight, scale)                 scale * weight[ids]
    layer_norm(x, weight, bias)                   over the last axis, any width
    linear_cross_entropy(hidden, weight, target)  cross entropy of hidden @ weight.T

Each runs hand-written kernels of libtheria_sm100.so (``include/theria_lm.h``)
on float32, float16 and bfloat16 CUDA tensors, on torch's current stream, and
each has its gradient.  Sums, softmax statistics and weight gradients are
float32 whatever the type, every result is rounded once, and the same inputs
give the same bits: no result depends on the order of atomics.  There is no
CPU path.

A token id or target outside the vocabulary is found on the device, where it
cannot raise: it counts as a row of zeros (an ignored row in the loss), and
``theria_b200.check_device_error()`` then raises.

There is no forward mode: a tensor that carries a tangent is refused with
NotImplementedError, as an input or as a gradient that arrives.

The reference library has no such operators; its decoder example composes them
from torch modules (``examples/minimal_decoder_transformer.py:82-263``).
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from theria_b200 import _lib

IGNORE_INDEX = -100
EPS = 1e-5
_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_opaque = torch.compiler.disable


_fns = {}


def _ptr(t):
    return None if t is None else t.data_ptr()


def _fn(name):
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(_lib.load(), name)
    return fn


def _call(name, device, *args):
    """One library call on `device` and torch's current stream there."""
    i = device.index
    if i == torch.cuda.current_device():
        st = _fn(name)(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(device):
            st = _fn(name)(*args, torch._C._cuda_getCurrentRawStream(i))
    if st:
        _lib.check(st, name)


def _workspace(name, device, *sizes):
    n = _fn(name)(*sizes)
    return torch.empty(n, dtype=torch.uint8, device=device), n


def _check(what, name, t, device=None):
    if not t.is_cuda:
        raise AssertionError(f"{what} requires CUDA tensors")
    if t.dtype not in _DTYPES:
        raise AssertionError(f"Unsupported dtype for {name}: {t.dtype}")
    if device is not None and t.device != device:
        raise AssertionError(f"{what}: {name} is on {t.device}, not {device}")


def _check_ids(what, name, ids, device):
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        raise AssertionError(f"{what}: {name} must be int64 or int32, got {ids.dtype}")
    if ids.device != device:
        raise AssertionError(f"{what}: {name} is on {ids.device}, not {device}")


def _no_tangents(what, *tensors):
    """Forward mode is refused: a tangent left out would read as a derivative of 0."""
    if forward_ad._current_level < 0:  # no tensor carries one (looking at each costs 0.3 us)
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} has no forward mode derivative")


def _wide(ids):
    return int(ids.dtype == torch.int64)


# Each operator's backward is a Function of its own, entered only while a graph
# of the gradients is being made (create_graph=True), so that a second
# derivative is either right or refused, never silently cut.

# ------------------------------------------------------------------ embedding
def _embed(ids, weight, scale, zero_idx):
    V, D = weight.shape
    out = torch.empty((*ids.shape, D), dtype=weight.dtype, device=weight.device)
    _call("theria_embed_fwd", weight.device, ids.data_ptr(), _wide(ids), weight.data_ptr(),
          out.data_ptr(), ids.numel(), V, D, _DTYPES[weight.dtype], scale, zero_idx)
    return out


def _embed_grad(gy, ids, V, scale, padding):
    gy = gy.contiguous()
    D, n = gy.shape[-1], ids.numel()
    gw = torch.empty(V, D, dtype=gy.dtype, device=gy.device)
    ws, size = _workspace("theria_embed_bwd_workspace_bytes", gy.device, n, V, D)
    _call("theria_embed_bwd", gy.device, ids.data_ptr(), _wide(ids), gy.data_ptr(), gw.data_ptr(),
          ws.data_ptr(), size, n, V, D, _DTYPES[gy.dtype], scale, padding)
    return gw


class _EmbeddingBackward(torch.autograd.Function):
    """gy -> gw, linear: its backward is the lookup of the cotangent's rows
    (zeros at the padding tokens, which gw leaves out)."""

    @staticmethod
    def forward(ctx, gy, ids, V, scale, padding):
        ctx.save_for_backward(ids)
        ctx.scale, ctx.padding = scale, padding
        return _embed_grad(gy, ids, V, scale, padding)

    @staticmethod
    @once_differentiable
    def backward(ctx, u):
        _no_tangents("theria embedding", u)
        (ids,) = ctx.saved_tensors
        return _embed(ids, u.contiguous(), ctx.scale, ctx.padding), None, None, None, None


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding):
        ctx.save_for_backward(ids)
        ctx.V, ctx.scale, ctx.padding = weight.shape[0], scale, padding
        return _embed(ids, weight, scale, -1)

    @staticmethod
    def backward(ctx, gy):
        _no_tangents("theria embedding", gy)
        (ids,) = ctx.saved_tensors
        grad = _EmbeddingBackward.apply if torch.is_grad_enabled() else _embed_grad
        return grad(gy, ids, ctx.V, ctx.scale, ctx.padding), None, None, None


@_opaque
def embedding(ids, weight, scale=1.0, padding_idx=None):
    """``scale * weight[ids]`` for ids of any shape (int64 or int32), weight
    [V, D]; differentiable twice in weight.

    The weight's gradient (dense) sums each token's rows in token order; the
    row ``padding_idx`` (negative: from the end) gets none.
    """
    _check("theria embedding", "weight", weight)
    _check_ids("theria embedding", "ids", ids, weight.device)
    if weight.ndim != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise AssertionError("weight must have shape (V,D)")
    _no_tangents("theria embedding", weight)
    V = weight.shape[0]
    padding = -1
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise AssertionError(f"padding_idx must be within the {V} rows of weight")
        padding = padding_idx % V
    ids, weight, scale = ids.contiguous(), weight.contiguous(), float(scale)
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embedding.apply(weight, ids, scale, padding)
    return _embed(ids, weight, scale, -1)


# ----------------------------------------------------------------- layer norm
def _norm(x, w, b, eps, need_stats):
    D = x.shape[-1]
    N = x.numel() // D
    y = torch.empty_like(x)
    stats = torch.empty(N, 4, dtype=torch.float32, device=x.device) if need_stats else None
    _call("theria_norm_fwd", x.device, x.data_ptr(), _ptr(w), _ptr(b), _affine_dtype(x, w, b),
          y.data_ptr(), _ptr(stats), N, D, _DTYPES[x.dtype], eps)
    return y, stats


def _affine_dtype(x, w, b):
    return _DTYPES[(w if w is not None else b if b is not None else x).dtype]


def _norm_grad(x, w, b, stats, gy, need):
    gy = gy.contiguous()
    D = x.shape[-1]
    N = x.numel() // D
    gx = torch.empty_like(x) if need[0] else None
    gw = gb = ws = None
    size = 0
    if need[1] or need[2]:
        like = w if w is not None else b
        gw, gb = torch.empty_like(like), torch.empty_like(like)
        ws, size = _workspace("theria_norm_bwd_workspace_bytes", x.device, N, D)
    _call("theria_norm_bwd", x.device, x.data_ptr(), _ptr(w), _affine_dtype(x, w, b),
          gy.data_ptr(), stats.data_ptr(), _ptr(gx), _ptr(gw), _ptr(gb), _ptr(ws), size, N, D,
          _DTYPES[x.dtype])
    return gx, gw if need[1] else None, gb if need[2] else None


def _norm_grad2(x, w, b, gy, stats, u, a, c):
    D = x.shape[-1]
    N = x.numel() // D
    u, a, c = (None if t is None else t.contiguous() for t in (u, a, c))
    dx, dgy = torch.empty_like(x), torch.empty_like(x)
    dw = None if w is None else torch.empty_like(w)
    ws, size = _workspace("theria_norm_bwd_workspace_bytes", x.device, N, D)
    _call("theria_norm_bwd2", x.device, x.data_ptr(), _ptr(w), _affine_dtype(x, w, b),
          gy.data_ptr(), stats.data_ptr(), _ptr(u), _ptr(a), _ptr(c), dx.data_ptr(),
          _ptr(dw), dgy.data_ptr(), ws.data_ptr(), size, N, D, _DTYPES[x.dtype])
    return dx, dw, dgy


class _LayerNormBackward2(torch.autograd.Function):
    """Cotangents of the backward -> (dx, dw, dgy); a third derivative is refused
    (once_differentiable would cut it off where no cotangent needs a gradient)."""

    @staticmethod
    def forward(ctx, *args):
        return _norm_grad2(*args)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("theria layer_norm is differentiable twice: its second derivatives "
                           "have no derivative here")


class _LayerNormBackward(torch.autograd.Function):
    """(x, w, gy) -> (gx, gw, gb); its backward is the second derivative.
    The statistics are functions of x, differentiated through there."""

    @staticmethod
    def forward(ctx, x, w, b, gy, stats, need):
        gy = gy.contiguous()
        ctx.save_for_backward(x, w, b, gy, stats)
        return _norm_grad(x, w, b, stats, gy, need)

    @staticmethod
    def backward(ctx, u, a, c):
        _no_tangents("theria layer_norm", u, a, c)
        grad = _LayerNormBackward2.apply if torch.is_grad_enabled() else _norm_grad2
        dx, dw, dgy = grad(*ctx.saved_tensors, u, a, c)
        return dx, dw, None, dgy, None, None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps):
        y, stats = _norm(x, w, b, eps, True)
        ctx.save_for_backward(x, w, b, stats)
        return y

    @staticmethod
    def backward(ctx, gy):
        _no_tangents("theria layer_norm", gy)
        x, w, b, stats = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        if torch.is_grad_enabled():
            grads = _LayerNormBackward.apply(x, w, b, gy, stats, need)
        else:
            grads = _norm_grad(x, w, b, stats, gy, need)
        return (*grads, None)


@_opaque
def layer_norm(x, weight=None, bias=None, eps=EPS):
    """Layer norm over the last axis of x [..., D]; weight, bias [D] (either
    may be None) of x's type or float32.  Differentiable twice."""
    what = "theria layer_norm"
    _check(what, "x", x)
    if x.ndim == 0 or x.shape[-1] == 0:
        raise AssertionError("x must have shape (...,D)")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _check(what, name, t, x.device)
        if t.ndim != 1 or t.shape[0] != x.shape[-1]:
            raise AssertionError(f"{name} must have shape ({x.shape[-1]},)")
        if t.dtype is not x.dtype and t.dtype is not torch.float32:
            raise AssertionError(f"{name} dtype must be {x.dtype} or float32")
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise AssertionError("weight and bias must share one dtype")
    _no_tangents(what, x, weight, bias)
    x = x.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad
                                    or weight is not None and weight.requires_grad
                                    or bias is not None and bias.requires_grad):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _norm(x, weight, bias, float(eps), False)[0]


# ------------------------------------------------------- linear cross entropy
def _loss(h, w, target, ignore_index, reduction):
    V, D = w.shape
    N, dt, dev = target.numel(), _DTYPES[h.dtype], h.device
    loss = torch.empty(target.shape if reduction == 0 else (), dtype=torch.float32, device=dev)
    stats = torch.empty(3 * N + 1, dtype=torch.float32, device=dev)  # lse [3, N], count
    ws, size = _workspace("theria_xent_fwd_workspace_bytes", dev, N, V, D, dt)
    lse = stats.data_ptr()
    _call("theria_xent_fwd", dev, h.data_ptr(), w.data_ptr(), target.data_ptr(), _wide(target),
          ignore_index, reduction, loss.data_ptr(), lse, lse + 12 * N, ws.data_ptr(), size, N, V,
          D, dt)
    return loss, stats


def _loss_grad(h, w, g, target, stats, ignore_index, reduction, need):
    V, D = w.shape
    N, dt, dev = target.numel(), _DTYPES[h.dtype], h.device
    g = g.to(torch.float32).contiguous()
    dh = torch.empty_like(h) if need[0] else None
    dw = torch.empty_like(w) if need[1] else None
    ws, size = _workspace("theria_xent_bwd_workspace_bytes", dev, N, V, D, dt)
    lse = stats.data_ptr()
    _call("theria_xent_bwd", dev, h.data_ptr(), w.data_ptr(), target.data_ptr(), _wide(target),
          ignore_index, reduction, g.data_ptr(), lse, lse + 12 * N, _ptr(dh), _ptr(dw),
          ws.data_ptr(), size, N, V, D, dt)
    return dh, dw


class _LinearCrossEntropyBackward(torch.autograd.Function):
    """(h, w, g) -> (dh, dw); a second derivative is refused."""

    @staticmethod
    def forward(ctx, h, w, g, *rest):
        return _loss_grad(h, w, g, *rest)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("theria linear_cross_entropy is differentiable once: its gradients "
                           "have no second derivative here")


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, target, ignore_index, reduction):
        loss, stats = _loss(h, w, target, ignore_index, reduction)
        ctx.save_for_backward(h, w, target, stats)
        ctx.rest = ignore_index, reduction
        return loss

    @staticmethod
    def backward(ctx, g):
        _no_tangents("theria linear_cross_entropy", g)
        h, w, target, stats = ctx.saved_tensors
        grad = _LinearCrossEntropyBackward.apply if torch.is_grad_enabled() else _loss_grad
        dh, dw = grad(h, w, g, target, stats, *ctx.rest, ctx.needs_input_grad[:2])
        return dh, dw, None, None, None


def _aligned(t):
    # the tensor-core kernels read 16 bytes at a time
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


@_opaque
def linear_cross_entropy(hidden, weight, target, ignore_index=IGNORE_INDEX, reduction="mean"):
    """Softmax cross entropy of the scores ``hidden @ weight.T`` without
    keeping them: hidden [..., D], weight [V, D] of one type, target [...]
    (int64 or int32).  Differentiable once, in hidden and weight.

    Rows whose target is ``ignore_index`` are left out: loss 0, no gradient,
    and nothing that their hidden states hold reaches a result.  The loss is
    float32: one per row for ``reduction="none"`` (target's shape), else a
    scalar; the mean over no row at all is NaN, with zero gradients.
    """
    what = "theria linear_cross_entropy"
    _check(what, "hidden", hidden)
    _check(what, "weight", weight, hidden.device)
    _check_ids(what, "target", target, hidden.device)
    if weight.dtype != hidden.dtype:
        raise AssertionError("hidden and weight must share one dtype")
    if weight.ndim != 2 or 0 in weight.shape:
        raise AssertionError("weight must have shape (V,D)")
    if hidden.ndim == 0 or hidden.shape[-1] != weight.shape[1]:
        raise AssertionError("hidden must have shape (...,D) with D matching weight")
    if target.shape != hidden.shape[:-1]:
        raise AssertionError(f"target shape must be {tuple(hidden.shape[:-1])}")
    if reduction not in _REDUCTIONS:
        raise AssertionError(f"reduction must be one of {sorted(_REDUCTIONS)}")
    _no_tangents(what, hidden, weight)
    h, w, t = hidden.contiguous(), _aligned(weight), target.contiguous()
    if torch.is_grad_enabled() and (h.requires_grad or w.requires_grad):
        return _LinearCrossEntropy.apply(h, w, t, int(ignore_index), _REDUCTIONS[reduction])
    return _loss(h, w, t, int(ignore_index), _REDUCTIONS[reduction])[0]


__all__ = ["embedding", "layer_norm", "linear_cross_entropy"]
