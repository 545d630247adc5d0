"""Language-model operators around the attention: what stands before, between
and after the blocks of a pre-LN decoder, and at the end of its training step.

    embedding(ids, weight, scale)                 scale * weight[ids]
    layer_norm(x, weight, bias)                   over the last axis, any width
    linear_cross_entropy(hidden, weight, target)  cross entropy of hidden @ weight.T
    rotary(q, k, frequencies)                     rotary positions of queries and keys
    clip_gradients(tensors, max_norm)             by their global norm

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

import ctypes
import math

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
    if i == torch._C._cuda_getDevice():
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


# --------------------------------------------------------------------- rotary
SCALINGS = (None, "linear", "ntk", "by_parts")
_Strides12 = ctypes.c_int64 * 12


def rotary_frequencies(dim, base=10000.0, scaling=None, factor=1.0, original_length=None,
                       low=1.0, high=32.0, device="cuda"):
    """The angular frequencies ``base ** (-2 m / dim)`` of the dim / 2 pairs, float64,
    for ``rotary``; made once and kept, like a weight.

    ``scaling`` stretches them for contexts ``factor`` times as long as the
    model was trained on:

    - "linear": all frequencies divided by factor (positions interpolated);
    - "ntk": base times factor ** (dim / (dim - 2)), which divides the lowest
      frequency by factor and keeps the highest;
    - "by_parts": a pair that turns fewer than ``low`` times within
      ``original_length`` is divided by factor, one that turns more than ``high``
      times is kept, with a linear passage between them (its scores are usually
      also sharpened by ``rotary(..., amplitude=0.1 * log(factor) + 1)``).
    """
    if dim <= 0 or dim % 2:
        raise AssertionError(f"dim must be positive and even, got {dim}")
    if scaling not in SCALINGS:
        raise AssertionError(f"scaling must be one of {SCALINGS}")
    if not factor > 0 or not base > 0:
        raise AssertionError("base and factor must be positive")
    if scaling == "ntk" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    m = torch.arange(0, dim, 2, dtype=torch.float64)
    f = base ** (-m / dim)
    if scaling == "linear":
        f = f / factor
    if scaling == "by_parts":
        if original_length is None or original_length <= 0 or not high > low:
            raise AssertionError("by_parts needs original_length, and low < high")
        keep = ((original_length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
    return f.to(device)


def _rotary_layout(t):
    return t if t.stride(-1) == 1 else t.contiguous()


def _rotate(q, k, frequencies, positions, offsets, interleaved, amplitude, back):
    """Rotated q and k (each may be None)."""
    out, strides, pointers, heads = [None, None], [], [], []
    x = [None if t is None else _rotary_layout(t) for t in (q, k)]  # copies live to the launch
    for i, xi in enumerate(x):
        if xi is None:
            strides += (0, 0, 0, 0, 0, 0)
            pointers += (None, None)
            heads.append(0)
            continue
        y, a = torch.empty_like(xi), xi.stride()
        b, shape = y.stride(), xi.shape
        if b[-1] != 1:
            y = torch.empty(shape, dtype=xi.dtype, device=xi.device)
            b = y.stride()
        out[i], last = y, xi
        strides += (*a[:3], *b[:3]) if len(a) == 4 else (0, a[0], a[1], 0, b[0], b[1])
        pointers += (xi.data_ptr(), y.data_ptr())
        heads.append(shape[-2])
    at = positions if positions is not None else offsets
    _call("theria_rotary", last.device, pointers[0], pointers[2], pointers[1], pointers[3],
          _Strides12(*strides), shape[0] if len(shape) == 4 else 1, shape[-3], *heads,
          shape[-1], _DTYPES[last.dtype], _ptr(positions),
          0 if positions is None else positions.numel(), _ptr(offsets),
          0 if offsets is None else offsets.numel() - 1, 0 if at is None else _wide(at),
          frequencies.data_ptr(), frequencies.numel(), amplitude, interleaved, back)
    return tuple(out)


class _Rotary(torch.autograd.Function):
    """Linear in (q, k): its backward is itself with the angles negated."""

    @staticmethod
    def forward(ctx, q, k, frequencies, positions, offsets, *rest):
        ctx.save_for_backward(frequencies, positions, offsets)
        ctx.rest = rest
        ctx.set_materialize_grads(False)
        out = _rotate(q, k, frequencies, positions, offsets, *rest)
        ctx.mark_non_differentiable(*(y for y, need in zip(out, ctx.needs_input_grad)
                                      if y is not None and not need))
        return out

    @staticmethod
    def backward(ctx, gq, gk):
        what = "theria rotary"
        _no_tangents(what, gq, gk)
        if gq is None and gk is None:
            return (None,) * 8
        *rest, back = ctx.rest
        turn = _Rotary.apply if torch.is_grad_enabled() else _rotate
        gq, gk = turn(gq, gk, *ctx.saved_tensors, *rest, 1 - back)
        return gq, gk, None, None, None, None, None, None


@_opaque
def rotary(q, k, frequencies, positions=None, offsets=None, interleaved=False, amplitude=1.0):
    """Rotary positions: q [T, Hq, D] and k [T, Hk, D], or [B, T, H, D] each, any
    strides (heads-first tensors are passed as ``q.transpose(1, 2)``, and come back
    in the same order of memory); k may be None.  Returns the pair, or q alone.

    The pair m of each head's first ``2 * len(frequencies)`` values turns by
    ``position * frequencies[m]`` and is multiplied by ``amplitude``; the values
    behind pass through.  Pairs are (m, m + len(frequencies)), or with
    ``interleaved`` (2 m, 2 m + 1).  ``frequencies`` is float64 (see
    ``rotary_frequencies``); angles are reduced in float64, so positions may be far,
    and their cosines, sines and products are float32.

    Positions: ``positions`` (int64 or int32) [T] or [B, T]; or ``offsets`` [S + 1]
    of packed sequences, each counted from its first token (tokens of no sequence
    stand at 0); else 0 .. T - 1.  Differentiable in q and k, any number of times.
    """
    what, device, shape = "theria rotary", q.device, tuple(q.shape)
    _check(what, "q", q)
    if len(shape) not in (3, 4) or shape[-1] == 0:
        raise AssertionError("q must have shape (T,H,D) or (B,T,H,D)")
    tokens = shape[:-2]
    if k is not None:
        _check(what, "k", k, device)
        ks = tuple(k.shape)
        if len(ks) != len(shape) or ks[:-2] != tokens or ks[-1] != shape[-1]:
            raise AssertionError("k must have q's shape up to the number of heads")
        if k.dtype != q.dtype:
            raise AssertionError("q and k must share one dtype")
    if frequencies.dtype is not torch.float64 or frequencies.device != device:
        raise AssertionError("frequencies must be float64 on q's device")
    if frequencies.ndim != 1 or 2 * frequencies.numel() > shape[-1]:
        raise AssertionError("frequencies must have shape (pairs,) with 2 * pairs <= D")
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise AssertionError("theria rotary has no gradient for its frequencies")
    if positions is not None and offsets is not None:
        raise AssertionError("theria rotary takes positions or offsets, not both")
    for name, t in (("positions", positions), ("offsets", offsets)):
        if t is not None:
            _check_ids(what, name, t, device)
    if positions is not None and tuple(positions.shape) not in (tokens, tokens[-1:]):
        raise AssertionError(f"positions must have shape {tokens} or {tokens[-1:]}")
    if offsets is not None and (offsets.ndim != 1 or offsets.shape[0] == 0):
        raise AssertionError("offsets must have shape (S+1,)")
    _no_tangents(what, q, k)
    if q.numel() == 0 and (k is None or k.numel() == 0):
        out = torch.empty_like(q), None if k is None else torch.empty_like(k)
        return out if k is not None else out[0]
    positions = None if positions is None else positions.contiguous()
    offsets = None if offsets is None else offsets.contiguous()
    args = (q, k, frequencies.contiguous(), positions, offsets, int(bool(interleaved)),
            float(amplitude), 0)
    if torch.is_grad_enabled() and (q.requires_grad or k is not None and k.requires_grad):
        out = _Rotary.apply(*args)
    else:
        out = _rotate(*args)
    return out if k is not None else out[0]


# ------------------------------------------------------ gradient norm, clipping
def _grads_table(tensors):
    n = len(tensors)
    return ((ctypes.c_int64 * n)(*[t.numel() for t in tensors]),
            (ctypes.c_int * n)(*[_DTYPES[t.dtype] for t in tensors]))


def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def _grads_dot(x, u, sizes, dtypes, dev):
    parts = torch.empty(max(1, _fn("theria_grads_parts")(sizes, len(x))), dtype=torch.float64,
                        device=dev)
    _call("theria_grads_dot", dev, _pointers(x), None if u is None else _pointers(u), sizes,
          dtypes, len(x), parts.data_ptr())
    return parts


def _clip(x, out, max_norm):
    """norm [] of x, and its stats; out (None: not wanted) receives x clipped."""
    dev, (sizes, dtypes) = x[0].device, _grads_table(x)
    parts = _grads_dot(x, None, sizes, dtypes, dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    stats = torch.empty(2, dtype=torch.float64, device=dev)
    _call("theria_grads_clip", dev, _pointers(x), None if out is None else _pointers(out), sizes,
          dtypes, len(x), parts.data_ptr(), max_norm, norm.data_ptr(), stats.data_ptr())
    return norm, stats


def _clip_grad(x, u, gnorm, stats):
    dev, (sizes, dtypes) = x[0].device, _grads_table(x)
    parts = None
    if u is not None:
        u = [t.contiguous() for t in u]
        parts = _grads_dot(x, u, sizes, dtypes, dev)
    dx = [torch.empty_like(t) for t in x]
    gnorm = None if gnorm is None else gnorm.to(torch.float32).contiguous()
    _call("theria_grads_clip_bwd", dev, _pointers(x), None if u is None else _pointers(u),
          _pointers(dx), sizes, dtypes, len(x), _ptr(parts), stats.data_ptr(), _ptr(gnorm))
    return dx


class _ClipBackward(torch.autograd.Function):
    """(x, u, gnorm) -> dx; a second derivative is refused."""

    @staticmethod
    def forward(ctx, n, stats, gnorm, *xu):
        return tuple(_clip_grad(xu[:n], xu[n:] or None, gnorm, stats))

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("theria clip_gradients is differentiable once: its gradients have no "
                           "second derivative here")


class _Clip(torch.autograd.Function):
    """tensors -> (norm, *clipped); clip false: the norm alone."""

    @staticmethod
    def forward(ctx, max_norm, clip, *x):
        y = [torch.empty_like(t) for t in x] if clip else None
        norm, stats = _clip(x, y, max_norm)
        ctx.save_for_backward(stats, *x)
        ctx.set_materialize_grads(False)
        return (norm, *y) if clip else norm

    @staticmethod
    def backward(ctx, gnorm, *gy):
        _no_tangents("theria clip_gradients", gnorm, *gy)
        stats, *x = ctx.saved_tensors
        some = any(g is not None for g in gy)
        if not some and gnorm is None:
            return (None, None, *(None for _ in x))
        u = [torch.zeros_like(t) if g is None else g for t, g in zip(x, gy)] if some else []
        if torch.is_grad_enabled():
            dx = _ClipBackward.apply(len(x), stats, gnorm, *x, *u)
        else:
            dx = _clip_grad(x, u or None, gnorm, stats)
        return (None, None, *dx)


def _check_grads(what, tensors):
    tensors = list(tensors)
    if not tensors:
        raise AssertionError(f"{what} needs at least one tensor")
    for i, t in enumerate(tensors):
        _check(what, f"tensor {i}", t, tensors[0].device)
    _no_tangents(what, *tensors)
    return tensors


def _reach(dims):
    """How far behind the first address the last one lies."""
    return sum(s * (n - 1) for s, n in dims)


def _dims(t):
    """(stride, size) of t's addresses in bytes, its values' own bytes among them."""
    e = t.element_size()
    return [(s * e, n) for s, n in zip(t.stride(), t.shape) if n > 1] + [(1, e)]


def _folded(t):
    """Whether two indices of t may be one address (never missed; where strides
    interleave it may be said of a tensor without any)."""
    dims = sorted(_dims(t))
    return any(s <= _reach(dims[:i]) for i, (s, _) in enumerate(dims))


def _chains(sets):
    """The sets (address, dims) in runs whose ranges of addresses meet."""
    runs, end = [], None
    for one in sorted(sets, key=lambda s: s[0]):
        if end is None or one[0] > end:
            runs.append([])
            end = one[0]
        runs[-1].append(one)
        end = max(end, one[0] + _reach(one[1]))
    return runs


def _apart(sets):
    """Whether no two of the sets of addresses have one in common (never said where two
    do).  Written as m Q + R with R < m, for m one of the strides, two addresses differ
    where their Q or their R do: so slices of the same rows, of every second row, of
    single heads are found to be apart."""
    return all(len(run) == 1 or _run_apart(run) for run in _chains(sets))


def _run_apart(run):
    for m in sorted({s for _, dims in run for s, _ in dims if s > 1}, reverse=True):
        parts = []  # (R's first, R's dims, Q's set)
        for a, dims in run:
            a -= run[0][0]
            rest = [d for d in dims if d[0] % m]
            if a % m + _reach(rest) >= m:
                break
            parts.append((a % m, rest, (a // m, [(s // m, n) for s, n in dims if s % m == 0])))
        else:
            if all(len(r) == 1 or _apart([p[2] for p in r]) or _apart([p[:2] for p in r])
                   for r in _chains(parts)):
                return True
    return len(run) > 2 and all(_apart([x, y]) for i, x in enumerate(run) for y in run[:i])


def _overlap(tensors):
    """Whether two of the tensors may share an address."""
    some = [t for t in tensors if t.numel()]
    spans = []
    for t in some:
        at = t.data_ptr()
        spans.append((at, at + (t.nbytes if t.is_contiguous() else _reach(_dims(t)) + 1)))
    spans.sort()
    # (most calls end here: no two ranges meet)
    return (any(a[1] > b[0] for a, b in zip(spans, spans[1:]))
            and not _apart([(t.data_ptr(), [(1, t.nbytes)] if t.is_contiguous() else _dims(t))
                            for t in some]))


def _check_max(max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise AssertionError(f"max_norm must not be negative, got {max_norm}")
    return max_norm


@_opaque
def gradient_norm(tensors):
    """The 2-norm of all values of the tensors together (float32, on the device);
    differentiable once.  Any shapes and mixed types; sums are taken to float64, so
    very large and very small gradients neither overflow nor vanish."""
    x = [t.contiguous() for t in _check_grads("theria gradient_norm", tensors)]
    if torch.is_grad_enabled() and any(t.requires_grad for t in x):
        return _Clip.apply(0.0, False, *x)
    return _clip(x, None, 0.0)[0]


@_opaque
def clip_gradients(tensors, max_norm):
    """``([t * c for t in tensors], norm)`` with ``norm = gradient_norm(tensors)`` and
    ``c = min(1, max_norm / norm)``; differentiable once, so that clipped steps can be
    part of an adapted model.  A norm that is NaN makes every value NaN, an
    infinite one makes c 0 (1 where max_norm is infinite too)."""
    what = "theria clip_gradients"
    x = [t.contiguous() for t in _check_grads(what, tensors)]
    max_norm = _check_max(max_norm)
    if torch.is_grad_enabled() and any(t.requires_grad for t in x):
        norm, *y = _Clip.apply(max_norm, True, *x)
        return y, norm
    y = [torch.empty_like(t) for t in x]
    return y, _clip(x, y, max_norm)[0]


@_opaque
def clip_gradients_(tensors, max_norm):
    """clip_gradients in place; returns the norm.  No two tensors may overlap, none
    itself, and none may need a gradient (under ``torch.no_grad()`` they may).  Views of
    one tensor that share no value (columns, heads, every second row) are taken; such
    whose strides do not show it are refused."""
    what = "theria clip_gradients_"
    tensors = _check_grads(what, tensors)
    max_norm = _check_max(max_norm)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise AssertionError(f"{what} changes its tensors: none may require a gradient")
    x = [t.contiguous() for t in tensors]
    for t, c in zip(tensors, x):
        if t is not c and any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
            raise AssertionError(f"{what} changes its tensors: none may be an expanded view")
        if t is not c and _folded(t):
            raise AssertionError(f"{what} changes its tensors: none may overlap itself")
    if _overlap(tensors):
        raise AssertionError(f"{what} changes its tensors: no two may overlap")
    norm, _ = _clip(x, x, max_norm)
    for t, c in zip(tensors, x):
        if t is not c:
            t.copy_(c)
        elif not t.is_inference():
            torch.autograd.graph.increment_version(t)
    return norm


__all__ = ["embedding", "layer_norm", "linear_cross_entropy", "rotary", "rotary_frequencies",
           "gradient_norm", "clip_gradients", "clip_gradients_"]
