"""Host-side checks of the attention over packed sequences, the rotary positions
and the gradient clipping: statuses for bad arguments before anything is
launched, workspace sizes, refusals without a GPU.  No GPU needed."""

import ctypes

import pytest
import torch

from theria_b200 import _lib, lm, sdpa_ragged

P = ctypes.c_void_p(16)  # never dereferenced: validation fails first


def test_ragged_arguments():
    lib = _lib.load()
    st = (ctypes.c_int64 * 6)(64, 16, 32, 16, 32, 16)

    def fwd(**k):
        return lib.theria_ragged_fwd(k.get("q", P), P, P, k.get("st", st), k.get("off", P), 0,
                                     k.get("o", P), None, None, k.get("ws", P), k.get("size", 0),
                                     k.get("T", 8), k.get("S", 2), k.get("H", 4), k.get("Hkv", 2),
                                     k.get("D", 16), k.get("dtype", 0), 1.0, 1, None)

    def bwd(**k):
        return lib.theria_ragged_bwd(P, P, P, st, P, 0, P, None, P, k.get("lse", P), k.get("dq", P),
                                     k.get("dk", P), k.get("dv", P), k.get("ws", P),
                                     k.get("size", 0), k.get("T", 8), 2, 4, 2, 16, 0, 1.0, 1, None)

    assert fwd(T=0) == _lib.THERIA_OK
    for bad in (dict(T=-1), dict(S=-1), dict(H=0), dict(Hkv=0), dict(Hkv=3), dict(D=0),
                dict(dtype=3), dict(q=None), dict(st=None), dict(off=None), dict(o=None)):
        assert fwd(**bad) == _lib.THERIA_ERR_INVALID_ARG
    for big in (dict(D=129), dict(T=1 << 30), dict(S=1 << 30), dict(T=1 << 29, H=8)):
        assert fwd(**big) == _lib.THERIA_ERR_UNSUPPORTED
    size = lib.theria_ragged_fwd_workspace_bytes(8, 2, 4, 2)
    assert size > 0 and size % 256 == 0
    assert fwd(size=size - 1) == fwd(ws=None, size=size) == _lib.THERIA_ERR_WORKSPACE
    assert bwd(T=0) == bwd(dq=None, dk=None, dv=None) == _lib.THERIA_OK
    assert bwd(dk=None) == bwd(dv=None) == bwd(lse=None) == _lib.THERIA_ERR_INVALID_ARG
    size = lib.theria_ragged_bwd_workspace_bytes(8, 2, 4, 2, 16)
    assert size >= 8 * 4 * 8 and bwd(size=size - 1) == _lib.THERIA_ERR_WORKSPACE


def test_rotary_arguments():
    lib = _lib.load()
    st = (ctypes.c_int64 * 12)()

    def call(**k):
        return lib.theria_rotary(k.get("q", P), k.get("k", None), k.get("yq", P), None,
                                 k.get("st", st), k.get("B", 1), k.get("T", 4), k.get("Hq", 2),
                                 k.get("Hk", 0), k.get("D", 16), k.get("dtype", 0),
                                 k.get("pos", None), k.get("n", 0), k.get("off", None), 1, 0,
                                 k.get("f", P), k.get("pairs", 8), 1.0, 0, 0, None)

    assert call(T=0) == call(B=0) == call(Hq=0) == _lib.THERIA_OK
    for bad in (dict(B=-1), dict(D=0), dict(pairs=9), dict(pairs=-1), dict(dtype=3), dict(q=None),
                dict(yq=None), dict(st=None), dict(f=None), dict(Hk=1), dict(pos=P),
                dict(pos=P, n=4, off=P)):
        assert call(**bad) == _lib.THERIA_ERR_INVALID_ARG
    for big in (dict(D=4097), dict(Hq=65536), dict(T=1 << 31), dict(B=1 << 40, T=2)):
        assert call(**big) == _lib.THERIA_ERR_UNSUPPORTED


def test_clip_arguments():
    lib = _lib.load()
    sizes, types = (ctypes.c_int64 * 2)(5, 20000), (ctypes.c_int * 2)(0, 2)
    ptrs = (ctypes.c_void_p * 2)(16, 16)
    assert lib.theria_grads_parts(sizes, 2) == 1 + 3  # chunks of 8192 values
    assert lib.theria_grads_parts((ctypes.c_int64 * 1)(1 << 33), 1) == 592
    assert lib.theria_grads_parts(sizes, 0) == 0
    bad_types, bad_sizes = (ctypes.c_int * 2)(0, 3), (ctypes.c_int64 * 2)(5, -1)
    inv = _lib.THERIA_ERR_INVALID_ARG
    assert lib.theria_grads_dot(ptrs, None, sizes, bad_types, 2, P, None) == inv
    assert lib.theria_grads_dot(ptrs, None, bad_sizes, types, 2, P, None) == inv
    assert lib.theria_grads_dot(ptrs, None, sizes, types, 2, None, None) == inv
    assert lib.theria_grads_dot(ptrs, None, sizes, types, 0, None, None) == _lib.THERIA_OK
    assert lib.theria_grads_clip(ptrs, ptrs, sizes, types, 2, P, -1.0, P, P, None) == inv
    assert lib.theria_grads_clip(ptrs, ptrs, sizes, types, 2, P, float("nan"), P, P, None) == inv
    assert lib.theria_grads_clip(ptrs, ptrs, sizes, types, 2, P, 1.0, None, None, None) == inv
    assert lib.theria_grads_clip_bwd(ptrs, None, ptrs, sizes, types, 2, None, P, None, None) == inv
    huge = (ctypes.c_int64 * 1)(1 << 60)
    assert lib.theria_grads_dot(ptrs, None, huge, types, 1, P, None) == _lib.THERIA_ERR_UNSUPPORTED


def test_there_is_no_cpu_path():
    q, off = torch.randn(3, 2, 16), torch.tensor([0, 3])
    f = lm.rotary_frequencies(16, device="cpu")
    for call in (lambda: sdpa_ragged(q, q, q, off), lambda: lm.rotary(q, q, f),
                 lambda: lm.gradient_norm([q]), lambda: lm.clip_gradients([q], 1.0),
                 lambda: lm.clip_gradients_([q], 1.0)):
        with pytest.raises(AssertionError, match="requires CUDA"):
            call()
