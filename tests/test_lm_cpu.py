"""Host-side checks of the language-model entry points (include/theria_lm.h):
statuses for bad arguments before anything is launched, workspace sizes, and
no CPU path.  No GPU needed."""

import ctypes

import pytest
import torch

from theria_b200 import _lib, lm

P = ctypes.c_void_p(16)  # never dereferenced: validation fails first


def test_embedding_arguments():
    lib = _lib.load()
    fwd = lambda **k: lib.theria_embed_fwd(  # noqa: E731
        k.get("ids", P), 1, P, k.get("out", P), k.get("n", 4), k.get("V", 8), k.get("D", 16),
        k.get("dtype", 0), 1.0, -1, None)
    assert fwd(n=0) == _lib.THERIA_OK
    for bad in (dict(n=-1), dict(V=0), dict(D=0), dict(dtype=3), dict(ids=None), dict(out=None)):
        assert fwd(**bad) == _lib.THERIA_ERR_INVALID_ARG
    assert fwd(n=1 << 30) == _lib.THERIA_ERR_UNSUPPORTED
    assert fwd(V=(1 << 31) - 1) == _lib.THERIA_ERR_UNSUPPORTED
    size = lib.theria_embed_bwd_workspace_bytes(1000, 500, 16)
    assert size >= 2 * 1000 * 4 and size % 256 == 0
    bwd = lambda ws, n: lib.theria_embed_bwd(  # noqa: E731
        P, 1, P, P, ws, n, 1000, 500, 16, 0, 1.0, -1, None)
    assert bwd(None, size) == _lib.THERIA_ERR_WORKSPACE
    assert bwd(P, size - 1) == _lib.THERIA_ERR_WORKSPACE


def test_layer_norm_arguments():
    lib = _lib.load()
    fwd = lambda **k: lib.theria_norm_fwd(  # noqa: E731
        k.get("x", P), P, P, k.get("wdtype", 0), k.get("y", P), None, k.get("N", 4),
        k.get("D", 16), k.get("dtype", 0), 1e-5, None)
    assert fwd(N=0) == _lib.THERIA_OK
    for bad in (dict(N=-1), dict(D=0), dict(dtype=3), dict(x=None), dict(y=None),
                dict(wdtype=2), dict(dtype=1, wdtype=2)):
        assert fwd(**bad) == _lib.THERIA_ERR_INVALID_ARG
    bwd = lambda gw, gb, ws: lib.theria_norm_bwd(  # noqa: E731
        P, P, 0, P, P, P, gw, gb, ws, 0, 4, 16, 0, None)
    assert bwd(P, None, P) == _lib.THERIA_ERR_INVALID_ARG
    assert bwd(P, P, P) == _lib.THERIA_ERR_WORKSPACE
    assert bwd(P, P, None) == _lib.THERIA_ERR_WORKSPACE


def test_linear_cross_entropy_arguments():
    lib = _lib.load()

    def fwd(**k):
        return lib.theria_xent_fwd(k.get("h", P), P, P, 1, -100, k.get("red", 2),
                                   k.get("loss", P), P, k.get("count", P), k.get("ws", P),
                                   k.get("size", 0), k.get("N", 4), k.get("V", 8), k.get("D", 16),
                                   k.get("dtype", 0), None)

    for bad in (dict(N=-1), dict(V=0), dict(D=0), dict(dtype=3), dict(red=3), dict(h=None),
                dict(loss=None), dict(count=None)):
        assert fwd(**bad) == _lib.THERIA_ERR_INVALID_ARG
    assert fwd() == _lib.THERIA_ERR_WORKSPACE
    assert fwd(ws=None, size=1 << 30) == _lib.THERIA_ERR_WORKSPACE
    assert fwd(N=1 << 40) == _lib.THERIA_ERR_UNSUPPORTED
    size = lib.theria_xent_bwd_workspace_bytes(100, 1000, 64, _lib.BF16)
    assert size > 0 and size % 256 == 0
    assert lib.theria_xent_bwd(P, P, P, 1, -100, 2, P, P, P, P, P, P, size - 1, 100, 1000, 64,
                               _lib.BF16, None) == _lib.THERIA_ERR_WORKSPACE
    assert lib.theria_xent_bwd(P, P, P, 1, -100, 2, P, P, None, P, P, P, size, 100, 1000, 64,
                               _lib.BF16, None) == _lib.THERIA_ERR_INVALID_ARG


def test_there_is_no_cpu_path():
    w, x = torch.randn(8, 16), torch.randn(3, 16)
    ids = torch.zeros(3, dtype=torch.long)
    for call in (lambda: lm.embedding(ids, w), lambda: lm.layer_norm(x),
                 lambda: lm.linear_cross_entropy(x, w, ids)):
        with pytest.raises(AssertionError, match="requires CUDA"):
            call()
