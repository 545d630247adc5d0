"""sdpa_ragged in float16 with cotangents and values that are not of order 1: its
gradients are linear in both, and float16's range is short.

Tolerance on the 2-norm of dq, dk: each is rounded once, and is a sum of as many
products of ds, rounded once too.  With independent values the sum of the products'
roundings is to the sum itself as one rounding is to its value, so 2 u (u = 2^-11, half
a step) covers both, each of them u at most.  Inputs are such that the results lie in
float16's normal range; those of a row's that do not are off by 2^-25 besides."""

import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

from theria_b200 import sdpa_ragged  # noqa: E402

U = 2.0 ** -11


def _inputs(n, H, Hkv, D, std_q, std_k, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    mk = lambda h, std: (torch.randn(n, h, D, generator=g, device="cuda") * std).half()  # noqa: E731
    do = torch.randn(n, H, D, generator=g, device="cuda")
    return mk(H, std_q), mk(Hkv, std_k), mk(Hkv, 1.0), do


def _grads(q, k, v, do, lengths, causal):
    off = torch.tensor([0] + lengths, device="cuda").cumsum(0)
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    return torch.autograd.grad(sdpa_ragged(*x, off, causal=causal), x, do)


def _plain(q, k, v, do, lengths, causal):
    """dq, dk, dv in float64, one head at a time, and what z's error does to each row of dq."""
    out = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (q, k, v)]
    moved = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    G, scale, a = q.shape[1] // k.shape[1], q.shape[2] ** -0.5, 0
    for n in lengths:
        for h in range(q.shape[1]):
            qs, ks, vs, ds_o = (t[a:a + n, j].double() for t, j in
                                ((q, h), (k, h // G), (v, h // G), (do, h)))
            s = qs @ ks.t() * scale
            if causal:
                s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1),
                                  float("-inf"))
            p = s.softmax(-1)
            dp = ds_o @ vs.t()
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
            out[0][a:a + n, h] = ds @ ks
            moved[a:a + n, h] = U * (p * dp.abs()).sum(-1) * scale * (p @ ks).norm(dim=-1)
            out[1][a:a + n, h // G] += ds.t() @ qs
            out[2][a:a + n, h // G] += p.t() @ ds_o
        a += n
    return out, moved


def _error(got, want):
    """How far got is off beyond float16's smallest step."""
    assert torch.isfinite(got).all()
    return ((got.double() - want).abs() - 2.0 ** -25).clamp(min=0)


def _off(got, want):
    return (_error(got, want).norm() / want.norm()).item()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,std", [(4096, 1e-3), (1024, 1e-4), (1024, 1e-3), (1024, 1.0),
                                   (2048, 1e3), (64, 1e4), (700, 3e3)])
def test_sizes_of_cotangents(n, std, causal, D):
    lengths, H, Hkv = [n, n // 3], 4, 2
    for which, (std_q, std_k) in enumerate(((1 / 16, 16.0), (16.0, 1 / 16))):
        if std >= 1.0:
            std_q = std_k = 1.0
        q, k, v, do = _inputs(sum(lengths), H, Hkv, D, std_q, std_k)
        do = (do * std).clamp(-60000, 60000).half()
        want, _ = _plain(q, k, v, do, lengths, causal)
        assert want[which].abs().max().item() < 65504
        got = _grads(q, k, v, do, lengths, causal)
        assert _off(got[which], want[which]) <= 2 * U


@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 64), (6, 2, 80), (8, 1, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_different_sizes(H, Hkv, D, causal):
    # each row of dq goes by its own cotangent; a row's values are fewer: 3 u
    lengths = [500, 1, 203]
    q, k, v, do = _inputs(sum(lengths), H, Hkv, D, 1 / 16, 16.0)
    size = 2.0 ** -(torch.arange(sum(lengths), device="cuda") % 11).float()
    do = (do * size[:, None, None]).half()
    want, moved = _plain(q, k, v, do, lengths, causal)
    got = _grads(q, k, v, do, lengths, causal)
    assert (_error(got[0], want[0]).norm(dim=-1) <= 3 * U * want[0].norm(dim=-1) + moved).all()
    # a whole sequence of small ones beside one of large ones
    do = torch.cat([do[:500], do[500:] * 2.0 ** -12])
    want, _ = _plain(q, k, v, do, lengths, causal)
    got = _grads(q, k, v, do, lengths, causal)
    for part in (slice(0, 500), slice(501, None)):
        assert _off(got[0][part], want[0][part]) <= 2 * U


def test_cotangents_of_zero():
    lengths = [300, 40]
    q, k, v, do = _inputs(340, 4, 2, 64, 1.0, 1.0)
    assert not any(g.any() for g in _grads(q, k, v, torch.zeros_like(do).half(), lengths, True))
    do[:300] = 0
    do[300:, 1] = 0
    got = _grads(q, k, v, do.half(), lengths, True)
    want, _ = _plain(q, k, v, do.half(), lengths, True)
    assert not any(g[:300].any() for g in got) and not got[0][:, 1].any()
    for g, w in zip(got, want):
        assert _off(g, w) <= 2 * U


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,std,std_v", [(64, 1e-2, 3e3), (40, 0.5, 1e4), (512, 1e-3, 5e3),
                                         (4096, 1.0, 1e-3), (4096, 1e2, 1e-4), (300, 1.0, 300.0)])
def test_sizes_of_values(n, std, std_v, causal, D):
    lengths, H, Hkv = [n, n // 3], 4, 2
    small = std * std_v < 1
    for which, (std_q, std_k) in enumerate(((1 / 16, 16.0), (16.0, 1 / 16))):
        if not small:
            std_q = std_k = 1.0
        q, k, v, do = _inputs(sum(lengths), H, Hkv, D, std_q, std_k)
        do, v = ((t.float() * s).clamp(-60000, 60000).half() for t, s in ((do, std), (v, std_v)))
        want, _ = _plain(q, k, v, do, lengths, causal)
        assert want[which].abs().max().item() < 65504
        got = _grads(q, k, v, do, lengths, causal)
        assert _off(got[which], want[which]) <= 2 * U


@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (4, 4, 128)])
def test_a_single_large_row(H, Hkv, D):
    # the tokens behind it do not see it, though they share its tile of keys
    for what in ("cotangent", "value"):
        q, k, v, do = _inputs(3000, H, Hkv, D, 1.0, 1.0)
        if what == "cotangent":
            do[10] *= 1000
        else:
            v[10] *= 1000
        do = (do * 4).half()
        want, _ = _plain(q, k, v, do, [3000], True)
        got = _grads(q, k, v, do, [3000], True)
        for g, w in zip(got[:2], want[:2]):
            assert _off(g, w) <= 2 * U
        if what == "cotangent":
            assert _off(got[1][11:], want[1][11:]) <= 2 * U


def test_values_of_zero():
    q, k, v, do = _inputs(200, 4, 2, 64, 1.0, 1.0)
    got = _grads(q, k, torch.zeros_like(v), do.half(), [200], True)
    want, _ = _plain(q, k, torch.zeros_like(v), do.half(), [200], True)
    assert not got[0].any() and not got[1].any() and _off(got[2], want[2]) <= 2 * U


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_cotangent_that_is_not_finite_leaves_the_others_their_bits(value):
    # a small sequence of cotangents of 1e-3; the keys behind row 5 share its tile
    q, k, v, do = _inputs(700, 4, 2, 64, 16.0, 1 / 16)
    do = (do * 1e-3).half()
    want = _grads(q, k, v, do, [700], True)
    do[5] = value
    got = _grads(q, k, v, do, [700], True)
    assert torch.equal(got[0][:5], want[0][:5]) and torch.equal(got[0][6:], want[0][6:])
    without = do.clone()
    without[5] = 0
    exact, _ = _plain(q, k, v, without, [700], True)
    assert _off(got[1][6:], exact[1][6:]) <= 2 * U
