"""lm.rotary against the rotation in float64.

Tolerance: the angle is good to 2^-52 t w turns and half a float32 unit of its
remainder; sincospi adds at most 2 units of 2^-24, the two products and their sum
3 half units of the pair's length, and the result's rounding half a step u of its
type: |a| + |b| times (2^-24 * 8 + ...) with far angles' 2^-50 t w, and u."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

from theria_b200 import lm, sdpa, sdpa_ragged  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _check(x, y, at, f, interleaved, amplitude=1.0, sign=1):
    """y: x [..., T, H, D] turned at positions at [..., T]."""
    dim, xd = 2 * f.numel(), x.detach().double()
    ang = sign * at.double()[..., None, None] * f
    c, s = ang.cos() * amplitude, ang.sin() * amplitude
    a, b = ((slice(0, dim, 2), slice(1, dim, 2)) if interleaved
            else (slice(0, dim // 2), slice(dim // 2, dim)))
    want = xd.clone()
    want[..., a] = xd[..., a] * c - xd[..., b] * s
    want[..., b] = xd[..., b] * c + xd[..., a] * s
    size = torch.zeros_like(xd)
    size[..., a] = size[..., b] = (xd[..., a].abs() + xd[..., b].abs()) * amplitude
    far = at.double().abs().max().item() if at.numel() else 0.0
    tol = size * (2.0 ** -21 + far * 2.0 ** -50) + want.abs() * torch.finfo(x.dtype).eps / 2
    if x.dtype is torch.float16:
        tol = tol + 2.0 ** -25
    err = (y.double() - want).abs()
    assert y.dtype is x.dtype and y.shape == x.shape
    assert (err <= tol).all(), (err - tol).max().item()
    assert torch.equal(y[..., dim:], x[..., dim:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,dim", [(64, 64), (128, 128), (128, 64), (80, 30), (16, 2), (9, 6), (100, 100),
                                   (72, 0), (2, 2), (1000, 998), (4096, 4096)])
def test_rotation_and_gradient(D, dim, interleaved, dtype):
    for T, Hq, Hk in ((1, 1, 1), (37, 5, 2), (700, 3, 1), (2100, 1, 1)):
        if T * D > 400000:
            continue
        g = torch.Generator("cuda").manual_seed(T)
        q, k = (torch.randn(T, h, D, generator=g, device="cuda").to(dtype).requires_grad_(True)
                for h in (Hq, Hk))
        f = lm.rotary_frequencies(dim) if dim else torch.zeros(0, dtype=torch.float64, device="cuda")
        at = torch.randint(0, 1 << 20, (T,), generator=g, device="cuda")
        yq, yk = lm.rotary(q, k, f, at, interleaved=interleaved, amplitude=1.25)
        _check(q, yq, at, f, interleaved, 1.25 if dim else 1.0)
        _check(k, yk, at, f, interleaved, 1.25)
        gq, gk = torch.randn_like(q), torch.randn_like(k)
        dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
        _check(gq, dq, at, f, interleaved, 1.25, -1)
        _check(gk, dk, at, f, interleaved, 1.25, -1)
        alone = lm.rotary(q.detach(), None, f, at.int(), interleaved=interleaved, amplitude=1.25)
        assert torch.equal(alone, yq)
        none = lm.rotary(q.detach()[:, :0], k.detach(), f, at, interleaved=interleaved,
                         amplitude=1.25)
        assert none[0].numel() == 0 and torch.equal(none[1], yk)


@pytest.mark.parametrize("heads", [1, 2, 3, 7, 64, 1000, 8192, 8193, 60000])
def test_numbers_of_heads(heads):
    f = lm.rotary_frequencies(8)
    for T in (1, 5, 1500 if heads < 100 else 2):
        x = torch.randn(T, heads, 8, device="cuda")
        _check(x, lm.rotary(x, None, f), torch.arange(T, device="cuda"), f, False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_positions(dtype):
    f = lm.rotary_frequencies(64)
    q, k = (torch.randn(3, 50, h, 64, device="cuda").to(dtype) for h in (4, 2))
    i = torch.arange(50, device="cuda")
    for y, x in zip(lm.rotary(q, k, f), (q, k)):
        _check(x, y, i.expand(3, 50), f, False)
    far = torch.randint(-(1 << 40), 1 << 40, (3, 50), device="cuda")
    for y, x in zip(lm.rotary(q, k, f, far), (q, k)):
        _check(x, y, far, f, False)
    for y, x in zip(lm.rotary(q, k, f, far[0]), (q, k)):
        _check(x, y, far[0].expand(3, 50), f, False)
    for dt in (torch.int32, torch.int64):
        off = torch.tensor([3, 3, 10, 11, 11, 40], device="cuda", dtype=dt)
        at = torch.cat([torch.zeros(3), torch.arange(7), torch.zeros(1), torch.arange(29),
                        torch.zeros(10)]).long().cuda()
        for y, x in zip(lm.rotary(q, k, f, offsets=off), (q, k)):
            _check(x, y, at.expand(3, 50), f, False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_and_memory_order(dtype, interleaved):
    f = lm.rotary_frequencies(48)
    i = torch.arange(20, device="cuda")
    rows = torch.randn(2, 20, 9, 64, device="cuda").to(dtype)
    heads = torch.randn(2, 5, 20, 64, device="cuda").to(dtype)
    odd = torch.randn(2, 20, 5 * 64 + 1, device="cuda").to(dtype)[..., 1:].unflatten(-1, (5, 64))
    last = torch.randn(2, 20, 64, 5, device="cuda").to(dtype).transpose(2, 3)
    for x in (rows[:, :, 2:7], heads.transpose(1, 2), odd, last, rows[:1].expand(2, 20, 9, 64),
              rows[:, :, :1].expand(2, 20, 5, 64), rows.flip(0)[:, 1:], rows[..., 1:63]):
        at = i[:x.shape[1]].expand(2, x.shape[1])
        y, _ = lm.rotary(x, x[:, :, :1], f, interleaved=interleaved)
        _check(x, y, at, f, interleaved)
    y = lm.rotary(heads.transpose(1, 2), None, f)
    assert y.transpose(1, 2).is_contiguous()  # heads first, as the dense attention takes them


def test_derivatives_of_any_order():
    f = lm.rotary_frequencies(8)
    q, k = (torch.randn(6, 2, 8, device="cuda", requires_grad=True) for _ in range(2))
    yq, yk = lm.rotary(q, k, f)
    (g,) = torch.autograd.grad((yq.pow(3).sum() + (yk * yq).sum()), q, create_graph=True)
    (h,) = torch.autograd.grad((g * q).sum(), q, create_graph=True)
    (h3,) = torch.autograd.grad((h * q).sum(), q)
    x = q.detach().double().requires_grad_(True)
    kd = k.detach().double()
    ang = torch.arange(6, device="cuda").double()[:, None, None] * f
    rot = lambda t: torch.cat([t[..., :4] * ang.cos() - t[..., 4:] * ang.sin(),  # noqa: E731
                               t[..., 4:] * ang.cos() + t[..., :4] * ang.sin()], -1)
    (a,) = torch.autograd.grad(rot(x).pow(3).sum() + (rot(kd) * rot(x)).sum(), x, create_graph=True)
    (b,) = torch.autograd.grad((a * x).sum(), x, create_graph=True)
    (c,) = torch.autograd.grad((b * x).sum(), x)
    for got, want in ((g, a), (h, b), (h3, c)):
        # a few products of values of order 10 deep, each 2^-21 of the sums' sizes
        assert (got.double() - want).abs().max() <= 2.0 ** -16 * want.abs().max()
    only = torch.autograd.grad(lm.rotary(q.detach(), k, f)[1].sum(), k)[0]
    assert torch.isfinite(only).all()
    assert not lm.rotary(q.detach(), k, f)[0].requires_grad
    qd = q.detach().requires_grad_(True)
    yq, yk = lm.rotary(qd, k.detach(), f)
    assert torch.equal(torch.autograd.grad(yq.sum(), qd)[0], lm.rotary(
        torch.ones_like(q), None, -f))


def test_frequencies():
    f = lm.rotary_frequencies(64, 500.0)
    m = torch.arange(32, device="cuda", dtype=torch.float64)
    assert f.dtype is torch.float64 and torch.allclose(f, 500.0 ** (-m / 32), rtol=1e-14)
    assert torch.allclose(lm.rotary_frequencies(64, 500.0, "linear", 4.0), f / 4, rtol=1e-14)
    ntk = lm.rotary_frequencies(64, 500.0, "ntk", 4.0)
    assert math.isclose(ntk[0].item(), 1.0) and math.isclose(ntk[-1].item(), f[-1].item() / 4)
    part = lm.rotary_frequencies(64, 500.0, "by_parts", 4.0, original_length=128)
    turns = 128 * f / (2 * math.pi)
    assert (part[turns < 1] == f[turns < 1] / 4).all()
    assert (turns < 1).any() and ((part >= f / 4 * (1 - 1e-12)) & (part <= f)).all()
    assert lm.rotary_frequencies(2, scaling="ntk", factor=8.0).tolist() == [1.0]


def test_relative_positions_only():
    # scores of rotated queries and keys depend on the distance alone: through the attention
    # of two packed sequences, and of the same sequence moved
    T, f = 60, lm.rotary_frequencies(64)
    q, k, v = (torch.randn(T, 2, 64, device="cuda") for _ in range(3))
    off = torch.tensor([0, 25, T], device="cuda")
    o = sdpa_ragged(*lm.rotary(q, k, f, offsets=off), v, off)
    moved = sdpa_ragged(*lm.rotary(q, k, f, positions=torch.arange(T, device="cuda") + 100000), v, off)
    # both sides' rotations are off by 2^-21 of |a| + |b| <= 10: scores by 64 * 10 * 2^-20 / 8
    assert (o - moved).abs().max() < 1e-3
    dense = sdpa(*(t.transpose(0, 1)[None].contiguous()
                   for t in (*lm.rotary(q[25:], k[25:], f), v[25:])), causal=True)
    assert (dense[0].transpose(0, 1) - o[25:]).abs().max() < 1e-4


def test_capture_and_streams():
    f = lm.rotary_frequencies(64)
    q = torch.randn(40, 3, 64, device="cuda").bfloat16().requires_grad_(True)
    at = torch.arange(40, device="cuda")

    def step():
        y = lm.rotary(q, None, f, at)
        return y.detach(), torch.autograd.grad(y, q, torch.ones_like(y))[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    at.add_(7)
    graph.replay()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


def test_refusals_and_empty():
    f = lm.rotary_frequencies(16)
    q = torch.randn(8, 2, 16, device="cuda")
    i = torch.arange(8, device="cuda")
    bad = [
        (dict(q=q.cpu()), "requires CUDA"), (dict(q=q.double()), "Unsupported dtype"),
        (dict(q=q[0]), "q must"), (dict(k=q[:7]), "k must"), (dict(k=q[..., :8]), "k must"),
        (dict(k=q.half()), "share one"), (dict(frequencies=f.float()), "float64"),
        (dict(frequencies=f.cpu()), "float64"), (dict(frequencies=f[None]), "pairs"),
        (dict(frequencies=lm.rotary_frequencies(18)), "pairs"), (dict(positions=i[:7]), "positions must"),
        (dict(positions=i.float()), "int64 or int32"), (dict(positions=i, offsets=i), "not both"),
        (dict(offsets=i.cpu()), "offsets is on"), (dict(offsets=i[:0]), "offsets must"),
        (dict(frequencies=f.clone().requires_grad_(True)), "no gradient"),
    ]
    for change, match in bad:
        with pytest.raises(AssertionError, match=match):
            lm.rotary(**{**dict(q=q, k=q, frequencies=f), **change})
    for kw, match in ((dict(dim=7), "even"), (dict(dim=0), "even"), (dict(dim=8, scaling="x"), "scaling"),
                      (dict(dim=8, factor=0.0), "positive"), (dict(dim=8, scaling="by_parts"), "by_parts")):
        with pytest.raises(AssertionError, match=match):
            lm.rotary_frequencies(**kw)
    assert lm.rotary(q[:0], q[:0], f)[1].shape == (0, 2, 16)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, q)
        with pytest.raises(NotImplementedError):
            lm.rotary(dual, None, f)
