"""lm.clip_gradients and lm.gradient_norm, with their gradients, at norms near both
ends of float32's range, where the factors c = max / n and x . u / n^2 leave it.

Tolerances as in test_gpu_clip: E = 2^-21 of sums of sizes, and half a step of the
result's type; results below the type's smallest normal number are off by half its
smallest step instead."""

import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

from theria_b200 import lm  # noqa: E402

E = 2.0 ** -21
STEP = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133}  # between subnormal numbers
SHAPES = [(3000,), (50, 7), (8193,)]


def _tensors(dtype, seed, std):
    g = torch.Generator("cuda").manual_seed(seed)
    return [(torch.randn(s, generator=g, device="cuda").clamp(-3, 3).double() * std).to(dtype)
            for s in SHAPES]


def _check(dtype, std, most, gy_std, gn):
    x = [t.requires_grad_(True) for t in _tensors(dtype, 0, std)]
    x[0].data[:5] = 0.0
    xd = [t.detach().double() for t in x]
    n = torch.cat([t.flatten() for t in xd]).norm().item()
    most = most if most else n / 4
    c, u, tiny = min(1.0, most / n), torch.finfo(dtype).eps / 2, STEP[dtype] / 2
    y, norm = lm.clip_gradients(x, most)
    for a, b in zip(y, xd):
        want = b * c
        assert ((a.double() - want).abs() <= want.abs() * (u + 2 * E) + tiny).all()
    gy = _tensors(dtype, 1, gy_std)
    gd = [t.double() for t in gy]
    got = torch.autograd.grad([*y, norm], x, [*gy, torch.tensor(gn, device="cuda")])
    dot = sum((a * b).sum().item() for a, b in zip(xd, gd))
    size = sum((a * b).abs().sum().item() for a, b in zip(xd, gd))
    back = (-c * dot / n / n if c < 1 else 0.0) + gn / n
    for g, a, b in zip(got, xd, gd):
        want = c * b + back * a
        slack = (c * b.abs() + (abs(back) + c * size / n / n) * a.abs()) * 4 * E
        assert ((g.double() - want).abs() <= want.abs() * u + slack + tiny).all()
    alone = [t.detach().requires_grad_(True) for t in x]
    gn = torch.tensor(0.7, device="cuda")
    for g, a in zip(torch.autograd.grad(lm.gradient_norm(alone), alone, gn), xd):
        want = 0.7 / n * a
        assert ((g.double() - want).abs() <= want.abs() * (u + 4 * E) + tiny).all()
    inside = [t.detach().clone() for t in x]
    lm.clip_gradients_(inside, most)
    assert all(torch.equal(a, b) for a, b in zip(inside, y))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("most", [1.0, 1e-3])
@pytest.mark.parametrize("std", [1e20, 1e30, 1e37, 1e38])
def test_large_norms_to_ordinary_ones(std, most, dtype):
    _check(dtype, std, most, 1.0, 0.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("std", [1e-37, 1e-39, 1e-41])
def test_norms_of_subnormal_values(std, dtype):
    if dtype is torch.bfloat16 and std < 2.0 ** -131:
        std = 2.0 ** -131  # a few of its smallest steps
    _check(dtype, std, None, 1.0, 0.7)
    _check(dtype, std, None, 1e-37, 0.0)


def test_gradients_between_the_ends():
    # c of 1e-30, cotangents of 1e30: each factor within float32, products of order 1
    _check(torch.float32, 1e25, 1e-5, 1e30, 0.7)
    _check(torch.float32, 1e-25, None, 1e30, 0.7)
    # cotangents at float32's end: b x alone may pass it
    _check(torch.float32, 1.0, None, 1e38, 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("std", [1e20, 1e30])
def test_large_norms_without_a_gradient_of_their_own(std, dtype):
    # the values' gradient alone: c x . u / n^2 is far below float32's smallest number,
    # times x it is of the size of c u
    _check(dtype, std, 1.0, 1.0, 0.0)
