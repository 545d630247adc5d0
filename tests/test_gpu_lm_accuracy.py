"""Language-model operators where their arithmetic has most to lose, against
float64 on the CPU: nearly certain tokens, large means, one scored row, rows
that do not count beside gradients that are not finite, and the widest rows.
"""

import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

from theria_b200 import lm  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator("cpu").manual_seed(seed)


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    return ((got - want).norm() / want.norm()).item()


# ------------------------------------------------------- linear cross entropy
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("up", [math.nan, math.inf])
def test_ignored_rows_get_no_gradient_whatever_arrives(up, reduction, dtype):
    g = _gen(30)
    h = torch.randn(70, 48, generator=g).to("cuda", dtype).requires_grad_(True)
    w = torch.randn(90, 48, generator=g).to("cuda", dtype).requires_grad_(True)
    t = torch.randint(90, (70,), generator=g).cuda()
    t[::3] = -100
    up = torch.tensor(up, device="cuda")
    gh, gw = torch.autograd.grad(lm.linear_cross_entropy(h, w, t, reduction=reduction), (h, w), up)
    assert (gh[t == -100] == 0).all()
    assert not gh[t != -100].isfinite().any() and not gw.isfinite().any()
    t[:] = -100
    gh, gw = torch.autograd.grad(lm.linear_cross_entropy(h, w, t, reduction=reduction), (h, w), up)
    assert (gh == 0).all() and (gw == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_row_beside_weights_that_are_not_finite(dtype):
    w = torch.randn(9, 16, device="cuda").to(dtype)
    w[2, 3], w[5, 0] = math.inf, math.nan
    h = torch.randn(6, 16, device="cuda").to(dtype).requires_grad_(True)
    w.requires_grad_(True)
    loss = lm.linear_cross_entropy(h, w, torch.full((6,), -100, device="cuda"), reduction="sum")
    assert loss.item() == 0
    for grad in torch.autograd.grad(loss, (h, w)):
        assert (grad == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_word_whose_scores_are_minus_infinity(dtype):
    # probability 0, no gradient; the rows that fill up a tile of 70 leave none either
    g = _gen(31)
    h = torch.rand(70, 48, generator=g).to(dtype) + 0.5
    w = torch.randn(90, 48, generator=g).to(dtype) * 0.3
    t = torch.randint(1, 90, (70,), generator=g)
    hr, wr = h.double(), w[1:].double().requires_grad_(True)
    loss = F.cross_entropy(hr @ wr.t(), t - 1, reduction="sum")
    (want,) = torch.autograd.grad(loss, wr)
    w[0] = -math.inf
    wd = w.cuda().requires_grad_(True)
    got = lm.linear_cross_entropy(h.cuda(), wd, t.cuda(), reduction="sum")
    (gw,) = torch.autograd.grad(got, wd)
    assert abs(got.item() / loss.item() - 1) <= 4e-6
    assert (gw[0] == 0).all()
    assert _rel(gw[1:], want) <= {torch.float16: 8e-4, torch.bfloat16: 6e-3}[dtype]
