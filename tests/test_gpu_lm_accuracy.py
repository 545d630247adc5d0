"""Language-model operators where their arithmetic has most to lose, against
float64 on the CPU: nearly certain tokens, large means, one scored row, rows
that do not count beside gradients that are not finite, and the widest rows.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

from theria_b200 import lm  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator("cpu").manual_seed(seed)


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
