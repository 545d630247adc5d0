"""lm.clip_gradients_ on views of one tensor: those that share no value are clipped,
others are refused before anything changes."""

import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

from theria_b200 import lm  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_without_a_common_value(dtype):
    g = torch.Generator("cuda").manual_seed(0)
    w = torch.randn(60, 90, generator=g, device="cuda").to(dtype)
    flat = w.clone()
    for views in ([w[:, :20], w[:, 20:33].t(), w[:, 33:]], [w[::2], w[1::2]],
                  [w.view(60, 3, 30)[:, 1:], w.view(60, 3, 30)[:, 0]]):
        before = w.clone()
        most = before.double().norm().item() / 3
        norm = lm.clip_gradients_(views, most)
        # 2^-21 of sums of squares, as in test_gpu_clip
        assert abs(norm.item() - 3 * most) <= 2.0 ** -21 * norm.item()
        want = before.double() / 3
        assert ((w.double() - want).abs()
                <= want.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -20)).all()
    assert not torch.equal(w, flat)


def test_views_with_common_values_are_refused():
    w = torch.randn(12, 12, device="cuda")
    keep = w.clone()
    for views in ([w, w.t()], [w.t(), w.t()], [w[:, :5], w[:, 4:]], [w[3], w[:, 3]]):
        with pytest.raises(AssertionError, match="no two may overlap"):
            lm.clip_gradients_(views, 0.1)
    for view in (w.as_strided((4, 4), (2, 1)), w.flatten().unfold(0, 4, 2)):
        with pytest.raises(AssertionError, match="overlap itself"):
            lm.clip_gradients_([view], 0.1)
    assert torch.equal(w, keep)
