"""Which tensors lm.clip_gradients_ takes as sharing no address.  No GPU needed."""

import random

import pytest
import torch

from theria_b200 import lm


def _addresses(t):
    e = t.element_size()
    at = torch.arange(t.untyped_storage().nbytes() // e).as_strided(
        t.shape, t.stride(), t.storage_offset())
    return [e * i + b for i in at.flatten().tolist() for b in range(e)]


def test_random_views_never_share_an_address_unseen():
    rng = random.Random(0)
    base = torch.zeros(400)
    found = apart = 0
    for _ in range(4000):
        views = []
        while len(views) < 2:
            nd = rng.randint(0, 3)
            shape = [rng.randint(1, 5) for _ in range(nd)]
            stride = [rng.choice([1, 2, 3, 4, 5, 6, 8, 10, 12, 20, 24, 40]) for _ in range(nd)]
            off = rng.randint(0, 60)
            if off + sum(s * (n - 1) for s, n in zip(stride, shape)) >= 200:
                continue
            v = base.as_strided(shape, stride, off)
            if rng.random() < 0.3 and nd and stride[-1] == 1:
                v = v.view(torch.float16)
            views.append(v)
        sets = [_addresses(v) for v in views]
        for v, s in zip(views, sets):
            if len(set(s)) < len(s):
                assert lm._folded(v)
        if set(sets[0]) & set(sets[1]):
            assert lm._overlap(views)
            found += 1
        elif not lm._overlap(views):
            apart += 1
    assert found > 500 and apart > 1500


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_that_share_nothing_are_seen_to(dtype):
    w = torch.zeros(12, 40, dtype=dtype)
    h = torch.zeros(5, 4, 6, 8, dtype=dtype)
    for views in (
        [w[:, :8], w[:, 8:20], w[:, 20:]], [w[::2], w[1::2]], [w[:, ::2], w[:, 1::2]],
        [w[:6].t(), w[6:].t()], [w[:, 3:7].t(), w[:, 7:9], w[:, :3]], [w[1:, 30:], w[:, :5]],
        [h[:, 0], h[:, 1:]], [h[:, :, ::2], h[:, :, 1::2]], [h[..., :4], h[..., 4:]],
        [h.transpose(1, 2)[:, :3], h.transpose(1, 2)[:, 3:]], [h[:, 1, :, 2], h[:, 1, :, 3:]],
        [w[0], w[1], w[2, :0], w[5:, 0]], [w[0, 0], w[0, 1]],
    ):
        assert not lm._overlap(views) and not any(lm._folded(v) for v in views)


def test_views_that_share_values_are_found():
    w = torch.zeros(12, 12)
    for views in ([w, w.t()], [w.t(), w.t()], [w[:, :5], w[:, 4:]], [w[:, ::2], w[:, ::3]],
                  [w[3], w[:, 3]], [w[0, 0], w[0, :1]], [w, w.view(torch.float16)[:, 5:7]],
                  [w[:4], w[8:], w[3:9, 1:2]]):
        assert lm._overlap(views)
    assert lm._folded(w.as_strided((4, 4), (2, 1))) and lm._folded(torch.zeros(20).unfold(0, 4, 2))
    assert not lm._folded(w.t()) and not lm._folded(w[::3, ::2])
