"""Derivatives that the language-model operators do not have are refused, never
left out of a result."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

from theria_b200 import lm  # noqa: E402


def _calls():
    """name -> (function of its differentiable inputs, those inputs)."""
    ids = torch.tensor([1, 0, 5, 1], device="cuda")
    rand = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    return {
        "embedding": (lambda w: lm.embedding(ids, w), [rand(8, 16)]),
        "layer_norm": (lm.layer_norm, [rand(4, 16), rand(16), rand(16)]),
        "linear_cross_entropy": (lambda h, w: lm.linear_cross_entropy(h, w, ids),
                                 [rand(4, 16), rand(8, 16)]),
    }


@pytest.mark.parametrize("name", ["embedding", "layer_norm", "linear_cross_entropy"])
def test_forward_mode_is_refused(name):
    fn, args = _calls()[name]
    want = fn(*args)
    for k in range(len(args)):
        for grad in (False, True):
            xs = [a.clone().requires_grad_(grad) for a in args]
            with fwAD.dual_level():
                xs[k] = fwAD.make_dual(xs[k], torch.ones_like(xs[k]))
                with pytest.raises(NotImplementedError, match="forward mode"):
                    fn(*xs)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
                    fn(*xs)
    with fwAD.dual_level():  # nothing to carry
        assert torch.equal(fn(*args), want)
    with pytest.raises(RuntimeError):
        torch.func.jvp(fn, tuple(args), tuple(torch.ones_like(a) for a in args))


@pytest.mark.parametrize("name", ["embedding", "layer_norm", "linear_cross_entropy"])
@pytest.mark.parametrize("create_graph", [False, True])
def test_a_cotangent_with_a_tangent_is_refused(name, create_graph):
    fn, args = _calls()[name]
    xs = [a.requires_grad_(True) for a in args]
    y = fn(*xs)
    with fwAD.dual_level():
        g = fwAD.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="forward mode"):
            torch.autograd.grad(y, xs, g, create_graph=create_graph)


def test_a_second_cotangent_with_a_tangent_is_refused():
    calls = _calls()
    for name in ("embedding", "layer_norm"):
        fn, args = calls[name]
        xs = [a.requires_grad_(True) for a in args]
        y = fn(*xs)
        g = torch.ones_like(y).requires_grad_(True)
        first = torch.autograd.grad(y, xs, g, create_graph=True)
        with fwAD.dual_level():
            u = [fwAD.make_dual(torch.ones_like(t), torch.ones_like(t)) for t in first]
            with pytest.raises(NotImplementedError, match="forward mode"):
                torch.autograd.grad(first, g, u)


def test_layer_norm_refuses_a_third_derivative():
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    r = torch.randn(4, 16, device="cuda")
    (gx,) = torch.autograd.grad((lm.layer_norm(x) * r).sum(), x, create_graph=True)
    (g2,) = torch.autograd.grad((gx * r).sum(), x, create_graph=True)
    assert g2.requires_grad  # not silently cut off
    with pytest.raises(RuntimeError, match="differentiable twice"):
        g2.sum().backward()


def test_embedding_has_every_derivative_of_a_linear_map():
    # the second derivative's own: linear in its cotangent, constant in the table
    ids = torch.tensor([1, 0, 5, 1], device="cuda")
    w = torch.randn(8, 16, device="cuda", requires_grad=True)
    g = torch.randn(4, 16, device="cuda", requires_grad=True)
    (gw,) = torch.autograd.grad(lm.embedding(ids, w, scale=2.0), w, g, create_graph=True)
    (gg,) = torch.autograd.grad(gw, g, torch.ones_like(gw), create_graph=True)
    assert not gg.requires_grad and (gg == 2).all()
