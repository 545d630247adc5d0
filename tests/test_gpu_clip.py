"""lm.gradient_norm, clip_gradients and clip_gradients_ against float64.

Tolerances: sums of eight products in float32 (8 roundings of 2^-24 of values of
one sign: 2^-21 of the sum, half of it in the root), the rest in float64; the
factor's rounding to float32 and the product's are 2^-24 each, the result's half
a step of its type.  Gradients: x . u as above of its sum of sizes."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

from theria_b200 import lm  # noqa: E402
from theria_b200.maml.loops import inner_adapt, meta_loss_on_tasks, named_buffers, named_params  # noqa: E402
from theria_b200.maml.model import MAMLClassifier  # noqa: E402
from theria_b200.maml.distributed import GraphedMetaStep, MetaStep  # noqa: E402
from theria_b200.maml.tasks import sample_tasks, stack_tasks  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
E = 2.0 ** -21


def _norm(x):
    return torch.cat([t.detach().double().flatten() for t in x]).norm().item()


def _tensors(shapes, dtype, seed=0, std=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return [(torch.randn(s, generator=g, device="cuda") * std).to(dtype) for s in shapes]


SHAPES = [
    [(1,)], [(), (3,), (0,), (7, 5)], [(8192,), (8193,), (1, 8191)], [(100003,), (64, 64)],
    [(2, 3)] * 700, [(1000, 1000), (17,)] * 3,
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shapes", SHAPES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("ratio", [0.5, 3.0])
def test_clip_and_gradient(shapes, ratio, dtype):
    x = [t.requires_grad_(True) for t in _tensors(shapes, dtype)]
    n = _norm(x)
    most = n / ratio
    y, norm = lm.clip_gradients(x, most)
    assert norm.dtype is torch.float32 and abs(norm.item() - n) <= E * n
    assert abs(lm.gradient_norm([t.detach() for t in x]).item() - n) <= E * n
    c, u = min(1.0, 1 / ratio), torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype is torch.float16 else 0.0
    for a, b in zip(y, x):
        want = b.detach().double() * c
        assert a.dtype is dtype and a.shape == b.shape
        assert ((a.double() - want).abs() <= want.abs() * (u + 2 * E) + tiny).all()
    gy = _tensors(shapes, dtype, 1)
    gn = torch.tensor(0.7, device="cuda")
    got = torch.autograd.grad([*y, norm], x, [*gy, gn])
    xd, gd = ([t.detach().double() for t in s] for s in (x, gy))
    dot = sum((a * b).sum().item() for a, b in zip(xd, gd))
    size = sum((a * b).abs().sum().item() for a, b in zip(xd, gd))
    for g, a, b in zip(got, xd, gd):
        back = (-c * dot / n ** 2 if ratio > 1 else 0.0) + 0.7 / n
        want = c * b + back * a
        slack = (c * b.abs() + (abs(back) + c * size / n ** 2) * a.abs()) * 4 * E
        assert ((g.double() - want).abs() <= want.abs() * u + slack + tiny).all()
    assert torch.equal(torch.stack([a.sum() for a in y]),
                       torch.stack([a.sum() for a in lm.clip_gradients(x, most)[0]]))


def test_mixed_types_strides_and_alignment():
    base = torch.randn(5001, device="cuda")
    x = [base[1:], base[:4000].view(40, 100).t(), torch.randn(33, device="cuda").half()[1:],
         torch.randn(65, device="cuda").bfloat16(), base[:1].expand(7)]
    n = _norm(x)
    y, norm = lm.clip_gradients(x, n / 2)
    assert abs(norm.item() - n) <= E * n
    for a, b in zip(y, x):
        assert a.dtype is b.dtype
        want = b.double() / 2
        assert ((a.double() - want).abs() <= want.abs() * (torch.finfo(b.dtype).eps / 2 + 2 * E)
                + 1e-7).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("std", [1e-30, 1e-22, 1e18, 1e30])
def test_very_small_and_very_large(dtype, std):
    x = _tensors([(3000,), (50, 7)], dtype, std=std)
    n = _norm(x)
    y, norm = lm.clip_gradients(x, n / 4)
    assert abs(norm.item() - n) <= E * n
    assert abs(_norm(y) - n / 4) <= n / 4 * (2 * E + torch.finfo(dtype).eps / 2)


def test_zero_nan_and_infinity():
    z = [torch.zeros(100, device="cuda", requires_grad=True)]
    y, norm = lm.clip_gradients(z, 1.0)
    assert norm.item() == 0 and not y[0].any()
    assert not torch.autograd.grad(norm, z)[0].any()
    y, norm = lm.clip_gradients([torch.zeros(100, device="cuda")], 0.0)
    assert not y[0].any()
    x = [torch.ones(100, device="cuda"), torch.ones(9000, device="cuda")]
    x[1][8999] = math.nan
    y, norm = lm.clip_gradients(x, 1.0)
    assert norm.isnan() and all(t.isnan().all() for t in y)
    x[1][8999] = math.inf
    y, norm = lm.clip_gradients(x, 1.0)
    assert norm.isinf() and not y[0].any() and y[1].isnan().sum() == 1
    y, norm = lm.clip_gradients(x[:1], math.inf)
    assert torch.equal(y[0], x[0])


def test_in_place():
    x = _tensors([(100, 30), (8193,), (7,)], torch.float32)
    x.append(torch.randn(30, 50, device="cuda").t())
    keep = [t.clone() for t in x]
    n = _norm(x)
    version = [t._version for t in x]
    norm = lm.clip_gradients_(x, n / 3)
    want, _ = lm.clip_gradients(keep, n / 3)
    assert abs(norm.item() - n) <= E * n
    for a, b, c in zip(x, want, version):
        assert torch.equal(a, b) and a._version > c
    again = [t.clone() for t in x]
    lm.clip_gradients_(x, n)  # below the limit: unchanged
    assert all(torch.equal(a, b) for a, b in zip(x, again))
    p = torch.randn(8, device="cuda", requires_grad=True)
    with torch.no_grad():
        lm.clip_gradients_([p], 0.1)
    assert abs(p.norm().item() - 0.1) < 1e-6
    for bad, match in (([p], "require a gradient"), ([x[0], x[0]], "overlap"),
                       ([x[1][:5], x[1][4:9]], "overlap"), ([x[0][:1].expand(4, 30)], "expanded")):
        with pytest.raises(AssertionError, match=match):
            lm.clip_gradients_(bad, 1.0)


def test_refusals():
    x = torch.randn(4, device="cuda")
    for call in (lambda t, m: lm.clip_gradients(t, m), lambda t, m: lm.clip_gradients_(t, m),
                 lambda t, m: lm.gradient_norm(t)):
        for bad, match in (([], "at least one"), ([x.cpu()], "requires CUDA"),
                           ([x.double()], "Unsupported dtype"), ([x, x.long()], "Unsupported")):
            with pytest.raises(AssertionError, match=match):
                call(bad, 1.0)
    for m in (-1.0, math.nan):
        with pytest.raises(AssertionError, match="max_norm"):
            lm.clip_gradients([x], m)
    x.requires_grad_(True)
    (g,) = torch.autograd.grad(lm.clip_gradients([x], 0.1)[0][0].square().sum(), x,
                               create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            lm.gradient_norm([dual])


def test_capture_and_streams():
    x = _tensors([(5000,), (64, 64)], torch.float32)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        lm.clip_gradients(x, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, norm = lm.clip_gradients(x, 1.0)
    for t in x:
        t.mul_(3)
    graph.replay()
    want, n = lm.clip_gradients(x, 1.0)
    assert torch.equal(norm, n) and all(torch.equal(a, b) for a, b in zip(y, want))


def _model(seed=0):
    torch.manual_seed(seed)
    return MAMLClassifier().cuda()


def test_clipped_inner_steps_of_maml():
    """inner_adapt(max_norm) against the same steps with the clip in torch operations:
    float32 both, two second-order steps; the clip's own error is 2^-20 of each
    gradient, and the chain may grow it a thousandfold."""
    model = _model()
    tasks = [t.to("cuda") for t in sample_tasks(0, 2)]
    loss = meta_loss_on_tasks(model, tasks, inner_lr=0.4, inner_steps=2, max_norm=0.5)
    got = torch.autograd.grad(loss, list(model.parameters()))
    import theria_b200.maml.loops as loops
    ref = []
    for t in tasks:
        phi = named_params(model)
        for _ in range(2):
            ls = loops.loss_fn(torch.func.functional_call(model, (phi, named_buffers(model)), (t.x_s,)), t.y_s)
            grads = torch.autograd.grad(ls, tuple(phi.values()), create_graph=True)
            n = torch.stack([g.square().sum() for g in grads]).sum().sqrt()
            assert n > 0.5  # the clip acts
            phi = type(phi)((k, p - 0.4 * (g * (0.5 / n))) for (k, p), g in zip(phi.items(), grads))
        ref.append(loops.outer_loss(model, phi, named_buffers(model), t))
    want_loss = torch.stack(ref).mean()
    want = torch.autograd.grad(want_loss, list(model.parameters()))
    assert abs(loss.item() - want_loss.item()) <= 1e-5 * abs(want_loss.item())
    num = sum((a - b).double().square().sum() for a, b in zip(got, want)).sqrt()
    assert num / _norm(want) < 1e-3
    plain = inner_adapt(model, named_params(model), named_buffers(model), tasks[0], inner_lr=0.4)
    none = inner_adapt(model, named_params(model), named_buffers(model), tasks[0], inner_lr=0.4,
                       max_norm=1e9)
    for a, b in zip(plain.values(), none.values()):
        assert torch.equal(a, b)


def test_clipped_meta_step():
    batch = stack_tasks(sample_tasks(0, 2)).to("cuda")
    plain, clipped = (MetaStep(_model(), meta_batch=2, inner_steps=1, max_norm=m)
                      for m in (None, 1e-3))
    plain.loss_and_grad(batch)
    n = plain.bucket.double().norm().item()
    assert n > 1e-3
    clipped.step(batch)
    assert abs(clipped.grad_norm.item() - n) <= E * n
    want = plain.bucket.double() * (1e-3 / n)
    assert ((clipped.bucket.double() - want).abs() <= want.abs() * 2.0 ** -22).all()
    ms = MetaStep(_model(), meta_batch=2, inner_steps=1, max_norm=1e-3, capturable=True)
    graphed = GraphedMetaStep(ms, batch)
    graphed.step(batch)
    assert abs(ms.bucket.double().norm().item() - 1e-3) <= 1e-9


@pytest.mark.parametrize("most", [1e6, 0.5])
def test_some_in_place(most):
    # the C entry writes each y, also where only the first is its x
    x = _tensors([(100,), (9000,)], torch.float32)
    want, _ = lm.clip_gradients(x, most)
    out = [x[0], torch.full_like(x[1], 7.0)]
    lm._clip(x, out, most)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
