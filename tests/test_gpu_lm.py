"""Language-model operators (include/theria_lm.h) against plain forms in
float64 on the CPU.

Tolerances, per element type with unit roundoff u (2^-24, 2^-11, 2^-8 for
float32, float16, bfloat16): a result that is float32 arithmetic rounded once
is within u of the exact one plus the float32 arithmetic's own error, taken as
K * 2^-24 of the sum of the terms' sizes for sums of K terms (bounded below by
their random walk, so the bound is not tight).  Comparisons are by the 2-norm
over each output, where roundings of single elements average to less than u:
    float32 4e-6, float16 8e-4, bfloat16 6e-3,
i.e. 2^-24 * 64, 2^-11 * 1.6 and 2^-8 * 1.5: room for the one extra rounding
to the operands' type that the score gradients take on the tensor cores.  The
loss's gradients sum terms p - 1 that cancel where a word is nearly certain; to
them the float32 arithmetic's error of the terms' sizes (4 roundings, 2^-22) is
added, as above.
"""

import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

import theria_b200  # noqa: E402
from theria_b200 import _lib, lm  # noqa: E402

TOL = {torch.float32: 4e-6, torch.float16: 8e-4, torch.bfloat16: 6e-3}
DTYPES = list(TOL)


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    den = want.norm().item()
    return (got - want).norm().item() / (den if den > 0 else 1.0)


def _near(got, want, dtype, terms=None):
    """`terms`: the sizes of the terms that cancel in each value, where they do."""
    rel, tol = _rel(got, want), TOL[dtype]
    if terms is not None:
        tol += 2 ** -22 * terms.norm().item() / max(want.norm().item(), 1e-300)
    assert rel <= tol, (rel, tol)


def _gen(seed):
    return torch.Generator("cpu").manual_seed(seed)


# ------------------------------------------------------------------ embedding
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 5, 64), (33, 7, 40), (2049, 300, 65),
                                   (5000, 3, 24), (4096, 70000, 16), (70, 1000, 2052),
                                   (6000, 65536, 8)])
def test_embedding_and_its_gradient(n, V, D, dtype):
    g = _gen(n + V)
    w = torch.randn(V, D, generator=g).to(dtype)
    # a third of the tokens are token 0, the rest spread over the vocabulary
    ids = torch.where(torch.rand(n, generator=g) < 0.34, torch.zeros(n, dtype=torch.long),
                      torch.randint(V, (n,), generator=g))
    gy = torch.randn(n, D, generator=g).to(dtype)
    scale = math.sqrt(D)
    wd = w.cuda().requires_grad_(True)
    y = lm.embedding(ids.cuda(), wd, scale=scale)
    (gw,) = torch.autograd.grad(y, wd, gy.cuda())
    _near(y, w.double()[ids] * scale, dtype)
    want = torch.zeros(V, D, dtype=torch.float64).index_add_(0, ids, gy.double() * scale)
    _near(gw, want, dtype)
    # the same bits again
    (again,) = torch.autograd.grad(lm.embedding(ids.cuda(), wd, scale=scale), wd, gy.cuda())
    assert torch.equal(gw, again)


def test_embedding_sums_every_token_of_one_row():
    # one row takes all 100,000 tokens: ones sum exactly in float32
    ids = torch.full((100_000,), 2, device="cuda")
    w = torch.zeros(4, 8, device="cuda", requires_grad=True)
    (gw,) = torch.autograd.grad(lm.embedding(ids, w), w, torch.ones(100_000, 8, device="cuda"))
    assert gw[2].tolist() == [100_000.0] * 8 and gw[[0, 1, 3]].abs().max() == 0


@pytest.mark.parametrize("V", [1, 2, 500, 600, 300_000])
@pytest.mark.parametrize("n", [31, 1024, 4096, 4097, 9000, 20_000, 40_000, 131_072, 131_073,
                               150_001])
def test_embedding_gradient_over_token_counts(n, V):
    # every shape of the sort, with odd row widths; whole numbers, which
    # float32 adds exactly in any order (sums stay below 2^24)
    g = _gen(n + V)
    ids = (torch.rand(n, generator=g) ** 4 * V).long().clamp_(max=V - 1)
    gy = torch.randint(-8, 9, (n, 3), generator=g).float()
    w = torch.zeros(V, 3, device="cuda", requires_grad=True)
    (gw,) = torch.autograd.grad(lm.embedding(ids.cuda(), w), w, gy.cuda())
    want = torch.zeros(V, 3, dtype=torch.float64).index_add_(0, ids, gy.double())
    assert torch.equal(gw.cpu().double(), want)


@pytest.mark.parametrize("padding", [0, 3, -1])
def test_embedding_padding_row_gets_no_gradient(padding):
    g = _gen(3)
    w, ids = torch.randn(10, 12, generator=g).double(), torch.randint(10, (5, 40), generator=g)
    gy = torch.randn(5, 40, 12, generator=g).double()
    wr = w.clone().requires_grad_(True)
    y = F.embedding(ids, wr, padding_idx=padding)
    (want,) = torch.autograd.grad(y, wr, gy)
    wd = w.float().cuda().requires_grad_(True)
    yd = lm.embedding(ids.cuda().int(), wd, padding_idx=padding)
    (got,) = torch.autograd.grad(yd, wd, gy.float().cuda())
    _near(yd, y, torch.float32)
    _near(got, want, torch.float32)
    assert got[padding].abs().max() == 0


def test_embedding_strides_shapes_and_empty():
    g = _gen(4)
    table = torch.randn(50, 48, generator=g).cuda()
    w = table[:, 8:24]                                    # strided rows
    ids = torch.randint(50, (6, 9), generator=g).cuda().t()  # transposed ids
    assert torch.equal(lm.embedding(ids, w, scale=2.0), w[ids] * 2.0)
    assert lm.embedding(ids[:0], w).shape == (0, 6, 16)
    wd = w.contiguous().requires_grad_(True)
    y = lm.embedding(ids[:0], wd)
    assert torch.autograd.grad(y, wd, torch.empty_like(y))[0].abs().max() == 0
    # a misaligned table (rows of 16 bytes that start 4 bytes off)
    flat = torch.randn(41, generator=g).cuda()[1:].view(10, 4)
    assert torch.equal(lm.embedding(ids % 10, flat), flat[ids % 10])
    # gradients that arrive broadcast over the tokens
    y = lm.embedding(ids, wd)
    (gw,) = torch.autograd.grad(y.sum(), wd)
    assert torch.equal(gw[:, 0].cpu(), torch.bincount(ids.flatten().cpu(), minlength=50).float())


def test_embedding_second_derivative():
    g = _gen(5)
    ids, w = torch.randint(9, (30,), generator=g), torch.randn(9, 6, generator=g)
    r, u = torch.randn(30, 6, generator=g), torch.randn(9, 6, generator=g)

    def run(fn, dev, dt):
        wd = w.to(dev, dt).requires_grad_(True)
        rd = r.to(dev, dt).requires_grad_(True)
        y = fn(ids.to(dev), wd)
        (gw,) = torch.autograd.grad(y.square(), wd, rd, create_graph=True)
        return torch.autograd.grad(gw, (wd, rd), u.to(dev, dt))

    got = run(lambda i, t: lm.embedding(i, t, scale=3.0, padding_idx=4), "cuda", torch.float32)
    want = run(lambda i, t: F.embedding(i, t, padding_idx=4) * 3.0, "cpu", torch.float64)
    for a, b in zip(got, want):
        _near(a, b, torch.float32)


def test_ids_outside_the_vocabulary_are_reported():
    w = torch.ones(4, 8, device="cuda", requires_grad=True)
    ids = torch.tensor([0, 4, -1, 3], device="cuda")
    y = lm.embedding(ids, w)
    assert y[:, 0].tolist() == [1, 0, 0, 1]
    with pytest.raises(theria_b200._lib.TheriaError, match="invalid"):
        theria_b200.check_device_error()
    (gw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert gw[:, 0].tolist() == [1, 0, 0, 1]
    with pytest.raises(theria_b200._lib.TheriaError):
        theria_b200.check_device_error()
    loss = lm.linear_cross_entropy(torch.zeros(3, 8, device="cuda"), w.detach(),
                                   torch.tensor([1, 9, -7], device="cuda"))
    assert abs(loss.item() - math.log(4)) < 1e-6
    with pytest.raises(theria_b200._lib.TheriaError):
        theria_b200.check_device_error()


def test_embedding_offsets_past_32_bits():
    # 4.5e9 elements: the last rows lie beyond 2^32
    V, D = 2_200_000, 2048
    w = torch.zeros(V, D, device="cuda", dtype=torch.bfloat16)
    w[V - 2:] = torch.randn(2, D, device="cuda").bfloat16()
    w.requires_grad_(True)
    ids = torch.tensor([V - 1, 0, V - 2, V - 1], device="cuda")
    y = lm.embedding(ids, w)
    assert torch.equal(y[0], w[V - 1]) and torch.equal(y[2], w[V - 2]) and y[1].abs().max() == 0
    (gw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert (gw[V - 1] == 2).all() and (gw[V - 2] == 1).all() and (gw[0] == 1).all()
    assert gw[1:V - 2].any().item() is False


# ----------------------------------------------------------------- layer norm
NORM_SHAPES = [(1, 1), (1, 64), (5, 31), (300, 33), (17, 64), (3, 256), (9, 257), (4, 1000),
               (33, 1111), (7, 2048), (300, 4096), (3, 8192), (5, 8200), (2, 20001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D", NORM_SHAPES)
def test_layer_norm_and_its_gradients(N, D, dtype):
    g = _gen(N + D)
    x = (torch.randn(N, D, generator=g) * 1.5 + torch.randn(D, generator=g) + 0.5).to(dtype)
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(dtype)
    b, gy = torch.randn(D, generator=g).to(dtype), torch.randn(N, D, generator=g).to(dtype)
    ref = [t.double().requires_grad_(True) for t in (x, w, b)]
    yr = F.layer_norm(ref[0], (D,), ref[1], ref[2], 1e-5)
    want = torch.autograd.grad(yr, ref, gy.double())
    dev = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = lm.layer_norm(*dev)
    got = torch.autograd.grad(y, dev, gy.cuda())
    _near(y, yr, dtype)
    if D > 1:
        _near(got[0], want[0], dtype)
        _near(got[1], want[1], dtype)
    else:  # one column: xhat and these gradients are exactly 0
        assert got[0].abs().max() == 0 and got[1].abs().max() == 0
    _near(got[2], want[2], dtype)
    with torch.no_grad():
        assert torch.equal(lm.layer_norm(*dev), y)
    assert all(torch.equal(p, q) for p, q in zip(
        torch.autograd.grad(lm.layer_norm(*dev), dev, gy.cuda()), got))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("affine", ["wb", "w", "b", ""])
def test_layer_norm_float32_affine_and_missing_parts(dtype, affine):
    g = _gen(6)
    x, gy = (torch.randn(6, 50, 96, generator=g).to(dtype) for _ in range(2))
    w = torch.randn(96, generator=g) if "w" in affine else None
    b = torch.randn(96, generator=g) if "b" in affine else None
    ref = [None if t is None else t.double().requires_grad_(True) for t in (x, w, b)]
    dev = [None if t is None else t.cuda().requires_grad_(True) for t in (x, w, b)]
    yr, y = F.layer_norm(ref[0], (96,), ref[1], ref[2], 1e-3), lm.layer_norm(*dev, eps=1e-3)
    assert y.dtype == dtype
    want = torch.autograd.grad(yr, [t for t in ref if t is not None], gy.double())
    got = torch.autograd.grad(y, [t for t in dev if t is not None], gy.cuda())
    _near(y, yr, dtype)
    for p, q in zip(got, want):
        _near(p, q, dtype if p.ndim == 3 else torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D", [(3, 64), (70, 33), (9, 1111), (5, 4096), (2, 8200)])
def test_layer_norm_second_derivative(N, D, dtype):
    g = _gen(N * D)
    x, r, v = (torch.randn(N, D, generator=g).to(dtype) for _ in range(3))
    w, b, vw, vb = (torch.randn(D, generator=g).to(dtype) for _ in range(4))

    def run(fn, dev, dt):
        xs = [t.to(dev, dt or t.dtype).requires_grad_(True) for t in (x, w, b, r)]
        y = fn(xs[0], (D,), xs[1], xs[2])
        grads = torch.autograd.grad(y, xs[:3], xs[3], create_graph=True)
        return torch.autograd.grad(grads, (xs[0], xs[1], xs[3]),
                                   [t.to(dev, dt or t.dtype) for t in (v, vw, vb)])

    want = run(F.layer_norm, "cpu", torch.float64)
    got = run(lambda x, _, w, b: lm.layer_norm(x, w, b), "cuda", None)
    for p, q in zip(got, want):
        _near(p, q, dtype)


def test_layer_norm_second_derivative_of_one_gradient():
    # only gx is used downstream, from a sum: its cotangent arrives broadcast
    g = _gen(17)
    x, r = torch.randn(8, 80, generator=g), torch.randn(8, 80, generator=g)

    def run(fn, dev, dt):
        xd = x.to(dev, dt).requires_grad_(True)
        (gx,) = torch.autograd.grad((fn(xd) * r.to(dev, dt)).sum(), xd, create_graph=True)
        return torch.autograd.grad(gx.square().sum(), xd)[0]

    _near(run(lm.layer_norm, "cuda", torch.float32),
          run(lambda t: F.layer_norm(t, (80,)), "cpu", torch.float64), torch.float32)


def test_layer_norm_keeps_a_large_mean_and_a_flat_row():
    # mean 1000, deviation 1: a variance from E[x^2] - mean^2 would lose it.
    # x itself is float32 (spacing 6e-5 at 1000), the reference takes the same x.
    x = 1000 + torch.randn(4, 512, generator=_gen(7))
    _near(lm.layer_norm(x.cuda()), F.layer_norm(x.double(), (512,)), torch.float32)
    flat = torch.full((2, 64), 3.0, device="cuda")
    assert lm.layer_norm(flat).abs().max() == 0


def test_layer_norm_nan_and_inf_stay_in_their_rows():
    x = torch.randn(5, 300, generator=_gen(8))
    x[1, 7], x[3, 9] = float("nan"), float("inf")
    y = lm.layer_norm(x.cuda())
    assert y[1].isnan().all() and y[3].isnan().all()
    _near(y[[0, 2, 4]], F.layer_norm(x.double(), (300,))[[0, 2, 4]], torch.float32)


def test_layer_norm_strides_empty_and_streams():
    g = _gen(9)
    big = torch.randn(64, 40, 32, generator=g).cuda()
    x = big.transpose(0, 1)[:, ::2]
    _near(lm.layer_norm(x), F.layer_norm(x.double(), (32,)), torch.float32)
    w = torch.ones(32, device="cuda", requires_grad=True)
    y = lm.layer_norm(x[:0], w)
    assert y.shape == (0, 32, 32)
    assert torch.autograd.grad(y, w, torch.empty_like(y))[0].abs().max() == 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = lm.layer_norm(x)
    torch.cuda.current_stream().wait_stream(side)
    _near(y, F.layer_norm(x.double(), (32,)), torch.float32)


def test_layer_norm_offsets_past_32_bits():
    N, D = 1_050_000, 4096
    x = torch.empty(N, D, device="cuda", dtype=torch.bfloat16).normal_().requires_grad_(True)
    y = lm.layer_norm(x)
    _near(y[-3:], F.layer_norm(x.detach()[-3:].double(), (D,)), torch.bfloat16)
    (gx,) = torch.autograd.grad(y, x, x.detach())
    xr = x.detach()[-3:].double().requires_grad_(True)
    (want,) = torch.autograd.grad(F.layer_norm(xr, (D,)), xr, xr.detach())
    # the upstream gradient x is nearly all mean and xhat: gx is what is left,
    # the rounding of x's own 8 bits cancels in it to float32's
    assert (gx[-3:].double() - want).abs().max() <= 2 ** -8 * want.abs().max() + 2 ** -20


def test_layer_norm_gradient_against_differences():
    # float32 central differences of <y, r> along a direction: with step 1e-2
    # the truncation error is ~ 1e-4 of the slope and the float32 sum's
    # rounding ~ 1e-5 / 1e-2; 5e-3 holds both
    g = _gen(10)
    x, r, u = (torch.randn(20, 96, generator=g).cuda() for _ in range(3))
    w, b = (torch.randn(96, generator=g).cuda() for _ in range(2))
    xd = x.clone().requires_grad_(True)
    (gx,) = torch.autograd.grad(lm.layer_norm(xd, w, b), xd, r)
    f = lambda t: (lm.layer_norm(x + t * u, w, b).double() * r.double()).sum()  # noqa: E731
    slope = ((f(1e-2) - f(-1e-2)) / 2e-2).item()
    assert abs((gx * u).sum().item() - slope) <= 5e-3 * max(1.0, abs(slope))


# ------------------------------------------------------- linear cross entropy
def _reference_loss(h, w, t, reduction, g=None):
    h, w = (x.double().requires_grad_(True) for x in (h, w))
    loss = F.cross_entropy(h @ w.t(), t, ignore_index=-100, reduction=reduction)
    return loss, torch.autograd.grad(loss, (h, w), g)


def _terms(h, w, t, c):
    """Sizes of the sums dh = dz w, dw = dz^T h with |dz| taken as c (p + onehot)."""
    h, w, live = h.double(), w.double(), t != -100
    dz = torch.softmax(h @ w.t(), 1)
    dz[live] += F.one_hot(t[live], w.shape[0])
    dz *= (live * c).view(-1, 1)
    return dz @ w.abs(), dz.t() @ h.abs()


XENT_SHAPES = [(1, 1, 1), (1, 2, 8), (3, 32, 64), (64, 32, 64), (65, 33, 63), (130, 257, 72),
               (300, 1000, 136), (7, 5001, 40), (513, 700, 512), (128, 256, 64),
               (1025, 129, 24), (40, 20000, 100)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,D", XENT_SHAPES)
def test_linear_cross_entropy_and_its_gradients(N, V, D, dtype):
    g = _gen(N + V + D)
    h = torch.randn(N, D, generator=g).to(dtype)
    w = (torch.randn(V, D, generator=g) / math.sqrt(D) * 2).to(dtype)
    t = torch.randint(V, (N,), generator=g)
    if N > 2:
        t[torch.randperm(N, generator=g)[:N // 3]] = -100
    # an upstream gradient that keeps float16 results in its normal range
    up = torch.tensor(64.0 * max(1, N // 8))
    loss, (dh, dw) = _reference_loss(h, w, t, "mean", up.double())
    hd, wd = h.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    got = lm.linear_cross_entropy(hd, wd, t.cuda())
    assert got.dtype == torch.float32 and got.shape == ()
    # the loss: float32 sums of exact products
    assert abs(got.item() - loss.item()) <= 4e-6 * max(1.0, abs(loss.item()))
    gh, gw = torch.autograd.grad(got, (hd, wd), up.cuda())
    if V > 1:  # one word: the gradient is exactly 0
        th, tw = _terms(h, w, t, up.item() / (t != -100).sum().item())
        _near(gh, dh, dtype, th)
        _near(gw, dw, dtype, tw)
    else:
        assert gh.abs().max() <= 1e-3 and gw.abs().max() <= 1e-3
    assert gh[t.cuda() == -100].abs().sum() == 0
    with torch.no_grad():
        assert torch.equal(lm.linear_cross_entropy(hd, wd, t.cuda()), got)
    again = torch.autograd.grad(lm.linear_cross_entropy(hd, wd, t.cuda()), (hd, wd), up.cuda())
    assert torch.equal(again[0], gh) and torch.equal(again[1], gw)


@pytest.mark.parametrize("dtype,N,V,D", [(torch.bfloat16, 16384, 20000, 64),
                                         (torch.float32, 8192, 12000, 40)])
def test_linear_cross_entropy_in_pieces_of_the_vocabulary(dtype, N, V, D):
    # dz of all words would take over 512 MB: two pieces, dh added up over them
    g = _gen(18)
    h = torch.randn(N, D, generator=g).to(dtype).cuda().requires_grad_(True)
    w = (torch.randn(V, D, generator=g) / math.sqrt(D)).to(dtype).cuda().requires_grad_(True)
    t = torch.randint(V, (N,), generator=g).cuda()
    t[::7] = -100
    got = lm.linear_cross_entropy(h, w, t, reduction="sum")
    gh, gw = torch.autograd.grad(got, (h, w))
    hr, wr = (x.detach().double().requires_grad_(True) for x in (h, w))
    want = F.cross_entropy(hr @ wr.t(), t, reduction="sum")
    dh, dw = torch.autograd.grad(want, (hr, wr))
    assert abs(got.item() / want.item() - 1) <= 4e-6
    _near(gh, dh, dtype)
    _near(gw, dw, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_linear_cross_entropy_reductions(dtype, reduction):
    g = _gen(12)
    h = torch.randn(4, 50, 96, generator=g).to(dtype)
    w = (torch.randn(300, 96, generator=g) * 0.1).to(dtype)
    t = torch.randint(300, (4, 50), generator=g)
    t[1, 3:20] = -100
    up = torch.randn(4, 50, generator=g) * 10 if reduction == "none" else torch.tensor(3.0)
    if reduction == "none":
        up[..., :1] *= 100
    loss, (dh, dw) = _reference_loss(h.view(-1, 96), w, t.view(-1), reduction,
                                     up.double().view(-1) if up.ndim else up.double())
    hd, wd = h.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    got = lm.linear_cross_entropy(hd, wd, t.cuda().int(), reduction=reduction)
    gh, gw = torch.autograd.grad(got, (hd, wd), up.cuda())
    assert _rel(got.view(-1), loss.view(-1)) <= 4e-6
    _near(gh.view(-1, 96), dh, dtype)
    _near(gw, dw, dtype)


def test_linear_cross_entropy_ignored_rows_may_hold_anything():
    g = _gen(13)
    h, w = torch.randn(200, 64, generator=g), torch.randn(500, 64, generator=g) * 0.2
    t = torch.randint(500, (200,), generator=g)
    drop = torch.rand(200, generator=g) < 0.5
    t[drop] = -100
    clean, (dh, dw) = _reference_loss(h, w, t, "sum")
    for dtype in (torch.float32, torch.bfloat16):
        hd = h.clone()
        hd[drop] = float("nan")
        hd[drop.nonzero()[0, 0]] = float("inf")
        hd = hd.to("cuda", dtype).requires_grad_(True)
        wd = w.to("cuda", dtype).requires_grad_(True)
        got = lm.linear_cross_entropy(hd, wd, t.cuda(), reduction="sum")
        gh, gw = torch.autograd.grad(got, (hd, wd))
        # bfloat16: inputs rounded as well, by 2^-9 each on average
        tol = 4e-6 if dtype == torch.float32 else 1.2e-2
        assert abs(got.item() / clean.item() - 1) <= tol
        assert _rel(gh, dh) <= tol and _rel(gw, dw) <= tol


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_cross_entropy_of_no_row(dtype):
    h = torch.randn(6, 16, device="cuda").to(dtype).requires_grad_(True)
    w = torch.randn(9, 16, device="cuda").to(dtype).requires_grad_(True)
    t = torch.full((6,), -100, device="cuda")
    loss = lm.linear_cross_entropy(h, w, t)
    assert loss.isnan()
    assert all(x.abs().max() == 0 for x in torch.autograd.grad(loss, (h, w)))
    assert lm.linear_cross_entropy(h, w, t, reduction="sum").item() == 0
    assert lm.linear_cross_entropy(h, w, t, reduction="none").tolist() == [0.0] * 6
    empty = lm.linear_cross_entropy(h[:0], w, t[:0], reduction="sum")
    assert empty.item() == 0
    assert torch.autograd.grad(empty, w)[0].abs().max() == 0
    assert lm.linear_cross_entropy(h[:0], w, t[:0]).isnan()
    assert lm.linear_cross_entropy(h[:0], w, t[:0], reduction="none").shape == (0,)


def test_linear_cross_entropy_extreme_scores():
    # scores of +-30000: the running maximum keeps the exponentials finite
    h = torch.tensor([[1.0, 0.0], [0.0, 1.0], [1.0, 1.0]])
    w = torch.tensor([[30000.0, -30000.0], [-30000.0, 30000.0], [0.0, 0.0]])
    t = torch.tensor([0, 0, 2])
    want = F.cross_entropy(h.double() @ w.double().t(), t, reduction="none")
    got = lm.linear_cross_entropy(h.cuda(), w.cuda(), t.cuda(), reduction="none")
    assert (got.cpu().double() - want).abs().max() <= 1e-6 * 60000


def test_linear_cross_entropy_strides_and_one_sided_gradients():
    g = _gen(15)
    big = torch.randn(80, 3, 128, generator=g).bfloat16()
    h, w = big[:, 1, 32:96], torch.randn(64, 150, generator=g).bfloat16().t() * 0.2
    t = torch.randint(150, (80,), generator=g)
    loss, (dh, dw) = _reference_loss(h, w, t, "sum")
    hd, wd = big.cuda()[:, 1, 32:96], w.cuda()
    for need_h, need_w in ((True, False), (False, True), (True, True)):
        a, b = hd.detach().requires_grad_(need_h), wd.detach().requires_grad_(need_w)
        out = lm.linear_cross_entropy(a, b, t.cuda(), reduction="sum")
        got = torch.autograd.grad(out, [x for x, n in ((a, need_h), (b, need_w)) if n])
        for x, y in zip(got, [x for x, n in ((dh, need_h), (dw, need_w)) if n]):
            _near(x, y, torch.bfloat16)


def test_linear_cross_entropy_gradient_against_differences():
    # central differences of the float32 loss (sum over 40 rows, ~ 200) with
    # step 1e-2: rounding 200 * 2^-24 / 1e-2 ~ 1e-3, truncation ~ 1e-4 of the
    # third derivative; 1e-2 holds both for slopes of order one
    g = _gen(16)
    h, u = torch.randn(40, 64, generator=g).cuda(), torch.randn(40, 64, generator=g).cuda()
    w, p = ((torch.randn(200, 64, generator=g) * 0.2).cuda() for _ in range(2))
    t = torch.randint(200, (40,), generator=g).cuda()
    hd, wd = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    gh, gw = torch.autograd.grad(lm.linear_cross_entropy(hd, wd, t, reduction="sum"), (hd, wd))
    f = lambda s: lm.linear_cross_entropy(h + s * u, w + s * p, t, reduction="none").double().sum()  # noqa: E731
    slope = ((f(1e-2) - f(-1e-2)) / 2e-2).item()
    assert abs(((gh * u).sum() + (gw * p).sum()).item() - slope) <= 1e-2 * max(1.0, abs(slope))


def test_linear_cross_entropy_refuses_a_second_derivative():
    h = torch.randn(4, 16, device="cuda", requires_grad=True)
    w = torch.randn(9, 16, device="cuda", requires_grad=True)
    loss = lm.linear_cross_entropy(h, w, torch.arange(4, device="cuda"))
    (gh,) = torch.autograd.grad(loss, h, create_graph=True)
    assert gh.requires_grad  # not silently cut off
    with pytest.raises(RuntimeError, match="differentiable once"):
        gh.sum().backward()


# --------------------------------------------------------- streams and graphs
def _step(ids, target, table, w, b):
    x = lm.embedding(ids, table, scale=4.0)
    loss = lm.linear_cross_entropy(lm.layer_norm(x, w, b), table, target)
    return (loss, *torch.autograd.grad(loss, (table, w, b)))


def _step_inputs(seed):
    g = _gen(seed)
    ids, target = (torch.randint(700, (6, 90), generator=g).cuda() for _ in range(2))
    target[2, 10:] = -100
    table = (torch.randn(700, 64, generator=g) * 0.2).cuda().bfloat16().requires_grad_(True)
    w, b = (torch.randn(64, generator=g).cuda().requires_grad_(True) for _ in range(2))
    return ids, target, table, w, b


def test_training_step_in_a_cuda_graph():
    # captured once, replayed on other tokens: the number of rows that count and
    # the splits chosen from it are found on the device
    ids, target, table, w, b = _step_inputs(20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(ids, target, table, w, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(ids, target, table, w, b)
    ids2, target2, *_ = _step_inputs(21)
    target2[4:] = -100
    for i, t in ((ids2, target2), (ids.clone(), target.clone())):
        ids.copy_(i)
        target.copy_(t)
        graph.replay()
        for x, y in zip(out, _step(i, t, table, w, b)):
            assert torch.equal(x, y)


def test_training_steps_on_two_streams():
    first, second = _step_inputs(22), _step_inputs(23)
    want = [[t.clone() for t in _step(*x)] for x in (first, second)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for k, x in enumerate((first, second)):
            with torch.cuda.stream(streams[k]):
                got[k] = _step(*x)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------ refusals
def test_refusals():
    w = torch.randn(8, 16, device="cuda")
    x, ids = torch.randn(3, 16, device="cuda"), torch.zeros(3, dtype=torch.long, device="cuda")
    cases = [
        (lambda: lm.embedding(ids, w.cpu()), "requires CUDA"),
        (lambda: lm.embedding(ids, w.double()), "Unsupported dtype"),
        (lambda: lm.embedding(ids.float(), w), "int64 or int32"),
        (lambda: lm.embedding(ids.cpu(), w), "ids is on"),
        (lambda: lm.embedding(ids, w[0]), r"\(V,D\)"),
        (lambda: lm.embedding(ids, w, padding_idx=8), "padding_idx"),
        (lambda: lm.layer_norm(x.cpu()), "requires CUDA"),
        (lambda: lm.layer_norm(x.double()), "Unsupported dtype"),
        (lambda: lm.layer_norm(x, w), "weight must have shape"),
        (lambda: lm.layer_norm(x.half(), w[0].bfloat16()), "weight dtype"),
        (lambda: lm.layer_norm(x.half(), w[0].half(), w[0]), "share one dtype"),
        (lambda: lm.linear_cross_entropy(x, w.half(), ids), "share one dtype"),
        (lambda: lm.linear_cross_entropy(x[:, :8], w, ids), "D matching"),
        (lambda: lm.linear_cross_entropy(x, w, ids[:2]), "target shape"),
        (lambda: lm.linear_cross_entropy(x, w, ids.float()), "int64 or int32"),
        (lambda: lm.linear_cross_entropy(x, w, ids, reduction="avg"), "reduction"),
        (lambda: lm.linear_cross_entropy(x.double(), w.double(), ids), "Unsupported dtype"),
    ]
    for call, match in cases:
        with pytest.raises(AssertionError, match=match):
            call()
    assert _lib.device_error() == _lib.THERIA_OK
