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
# Scores are sums of D products to which the tensor cores add 16 at a time; each
# addition cuts the sum by less than a unit in its last place, 2^-23 of the next
# power of two above the largest score: `_score_error` for the difference of two
# scores.  Against that, and relative to the result, stands what float32 softmax
# arithmetic around the maximum costs in absolute terms: sums of V exponentials
# beside a 1 go through at most 20 roundings of 2^-24 (8 in a chain of a row's 32
# columns, 5 for joining chains and blocks, 7 for the tiles and the logarithm),
# which over many rows average to the size of 3.
def _score_error(top, D):
    return 2 * math.ceil(D / 16) * 2.0 ** -23 * 2.0 ** math.ceil(math.log2(top))


def _certain(N, V, D, score, gap, dtype, seed):
    """Targets whose score is about `score`, `gap` above all others'."""
    g = _gen(seed)
    w = torch.randn(V, D, generator=g) / math.sqrt(D)
    t = torch.randint(V, (N,), generator=g)
    h = gap * w[t]
    h[:, 0], w[:, 0] = 8.0, (score - gap) / 8  # the others' common score
    return h.to(dtype), w.to(dtype), t


def _exact_loss(h, w, t):
    """loss, dz and z_t - lse of each row, in float64 without cancellation."""
    z = h.double() @ w.double().t()
    z = z - z.gather(1, t[:, None])
    others = z.exp().scatter(1, t[:, None], 0.0).sum(1)
    dz = z.exp() / (1 + others)[:, None]
    dz.scatter_(1, t[:, None], (-others / (1 + others))[:, None])
    return torch.log1p(others), dz


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score,gap", [(20, 8), (20, 20), (60, 14), (100, 8), (100, 20)])
@pytest.mark.parametrize("N,V,D", [(200, 256, 64), (300, 1000, 72)])
def test_loss_and_gradients_of_nearly_certain_tokens(N, V, D, score, gap, dtype):
    h, w, t = _certain(N, V, D, float(score), float(gap), dtype, score + gap + N)
    want, dz = _exact_loss(h, w, t)
    rel = _score_error(2 * score, D) + 2 ** -21  # of a small loss, and of its gradient
    hd, wd = h.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    loss = lm.linear_cross_entropy(hd, wd, t.cuda(), reduction="none")
    err = (loss.detach().cpu().double() - want).abs()
    assert (loss >= 0).all()
    assert (err <= rel * want + 20 * 2 ** -24).all()
    assert err.mean() <= rel * want.mean() + 3 * 2 ** -24
    # an upstream gradient that keeps float16 results above their smallest numbers
    (gh,) = torch.autograd.grad(loss, hd, torch.full_like(loss, 1024.0))
    dh = dz @ w.double()
    size = dz.abs() @ w.double().abs()  # of dh's terms
    # dz in 16 bits: 2^-8 and 2^-11 of each, and the result's own rounding
    unit = {torch.float32: 2 ** -22, torch.float16: 2 ** -10, torch.bfloat16: 2 ** -7}[dtype]
    err = (gh.cpu().double() / 1024 - dh).abs()
    p = 2 ** -24 * w.double().abs()[t]  # the absolute error is that of the target's term
    tiny = 2 ** -34 if dtype == torch.float16 else 0.0  # the spacing of its smallest numbers
    assert (err <= (rel + unit) * size + 20 * p + tiny).all()
    assert err.mean() <= (rel + unit) * size.mean() + 3 * p.mean() + tiny


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 2048])
def test_loss_of_one_word_is_exactly_zero(D, dtype):
    g = _gen(D)
    h, w = torch.randn(90, D, generator=g).to(dtype), torch.randn(1, D, generator=g).to(dtype)
    hd, wd = h.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    loss = lm.linear_cross_entropy(hd, wd, torch.zeros(90, dtype=torch.long, device="cuda"),
                                   reduction="none")
    assert (loss == 0).all()
    for grad in torch.autograd.grad(loss, (hd, wd), torch.ones_like(loss)):
        assert (grad == 0).all()


def test_loss_of_extreme_scores_to_its_own_size():
    h = torch.tensor([[1.0, 0.0], [0.0, 1.0], [1.0, 1.0], [0.0, 1.0]])
    w = torch.tensor([[30000.0, -30000.0], [-30000.0, 30000.0], [0.0, 0.0]])
    t = torch.tensor([0, 0, 2, 1])
    want = torch.tensor([0.0, 60000.0, math.log(3.0), 0.0], dtype=torch.float64)
    for dtype in (torch.float32, torch.bfloat16):
        wd = w.to(dtype)
        scale = wd[0, 0].item() / 30000  # bfloat16 has no 30000
        got = lm.linear_cross_entropy(h.to("cuda", dtype), wd.cuda(), t.cuda(), reduction="none")
        want_d = want * torch.tensor([1, scale, 1, 1])
        assert ((got.cpu().double() - want_d).abs() <= 2 ** -22 * want_d).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,V", [(70, 512), (3, 300)])
def test_gradients_of_certain_tokens_in_wide_rows(N, V, dtype):
    # few tiles of wide 16-bit rows: the backward's scores have to be the
    # forward's to the bit, or their difference is what is left of p - 1
    D = 2048
    h, w, t = _certain(N, V, D, 60.0, 14.0, dtype, V)
    want, dz = _exact_loss(h, w, t)
    hd, wd = h.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    loss = lm.linear_cross_entropy(hd, wd, t.cuda(), reduction="none")
    (gh,) = torch.autograd.grad(loss, hd, torch.full_like(loss, 1024.0))
    dh, size = dz @ w.double(), dz.abs() @ w.double().abs()
    unit = {torch.float16: 2 ** -10, torch.bfloat16: 2 ** -7}[dtype]
    err = (gh.cpu().double() / 1024 - dh).abs()
    p = 2 ** -24 * w.double().abs()[t]
    assert (err <= (_score_error(120, D) + unit) * size + 20 * p + 2 ** -34).all()
    assert err.mean() <= (_score_error(120, D) + unit) * size.mean() + 3 * p.mean() + 2 ** -34


def test_float32_products_keep_their_low_bits():
    # 1 + 2^-7 - 2^-23 as bfloat16 parts cut toward zero leaves products 7.8 * 2^-24
    # short.  Here: at most one unit for what three parts rounded to nearest leave
    # out, one for the accumulator's cut, half a one for the last rounding.
    x = 1 + 2.0 ** -7 - 2.0 ** -23
    bound = 2.5 * 2.0 ** -23
    h = torch.full((8, 16), x, device="cuda")
    w = torch.zeros(2, 16, device="cuda")
    w[0] = x
    one = torch.ones(8, dtype=torch.long, device="cuda")
    loss = lm.linear_cross_entropy(h, w, one, reduction="none").cpu().double()
    z = 16 * x * x
    assert (loss / (z + math.log1p(math.exp(-z))) - 1).abs().max() <= bound
    # scores of 0: dz = +-x for the upstream gradient 2 x, and dh = x * x
    hz = torch.zeros(8, 16, device="cuda", requires_grad=True)
    w = torch.zeros(2, 16, device="cuda")
    w[1] = -x
    loss = lm.linear_cross_entropy(hz, w, one, reduction="none")
    (gh,) = torch.autograd.grad(loss, hz, torch.full_like(loss, 2 * x))
    assert (gh.cpu().double() / (x * x) - 1).abs().max() <= bound


def test_float32_loss_of_the_largest_numbers():
    # rounded to nearest, the leading part of the largest float32 would be infinite
    big = torch.finfo(torch.float32).max
    h = torch.tensor([[big], [-big]], device="cuda")
    w = torch.tensor([[2.0 ** -120], [0.0]], device="cuda", requires_grad=True)
    loss = lm.linear_cross_entropy(h, w, torch.tensor([1, 0], device="cuda"), reduction="none")
    assert ((loss.detach().cpu().double() / (big * 2.0 ** -120)) - 1).abs().max() <= 2 ** -20
    (gw,) = torch.autograd.grad(loss, w, torch.tensor([1.0, 0.0], device="cuda"))
    want = torch.tensor([big, -big]).double()
    assert (gw[:, 0].cpu().double() / want - 1).abs().max() <= 2 ** -20
    hs = torch.zeros(1, 1, device="cuda", requires_grad=True)
    ws = torch.tensor([[0.5], [-0.5]], device="cuda")
    loss = lm.linear_cross_entropy(hs, ws, torch.zeros(1, dtype=torch.long, device="cuda"),
                                   reduction="none")
    (gh,) = torch.autograd.grad(loss, hs, torch.full_like(loss, big))
    assert abs(gh.item() / (-0.5 * big) - 1) <= 2 ** -20


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,live", [(64, 64), (65, 1), (500, 3), (1000, 64)])
def test_few_scored_rows_among_many_keep_their_gradients(N, live, dtype):
    # The rows that count decide how finely dz is held: the error is that of the
    # results' own rounding (a fifth more for results that round the other way).
    g = _gen(N + live)
    D, V = 256, 700
    h = torch.randn(N, D, generator=g).to(dtype)
    w = (torch.randn(V, D, generator=g) * 0.2).to(dtype)
    t = torch.full((N,), -100)
    t[torch.randperm(N, generator=g)[:live]] = torch.randint(V, (live,), generator=g)
    up = 64.0
    hr, wr = h.double().requires_grad_(True), w.double().requires_grad_(True)
    want = torch.autograd.grad(F.cross_entropy(hr @ wr.t(), t, reduction="sum"), (hr, wr),
                               torch.tensor(up).double())
    hd, wd = h.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    loss = lm.linear_cross_entropy(hd, wd, t.cuda(), reduction="sum")
    got = torch.autograd.grad(loss, (hd, wd), torch.tensor(up, device="cuda"))
    for a, b in zip(got, want):
        assert _rel(a, b) <= 1.2 * _rel(b.to(dtype), b)


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


# ----------------------------------------------------------------- layer norm
def _norm_grads(fn, x, w, b, gy, dev, dt):
    xs = [t.to(dev, dt).requires_grad_(True) for t in (x, w, b)]
    g = gy.to(dev, dt).requires_grad_(True)
    y = fn(*xs)
    first = torch.autograd.grad(y, xs, g, create_graph=True)
    second = torch.autograd.grad(first[0], (xs[0], xs[1], g), g.detach().roll(1, 0))
    return [t.detach() for t in (y, *first, *second)]


@pytest.mark.parametrize("N,D", [(64, 512), (70, 64), (64, 511), (33, 4096), (5, 16392),
                                 (3, 33001)])
@pytest.mark.parametrize("mean", [100.0, 1000.0, 10000.0])
def test_layer_norm_gradients_of_rows_with_a_large_mean(N, D, mean):
    # x - mean is exact near the mean: nothing is lost that float32 rows around
    # zero would keep, so the bound is theirs (64 units of 2^-24)
    g = _gen(N + D)
    x = mean + torch.randn(N, D, generator=g)
    w, b = 1 + 0.3 * torch.randn(D, generator=g), torch.randn(D, generator=g)
    gy = torch.randn(N, D, generator=g)
    got = _norm_grads(lm.layer_norm, x, w, b, gy, "cuda", torch.float32)
    want = _norm_grads(lambda x, w, b: F.layer_norm(x, (D,), w, b), x, w, b, gy, "cpu",
                       torch.float64)
    for p, q in zip(got, want):
        assert _rel(p, q) <= 4e-6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,D", [(5, 12808), (3, 16384), (4, 16385), (2, 32768), (3, 32776),
                                 (2, 40001)])
def test_layer_norm_of_the_widest_rows(N, D, dtype):
    # past each width that a kernel keeps in registers or in its ring: forward up
    # to 32768, backward and second derivative up to 16384
    tol = {torch.float32: 4e-6, torch.float16: 8e-4, torch.bfloat16: 6e-3}[dtype]
    g = _gen(N + D)
    x, w, b, gy = (torch.randn(*s, generator=g).to(dtype) for s in ((N, D), (D,), (D,), (N, D)))
    got = _norm_grads(lm.layer_norm, x, w, b, gy, "cuda", dtype)
    want = _norm_grads(lambda x, w, b: F.layer_norm(x, (D,), w, b), x, w, b, gy, "cpu",
                       torch.float64)
    for p, q in zip(got, want):
        assert _rel(p, q) <= tol
