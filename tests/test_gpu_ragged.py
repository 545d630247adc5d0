"""sdpa_ragged against a plain float64 attention per sequence and head.

Tolerances, element by element, from the formulas.  u is half a step of the
type (float32: 2^-24).  16-bit kernels round p before p v and p^T do, ds before
ds k and ds^T q, and every result: each is off by u times the same sum of
absolute values.  z = o . do is taken from the rounded o, which is off by
u (p |v| + |o|), so ds is off by p * dz besides.  What float32 adds is at most
(terms of the sum + 8 max|s| + 32) 2^-24 of the sums of absolute values: one
rounding a term, the scores' own error in the exponent, and the exponential's.

float16 has no relative precision below 2^-14: p and ds are off by 2^-25 besides
there (half its smallest step), each time the sum of the sizes that it multiplies;
in the forward p is at least 1 in each row's maximum, and the row's sum l >= 1."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

import theria_b200  # noqa: E402
from theria_b200 import _lib, sdpa_ragged  # noqa: E402
from theria_b200.attention import ragged  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _offsets(lengths, lead=0, dtype=torch.int32):
    return (torch.tensor([0] + list(lengths)).cumsum(0) + lead).to("cuda", dtype)


def _inputs(lengths, H, Hkv, D, dtype, seed=0, lead=0, tail=0):
    g = torch.Generator("cuda").manual_seed(seed)
    T = sum(lengths) + lead + tail
    mk = lambda h: torch.randn(T, h, D, generator=g, device="cuda").to(dtype)  # noqa: E731
    return mk(H), mk(Hkv), mk(Hkv), mk(H)


def _plain(q, k, v, do, lengths, lead, causal, scale):
    """Results, and how far each may be off, in float64."""
    u = torch.finfo(q.dtype).eps / 2
    half, q_type = q.dtype != torch.float32, q.dtype
    q, k, v, do = (t.double() for t in (q, k, v, do))
    G = q.shape[1] // k.shape[1]
    D = q.shape[2]
    out = [torch.zeros_like(t) for t in (q, q, k, v)]
    off = [torch.zeros_like(t) for t in (q, q, k, v)]
    a = lead
    for n in lengths:
        b = a + n
        if n:
            qs, ds_o = q[a:b].transpose(0, 1), do[a:b].transpose(0, 1)
            ks, vs = (t[a:b].transpose(0, 1).repeat_interleave(G, 0) for t in (k, v))
            s = qs @ ks.transpose(1, 2) * scale
            if causal:
                s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1),
                                  -math.inf)
            p = s.softmax(-1)
            o = p @ vs
            dp = ds_o @ vs.transpose(1, 2)
            z = (o * ds_o).sum(-1, keepdim=True)
            ds = p * (dp - z) * scale
            dq, dk, dv = ds @ ks, ds.transpose(1, 2) @ qs, p.transpose(1, 2) @ ds_o
            smax = s[s > -math.inf].abs().max().item()
            f = (max(n, n * G) + D + 8 * smax + 32) * 2.0 ** -24
            w = (u if half else 0.0) + f
            # float16's smallest half step, for each pair that is not masked
            sub = (s > -math.inf).double() * (2.0 ** -25 if q_type is torch.float16 else 0.0)
            a_o = p @ vs.abs()
            e_o = w * a_o + u * o.abs() + sub @ vs.abs()
            # dp - z: float32 sums of D terms, and z from the o that was stored
            e_dp = f * (ds_o.abs() @ vs.abs().transpose(1, 2))
            e_z = (ds_o.abs() * (e_o + f * o.abs())).sum(-1, keepdim=True)
            e_ds = w * ds.abs() + scale * sub + scale * p * (e_dp + e_z + f * (dp - z).abs())
            e_dq = (e_ds + f * ds.abs()) @ ks.abs() + u * dq.abs()
            e_dk = (e_ds + f * ds.abs()).transpose(1, 2) @ qs.abs()
            e_dv = (w * p + sub).transpose(1, 2) @ ds_o.abs()
            per = lambda t: t.unflatten(0, (-1, G)).sum(1)  # noqa: E731
            dk, dv = per(dk), per(dv)
            e_dk, e_dv = per(e_dk) + u * dk.abs(), per(e_dv) + u * dv.abs()
            for dst, t in zip(out + off, (o, dq, dk, dv, e_o, e_dq, e_dk, e_dv)):
                dst[a:b] = t.transpose(0, 1)
        a = b
    return out, off


def _check(lengths, H, Hkv, D, dtype, causal=True, lead=0, tail=0, seed=0, scale=None):
    q, k, v, do = _inputs(lengths, H, Hkv, D, dtype, seed, lead, tail)
    offsets = _offsets(lengths, lead)
    for t in (q, k, v):
        t.requires_grad_(True)
    o = sdpa_ragged(q, k, v, offsets, causal=causal, scale=scale)
    got = [o, *torch.autograd.grad(o, (q, k, v), do)]
    want, off = _plain(q.detach(), k.detach(), v.detach(), do, lengths, lead, causal,
                       scale or D ** -0.5)
    # fp16 results below its smallest normal number lose bits: half its smallest step
    tiny = 2.0 ** -25 if dtype is torch.float16 else 0.0
    for name, g, w, e in zip(("o", "dq", "dk", "dv"), got, want, off):
        assert g.dtype is dtype and g.shape == w.shape
        bad = ((g.double() - w).abs() > 1.01 * e + tiny) | ~torch.isfinite(g)
        assert not bad.any(), (name, bad.nonzero()[:3].tolist(),
                               ((g.double() - w).abs() - e).max().item())
    with torch.no_grad():
        assert torch.equal(o, sdpa_ragged(q, k, v, offsets, causal=causal, scale=scale))


LENGTHS = [[1], [2, 0, 1], [64], [17, 0, 65, 1], [128, 129, 127], [256, 31, 257], [300, 1, 0, 700, 64]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_lengths(lengths, causal, dtype):
    _check(lengths, 4, 2, 64, dtype, causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 9, 16, 20, 32, 40, 72, 80, 96, 100, 127, 128])
def test_head_widths(D, dtype):
    _check([200, 3, 77], 3, 3, D, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hkv", [(1, 1), (5, 1), (6, 2), (7, 1), (8, 1), (24, 2), (64, 1), (65, 1),
                                   (96, 1), (16, 16)])
@pytest.mark.parametrize("D", [64, 128])
def test_groups(H, Hkv, D, dtype):
    _check([150, 1, 40], H, Hkv, D, dtype)
    _check([70, 5], H, Hkv, D, dtype, causal=False, tail=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_long(D, dtype):
    _check([1500, 33, 700], 8, 2, D, dtype)
    _check([2100], 2, 1, D, dtype, causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_no_sequence_and_scale(dtype):
    _check([40, 130], 4, 2, 64, dtype, lead=7, tail=200)
    _check([40, 130], 4, 2, 128, dtype, lead=300, scale=0.3)
    q, k, v, _ = _inputs([5], 2, 1, 64, dtype)
    assert not sdpa_ragged(q, k, v, _offsets([])).any()
    assert sdpa_ragged(q[:0], k[:0], v[:0], _offsets([0, 0])).shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_beyond_32_bits(dtype):
    # heads in rows so long that the last sequence starts beyond 2^31 elements
    lengths, H, Hkv, D = [70000, 300, 129], 2, 1, 64
    T, wide = sum(lengths), 32768
    store = torch.empty(T * wide, dtype=dtype, device="cuda").view(T, wide)
    q, k, v, _ = _inputs(lengths[1:], H, Hkv, D, dtype)
    for t, at in ((q, 0), (k, 1000), (v, 2000)):
        store[lengths[0]:, at:at + t.shape[1] * D] = t.flatten(1)
    views = [store[:, at:at + h * D].view(T, h, D) for h, at in ((H, 0), (Hkv, 1000), (Hkv, 2000))]
    off = _offsets(lengths)[1:]  # the first 70000 tokens belong to none
    x = [t.detach().requires_grad_(True) for t in views]
    y = [t.requires_grad_(True) for t in (q, k, v)]
    a, b = sdpa_ragged(*x, off), sdpa_ragged(*y, _offsets(lengths[1:]))
    assert torch.equal(a[lengths[0]:], b) and not a[:lengths[0]].any()
    # dk and dv are split over another number of parts, so float32 sums of terms that
    # cancel run in another order: against the plain form, with its derived tolerances
    do = torch.ones_like(q)
    want, off_by = _plain(q.detach(), k.detach(), v.detach(), do, lengths[1:], 0, True, D ** -0.5)
    for g, w, e in zip(torch.autograd.grad(a.sum(), x), want[1:], off_by[1:]):
        assert not g[:lengths[0]].any()
        assert ((g[lengths[0]:].double() - w).abs() <= 1.01 * e).all()


def test_many_sequences():
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 9, (1500,), generator=g).tolist()
    for dtype in DTYPES:
        _check(lengths, 2, 1, 64, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hkv", [(4, 2), (6, 2)])
def test_nothing_outside_a_sequence_reaches_it(dtype, D, causal, H, Hkv):
    lengths = [70, 130, 50, 260]
    q, k, v, do = _inputs(lengths, H, Hkv, D, dtype, lead=9, tail=40)
    offsets = _offsets(lengths, 9)

    def run():
        x = [t.clone().requires_grad_(True) for t in (q, k, v)]
        o = sdpa_ragged(*x, offsets, causal=causal)
        return [o.detach(), *torch.autograd.grad(o, x, do)]

    before = run()
    rows = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    for a, b, value in ((0, 9, math.nan), (9, 79, math.nan), (209, 259, math.inf), (519, 559, -math.inf)):
        for t in (q, k, v, do):
            t[a:b] = value
        rows[a:b] = False
    for x, y in zip(before, run()):
        assert torch.equal(x[rows], y[rows])
        assert not y[:9].any() and not y[519:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    # heads split out of a fused projection, heads-first memory, expanded and reversed tensors
    lengths, H, Hkv, D = [90, 41, 6], 4, 2, 64
    T = sum(lengths)
    g = torch.Generator("cuda").manual_seed(1)
    rows = torch.randn(T, H + 2 * Hkv, D, generator=g, device="cuda").to(dtype)
    heads = torch.randn(H, T, D, generator=g, device="cuda").to(dtype)
    odd = torch.randn(T, H * D + 3, generator=g, device="cuda").to(dtype)[:, 1:1 + H * D]
    cases = [
        (rows[:, :H], rows[:, H:H + Hkv], rows[:, H + Hkv:]),
        (heads.transpose(0, 1), rows[:, :Hkv], rows[:, Hkv:2 * Hkv]),
        (odd.view(T, H, D), rows[:, :Hkv], rows[:, 1:1 + Hkv]),
        (rows[:, :H], rows[:, :1].expand(T, Hkv, D), rows[:, 2:3].expand(T, Hkv, D)),
        (rows[:, 0:8:2], rows[:, 0:4:2], rows.flip(0)[:, 1:5:2]),
        (rows.transpose(1, 2).contiguous().transpose(1, 2)[:, :H], rows[:, :Hkv], rows[:, :Hkv]),
    ]
    do = torch.randn(H, T, D, generator=g, device="cuda").to(dtype).transpose(0, 1)
    offsets = torch.stack([_offsets(lengths, dtype=torch.int64)] * 2, 1)[:, 0]  # strided, int64
    for case in cases:
        x = [t.detach().requires_grad_(True) for t in case]
        y = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
             for t in case]
        a = sdpa_ragged(*x, offsets)
        b = sdpa_ragged(*y, _offsets(lengths))
        assert torch.equal(a, b)
        for s, t in zip(torch.autograd.grad(a, x, do), torch.autograd.grad(b, y, do.contiguous())):
            assert torch.equal(s, t)


@pytest.mark.parametrize("dtype", DTYPES)
def test_partial_gradients_and_expanded_cotangent(dtype):
    lengths = [60, 200]
    q, k, v, _ = _inputs(lengths, 4, 2, 64, dtype)
    offsets = _offsets(lengths)
    full = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(sdpa_ragged(*full, offsets).sum(), full)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        x = [t.clone().requires_grad_(bool(n)) for t, n in zip((q, k, v), need)]
        got = torch.autograd.grad(sdpa_ragged(*x, offsets).sum(), [t for t, n in zip(x, need) if n])
        for g, w in zip(got, [w for w, n in zip(want, need) if n]):
            assert torch.equal(g, w)


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits_and_streams_and_capture(dtype):
    lengths = [500, 33, 700]
    q, k, v, do = _inputs(lengths, 8, 1, 64, dtype)
    offsets = _offsets(lengths)

    def step(x):
        o = sdpa_ragged(*x, offsets)
        return [o.detach(), *torch.autograd.grad(o, x, do)]

    first = step([t.clone().requires_grad_(True) for t in (q, k, v)])
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    both = []
    for s in side:
        with torch.cuda.stream(s):
            both.append(step([t.clone().requires_grad_(True) for t in (q, k, v)]))
    torch.cuda.synchronize()
    for res in both:
        for a, b in zip(first, res):
            assert torch.equal(a, b)
    # captured once; replayed with other values and other lengths of as many tokens
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    with torch.cuda.stream(side[0]):
        step(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x)
    new = _offsets([100, 1000, 133])
    with torch.no_grad():
        for t, s in zip(x, (q, k, v)):
            t.copy_(s * 0.5)
    offsets.copy_(new)
    graph.replay()
    graph.replay()
    want = step([(t * 0.5).requires_grad_(True) for t in (q, k, v)])
    for a, b in zip(out, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bad", [[0, 30, 20, 50], [-1, 20], [0, 20, 51], [5, 4]], ids=str)
def test_bad_offsets_give_zeros_and_an_error(bad):
    for dtype in DTYPES:
        x = [t.requires_grad_(True) for t in _inputs([50], 4, 2, 64, dtype)[:3]]
        for od in (torch.int32, torch.int64):
            o = sdpa_ragged(*x, torch.tensor(bad, device="cuda", dtype=od))
            grads = torch.autograd.grad(o.sum(), x)
            assert not o.any() and not any(g.any() for g in grads)
            with pytest.raises(_lib.TheriaError):
                theria_b200.check_device_error()


def test_derivatives_against_differences():
    # float64 differences of the plain form are not the kernels': take the kernels' own,
    # float32, along random directions; step 2^-6, third derivatives of order 1: 2^-12 and
    # float32's 2^-24 / 2^-6 of values of order 10
    lengths = [30, 75]
    q, k, v, do = _inputs(lengths, 4, 2, 32, torch.float32)
    offsets = _offsets(lengths)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    o = sdpa_ragged(*x, offsets)
    grads = torch.autograd.grad(o, x, do)
    g = torch.Generator("cuda").manual_seed(9)
    for i in range(3):
        u = torch.randn(x[i].shape, generator=g, device="cuda")
        u /= u.norm()
        vals = []
        for s in (2.0 ** -6, -2.0 ** -6):
            y = [t.detach() + (s * u if j == i else 0) for j, t in enumerate(x)]
            vals.append((sdpa_ragged(*y, offsets).double() * do.double()).sum().item())
        fd = (vals[0] - vals[1]) / 2.0 ** -5
        assert abs(fd - (grads[i].double() * u.double()).sum().item()) < 2e-3


def test_refusals():
    q, k, v, _ = _inputs([8], 4, 2, 16, torch.float32)
    off = _offsets([8])
    call = lambda *a, **kw: pytest.raises(AssertionError, match=kw.pop("match"))  # noqa: E731
    bad = [
        ((q.cpu(), k, v, off), "requires CUDA"), ((q.double(), k, v, off), "Unsupported dtype"),
        ((q[0], k, v, off), "q must"), ((q, k[:7], v, off), "k must"),
        ((q, k[:, :1].expand(8, 3, 16), v, off), "k must"), ((q, k, v[:, :1], off), "v must"),
        ((q, k.half(), v, off), "share one dtype"), ((q, k, v, off.float()), "offsets must be"),
        ((q, k, v, off.cpu()), "offsets is on"), ((q, k, v, off[:0]), "offsets must have"),
        ((q, k, v, off[None]), "offsets must have"),
        ((torch.zeros(2, 1, 129, device="cuda"),) * 3 + (off,), "D<=128"),
    ]
    for args, match in bad:
        with call(match=match):
            sdpa_ragged(*args)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with call(match="scale must"):
            sdpa_ragged(q, k, v, off, scale=scale)


def test_second_derivative_and_forward_mode_are_refused():
    x = [t.requires_grad_(True) for t in _inputs([8], 2, 1, 16, torch.float32)[:3]]
    off = _offsets([8])
    (g,) = torch.autograd.grad(sdpa_ragged(*x, off).square().sum(), x[:1], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x[0].detach(), torch.ones_like(x[0]))
        with pytest.raises(NotImplementedError):
            sdpa_ragged(dual, x[1].detach(), x[2].detach(), off)


def test_workspace_and_arguments_at_the_c_entry():
    lib = _lib.load()
    assert lib.theria_ragged_fwd_workspace_bytes(100, 3, 4, 3) == 0  # H not a multiple
    assert lib.theria_ragged_fwd_workspace_bytes(100, 3, 4, 2) > 0
    assert ragged._strides(*(torch.zeros(2, 2, 4),) * 3)[0] == 8


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_that_no_address_uses(dtype):
    # a single key head, a single token: their strides may be any number
    q, k, v, _ = _inputs([70, 9], 4, 1, 64, dtype)
    odd = [t.as_strided(t.shape, (64, 5, 1)) for t in (k, v)]
    off = _offsets([70, 9])
    assert torch.equal(sdpa_ragged(q, *odd, off), sdpa_ragged(q, k, v, off))
    one = [t[:1].as_strided((1, *t.shape[1:]), (3, 64, 1)) for t in (q, k, v)]
    off = _offsets([1])
    assert torch.equal(sdpa_ragged(*one, off), sdpa_ragged(q[:1], k[:1], v[:1], off))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("G", [33, 48, 63])
def test_groups_of_one_token_a_tile(G, dtype):
    # a tile of 64 rows holds one token, and rows that no copy fills
    _check([90, 0, 33, 1], 2 * G, 2, 128, dtype)
    _check([50, 7], G, 1, 72, dtype, causal=False, lead=2)
