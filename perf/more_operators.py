"""Timed cases of the operators of a decoder's training step on packed text.

Sequences of different lengths lie one after the other in one row of tokens:
rotary positions of the queries and keys (``theria_b200.lm.rotary``), attention
within each sequence with grouped heads and its gradients
(``theria_b200.sdpa_ragged``), and at the step's end the gradients clipped by
their global norm, differentiable for adapted (inner-loop) steps
(``theria_b200.lm.clip_gradients``).  ``own`` chooses who computes a pass: the
plain forms below (elementary torch operations in float32, angles in float64,
rounded once), or the framework's operators as a user's program calls them.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------ the cases
# lengths: "64x25" is 25 sequences of 64 tokens, "," joins; padding: tokens
# behind the last sequence that belong to none.
def listed():
    return [
        # the MAML classifier's support set: 25 sequences of 64 tokens, 4 heads of 16
        dict(name="ragged train 25x64 f32", op="ragged", train=True, lengths="64x25", padding=0,
             heads=4, kv_heads=4, d=16, dtype="f32", causal=False),
        # one short prompt: latency
        dict(name="ragged prompt 17", op="ragged", train=False, lengths="17", padding=0, heads=8,
             kv_heads=2, d=64, dtype="bf16", causal=True),
        # a packed training batch of a mid-sized model, ragged, with padding behind it
        dict(name="ragged train 16k D64", op="ragged", train=True,
             lengths="4096,2500,2048x2,1111,1024x2,777,512x2,300,200,128,64,33,1,0,5", padding=105,
             heads=16, kv_heads=4, d=64, dtype="bf16", causal=True),
        # a large training batch of long sequences in a wide model
        dict(name="ragged train 32k D128", op="ragged", train=True,
             lengths="8192x2,4096x2,2048x2,1500,1000,900,500,196", padding=0, heads=32,
             kv_heads=8, d=128, dtype="bf16", causal=True),
        # one long prompt
        dict(name="ragged prompt 16384", op="ragged", train=False, lengths="16384", padding=0,
             heads=32, kv_heads=8, d=128, dtype="bf16", causal=True),
        # odd sizes: three heads a group, a head width between the tile widths
        dict(name="ragged train odd f16", op="ragged", train=True,
             lengths="1021,17,2003,640,5,333", padding=13, heads=6, kv_heads=2, d=80,
             dtype="f16", causal=True),
        # full precision, one key head for all query heads
        dict(name="ragged train odd f32", op="ragged", train=True, lengths="999,30,1301,64,1",
             padding=0, heads=5, kv_heads=1, d=72, dtype="f32", causal=True),
        # the next token of 8 sequences, far out in a context scaled eight times
        dict(name="rotary 8 tokens", op="rotary", train=False, tokens=8, sequences=0, heads=32,
             kv_heads=8, d=128, dim=128, dtype="bf16", interleaved=False, scaling="linear",
             far=1 << 20),
        # a training batch of packed sequences, positions counted within each
        dict(name="rotary train 32768", op="rotary", train=True, tokens=32768, sequences=11,
             heads=32, kv_heads=8, d=128, dim=128, dtype="bf16", interleaved=True, scaling="none",
             far=0),
        # part of an odd head in full precision, interpolated by wavelength
        dict(name="rotary train odd f32", op="rotary", train=True, tokens=5003, sequences=7,
             heads=6, kv_heads=2, d=80, dim=30, dtype="f32", interleaved=False,
             scaling="by_parts", far=0),
        # the inner-loop gradients of the MAML classifier, clipped and differentiated through
        dict(name="clip train 106565", op="clip", train=True, layers=2, width=64, vocab=32,
             dtype="f32", ratio=4.0),
        # all gradients of a small stack of wide layers and a large vocabulary
        dict(name="clip 403M", op="clip", train=False, layers=4, width=2048, vocab=98304,
             dtype="bf16", ratio=4.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ragged", "ragged", "ragged", "rotary", "clip"])
    train = rng.random() < 0.7
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 8])
    if op == "clip":
        width = _log_uniform(rng, 32, 1024 if train else 2048)
        return dict(op=op, train=train, layers=rng.randint(1, 2 if train else 4), width=width,
                    vocab=_log_uniform(rng, 32, 32768), dtype=dtype,
                    ratio=rng.choice([0.5, 2.0, 30.0]))
    if op == "rotary":
        d = rng.choice([16, 32, 64, 80, 96, 128, 128])
        dim = d if rng.random() < 0.6 else 2 * rng.randint(1, d // 2)
        tokens = _log_uniform(rng, 1, 32768 if dtype != "f32" else 16384)
        packed = rng.random() < 0.5
        return dict(op=op, train=train, tokens=tokens,
                    sequences=_log_uniform(rng, 1, 64) if packed else 0, heads=heads, kv_heads=kv,
                    d=d, dim=dim, dtype=dtype, interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "by_parts"]),
                    far=0 if packed else rng.choice([4096, 1 << 20]))
    d = rng.choice([16, 32, 64, 64, 72, 96, 100, 128, 128, rng.randint(9, 128)])
    # no costlier than the largest listed case (float32: a 256th of its products)
    cap = (2.8e12 if dtype != "f32" else 1.1e10) / (1.0 if train else 0.5)
    lengths, left = [], rng.choice([1, 2, 4, 12, 40])
    total = 0
    while left > 0:
        n = rng.choice([0, 1, _log_uniform(rng, 2, 300), _log_uniform(rng, 16, 8192),
                        _log_uniform(rng, 128, 8192)])
        left -= 1
        if total + heads * d * n * n > cap or sum(lengths) + n > 32768:
            continue
        total += heads * d * n * n
        lengths.append(n)
    if sum(lengths) == 0:
        lengths.append(rng.randint(1, 64))
    return dict(op=op, train=train, lengths=",".join(map(str, lengths)),
                padding=rng.choice([0, 0, rng.randint(1, 200)]), heads=heads, kv_heads=kv, d=d,
                dtype=dtype, causal=rng.random() < 0.8)


def _lengths(case):
    out = []
    for part in case["lengths"].split(","):
        n, _, times = part.partition("x")
        out += [int(n)] * int(times or 1)
    return out


def _shapes(case):
    """The parameters of a pre-LN decoder with tied embeddings."""
    w = case["width"]
    block = [(w,), (w,), (3 * w, w), (3 * w,), (w, w), (w,), (w,), (w,), (4 * w, w), (4 * w,),
             (w, 4 * w), (w,)]
    return [(case["vocab"], w), (64, w)] + block * case["layers"] + [(w,), (w,), (5, w), (5,)]


def work(case):
    e = SIZES[case["dtype"]]
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        # gradients in, clipped out; the cotangents in, their gradient out
        return {"bytes": (4 if case["train"] else 2) * n * e,
                "flops": (8 if case["train"] else 3) * n}
    if case["op"] == "rotary":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        passes = 4 if case["train"] else 2
        return {"bytes": passes * n * case["d"] * e + 8 * case["tokens"],
                "flops": (passes // 2) * 3 * n * case["dim"]}
    ns, d, h = _lengths(case), case["d"], case["heads"]
    rows = (sum(ns) + case["padding"]) * d * e * (2 * h + 2 * case["kv_heads"])
    pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in ns)
    return {"bytes": rows * (2 if case["train"] else 1) + 8 * len(ns),
            "flops": (14 if case["train"] else 4) * pairs * d * h}


# ----------------------------------------------------------------- the inputs
def _frequencies(case, g):
    """The angular frequencies of the pairs, in 64 bits."""
    dim, base, factor, original = case["dim"], 10000.0, 8.0, 4096
    i = torch.arange(0, dim, 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "ntk" and dim > 2:
        base *= factor ** (dim / (dim - 2))
    f = base ** (-i / dim)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "by_parts":
        turns = original * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
    return f


def _offsets(lengths):
    at = torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0)
    return at.to("cuda", torch.int32)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt, train = DTYPES[case["dtype"]], case["train"]

    def normal(*shape, std=1.0):
        return torch.empty(shape, device="cuda", dtype=dt).normal_(0.0, std, generator=g)

    s = dict(case)
    if case["op"] == "clip":
        scales = torch.rand(len(_shapes(case)), generator=g, device="cuda").tolist()
        grads = [normal(*shape, std=1e-3 * 10 ** (2 * x))
                 for shape, x in zip(_shapes(case), scales)]
        if train:
            s["cotangents"] = [normal(*shape) for shape in _shapes(case)]
        size = sum(math.prod(shape) * (1e-3 * 10 ** (2 * x)) ** 2
                   for shape, x in zip(_shapes(case), scales))
        s["max_norm"] = math.sqrt(size) / case["ratio"]
        s["grads"] = [t.requires_grad_(train) for t in grads]
        return s
    h, hk, d = case["heads"], case["kv_heads"], case["d"]
    if case["op"] == "rotary":
        n = case["tokens"]
        # queries and keys as a fused projection leaves them: heads side by side in a row
        rows = normal(n, h + 2 * hk, d)
        s["q"] = rows[:, :h].detach().requires_grad_(train)
        s["k"] = rows[:, h:h + hk].detach().requires_grad_(train)
        s["frequencies"] = _frequencies(case, g)
        s["amplitude"] = 0.1 * math.log(8.0) + 1.0 if case["scaling"] == "by_parts" else 1.0
        s["positions"] = s["offsets"] = None
        if case["sequences"]:
            cut = torch.randint(0, n + 1, (case["sequences"] - 1,), generator=g, device="cuda")
            cut = cut.sort().values.tolist()
            s["lengths"] = [b - a for a, b in zip([0] + cut, cut + [n])]
            s["offsets"] = _offsets(s["lengths"])
        else:
            s["positions"] = torch.randint(0, case["far"], (n,), generator=g, device="cuda")
        if train:
            s["gq"], s["gk"] = normal(n, h, d), normal(n, hk, d)
        return s
    s["lengths"] = _lengths(case)
    n = sum(s["lengths"]) + case["padding"]
    s["offsets"] = _offsets(s["lengths"])
    s["q"] = normal(n, h, d).requires_grad_(train)
    s["k"] = normal(n, hk, d).requires_grad_(train)
    s["v"] = normal(n, hk, d).requires_grad_(train)
    if train:
        s["go"] = normal(n, h, d)
    return s


# ---------------------------------------------------------------- plain forms
def _rotate(s, x, positions, back):
    dim, dt = s["dim"], x.dtype
    angle = positions.double()[:, None, None] * s["frequencies"]
    c = (angle.cos() * s["amplitude"]).float()
    n = (angle.sin() * s["amplitude"]).float()
    if back:
        n = -n
    y = x.float().clone()
    if s["interleaved"]:
        a, b = slice(0, dim, 2), slice(1, dim, 2)
    else:
        a, b = slice(0, dim // 2), slice(dim // 2, dim)
    y[..., a] = x[..., a].float() * c - x[..., b].float() * n
    y[..., b] = x[..., b].float() * c + x[..., a].float() * n
    return y.to(dt)


def _rotary(s):
    if s["positions"] is not None:
        at = s["positions"]
    else:
        i = torch.arange(s["tokens"], device="cuda")
        start = s["offsets"][torch.searchsorted(s["offsets"][1:], i, right=True)]
        at = i - start
    y = _rotate(s, s["q"], at, False), _rotate(s, s["k"], at, False)
    if not s["train"]:
        return y
    return (*y, _rotate(s, s["gq"], at, True), _rotate(s, s["gk"], at, True))


def _attend(s, q, k, v, go):
    """Sequences of one length side by side: q [N, Hkv, G, n, D], k, v [N, Hkv, 1, n, D]."""
    n, scale = q.shape[3], 1.0 / math.sqrt(s["d"])
    p = (q @ k.transpose(-1, -2)).mul_(scale)
    if s["causal"]:
        i = torch.arange(n, device=q.device)
        p.masked_fill_(i[None, :] > i[:, None], -math.inf)
    p = p.sub_(p.max(-1, keepdim=True).values).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    o = p @ v
    if go is None:
        return o, None, None, None
    dv = (p.transpose(-1, -2) @ go).sum(2)
    dp = go @ v.transpose(-1, -2)
    ds = p.mul_(dp.sub_((go * o).sum(-1, keepdim=True))).mul_(scale)
    return o, ds @ k, (ds.transpose(-1, -2) @ q).sum(2), dv


def _ragged(s):
    q, k, v, go = s["q"], s["k"], s["v"], s.get("go")
    h, hk, d = s["heads"], s["kv_heads"], s["d"]
    out = [torch.zeros_like(t) for t in (q, q, k, v)]
    starts = [0]
    for n in s["lengths"]:
        starts.append(starts[-1] + n)
    groups = {}
    for n, at in zip(s["lengths"], starts):
        groups.setdefault(n, []).append(at)
    for n, ats in groups.items():
        if n == 0:
            continue
        # one or all key heads and sequences at a time: at most 4 GB of scores
        heads = hk if 4 * h * n * n <= 2 ** 32 else 1
        some = max(1, 2 ** 32 // (4 * (h // hk) * heads * n * n))
        for j in range(0, len(ats), some):
            rows = (torch.tensor(ats[j:j + some], device="cuda")[:, None]
                    + torch.arange(n, device="cuda"))

            def take(t, c):
                t = t[rows].float().view(*rows.shape, hk, -1, d)[:, :, c:c + heads]
                return t.permute(0, 2, 3, 1, 4)

            for c in range(0, hk, heads):
                res = _attend(s, take(q, c), take(k, c), take(v, c),
                              None if go is None else take(go, c))
                for t, r in zip(out, res):
                    if r is None:
                        continue
                    r = r if r.ndim == 5 else r[:, :, None]
                    group = t.shape[1] // hk
                    t[rows, c * group:(c + heads) * group] = r.permute(0, 3, 1, 2, 4).flatten(
                        2, 3).to(t.dtype)
    return out if s["train"] else out[0]


def _clip(s):
    x, dt = s["grads"], s["grads"][0].dtype
    norm = torch.stack([t.float().square().sum(dtype=torch.float64) for t in x]).sum().sqrt()
    c = torch.where(norm > s["max_norm"], s["max_norm"] / norm, 1.0)
    y = [(t.float() * c.float()).to(dt) for t in x]
    if not s["train"]:
        return y, norm.float()
    dot = torch.stack([(t.float() * u.float()).sum(dtype=torch.float64)
                       for t, u in zip(x, s["cotangents"])]).sum()
    back = torch.where(norm > s["max_norm"], -c * dot / norm.square(), 0.0)
    g = [(u.float() * c.float() + t.float() * back.float()).to(dt)
         for t, u in zip(x, s["cotangents"])]
    return y, norm.float(), g


def _own(s):
    import theria_b200
    from theria_b200 import lm
    if s["op"] == "clip":
        y, norm = lm.clip_gradients(s["grads"], s["max_norm"])
        if not s["train"]:
            return y, norm
        return y, norm, list(torch.autograd.grad(y, s["grads"], s["cotangents"]))
    if s["op"] == "rotary":
        y = lm.rotary(s["q"], s["k"], s["frequencies"], positions=s["positions"],
                      offsets=s["offsets"], interleaved=s["interleaved"],
                      amplitude=s["amplitude"])
        if not s["train"]:
            return y
        return (*y, *torch.autograd.grad(y, (s["q"], s["k"]), (s["gq"], s["gk"])))
    o = theria_b200.sdpa_ragged(s["q"], s["k"], s["v"], s["offsets"], causal=s["causal"])
    if not s["train"]:
        return o
    return [o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["go"])]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"ragged": _ragged, "rotary": _rotary, "clip": _clip}[state["op"]](state)


# ------------------------------------------------------------------ in 64 bits
def _exact_rotary(s, x, at, sign):
    """Pairs as complex numbers, turned by their angle."""
    dim, y = s["dim"], x.detach().double()
    part = y[..., :dim]
    pairs = (part.unflatten(-1, (dim // 2, 2)) if s["interleaved"]
             else part.unflatten(-1, (2, dim // 2)).transpose(-1, -2))
    angle = sign * at.double()[:, None, None] * s["frequencies"]
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(
        torch.full_like(angle, s["amplitude"]), angle)
    z = torch.view_as_real(z)
    z = z.flatten(-2) if s["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return torch.cat([z, y[..., dim:]], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        x = torch.cat([t.detach().double().flatten() for t in s["grads"]])
        norm = torch.linalg.vector_norm(x)
        over = bool(norm > s["max_norm"])
        c = s["max_norm"] / norm if over else torch.ones_like(norm)
        sizes = [t.numel() for t in s["grads"]]
        part = lambda t: [a.view(b.shape) for a, b in zip(t.split(sizes), s["grads"])]  # noqa: E731
        if not case["train"]:
            return part(x * c), norm
        u = torch.cat([t.double().flatten() for t in s["cotangents"]])
        g = c * (u - x * (torch.dot(x, u) / norm ** 2)) if over else u
        return part(x * c), norm, part(g)
    if case["op"] == "rotary":
        at = s["positions"]
        if at is None:
            at = torch.cat([torch.arange(n, device="cuda") for n in s["lengths"]])
        y = _exact_rotary(s, s["q"], at, 1), _exact_rotary(s, s["k"], at, 1)
        if not case["train"]:
            return y
        return (*y, _exact_rotary(s, s["gq"], at, -1), _exact_rotary(s, s["gk"], at, -1))
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    group = case["heads"] // case["kv_heads"]
    o, grads = torch.zeros_like(q), [torch.zeros_like(t) for t in (q, k, v)]
    a = 0
    for n in s["lengths"]:
        for h in range(case["heads"] if n else 0):
            one = [t[a:a + n, j].clone().requires_grad_(case["train"])
                   for t, j in ((q, h), (k, h // group), (v, h // group))]
            w = one[0] @ one[1].t() / math.sqrt(case["d"])
            if case["causal"]:
                w = w + torch.full_like(w, -math.inf).triu(1)
            y = torch.softmax(w, -1) @ one[2]
            o[a:a + n, h] = y.detach()
            if case["train"]:
                got = torch.autograd.grad(y, one, s["go"][a:a + n, h].double())
                for t, r, j in zip(grads, got, (h, h // group, h // group)):
                    t[a:a + n, j] += r
            del w, y
        a += n
    return [o, *grads] if case["train"] else o
