"""Timed cases of the language-model operators of ``theria_b200.lm``.

The operators are the two ends of a pre-LN decoder and the norm between its
blocks: the scaled token embedding with its gradient, the layer norm with its
gradients, and the linear layer to the vocabulary with its softmax cross
entropy and their gradients.  ``own`` chooses who computes a pass: the plain
forms below (elementary torch operations in float32, rounded once), or the
framework's operators as a user's program calls them.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
IGNORE = -100
EPS = 1e-5


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one 64-token sequence of the 32-token MAML vocabulary looked up: latency
        dict(name="embedding lookup 64", op="embedding", train=False, n=64, vocab=32, d=64,
             dtype="f32", scaled=False, padded=False),
        # a ragged packed batch of an fp32 model, with padding tokens
        dict(name="embedding train 5003 odd", op="embedding", train=True, n=5003, vocab=50021,
             d=1001, dtype="f32", scaled=True, padded=True),
        # a large training batch: 32 sequences of 2048 tokens, a large vocabulary
        dict(name="embedding train 65536", op="embedding", train=True, n=65536, vocab=131072,
             d=2048, dtype="bf16", scaled=True, padded=False),
        # the norm of one decoded token
        dict(name="norm 1 row", op="norm", train=False, n=1, d=1024, dtype="bf16"),
        # the MAML classifier's query rows: 75 sequences of 64 tokens, width 64
        dict(name="norm train 4800x64", op="norm", train=True, n=4800, d=64, dtype="f32"),
        # an odd row count and an odd width
        dict(name="norm train 3001x1111", op="norm", train=True, n=3001, d=1111, dtype="f16"),
        # a training batch of 8 sequences of 2048 tokens in a wide model
        dict(name="norm train 16384x4096", op="norm", train=True, n=16384, d=4096,
             dtype="bf16"),
        # one 64-token sequence against the 32-token vocabulary: latency
        dict(name="loss train 64x32", op="loss", train=True, n=64, vocab=32, d=64, dtype="f32",
             ignored=0.0),
        # a training batch of a mid-sized model
        dict(name="loss train 8192x32768", op="loss", train=True, n=8192, vocab=32768, d=2048,
             dtype="bf16", ignored=0.0),
        # the same loss trained in full precision
        dict(name="loss train 2048x16384 f32", op="loss", train=True, n=2048, vocab=16384,
             d=512, dtype="f32", ignored=0.0),
        # odd sizes, a quarter of the tokens not scored (prompts, padding)
        dict(name="loss train 1021x50021 odd", op="loss", train=True, n=1021, vocab=50021,
             d=1000, dtype="f16", ignored=0.25),
        # the log-probability of each token of a text (no gradient), with a wide model and a
        # large vocabulary
        dict(name="loss score 4096x131072", op="loss", train=False, n=4096, vocab=131072,
             d=4096, dtype="bf16", ignored=0.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embedding", "norm", "loss", "loss"])
    train = rng.random() < 0.7
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op == "embedding":
        n, vocab = _log_uniform(rng, 1, 65536), _log_uniform(rng, 32, 131072)
        d = _log_uniform(rng, 16, min(1024 if dtype == "f32" else 2048, 2 ** 27 // n))
        if rng.random() < 0.6:
            d = -(-d // 16) * 16
        return dict(op=op, train=train, n=n, vocab=vocab, d=d, dtype=dtype,
                    scaled=rng.random() < 0.5, padded=rng.random() < 0.3)
    if op == "norm":
        n = _log_uniform(rng, 1, 65536)
        d = _log_uniform(rng, 32, min(8192, 16384 * 4096 // n))
        if rng.random() < 0.6:
            d = -(-d // 32) * 32
        return dict(op=op, train=train, n=n, d=d, dtype=dtype)
    n, vocab = _log_uniform(rng, 1, 16384), _log_uniform(rng, 32, 131072)
    # no costlier than the largest listed case (float32: an eighth of its flops)
    cap = (5e11 if dtype == "f32" else 4.3e12) / (6 if train else 2)
    while n * vocab > min(2 ** 30, cap / 64):
        n //= 2
    d = _log_uniform(rng, 32, min(1024 if dtype == "f32" else 4096, cap / (n * vocab),
                                  2 ** 28 // vocab))
    if rng.random() < 0.85:
        d = -(-d // 8) * 8
    return dict(op=op, train=train, n=n, vocab=vocab, d=d, dtype=dtype,
                ignored=rng.choice([0.0, 0.0, 0.25, 0.6]))


def work(case):
    e, d, n = SIZES[case["dtype"]], case["d"], case["n"]
    if case["op"] == "norm":
        passes, rows = (4, 4) if case["train"] else (2, 2)  # x, gy, y, gx; w, b, gw, gb
        return {"bytes": passes * n * d * e + rows * d * e,
                "flops": (18 if case["train"] else 8) * n * d}
    v = case["vocab"]
    if case["op"] == "embedding":
        b = 8 * n + min(n, v) * d * e + n * d * e
        return {"bytes": b + (n * d * e + v * d * e if case["train"] else 0),
                "flops": (2 if case["train"] else 1) * n * d}
    live = n - int(n * case["ignored"])
    b = 8 * n + (n + v) * d * e + (4 if case["train"] else 4 * n)
    return {"bytes": b + ((n + v) * d * e if case["train"] else 0),
            "flops": (6 if case["train"] else 2) * live * v * d}


# ----------------------------------------------------------------- the inputs
def _tokens(n, vocab, g):
    # word frequencies fall like 1 / rank
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return ((u * math.log(vocab + 1)).exp().long() - 1).clamp_(0, vocab - 1)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt, d, n, train = DTYPES[case["dtype"]], case["d"], case["n"], case["train"]

    def normal(*shape, std=1.0):
        x = torch.empty(shape, device="cuda", dtype=dt)
        return x.normal_(0.0, std, generator=g)

    s = dict(case)
    if case["op"] == "embedding":
        s["ids"] = _tokens(n, case["vocab"], g)
        s["weight"] = normal(case["vocab"], d, std=0.02).requires_grad_(train)
        s["scale"] = math.sqrt(d) if case["scaled"] else 1.0
        s["padding"] = 0 if case["padded"] else None
        if train:
            s["gy"] = normal(n, d)
    elif case["op"] == "norm":
        s["x"] = (normal(n, d, std=1.5) + normal(d, std=0.5)).requires_grad_(train)
        s["weight"] = (1 + normal(d, std=0.1)).requires_grad_(train)
        s["bias"] = normal(d, std=0.1).requires_grad_(train)
        if train:
            s["gy"] = normal(n, d)
    else:
        s["hidden"] = normal(n, d).requires_grad_(train)
        s["weight"] = normal(case["vocab"], d, std=1.0 / math.sqrt(d)).requires_grad_(train)
        t = _tokens(n, case["vocab"], g)
        order = torch.randperm(n, generator=g, device="cuda")
        t[order[:int(n * case["ignored"])]] = IGNORE
        s["target"] = t
    return s


# ---------------------------------------------------------------- plain forms
def _embedding(s):
    w, ids, scale = s["weight"], s["ids"], s["scale"]
    y = (w[ids].float() * scale).to(w.dtype)
    if not s["train"]:
        return y
    g = s["gy"].float() * scale
    if s["padding"] is not None:
        g = torch.where((ids == s["padding"])[:, None], torch.zeros_like(g), g)
    gw = torch.zeros(w.shape, device=w.device).index_add_(0, ids, g)
    return y, gw.to(w.dtype)


def _norm(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    dt = s["x"].dtype
    c = x - x.mean(-1, keepdim=True)
    r = ((c * c).mean(-1, keepdim=True) + EPS).rsqrt()
    h = c * r
    y = (h * w + b).to(dt)
    if not s["train"]:
        return y
    gy = s["gy"].float()
    gh = gy * w
    gx = r * (gh - gh.mean(-1, keepdim=True) - h * (gh * h).mean(-1, keepdim=True))
    return y, gx.to(dt), (gy * h).sum(0).to(dt), gy.sum(0).to(dt)


def _loss(s):
    h, w, t = s["hidden"].float(), s["weight"].float(), s["target"]
    live = t != IGNORE
    count = live.sum()
    at = torch.where(live, t, torch.zeros_like(t))[:, None]
    z = h @ w.t()
    top = z.max(-1, keepdim=True).values
    z = z - top
    picked = z.gather(1, at)
    p = z.exp_()
    total = p.sum(-1, keepdim=True)
    each = (total.log() - picked).squeeze(1)
    each = torch.where(live, each, torch.zeros_like(each))
    if not s["train"]:
        return each
    loss = each.sum() / count
    p = p.div_(total).scatter_add_(1, at, torch.full_like(picked, -1.0))
    p = p.mul_((live.float() / count)[:, None])
    dt = s["hidden"].dtype
    return loss, (p @ w).to(dt), (p.t() @ h).to(dt)


def _own(s):
    from theria_b200 import lm
    if s["op"] == "embedding":
        y = lm.embedding(s["ids"], s["weight"], scale=s["scale"], padding_idx=s["padding"])
        if not s["train"]:
            return y
        return (y, *torch.autograd.grad(y, s["weight"], s["gy"]))
    if s["op"] == "norm":
        y = lm.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
        if not s["train"]:
            return y
        return (y, *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["gy"]))
    loss = lm.linear_cross_entropy(s["hidden"], s["weight"], s["target"], ignore_index=IGNORE,
                                   reduction="mean" if s["train"] else "none")
    if not s["train"]:
        return loss
    return (loss, *torch.autograd.grad(loss, (s["hidden"], s["weight"])))


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"embedding": _embedding, "norm": _norm, "loss": _loss}[state["op"]](state)


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "embedding":
            table = s["weight"].double() * s["scale"]
            y = torch.nn.functional.embedding(s["ids"], table)
            if not case["train"]:
                return y
            rows = s["gy"].double() * s["scale"]
            if s["padding"] is not None:
                rows[s["ids"] == s["padding"]] = 0
            return y, torch.zeros_like(table).index_put_((s["ids"],), rows, accumulate=True)
    if case["op"] == "norm":
        x, w, b = (s[k].detach().double().requires_grad_(True) for k in ("x", "weight", "bias"))
        y = torch.nn.functional.layer_norm(x, (case["d"],), w, b, EPS)
        if not case["train"]:
            return y.detach()
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), s["gy"].double()))
    h, w = (s[k].detach().double().requires_grad_(case["train"]) for k in ("hidden", "weight"))
    loss = torch.nn.functional.cross_entropy(h @ w.t(), s["target"], ignore_index=IGNORE,
                                             reduction="mean" if case["train"] else "none")
    if not case["train"]:
        return loss
    return (loss.detach(), *torch.autograd.grad(loss, (h, w)))
