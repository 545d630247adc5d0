"""A training step on packed text, the operators together as a user runs them:
embedding, rotary positions, attention within each packed sequence with grouped
heads, loss, and the gradients clipped by their global norm.

The decoder of examples/decoder_lm.py against the same model in plain torch
operations in float64 on the CPU, sequence by sequence.  Tolerance: as for the
dense decoder's test, 5e-5 on each gradient's 2-norm: each float32 operator holds 1e-5
(rotary 2^-21), over two layers of them with float32 torch linears between."""

import importlib.util
import pathlib

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

from theria_b200 import lm  # noqa: E402

_path = pathlib.Path(__file__).resolve().parents[1] / "examples" / "decoder_lm.py"
_spec = importlib.util.spec_from_file_location("decoder_lm", _path)
decoder_lm = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(decoder_lm)


def _plain(model, p, ids, target, lengths):
    """The packed model's loss from parameters p in plain operations."""
    d = p["tok"].shape[1]
    m = torch.arange(model.pairs, dtype=torch.float64)
    freq = 10000.0 ** (-m / model.pairs)

    def turn(x):  # [n, H, e]
        ang = torch.arange(x.shape[0], dtype=torch.float64)[:, None, None] * freq
        a, b = x[..., :model.pairs], x[..., model.pairs:]
        return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)

    logits = []
    for part in ids.split(lengths):
        if not part.numel():
            continue
        x = F.embedding(part, p["tok"]) * model.scale
        n = x.shape[0]
        for i, block in enumerate(model.blocks):
            w = lambda s: p[f"blocks.{i}.{s}"]  # noqa: E731
            H, K = block.heads, block.kv_heads
            rows = (F.layer_norm(x, (d,), w("ln1_w"), w("ln1_b")) @ w("qkv.weight").t())
            q, k, v = rows.view(n, H + 2 * K, -1).split([H, K, K], 1)
            q, k = turn(q).transpose(0, 1), turn(k).transpose(0, 1).repeat_interleave(H // K, 0)
            v = v.transpose(0, 1).repeat_interleave(H // K, 0)
            s = q @ k.transpose(1, 2) / q.shape[-1] ** 0.5
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), float("-inf"))
            x = x + (s.softmax(-1) @ v).transpose(0, 1).reshape(n, d) @ w("out.weight").t()
            f = F.layer_norm(x, (d,), w("ln2_w"), w("ln2_b"))
            f = F.gelu(f @ w("up.weight").t() + w("up.bias"))
            x = x + f @ w("down.weight").t() + w("down.bias")
        logits.append(F.layer_norm(x, (d,), p["lnf_w"], p["lnf_b"]) @ p["tok"].t())
    return F.cross_entropy(torch.cat(logits), target)


@pytest.mark.parametrize("vocab,d,heads,kv_heads,seq_len", [(32, 64, 4, 2, 64), (1001, 72, 6, 1, 45)])
def test_packed_step_matches_plain_float64(vocab, d, heads, kv_heads, seq_len):
    torch.manual_seed(1)
    model = decoder_lm.PackedDecoderLM(vocab, d, heads, kv_heads, 2)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if name.endswith(("_w", "_b")):
                p.add_(0.1 * torch.randn_like(p))
    ids = torch.randint(1, vocab, (6, seq_len + 1))
    ids[1, seq_len // 2:] = 0
    ids[3, 3:] = 0
    ids[4, :] = 0  # a sequence without a token
    tokens, target, offsets = decoder_lm.pack(ids)
    lengths = offsets.diff().tolist()
    assert 0 in lengths and len(set(lengths)) > 2
    ref = {n: p.detach().double().requires_grad_(True) for n, p in model.named_parameters()}
    want = _plain(model, ref, tokens, target, lengths)
    grads = dict(zip(ref, torch.autograd.grad(want, list(ref.values()))))
    model.cuda()
    loss = model(tokens.cuda(), target.cuda(), offsets.cuda())
    loss.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * want.item()
    for name, p in model.named_parameters():
        err = (p.grad.double().cpu() - grads[name]).norm() / grads[name].norm()
        assert err <= 5e-5, (name, err.item())
    norm = torch.cat([g.flatten() for g in grads.values()]).norm().item()
    got = lm.clip_gradients_([p.grad for p in model.parameters()], norm / 3)
    assert abs(got.item() - norm) <= 5e-5 * norm
    for name, p in model.named_parameters():
        err = (p.grad.double().cpu() - grads[name] / 3).norm() / grads[name].norm()
        assert err <= 5e-5, (name, err.item())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_packed_training_runs(dtype):
    model, losses = decoder_lm.train(steps=3, dtype=dtype, log=None, packed=True)
    assert all(map(lambda x: x == x and abs(x) < 100, losses))
    assert all(torch.isfinite(p).all() for p in model.parameters())


def test_a_step_in_a_graph():
    """The packed step captured once: ids, targets and offsets of the same sizes change
    between replays, as do the sequences' lengths."""
    torch.manual_seed(2)
    model = decoder_lm.PackedDecoderLM(64, 64, 4, 2, 2).cuda().to(torch.bfloat16)
    params = list(model.parameters())
    T = 300

    def data(seed, lengths):
        g = torch.Generator().manual_seed(seed)
        ids = torch.randint(0, 64, (T,), generator=g)
        target = torch.where(torch.rand(T, generator=g) < 0.2, lm.IGNORE_INDEX, ids.roll(-1))
        return [t.cuda() for t in (ids, target, torch.tensor([0] + lengths).cumsum(0))]

    def step(ids, target, offsets):
        loss = model(ids, target, offsets)
        grads, norm = lm.clip_gradients(torch.autograd.grad(loss, params), 0.1)
        return [loss.detach(), norm, *grads]

    static = data(0, [100, 0, 50, 150])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for seed, lengths in ((1, [1, 298, 1, 0]), (2, [20, 60, 100, 120])):
        new = data(seed, lengths)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(*new)):
            assert torch.equal(a, b)
