"""examples/decoder_lm.py: the embedding, layer norm, causal attention and
linear cross entropy together in a small decoder, against the same model in
plain torch operations in float64 on the CPU.

Tolerance: the float32 operators hold 4e-6 or 1e-5 each (the attention's
contract); the chain is 2 layers of 3 of them deep, with float32 torch linears
of K <= 256 between: 5e-5 on each gradient's 2-norm is their sum with room for
the growth through the layers."""

import importlib.util
import pathlib

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("CUDA not available", allow_module_level=True)

_path = pathlib.Path(__file__).resolve().parents[1] / "examples" / "decoder_lm.py"
_spec = importlib.util.spec_from_file_location("decoder_lm", _path)
decoder_lm = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(decoder_lm)


def _plain(model, p, ids):
    """The model's loss from parameters p in plain operations."""
    d = p["tok"].shape[1]
    src, tgt = ids[:, :-1], ids[:, 1:]
    x = F.embedding(src, p["tok"]) * model.scale + p["pos"][:src.shape[1]]
    for i, block in enumerate(model.blocks):
        q = lambda s: p[f"blocks.{i}.{s}"]  # noqa: E731
        a = F.layer_norm(x, (d,), q("ln1_w"), q("ln1_b"))
        B, T, _ = a.shape
        qq, kk, vv = (a @ q("qkv.weight").t()).view(B, T, 3, block.heads, -1).permute(2, 0, 3, 1, 4)
        s = qq @ kk.transpose(-1, -2) / qq.shape[-1] ** 0.5
        s = s.masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), float("-inf"))
        o = (s.softmax(-1) @ vv).transpose(1, 2).reshape(B, T, d)
        x = x + o @ q("out.weight").t()
        f = F.layer_norm(x, (d,), q("ln2_w"), q("ln2_b"))
        f = F.gelu(f @ q("up.weight").t() + q("up.bias"))
        x = x + f @ q("down.weight").t() + q("down.bias")
    x = F.layer_norm(x, (d,), p["lnf_w"], p["lnf_b"])
    return F.cross_entropy((x @ p["tok"].t()).flatten(0, 1), tgt.flatten(),
                           ignore_index=model.pad)


@pytest.mark.parametrize("vocab,d,heads,seq_len", [(32, 64, 4, 64), (1001, 72, 3, 45)])
def test_decoder_loss_and_gradients_match_plain_float64(vocab, d, heads, seq_len):
    torch.manual_seed(1)
    model = decoder_lm.DecoderLM(vocab, d, heads, 2, seq_len)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if name.endswith(("_w", "_b", "pos")):
                p.add_(0.1 * torch.randn_like(p))
    ids = torch.randint(1, vocab, (5, seq_len + 1))
    ids[1, seq_len // 2:] = 0
    ids[3, 3:] = 0
    ref = {n: p.detach().double().requires_grad_(True) for n, p in model.named_parameters()}
    want = _plain(model, ref, ids)
    grads = dict(zip(ref, torch.autograd.grad(want, list(ref.values()))))
    model.cuda()
    loss = model(ids.cuda())
    loss.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * want.item()
    for name, p in model.named_parameters():
        err = (p.grad.double().cpu() - grads[name]).norm() / grads[name].norm()
        assert err <= 5e-5, (name, err.item())
    each = model.log_probs(ids.cuda())
    assert each.shape == ids[:, 1:].shape and (each[ids.cuda()[:, 1:] == 0] == 0).all()
    live = (ids[:, 1:] != 0).sum()
    assert abs(-each.sum().item() / live.item() - want.item()) <= 1e-5 * want.item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decoder_learns(dtype):
    # 32 words, the successor known nine times in ten: from log 31 = 3.43 down
    # to about 0.66; a hundred steps bring it well below half
    _, losses = decoder_lm.train(steps=100, dtype=dtype, log=None)
    assert losses[0] > 3.0 and losses[-1] < 1.7
