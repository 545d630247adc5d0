"""A small causal language model on the library's operators, trained for a few
steps on synthetic tokens.

    python examples/decoder_lm.py [--steps 50] [--dtype bf16] [--vocab 32768] [--packed] ...

A pre-LN decoder as in the reference's example
(``examples/minimal_decoder_transformer.py:82-263``): scaled token embedding,
blocks of layer norm, causal attention, layer norm and a GELU feed-forward, a
final layer norm, and the loss of the next token against the embedding table
itself (tied weights).  ``lm.embedding``, ``lm.layer_norm``, ``sdpa`` and
``lm.linear_cross_entropy`` run hand-written kernels; the scores of the
vocabulary are never stored.  Positions whose target is padding are not scored.

``--packed`` trains on the same sequences without their padding, one behind the
other in a row of tokens (``PackedDecoderLM``): rotary positions counted within each
sequence (``lm.rotary``), attention within each with heads that share keys and
values (``sdpa_ragged``), and gradients clipped by their global norm
(``lm.clip_gradients_``).

The token streams follow a fixed random successor table with noise, so that the
loss can fall from log(vocab) towards the noise's entropy.
"""

import argparse
import math
import pathlib
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))

from theria_b200 import lm, sdpa, sdpa_ragged  # noqa: E402


class Block(nn.Module):
    def __init__(self, d, heads):
        super().__init__()
        self.heads = heads
        self.ln1_w, self.ln1_b = nn.Parameter(torch.ones(d)), nn.Parameter(torch.zeros(d))
        self.ln2_w, self.ln2_b = nn.Parameter(torch.ones(d)), nn.Parameter(torch.zeros(d))
        self.qkv, self.out = nn.Linear(d, 3 * d, bias=False), nn.Linear(d, d, bias=False)
        self.up, self.down = nn.Linear(d, 4 * d), nn.Linear(4 * d, d)

    def forward(self, x):
        B, T, d = x.shape
        a = lm.layer_norm(x, self.ln1_w, self.ln1_b)
        q, k, v = self.qkv(a).view(B, T, 3, self.heads, d // self.heads).permute(2, 0, 3, 1, 4)
        o = sdpa(q, k, v, causal=True)
        x = x + self.out(o.transpose(1, 2).reshape(B, T, d))
        f = lm.layer_norm(x, self.ln2_w, self.ln2_b)
        return x + self.down(F.gelu(self.up(f)))


class DecoderLM(nn.Module):
    def __init__(self, vocab=32, d=64, heads=4, layers=2, seq_len=64, pad=0):
        super().__init__()
        self.pad, self.scale = pad, math.sqrt(d)
        self.tok = nn.Parameter(torch.randn(vocab, d) / math.sqrt(d))
        self.pos = nn.Parameter(torch.zeros(seq_len, d))
        self.blocks = nn.ModuleList(Block(d, heads) for _ in range(layers))
        self.lnf_w, self.lnf_b = nn.Parameter(torch.ones(d)), nn.Parameter(torch.zeros(d))

    def hidden(self, ids):
        x = lm.embedding(ids, self.tok, scale=self.scale) + self.pos[:ids.shape[1]]
        for block in self.blocks:
            x = block(x)
        return lm.layer_norm(x, self.lnf_w, self.lnf_b)

    def forward(self, ids, reduction="mean"):
        """Loss of each next token; targets that are padding are not scored."""
        return lm.linear_cross_entropy(self.hidden(ids[:, :-1]), self.tok, ids[:, 1:],
                                       ignore_index=self.pad, reduction=reduction)

    @torch.no_grad()
    def log_probs(self, ids):
        """log p(token | tokens before it), [B, T - 1]; 0 at padding."""
        return -self(ids, reduction="none")


class PackedBlock(nn.Module):
    def __init__(self, d, heads, kv_heads):
        super().__init__()
        self.heads, self.kv_heads, e = heads, kv_heads, d // heads
        self.ln1_w, self.ln1_b = nn.Parameter(torch.ones(d)), nn.Parameter(torch.zeros(d))
        self.ln2_w, self.ln2_b = nn.Parameter(torch.ones(d)), nn.Parameter(torch.zeros(d))
        self.qkv = nn.Linear(d, (heads + 2 * kv_heads) * e, bias=False)
        self.out = nn.Linear(d, d, bias=False)
        self.up, self.down = nn.Linear(d, 4 * d), nn.Linear(4 * d, d)

    def forward(self, x, offsets, frequencies):
        T, d = x.shape
        a = lm.layer_norm(x, self.ln1_w, self.ln1_b)
        # heads side by side, read in place: queries, keys, values
        rows = self.qkv(a).view(T, self.heads + 2 * self.kv_heads, -1)
        q, k, v = rows.split([self.heads, self.kv_heads, self.kv_heads], 1)
        q, k = lm.rotary(q, k, frequencies, offsets=offsets)
        x = x + self.out(sdpa_ragged(q, k, v, offsets).reshape(T, d))
        f = lm.layer_norm(x, self.ln2_w, self.ln2_b)
        return x + self.down(F.gelu(self.up(f)))


class PackedDecoderLM(nn.Module):
    """The decoder on packed sequences: ids [T], offsets [S + 1]."""

    def __init__(self, vocab=32, d=64, heads=4, kv_heads=2, layers=2):
        super().__init__()
        self.scale, self.pairs = math.sqrt(d), d // heads // 2
        self.tok = nn.Parameter(torch.randn(vocab, d) / math.sqrt(d))
        self.blocks = nn.ModuleList(PackedBlock(d, heads, kv_heads) for _ in range(layers))
        self.lnf_w, self.lnf_b = nn.Parameter(torch.ones(d)), nn.Parameter(torch.zeros(d))
        self.frequencies = None  # float64 whatever the parameters' type

    def forward(self, ids, target, offsets):
        """Mean loss of the targets [T]; those that are lm.IGNORE_INDEX are not scored."""
        if self.frequencies is None or self.frequencies.device != ids.device:
            self.frequencies = lm.rotary_frequencies(2 * self.pairs, device=ids.device)
        x = lm.embedding(ids, self.tok, scale=self.scale)
        for block in self.blocks:
            x = block(x, offsets, self.frequencies)
        return lm.linear_cross_entropy(lm.layer_norm(x, self.lnf_w, self.lnf_b), self.tok, target)


def pack(ids, pad=0):
    """Padded sequences [n, L + 1] as ids [T], their next tokens [T] and offsets."""
    src, tgt = ids[:, :-1], ids[:, 1:]
    live = src != pad
    offsets = F.pad(live.sum(1), (1, 0)).cumsum(0)
    target = torch.where(tgt == pad, lm.IGNORE_INDEX, tgt)
    return src[live], target[live], offsets


def batch(table, n, seq_len, g, pad=0):
    """Sequences that follow table[token] nine times in ten, of ragged lengths."""
    vocab, dev = table.numel(), table.device
    ids = torch.empty(n, seq_len + 1, dtype=torch.long, device=dev)
    ids[:, 0] = torch.randint(1, vocab, (n,), generator=g, device=dev)
    for t in range(seq_len):
        free = torch.randint(1, vocab, (n,), generator=g, device=dev)
        keep = torch.rand(n, generator=g, device=dev) < 0.9
        ids[:, t + 1] = torch.where(keep, table[ids[:, t]], free)
    length = torch.randint(seq_len // 2, seq_len + 2, (n, 1), generator=g, device=dev)
    return ids.masked_fill(torch.arange(seq_len + 1, device=dev) >= length, pad)


def train(steps=50, dtype=torch.float32, vocab=32, d=64, heads=4, layers=2, seq_len=64, size=32,
          lr=3e-3, seed=0, log=print, packed=False, max_norm=1.0):
    torch.manual_seed(seed)
    g = torch.Generator("cuda").manual_seed(seed)
    if packed:
        kv_heads = heads // 2 if heads % 2 == 0 else 1  # a divisor of the heads
        model = PackedDecoderLM(vocab, d, heads, kv_heads, layers).to("cuda", dtype)
    else:
        model = DecoderLM(vocab, d, heads, layers, seq_len).to("cuda", dtype)
    table = torch.randperm(vocab - 1, generator=g, device="cuda")
    table = torch.cat([table.new_zeros(1), table + 1])  # 0 is padding
    opt = torch.optim.Adam(model.parameters(), lr=lr)
    losses = []
    for step in range(steps):
        ids = batch(table, size, seq_len, g)
        loss = model(*pack(ids)) if packed else model(ids)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        if packed:
            lm.clip_gradients_([p.grad for p in model.parameters()], max_norm)
        opt.step()
        losses.append(loss.detach())
        if log and (step % 10 == 0 or step == steps - 1):
            log(f"step {step:4d}  loss {losses[-1].item():.4f}")
    return model, torch.stack(losses).tolist()


def main():
    ap = argparse.ArgumentParser()
    for name, value in (("steps", 50), ("vocab", 32), ("d", 64), ("heads", 4), ("layers", 2),
                        ("seq-len", 64), ("size", 32)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--lr", type=float, default=3e-3)
    ap.add_argument("--packed", action="store_true")
    ap.add_argument("--dtype", choices=["f32", "bf16"], default="f32")
    a = vars(ap.parse_args())
    a["dtype"] = {"f32": torch.float32, "bf16": torch.bfloat16}[a["dtype"]]
    train(**a)


if __name__ == "__main__":
    main()
