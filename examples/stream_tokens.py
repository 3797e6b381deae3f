"""Trains a small causal Mamba model on packed sequences of different lengths,
then serves it: prompts in pieces, and single tokens by a captured graph.

    python examples/stream_tokens.py [--steps 300] [--bf16]

The task: a sequence repeats a random word of 3 to 5 symbols; past its first
repetition every symbol can be foretold.  Served greedily from a prompt, the
model has to go on repeating it.
"""

import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import mlx_vision_mamba_amd as mvm  # noqa: E402
from mlx_vision_mamba_amd.optim import AdamW  # noqa: E402


class TokenModel(nn.Module):
    """Embedding, causal residual Mamba blocks, tied output."""

    def __init__(self, symbols=8, d_model=64, depth=2):
        super().__init__()
        self.embed = nn.Embedding(symbols, d_model)
        nn.init.normal_(self.embed.weight, std=d_model ** -0.5)
        self.blocks = nn.ModuleList([mvm.ResidualMambaBlock(d_model) for _ in range(depth)])
        self.norm = nn.LayerNorm(d_model)

    def head(self, x):
        return F.linear(self.norm(x), self.embed.weight).float()

    def forward(self, tokens, offsets, max_len):
        x = self.embed(tokens)
        for blk in self.blocks:
            x, _ = blk.forward_packed(x, offsets, max_len=max_len)
        return self.head(x)

    def init_states(self, rows):
        return [blk.init_states(rows) for blk in self.blocks]

    @torch.no_grad()
    def prefill(self, tokens, states, offsets, slots, fresh, max_len):
        """Logits after each sequence's last token; the cache advances."""
        x = self.embed(tokens)
        for blk, st in zip(self.blocks, states):
            x = blk.prefill(x, st, offsets, slots=slots, fresh=fresh, max_len=max_len)
        return self.head(x[offsets[1:].long() - 1])

    @torch.no_grad()
    def step(self, tokens, states, slots):
        x = self.embed(tokens)
        for blk, st in zip(self.blocks, states):
            x = blk.step(x, st, slots=slots)
        return self.head(x)


def words(lengths, symbols, gen):
    """One repeated word for each length, and the words' lengths."""
    out, period = [], []
    for n in lengths:
        p = int(torch.randint(3, 6, (1,), generator=gen))
        w = torch.randint(0, symbols, (p,), generator=gen)
        out.append(w.repeat(n // p + 1)[:n])
        period.append(p)
    return out, period


def pack(seqs, device):
    lens = [len(s) for s in seqs]
    off = torch.tensor([0] + lens).cumsum(0).int().to(device)
    return torch.cat(seqs).to(device), off, max(lens)


def train(model, steps, device, gen):
    opt = AdamW(model.parameters(), lr=3e-3)
    for i in range(steps):
        lens = torch.randint(20, 60, (16,), generator=gen).tolist()
        seqs, period = words(lens, model.embed.num_embeddings, gen)
        tokens, off, longest = pack(seqs, device)
        # the next symbol, where it can be foretold: past the first repetition
        target = torch.cat([torch.cat([s[1:], s[:1] * 0 - 100]) for s in seqs])
        for o, n, p in zip(off.tolist(), lens, period):
            target[o:o + p] = -100
        loss = F.cross_entropy(model(tokens, off, longest), target.to(device), ignore_index=-100)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        if i % 20 == 0 or i == steps - 1:
            print(f"step {i}: loss {loss.item():.3f}", flush=True)


def serve(model, device, gen, users=6, new=24):
    """Share of the served symbols that continue their word."""
    slots = torch.randperm(users + 2, generator=gen)[:users].int().to(device)
    states = model.init_states(users + 2)
    prompts, period = words(torch.randint(14, 30, (users,), generator=gen).tolist(), model.embed.num_embeddings, gen)
    for lo, hi in ((0, 8), (8, None)):  # the prompts come in two pieces
        tokens, off, longest = pack([p[lo:hi] for p in prompts], device)
        fresh = torch.full((users,), lo == 0, device=device)
        logits = model.prefill(tokens, states, off, slots, fresh, longest)
    token = logits.argmax(-1)
    # one step, captured: it reads its token from a fixed buffer and leaves the next one there
    graph, saved = torch.cuda.CUDAGraph(), [[t.clone() for t in st] for st in states]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model.step(token, states, slots)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        token.copy_(model.step(token, states, slots).argmax(-1))
    for st, old in zip(states, saved):  # the warm-up advanced them
        for t, o in zip(st, old):
            t.copy_(o)
    got = [token.clone()]
    for _ in range(new - 1):
        graph.replay()
        got.append(token.clone())
    got = torch.stack(got, 1).cpu()
    want = torch.stack([torch.stack([p[(len(p) + k) % q] for k in range(new)]) for p, q in zip(prompts, period)])
    return (got == want).float().mean().item()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--bf16", action="store_true", help="serve in bfloat16")
    args = ap.parse_args(argv)
    torch.manual_seed(0)
    gen, device = torch.Generator().manual_seed(0), torch.device("cuda")
    model = TokenModel().to(device)
    train(model, args.steps, device, gen)
    if args.bf16:
        model = model.bfloat16()
    right = serve(model, device, gen)
    print(f"served symbols that continue their word: {100 * right:.0f} %")
    return right


if __name__ == "__main__":
    main()
