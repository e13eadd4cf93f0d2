"""A small language model of retention layers: token ids to logits.

    x = embedding(ids);    per layer, on n = norm(x):
    x = x + (norm over each head of linear_attention(q, k, v, g) * silu(gate)) W_out

Trains on sequences whose next token follows from the one before the last, then
reads a prompt at once and goes on token by token from the layers' states:

    python examples/retention_lm.py --steps 200 --time 128 --dtype bfloat16
"""

import argparse
import os
import sys

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from mamba4_amd import embedding, group_norm, linear_attention, linear_attention_step_  # noqa: E402


class Retention(nn.Module):
    """x + the gated, normalised linear attention of x [B,T,D]; keys and queries
    are half as wide as values, and with fewer heads shared by the others."""

    def __init__(self, width, heads, key_heads):
        super().__init__()
        self.heads, self.key_heads = heads, key_heads
        self.p = width // heads
        self.n = self.p // 2
        sizes = [key_heads * self.n, key_heads * self.n, width, width]
        self.sizes = sizes
        self.norm = nn.Parameter(torch.ones(width))
        self.project = nn.Parameter(torch.randn(sum(sizes), width) / width**0.5)
        self.decay = nn.Parameter(torch.randn(heads, width) / width**0.5)
        self.decay_bias = nn.Parameter(torch.linspace(2.0, 6.0, heads))
        self.head_norm = nn.Parameter(torch.ones(width))
        self.out = nn.Parameter(torch.randn(width, width) / width**0.5)

    def _inputs(self, x):
        """Of x [rows,D]: q, k, v [rows,h,W], the gate and the log decays."""
        n = group_norm(x, 1, self.norm)
        # (Views of one projection: the kernels read them with its strides.)
        q, k, v, gate = F.linear(n, self.project.to(x.dtype)).split(self.sizes, -1)
        g = F.logsigmoid(F.linear(n, self.decay.to(x.dtype)).float() + self.decay_bias)
        return (q.unflatten(-1, (self.key_heads, self.n)),
                k.unflatten(-1, (self.key_heads, self.n)),
                v.unflatten(-1, (self.heads, self.p)), gate, g)

    def _result(self, x, attended, gate):
        y = group_norm(attended.flatten(1), self.heads, self.head_norm, gate=gate,
                       activation="silu")
        return x + F.linear(y, self.out.to(x.dtype))

    def forward(self, x, lengths=None):
        batch, time, _ = x.shape
        rows = x.flatten(0, 1)
        *qkv, gate, g = self._inputs(rows)
        q, k, v = (t.unflatten(0, (batch, time)) for t in qkv)
        r = linear_attention(q, k, v, g.unflatten(0, (batch, time)), lengths=lengths,
                             scale=self.n**-0.5)
        y = self._result(rows, r.output.flatten(0, 1), gate)
        return y.unflatten(0, (batch, time)), r.state

    def step(self, x, state, active=None):
        """One token of every row, x [B,D]; state is overwritten."""
        q, k, v, gate, g = self._inputs(x)
        o = linear_attention_step_(state, q, k, v, g, active=active, scale=self.n**-0.5).output
        return self._result(x, o, gate)


class RetentionLM(nn.Module):
    def __init__(self, vocab, width, heads, layers, key_heads=None, dtype=torch.float32):
        super().__init__()
        self.dtype = dtype
        self.scale = width**0.5
        self.table = nn.Parameter(torch.randn(vocab, width) / width**0.5)
        self.layers = nn.ModuleList(
            Retention(width, heads, key_heads or heads) for _ in range(layers))
        self.norm = nn.Parameter(torch.ones(width))

    def _logits(self, rows):
        return F.linear(group_norm(rows, 1, self.norm), self.table.to(self.dtype)).float()

    def forward(self, ids, lengths=None):
        """Logits [B,T,V] of ids [B,T] (-1: no token), and the layers' states."""
        x = embedding(ids, self.table, scale=self.scale, dtype=self.dtype)
        states = []
        for layer in self.layers:
            x, state = layer(x, lengths)
            states.append(state)
        return self._logits(x.flatten(0, 1)).unflatten(0, ids.shape), states

    @torch.no_grad()
    def step(self, ids, states, active=None):
        """Logits [B,V] after one more token of every row, ids [B]."""
        x = embedding(ids, self.table, scale=self.scale, dtype=self.dtype)
        for layer, state in zip(self.layers, states):
            x = layer.step(x, state, active)
        return self._logits(x)

    def loss(self, ids):
        logits, _ = self(ids[:, :-1])
        return F.cross_entropy(logits.flatten(0, 1), ids[:, 1:].flatten())

    @torch.no_grad()
    def generate(self, prompt, count, lengths=None):
        """The `count` most likely next tokens [B,count] of prompts [B,T] that end at
        lengths [B]."""
        logits, states = self(prompt, lengths)
        last = prompt.shape[1] - 1 if lengths is None else lengths.long() - 1
        ids = logits[torch.arange(len(prompt), device=prompt.device), last].argmax(-1)
        tokens = [ids]
        for _ in range(count - 1):
            ids = self.step(ids, states).argmax(-1)
            tokens.append(ids)
        return torch.stack(tokens, 1)


def chains(batch, time, vocab, device, generator=None):
    """Sequences [batch,time] of two interleaved walks over a fixed permutation: a
    token follows from the one before the last, which only the states remember."""
    follow = torch.randperm(vocab, generator=torch.Generator().manual_seed(0))
    tokens = list(torch.randint(vocab, (2, batch), generator=generator))
    for t in range(2, time):
        tokens.append(follow[tokens[t - 2]])
    return torch.stack(tokens[:time], 1).to(device)


def train(model, steps, batch, time, vocab, rate=2e-3, seed=0):
    """The losses of every step."""
    generator = torch.Generator().manual_seed(seed)
    optimizer = torch.optim.AdamW(model.parameters(), lr=rate, weight_decay=0.0)
    device = model.table.device
    losses = []
    for _ in range(steps):
        ids = chains(batch, time + 1, vocab, device, generator)
        optimizer.zero_grad(set_to_none=True)
        loss = model.loss(ids)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return [float(x) for x in losses]


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--batch", type=int, default=16)
    parser.add_argument("--time", type=int, default=128)
    parser.add_argument("--vocab", type=int, default=256)
    parser.add_argument("--width", type=int, default=256)
    parser.add_argument("--heads", type=int, default=8)
    parser.add_argument("--layers", type=int, default=2)
    parser.add_argument("--dtype", choices=["float32", "bfloat16"], default="bfloat16")
    args = parser.parse_args()
    torch.manual_seed(0)
    model = RetentionLM(args.vocab, args.width, args.heads, args.layers,
                        dtype=getattr(torch, args.dtype)).to("cuda")
    losses = train(model, args.steps, args.batch, args.time, args.vocab)
    for i in range(0, args.steps, max(1, args.steps // 10)):
        print(f"step {i}: loss {losses[i]:.3f}")
    print(f"step {args.steps - 1}: loss {losses[-1]:.3f}")
    ids = chains(args.batch, args.time + 32, args.vocab, "cuda")
    got = model.generate(ids[:, :args.time], 32)
    share = (got == ids[:, args.time:]).float().mean().item()
    print(f"continued {args.batch} prompts of {args.time} tokens by 32: {100 * share:.0f}% right")


if __name__ == "__main__":
    main()
