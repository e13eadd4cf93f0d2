"""A small language model of selective state space layers: token ids to logits.

    x = embedding(ids);  per layer:
    n, x = rms_norm(h + x);    u, z = n W_in;    u = silu(causal_conv(u))
    d, b, c = u W_x;    h = selective_scan(u, d W_d, a, b, c, gate=z) W_out

Trains on sequences that hold pairs of a key and its value and ask for the values
again, then reads a prompt at once and goes on token by token from the layers'
states:

    python examples/selective_lm.py --steps 1000 --time 128 --dtype bfloat16
"""

import argparse
import os
import sys

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from mamba4_amd import (  # noqa: E402
    causal_conv,
    causal_conv_step_,
    embedding,
    rms_norm,
    selective_scan,
    selective_scan_step_,
)


class Selective(nn.Module):
    """The layer's part of the residual stream from h and the stream, both [..., D]."""

    def __init__(self, width, inner, states, groups=1, taps=4, rank=None):
        super().__init__()
        self.inner, self.states, self.groups = inner, states, groups
        self.rank = rank or max(1, width // 16)
        self.sizes = [self.rank, groups * states, groups * states]
        self.norm = nn.Parameter(torch.ones(width))
        self.project = nn.Parameter(torch.randn(2 * inner, width) / width**0.5)
        self.taps = nn.Parameter((2 * torch.rand(inner, taps) - 1) / taps**0.5)
        self.taps_bias = nn.Parameter(torch.zeros(inner))
        self.select = nn.Parameter(torch.randn(sum(self.sizes), inner) / inner**0.5)
        self.steps = nn.Parameter(torch.randn(inner, self.rank) / self.rank**0.5)
        # Steps between 0.001 and 0.1 at the start (the inverse of softplus of them).
        dt = torch.exp(torch.empty(inner).uniform_(-6.9, -2.3))
        self.steps_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        self.log_rates = nn.Parameter(torch.log(torch.arange(1.0, states + 1)).repeat(inner, 1))
        self.skip = nn.Parameter(torch.ones(inner))
        self.out = nn.Parameter(torch.randn(width, inner) / inner**0.5)

    def _split(self, h, stream):
        """The convolution's input and the gate (views of one projection), and the stream."""
        n, stream = rms_norm(h, self.norm, residual=stream)
        u, z = F.linear(n, self.project.to(n.dtype)).split(self.inner, -1)
        return u, z, stream

    def _selected(self, u):
        """delta, b and c (views of one projection) of the convolved u."""
        low, b, c = F.linear(u, self.select.to(u.dtype)).split(self.sizes, -1)
        shape = (self.groups, self.states)
        return F.linear(low, self.steps.to(u.dtype)), b.unflatten(-1, shape), c.unflatten(-1, shape)

    def _options(self, z):
        return dict(skip=self.skip, gate=z, delta_bias=self.steps_bias, softplus=True)

    def forward(self, h, stream, lengths=None):
        u, z, stream = self._split(h, stream)
        u, rows = causal_conv(u, self.taps, self.taps_bias, activation="silu", lengths=lengths)
        delta, b, c = self._selected(u)
        y, state = selective_scan(u, delta, -torch.exp(self.log_rates), b, c, lengths=lengths,
                                  **self._options(z))
        return F.linear(y, self.out.to(y.dtype)), stream, (rows, state)

    def step(self, h, stream, states, active=None):
        """One token of every row; the states (of ``forward``) are overwritten."""
        rows, state = states
        u, z, stream = self._split(h, stream)
        u = causal_conv_step_(rows, u, self.taps, self.taps_bias, activation="silu",
                              active=active).output
        delta, b, c = self._selected(u)
        y = selective_scan_step_(state, u, delta, -torch.exp(self.log_rates), b, c, active=active,
                                 **self._options(z)).output
        return F.linear(y, self.out.to(y.dtype)), stream


class SelectiveLM(nn.Module):
    def __init__(self, vocab, width, layers, states=16, groups=1, dtype=torch.float32):
        super().__init__()
        self.dtype = dtype
        self.scale = width**0.5
        self.table = nn.Parameter(torch.randn(vocab, width) / width**0.5)
        self.layers = nn.ModuleList(
            Selective(width, 2 * width, states, groups) for _ in range(layers))
        self.norm = nn.Parameter(torch.ones(width))

    def _logits(self, h, stream):
        n = rms_norm(h, self.norm, residual=stream).output
        return F.linear(n, self.table.to(self.dtype)).float()

    def _start(self, ids):
        """No layer's output yet, and the float32 residual stream."""
        stream = embedding(ids, self.table, scale=self.scale, dtype=torch.float32)
        return torch.zeros(stream.shape, dtype=self.dtype, device=stream.device), stream

    def forward(self, ids, lengths=None):
        """Logits [B,T,V] of ids [B,T] (-1: no token), and the layers' states."""
        h, stream = self._start(ids)
        states = []
        for layer in self.layers:
            h, stream, state = layer(h, stream, lengths)
            states.append(state)
        return self._logits(h, stream), states

    @torch.no_grad()
    def step(self, ids, states, active=None):
        """Logits [B,V] after one more token of every row, ids [B]."""
        h, stream = self._start(ids)
        for layer, state in zip(self.layers, states):
            h, stream = layer.step(h, stream, state, active)
        return self._logits(h, stream)

    def loss(self, ids, asked):
        """Of the tokens that ``asked`` [B,T] marks."""
        logits, _ = self(ids[:, :-1])
        each = F.cross_entropy(logits.flatten(0, 1), ids[:, 1:].flatten(), reduction="none")
        mask = asked[:, 1:].flatten().to(each.dtype)
        return (each * mask).sum() / mask.sum()

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


def pairs(batch, time, vocab, count, device, generator=None):
    """Sequences [batch,time] of `count` pairs, a key of the first half of the vocabulary
    and a value of the second, drawn over and over; and which tokens are values of keys
    that have occurred."""
    half = vocab // 2
    keys = torch.stack([torch.randperm(half, generator=generator)[:count] for _ in range(batch)])
    values = half + torch.randint(half, (batch, count), generator=generator)
    drawn = torch.randint(count, (batch, (time + 1) // 2), generator=generator)
    ids = torch.stack([keys.gather(1, drawn), values.gather(1, drawn)], -1).flatten(1)[:, :time]
    seen = torch.stack([(drawn[:, :i] == drawn[:, i:i + 1]).any(1)
                        for i in range(drawn.shape[1])], 1)
    asked = torch.stack([torch.zeros_like(seen), seen], -1).flatten(1)[:, :time]
    return ids.to(device), asked.to(device)


def train(model, steps, batch, time, vocab, count, rate=2e-3, seed=0):
    """The losses of every step."""
    generator = torch.Generator().manual_seed(seed)
    optimizer = torch.optim.AdamW(model.parameters(), lr=rate, weight_decay=0.0)
    device = model.table.device
    losses = []
    for _ in range(steps):
        ids, asked = pairs(batch, time, vocab, count, device, generator)
        optimizer.zero_grad(set_to_none=True)
        loss = model.loss(ids, asked)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return [float(x) for x in losses]


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=1000)
    parser.add_argument("--batch", type=int, default=32)
    parser.add_argument("--time", type=int, default=128)
    parser.add_argument("--vocab", type=int, default=64)
    parser.add_argument("--pairs", type=int, default=8)
    parser.add_argument("--width", type=int, default=128)
    parser.add_argument("--layers", type=int, default=2)
    parser.add_argument("--dtype", choices=["float32", "bfloat16"], default="bfloat16")
    args = parser.parse_args()
    torch.manual_seed(0)
    model = SelectiveLM(args.vocab, args.width, args.layers,
                        dtype=getattr(torch, args.dtype)).to("cuda")
    losses = train(model, args.steps, args.batch, args.time, args.vocab, args.pairs)
    for i in range(0, args.steps, max(1, args.steps // 10)):
        print(f"step {i}: loss {losses[i]:.3f}")
    print(f"step {args.steps - 1}: loss {losses[-1]:.3f}")
    # Of each prompt the last token is a key: its value is the answer.
    time = args.time // 2 * 2 - 1
    ids, asked = pairs(args.batch, time + 1, args.vocab, args.pairs, "cuda")
    got = model.generate(ids[:, :time], 1)[:, 0]
    known = asked[:, time]
    share = (got == ids[:, time])[known].float().mean().item()
    print(f"answered {int(known.sum())} prompts of {time} tokens: {100 * share:.0f}% right")


if __name__ == "__main__":
    main()
