"""Linear attention over sequences long enough for every route of its segments."""

import pytest
import torch

from mamba4_amd import linear_attention
from tests.gpu_helpers import announce

pytestmark = pytest.mark.gpu


def test_more_segments_than_blocks_along_y(gpu_lib):
    """Past 67M tokens a segment grows, so that a launch still takes them all.  With a
    decay of e^-1/2 a token the last tokens are those of the sequence's end alone
    (e^-100 of what came before); bfloat16 results, within 2^-8 of the largest."""
    time, tail = 65535 * 1024 + 70, 70 + 64 * 5
    announce(f"linear attention T{time}")
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(1, time, 1, 8, device="cuda", generator=gen, dtype=torch.bfloat16)
               for _ in range(3))
    g = torch.full((1,), -0.5, device="cuda")
    d = torch.zeros_like(v)
    d[:, -100:] = torch.randn(1, 100, 1, 8, device="cuda", generator=gen)

    def run(first):
        x = [t[:, first:].clone().requires_grad_() for t in (q, k, v)] + [g.clone().requires_grad_()]
        r = linear_attention(*x)
        grads = torch.autograd.grad(r.output, x, d[:, first:].contiguous())
        return [t[:, -100:].detach().clone() for t in (r.output, *grads[:3])] + [r.state, grads[3]]

    whole, end = run(0), run(time - tail)
    for a, b in zip(whole, end):
        assert torch.isfinite(a).all()
        assert ((a.double() - b.double()).abs().max() <= 2.0 ** -8 * b.double().abs().max()).item()
