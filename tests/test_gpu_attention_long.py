"""Linear attention over sequences long enough for every route of its segments."""

import pytest
import torch

from mamba4_amd import linear_attention, linear_attention_step
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sums_of_shared_heads_over_many_elements(gpu_lib, dtype):
    """33M elements of a shared head's gradient, twice the threads of the launch that
    sums them: the sums of the heads' own gradients (float32: the same additions;
    bfloat16: of parts rounded before their sum, 2^-8 of them)."""
    time = 1 << 18
    announce(f"shared heads T{time} {dtype}")
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, v = (torch.randn(1, time, 2, 128, device="cuda", generator=gen).to(dtype) for _ in range(2))
    k = torch.randn(1, time, 1, 128, device="cuda", generator=gen).to(dtype)
    g = torch.full((2,), -0.1, device="cuda")
    d = torch.randn(1, time, 2, 128, device="cuda", generator=gen).to(dtype)
    k.requires_grad_()
    (shared,) = torch.autograd.grad(linear_attention(q, k, v, g).output, k, d)
    own = k.detach().expand(-1, -1, 2, -1).contiguous().requires_grad_()
    (parts,) = torch.autograd.grad(linear_attention(q, own, v, g).output, own, d)
    want = parts.float().sum(dim=2, keepdim=True)
    if dtype == torch.float32:
        assert torch.equal(shared, want)
    else:
        off = (shared.float() - want).abs().max()
        assert (off <= 3 * 2.0 ** -9 * parts.float().abs().max()).item()


def test_many_rows_of_odd_widths(gpu_lib):
    """34M pieces of 16 bytes to be copied, twice the threads of the launch that
    copies them: the results of the padded rows."""
    time = 1 << 21
    announce(f"odd widths T{time}")
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(1, time, 2, w, device="cuda", generator=gen, dtype=torch.bfloat16)
               for w in (63, 63, 61))
    g = torch.full((2,), -0.1, device="cuda")
    got = linear_attention(q, k, v, g)
    pad = torch.nn.functional.pad
    want = linear_attention(pad(q, (0, 1)), pad(k, (0, 1)), pad(v, (0, 3)), g)
    assert torch.equal(got.output, want.output[..., :61])
    assert torch.equal(got.state, want.state[..., :63, :61])


def test_the_largest_batches(gpu_lib):
    """Just under the 2^32 threads of a launch, which the entry points allow."""
    announce("largest batches")
    gen = torch.Generator(device="cuda").manual_seed(3)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    batch = 2**24 - 10
    s, q, k, v = normal(batch, 1, 1, 1), *(normal(batch, 1, 1) for _ in range(3))
    g = torch.tensor([-0.25], device="cuda")
    r = linear_attention_step(s, q, k, v, g)
    want = torch.exp(g) * s[..., 0] + k * v
    assert torch.allclose(r.state[..., 0], want, rtol=1e-6, atol=1e-6)
    assert torch.allclose(r.output, want * q, rtol=1e-6, atol=1e-6)
    batch = 2**23 - 9
    q, k, v = (normal(batch, 1, 1, 4) for _ in range(3))
    r = linear_attention(q, k, v, g)
    assert torch.allclose(r.state, k[:, 0, :, :, None] * v[:, 0, :, None, :], rtol=1e-5, atol=1e-5)
    assert torch.allclose(r.output, (q * k).sum(-1, keepdim=True) * v, rtol=1e-4, atol=1e-4)
