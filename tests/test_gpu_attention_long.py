"""Linear attention over sequences long enough for every route of its segments."""

import numpy as np
import pytest
import torch

from mamba4_amd import linear_attention, linear_attention_step
from oracle import retention as oracle
from tests.gpu_helpers import announce, host, normwise

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


NAMES = ("q", "k", "v", "log_decay", "initial")


def _problem(b, t, h, n, p, bf16, seed):
    rng = np.random.default_rng(seed)

    def f32(a):
        return a.astype(np.float32).astype(np.float64)

    def rows(a):
        return torch.tensor(a, dtype=torch.float32).to(
            torch.bfloat16 if bf16 else torch.float32).double().numpy()

    q, k = (rows(rng.normal(size=(b, t, h, n)) / np.sqrt(n)) for _ in range(2))
    v, d = (rows(rng.normal(size=(b, t, h, p))) for _ in range(2))
    g = f32(-np.log1p(np.exp(-rng.normal(3.0, 1.5, (b, t, h)))))
    s0, d_state = (f32(rng.normal(size=(b, h, n, p))) for _ in range(2))
    return [q, k, v, g, s0], d, d_state


def _device(a, bf16=False):
    return torch.tensor(a, dtype=torch.float32, device="cuda").to(
        torch.bfloat16 if bf16 else torch.float32)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("b,t,h,n,p,heads,lengths", [
    # Segments of 4, 8 and 16 chunks in the backward; 9, 5, 9 and 5 of them.
    (1, 2100, 8, 128, 128, (0, 7), None),
    (1, 2100, 32, 128, 128, (3,), None),
    (2, 8300, 32, 64, 64, (0, 31), (8300, 5003)),
    (1, 4200, 32, 128, 128, (9,), (4111,)),
])
def test_long_sequences(gpu_lib, monkeypatch, b, t, h, n, p, heads, lengths, bf16):
    """Segments of every length, more of them than a carry loads at once, decays'
    gradients over more tokens than a block: some heads against the oracle, and a
    walk and a split run bit by bit.  Tolerances as of short sequences (a decay of
    e^-1/20 a token forgets within a few hundred): float32 sums 2e-5, of differences
    over a segment 1e-4, bfloat16 results 2^-8."""
    announce(f"linear attention long B{b} T{t} H{h} N{n} P{p} bf16={bf16}")
    arrays, d, d_state = _problem(b, t, h, n, p, bf16, seed=t + h)
    lens = None if lengths is None else torch.tensor(lengths, device="cuda")
    results = []
    for route in ("walk", "split"):
        monkeypatch.setenv("M4RT_ATTENTION", route)
        x = [_device(a, bf16 and i < 3).requires_grad_() for i, a in enumerate(arrays)]
        r = linear_attention(*x[:4], initial=x[4], lengths=lens, scale=0.5)
        grads = torch.autograd.grad((r.output, r.state), x, (_device(d, bf16), _device(d_state)))
        results.append([r.output.detach(), r.state.detach(), *grads])
    for a, e in zip(*results):
        assert torch.equal(a, e)
    heads = list(heads)
    mine = [a[:, heads] if i == 4 else a[:, :, heads] for i, a in enumerate(arrays)]
    d, d_state = d[:, :, heads], d_state[:, heads]
    out, state = oracle.attention(*mine, lengths=lengths, scale=0.5)
    want = oracle.attention_backward(*mine[:4], d, d_state, mine[4], lengths, 0.5)
    rows = 2.0 ** -8 if bf16 else 2e-5
    limits = [rows, 2e-5, rows, rows, rows, 1e-4, 2e-5]
    for name, got, e, limit in zip(("output", "state") + NAMES, results[0], (out, state, *want),
                                   limits):
        got = got[:, heads] if name in ("state", "initial") else got[:, :, heads]
        error = normwise(host(got.float()), e)
        assert error <= limit, f"{name}: {error:.3g} > {limit:.3g}"


@pytest.mark.parametrize("bf16", [False, True])
def test_long_prompts(gpu_lib, monkeypatch, bf16):
    """The forward's segments of 16 chunks, 13 of them, by a constant decay of each head
    and keys that heads share."""
    announce(f"linear attention prompt T12300 bf16={bf16}")
    arrays, _, _ = _problem(1, 12300, 32, 128, 128, bf16, seed=5)
    q, k, v, _, s0 = arrays
    k = k[:, :, :8]
    g = -np.exp2(-3.0 - 5.0 * np.arange(32) / 31)
    results = []
    for route in ("walk", "split"):
        monkeypatch.setenv("M4RT_ATTENTION", route)
        with torch.no_grad():
            results.append(linear_attention(*(_device(a, bf16) for a in (q, k, v)), _device(g),
                                            initial=_device(s0)))
    for a, e in zip(*results):
        assert torch.equal(a, e)
    for head in (0, 17, 31):
        out, state = oracle.attention(q[:, :, [head]], k[:, :, [head // 4]], v[:, :, [head]],
                                      g.astype(np.float32)[[head]], s0[:, [head]])
        assert normwise(host(results[0].output[:, :, [head]].float()), out) <= (
            2.0 ** -8 if bf16 else 2e-5)
        assert normwise(host(results[0].state[:, [head]]), state) <= 2e-5


def test_strided_rows_of_a_long_sequence(gpu_lib):
    """Views of one projection, 17 segments, against the oracle."""
    announce("linear attention strided T4100")
    rng = np.random.default_rng(6)
    t, n = 4100, 64
    whole = rng.normal(size=(1, t, 3 * 2 * n)).astype(np.float32) / 8
    x = torch.tensor(whole, device="cuda")
    q, k, v = (x[..., i * 2 * n:(i + 1) * 2 * n].unflatten(-1, (2, n)) for i in range(3))
    g = -rng.uniform(0.0, 0.1, (1, t, 2)).astype(np.float32)
    r = linear_attention(q, k, v, torch.tensor(g, device="cuda"))
    rows = whole.astype(np.float64).reshape(1, t, 3, 2, n)
    out, state = oracle.attention(rows[:, :, 0], rows[:, :, 1], rows[:, :, 2], g)
    assert normwise(host(r.output), out) <= 2e-5
    assert normwise(host(r.state), state) <= 2e-5


@pytest.mark.parametrize("p", [128, 127])
def test_one_token_of_many_heads(gpu_lib, p):
    """More heads than a token stride could hold: o = (q . k) v for each, the gradients
    of the shared rows sums over the heads (70,000 terms, sqrt(n) 2^-24 = 2e-5)."""
    announce(f"linear attention one token P{p}")
    gen = torch.Generator(device="cuda").manual_seed(4)
    heads = 70_000
    q, k = (torch.randn(1, 1, h, 8, device="cuda", generator=gen).requires_grad_()
            for h in (1, heads))
    v = torch.randn(1, 1, 1, p, device="cuda", generator=gen).requires_grad_()
    d = torch.randn(1, 1, heads, p, device="cuda", generator=gen)
    r = linear_attention(q, k, v, torch.zeros(heads, device="cuda"))
    want = (q.double() * k.double()).sum(-1, keepdim=True) * v.double()
    assert (r.output.double() - want).abs().max() <= 1e-5 * want.abs().max()
    grads = torch.autograd.grad(r.output, (q, k, v), d)
    expected = torch.autograd.grad(want, (q, k, v), d.double())
    for a, e in zip(grads, expected):
        assert (a.double() - e.double()).abs().max() <= 5e-5 * e.double().abs().max()
