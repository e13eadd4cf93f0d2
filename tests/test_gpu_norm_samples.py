"""Group norm over positions with many samples: a sample's result does not depend on
how many there are beside it, and blocks that walk over several samples are right."""

import numpy as np
import pytest
import torch

from mamba4_amd import group_norm
from oracle import retention as oracle
from tests.gpu_helpers import announce, host, normwise

pytestmark = pytest.mark.gpu


def _run(x, w, b, gate, d, groups, activation="silu"):
    x, w, b = (t.clone().requires_grad_() for t in (x, w, b))
    gate = None if gate is None else gate.clone().requires_grad_()
    y = group_norm(x, groups, w, b, gate=gate, activation=activation)
    wanted = [x, w, b] + ([] if gate is None else [gate])
    return y.detach(), torch.autograd.grad(y, wanted, d)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("positions,channels,groups", [
    (200, 48, 6),       # a few rows a thread
    (600, 64, 4),
    (3, 96, 12),
    (5000, 16, 2),      # many parts
    (300, 4200, 1),     # groups of more than a block's vectors (float32)
    (1, 8200, 1),       # one position, too wide for a wave
])
@pytest.mark.parametrize("gated", [False, True])
def test_a_samples_bits_do_not_depend_on_the_number_of_samples(gpu_lib, positions, channels,
                                                               groups, dtype, gated):
    announce(f"norm samples L{positions} C{channels} G{groups} {dtype} gated={gated}")
    most = min(1500, 40_000_000 // (positions * channels))
    g = torch.Generator(device="cuda").manual_seed(0)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    x, gate, d = (normal(most, positions, channels).to(dtype) for _ in range(3))
    w, b = normal(channels), normal(channels)
    first = None
    for samples in (1, 2, 9, 60, 400, 1500):
        if samples > most:
            break
        y, (dx, _, _, *dgate) = _run(x[:samples], w, b, gate[:samples] if gated else None,
                                     d[:samples], groups)
        mine = [t[0].clone() for t in (y, dx, *dgate)]
        first = first or mine
        for a, e in zip(mine, first):
            assert torch.equal(a, e), samples


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("samples,positions,channels,groups", [
    (3000, 3, 48, 6), (1500, 40, 206, 2), (1200, 1, 4100, 1), (2100, 130, 12, 3),
])
@pytest.mark.parametrize("gated", [False, True])
def test_blocks_that_walk_over_samples(gpu_lib, samples, positions, channels, groups, dtype,
                                       gated):
    """More samples than the launch has blocks for, against the oracle.  Float32: sums
    of up to 4,100 terms in float32, about sqrt(n) 2^-24 = 4e-6 of the largest, 2e-5
    with what follows; of 270,000 for weight and bias, 3e-5, 1e-4 with it.  Bfloat16:
    results rounded, 2^-9 of the element, 2^-8 with what precedes."""
    announce(f"norm walk M{samples} L{positions} C{channels} G{groups} {dtype} gated={gated}")
    rng = np.random.default_rng(1)
    shape = (samples, positions, channels)

    def device(a, kind=torch.float32):
        return torch.tensor(a, dtype=torch.float32, device="cuda").to(kind)

    x, d, gate = (device(rng.normal(size=shape), dtype) for _ in range(3))
    w, b = device(rng.uniform(0.5, 1.5, channels)), device(rng.normal(size=channels))
    gate = gate if gated else None
    y, grads = _run(x, w, b, gate, d, groups)
    arrays = [None if t is None else host(t.float()) for t in (x, w, b, gate, d)]
    xs, ws, bs, gs, ds = arrays
    want = oracle.group_norm(xs, groups, ws, bs, gs, "silu")
    expected = oracle.group_norm_backward(xs, groups, ds, ws, bs, gs, "silu")
    rows = 2e-5 if dtype == torch.float32 else 2.0 ** -8
    limits = [rows, 1e-4, 1e-4, rows]
    assert normwise(host(y.float()), want) <= rows
    for got, e, limit in zip(grads, expected, limits):
        assert normwise(host(got.float()), e) <= limit
