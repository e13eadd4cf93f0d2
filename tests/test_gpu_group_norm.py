"""Group normalisation on the GPU against the float64 oracle.

Tolerances, as max |difference| / max |expected|.  Float32: a handful of
roundings of 2^-24 an element on values up to a few times the largest, and sums
of up to a few ten thousand terms: 1e-5.  Bfloat16 results: half a unit of 2^-8
of the element: 2^-8.  Gradients of weight and bias are float32 sums over
exact inputs: 2e-5.
"""

import numpy as np
import pytest
import torch

from mamba4_amd import group_norm
from oracle import retention as oracle
from tests.gpu_helpers import announce, host, normwise

pytestmark = pytest.mark.gpu


def _cast(x, bf16):
    t = torch.tensor(x, dtype=torch.float32)
    return (t.to(torch.bfloat16) if bf16 else t).double().numpy()


def _problem(shape, bf16, affine, gated, seed=0, mean=0.5):
    rng = np.random.default_rng(seed)
    c = shape[-1]
    x = _cast(rng.normal(mean, 1.5, shape), bf16)
    dy = _cast(rng.normal(size=shape), bf16)
    w = _cast(rng.uniform(0.5, 1.5, c), False) if affine else None
    b = _cast(rng.normal(size=c), False) if affine else None
    gate = _cast(rng.normal(size=shape), bf16) if gated else None
    return x, dy, w, b, gate


def _device(a, bf16=False, grad=True):
    if a is None:
        return None
    t = torch.tensor(a, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    return t.requires_grad_(grad)


def _check(label, got, want, limit):
    error = normwise(host(got.float()), want)
    assert error <= limit, f"{label}: {error:.3g} > {limit:.3g}"


def _compare(shape, groups, bf16, affine, gated, activation, eps=1e-5, **kw):
    x, dy, w, b, gate = _problem(shape, bf16, affine, gated, **kw)
    tx, tg = _device(x, bf16), _device(gate, bf16)
    tw, tb = _device(w), _device(b)
    y = group_norm(tx, groups, tw, tb, gate=tg, activation=activation, eps=eps)
    named = [(n, t) for n, t in (("x", tx), ("weight", tw), ("bias", tb), ("gate", tg))
             if t is not None]
    grads = torch.autograd.grad(y, [t for _, t in named], _device(dy, bf16, False))
    torch.cuda.synchronize()
    want = oracle.group_norm(x, groups, w, b, gate, activation, eps)
    wants = dict(zip(("x", "weight", "bias", "gate"),
                     oracle.group_norm_backward(x, groups, dy, w, b, gate, activation, eps)))
    rows = 2.0 ** -8 if bf16 else 1e-5
    assert y.dtype == tx.dtype
    _check("y", y, want, rows)
    for (name, _), g in zip(named, grads):
        _check("d_" + name, g, wants[name], rows if name in ("x", "gate") else 2e-5)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("shape,groups", [
    ((1, 8), 1), ((5, 1536), 12), ((1000, 768), 12), ((300, 96), 32), ((33, 100), 4),
    ((17, 130), 1), ((9, 21), 7), ((40, 64), 64), ((7, 1000), 1), ((3, 4096), 1),
    ((2050, 24), 3), ((6, 6000), 2),
    ((2, 2, 64), 4), ((3, 77, 96), 8), ((1, 5000, 32), 2), ((700, 3, 48), 6), ((2, 301, 35), 5),
    ((2, 9, 11, 40), 4), ((2, 40, 5200), 1), ((1, 3, 9000), 3), ((1, 2000, 7), 7),
])
def test_forward_and_gradients(gpu_lib, shape, groups, bf16):
    announce(f"group norm {shape} G{groups} bf16={bf16}")
    _compare(shape, groups, bf16, True, False, "silu")
    _compare(shape, groups, bf16, True, True, "silu", seed=1)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("shape,groups", [((50, 256), 4), ((3, 60, 64), 4)])
@pytest.mark.parametrize("activation", ["none", "silu", "gelu"])
@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_options(gpu_lib, shape, groups, activation, affine, gated, bf16):
    announce(f"group norm {shape} {activation} affine={affine} gated={gated} bf16={bf16}")
    _compare(shape, groups, bf16, affine, gated, activation, eps=1e-3, seed=2)


def test_large_means_keep_the_variance(gpu_lib):
    """Deviations of 1 about a mean of 1000: the inputs' own rounding is 2^-14 of
    a deviation, and the result no worse than a few of those."""
    announce("group norm large mean")
    for shape in ((64, 256), (2, 3000, 64)):
        x = _cast(np.random.default_rng(3).normal(1000.0, 1.0, shape), False)
        y = group_norm(_device(x, grad=False), 4)
        _check("y", y, oracle.group_norm(x, 4), 2.0 ** -12)


def test_weight_or_bias_alone_and_constant_rows(gpu_lib):
    announce("group norm weight or bias alone")
    x, dy, w, b, _ = _problem((20, 96), False, True, False, seed=4)
    for weight, bias in ((w, None), (None, b)):
        ts = [_device(x), _device(weight), _device(bias)]
        y = group_norm(ts[0], 6, ts[1], ts[2], activation="gelu")
        _check("y", y, oracle.group_norm(x, 6, weight, bias, None, "gelu"), 1e-5)
        wants = oracle.group_norm_backward(x, 6, dy, weight, bias, None, "gelu")
        some = [t for t in ts if t is not None]
        for g, want in zip(torch.autograd.grad(y, some, _device(dy, grad=False)),
                           [u for t, u in zip(ts, wants) if t is not None]):
            _check("gradient", g, want, 2e-5)
    same = torch.full((3, 50, 64), 7.0, device="cuda")
    assert (group_norm(same, 4) == 0).all()


def test_a_bad_value_stays_in_its_group(gpu_lib):
    """A NaN or infinity reaches its own group only, both ways."""
    announce("group norm NaN")
    for shape in ((30, 128), (4, 50, 128)):
        x, dy, w, b, gate = _problem(shape, False, True, True, seed=5)
        clean = group_norm(_device(x), 4, _device(w), _device(b), gate=_device(gate))
        x[1].reshape(-1, 128)[0, 40] = np.nan
        tx = _device(x)
        y = group_norm(tx, 4, _device(w), _device(b), gate=_device(gate))
        d = torch.autograd.grad(y, tx, _device(dy, grad=False))[0]
        bad = torch.zeros(y.shape, dtype=torch.bool, device="cuda")
        bad[1, ..., 32:64] = True
        assert torch.isnan(y[bad]).all() and torch.isnan(d[bad]).all()
        assert torch.equal(y[~bad], clean[~bad]) and torch.isfinite(d[~bad]).all()


def test_a_samples_bits_do_not_depend_on_the_others(gpu_lib):
    announce("group norm batch")
    x = torch.randn(5000, 384, device="cuda")
    gate = torch.randn(5000, 384, device="cuda")
    y = group_norm(x, 6, gate=gate, activation="silu")
    for n in (1, 3, 700):
        assert torch.equal(group_norm(x[:n], 6, gate=gate[:n], activation="silu"), y[:n])


def test_repeatable_gradients_views_and_streams(gpu_lib):
    announce("group norm repeat, views, stream")
    wide = torch.randn(3000, 2 * 384 + 1, device="cuda").to(torch.bfloat16)
    x, gate = wide[:, 1:385], wide[:, 385:]
    w = torch.randn(384, device="cuda")
    dy = torch.randn(3000, 384, device="cuda").to(torch.bfloat16)

    def both():
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        y = group_norm(leaves[0], 6, leaves[1], gate=gate, activation="silu")
        return [y, *torch.autograd.grad(y, leaves, dy)]

    want = both()
    copy = group_norm(x.detach().contiguous(), 6, w, gate=gate.contiguous(), activation="silu")
    assert torch.equal(copy, want[0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = both()
    stream.synchronize()
    for a, b, c in zip(want, both(), other):
        assert torch.equal(a, b) and torch.equal(a, c)
    # An address that allows single elements only.
    odd = torch.randn(40 * 384 + 1, device="cuda").to(torch.bfloat16)[1:].view(40, 384)
    _check("unaligned", group_norm(odd, 6), oracle.group_norm(host(odd.float()), 6), 2.0 ** -8)


def test_gradients_against_differences(gpu_lib):
    """Central differences with a step of 2^-7: curvature about 2^-14, rounding
    2^-24 * 2^7 times the terms of the loss, both relative to its scale."""
    announce("group norm differences")
    x, dy, w, b, gate = _problem((6, 10, 32), False, True, True, seed=6)
    arrays = [x, w, b, gate]

    def call(a, grad=False):
        ts = [_device(v, grad=grad) for v in a]
        return ts, group_norm(ts[0], 4, ts[1], ts[2], gate=ts[3], activation="gelu")

    ts, y = call(arrays, True)
    grads = torch.autograd.grad(y, ts, _device(dy, grad=False))
    rng = np.random.default_rng(7)
    step = 2.0 ** -7
    for i, g in enumerate(grads):
        direction = rng.normal(size=arrays[i].shape)
        moved = [[a if j != i else a + s * step * direction for j, a in enumerate(arrays)]
                 for s in (1, -1)]
        up, down = ((host(call(a)[1]) * dy).sum() for a in moved)
        got, scale = (host(g) * direction).sum(), np.abs(host(g) * direction).sum()
        assert abs(got - (up - down) / (2 * step)) <= 2e-3 * scale, i


def test_graph_replays(gpu_lib):
    announce("group norm graph")
    x = torch.randn(3, 400, 64, device="cuda")
    want = group_norm(x, 4, activation="silu")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = group_norm(x, 4, activation="silu")
    for _ in range(3):
        y.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    del graph


def test_empty_and_refusals(gpu_lib):
    x = torch.randn(4, 12, device="cuda")
    assert group_norm(x[:0], 3).shape == (0, 12)
    assert group_norm(torch.zeros(2, 0, 12, device="cuda"), 3).shape == (2, 0, 12)
    with pytest.raises(ValueError, match="ROCm device"):
        group_norm(x.cpu(), 3)
    with pytest.raises(ValueError, match="groups"):
        group_norm(x, 5)
    with pytest.raises(ValueError, match="groups"):
        group_norm(x, 0)
    with pytest.raises(ValueError, match="activation"):
        group_norm(x, 3, activation="relu6")
    with pytest.raises(ValueError, match="weight"):
        group_norm(x, 3, x)
    with pytest.raises(ValueError, match="gate"):
        group_norm(x, 3, gate=x[:2])
    with pytest.raises(ValueError, match="one device"):
        group_norm(x, 3, x[0].cpu())
