"""The root-mean-square norm on the GPU against the float64 oracle.

Tolerances, as max |difference| / max |expected|.  Float32: a handful of roundings of
2^-24 on values, means over up to 32,768 squares of one sign: 5e-6; the weight's
gradient sums rows: 2e-5.  The gradient of the sum is a difference, (dn - n mean(dn n))
/ deviation, that cancels where a row has few channels (all but eps / x^2 of it with one):
its float32 error is that of its terms, dn / deviation.  Bfloat16 results are rounded once: 2^-8 + 5e-6.  8-bit
results: half a step of 2^-3 of the value (2^-4), or of the smallest step, 2^-10 of the
scale, both with the float32 error of value and scale.
"""

import numpy as np
import pytest
import torch

from mamba4_amd import rms_norm, rms_norm_e4m3
from oracle import selective as oracle
from tests.gpu_helpers import announce, host, normwise

pytestmark = pytest.mark.gpu

F32 = 5e-6
SUMS = 2e-5
BF16 = 2.0 ** -8 + F32
TYPES = {"f": torch.float32, "b": torch.bfloat16}


def _limit(dtype):
    return BF16 if dtype == torch.bfloat16 else F32


def _rounded(dtype):
    return lambda s: torch.tensor(s).float().to(dtype).double().numpy()


def _problem(m, c, x, residual, weight=True, seed=0):
    rng = np.random.default_rng(seed)
    t = dict(x=torch.tensor(rng.normal(size=(m, c)), device="cuda").to(TYPES[x]))
    if residual:
        t["residual"] = torch.tensor(rng.normal(0.0, 2.0, (m, c)), device="cuda") \
            .to(TYPES[residual])
    if weight:
        t["weight"] = torch.tensor(rng.uniform(0.5, 1.5, c), device="cuda").float()
    return t, rng


def _arrays(t):
    return {k: host(v.float()) for k, v in t.items()}


def _check(label, got, want, limit, terms=0.0):
    got = host(got.float())
    error = normwise(got, want)
    if terms:
        error = np.abs(got - want).max() / max(np.abs(want).max(), terms)
    assert error <= limit, f"{label}: {error:.3g} > {limit:.3g}"


def _oracle(t, eps):
    kept = t["residual"].dtype if "residual" in t else t["x"].dtype
    return oracle.rms(**_arrays(t), eps=eps, rounded=_rounded(kept))


def _compare(t, rng, eps=1e-5):
    t = {k: v.detach().requires_grad_() for k, v in t.items()}
    y, s = rms_norm(t["x"], t.get("weight"), residual=t.get("residual"), eps=eps)
    d_y = torch.tensor(rng.normal(size=y.shape), device="cuda").to(y.dtype)
    outs, cots = [y], [d_y]
    d_s = None
    if "residual" in t:
        d_s = torch.tensor(rng.normal(size=y.shape), device="cuda").to(s.dtype)
        outs, cots = [y, s], [d_y, d_s]
    grads = dict(zip(t, torch.autograd.grad(outs, list(t.values()), cots)))
    torch.cuda.synchronize()
    want, total = _oracle(t, eps)
    assert y.dtype == t["x"].dtype
    _check("y", y, want, _limit(y.dtype))
    assert (host(s.float()) == total).all()
    weight = None if "weight" not in t else host(t["weight"])
    d_total, d_weight = oracle.rms_backward(
        total, host(d_y.float()), None if d_s is None else host(d_s.float()), weight, eps)
    terms = np.abs(host(d_y.float()) * (1.0 if weight is None else weight)
                   / np.sqrt((total * total).mean(-1, keepdims=True) + eps)).max()
    for name, g in grads.items():
        assert g.dtype == t[name].dtype and g.shape == t[name].shape
        if name == "weight":
            _check("d_weight", g, d_weight, SUMS)
        else:
            _check("d_" + name, g, d_total, _limit(g.dtype), terms)
    with torch.no_grad():
        plain, sum2 = rms_norm(t["x"], t.get("weight"), residual=t.get("residual"), eps=eps)
    assert torch.equal(plain, y) and torch.equal(sum2, s)


@pytest.mark.parametrize("x,residual", [("f", ""), ("b", ""), ("f", "f"), ("b", "f"), ("f", "b"),
                                        ("b", "b")])
@pytest.mark.parametrize("m,c", [
    (1, 1), (5, 8), (3, 7), (300, 64), (70, 100), (33, 512), (1000, 768), (9, 1000), (6, 1024),
    (4, 1032), (3, 4096), (2, 8191), (2, 12000), (1, 16384), (2, 32768), (1, 32767), (5000, 24),
])
def test_forward_and_gradients(gpu_lib, m, c, x, residual):
    announce(f"rms norm {m} x {c} x={x} residual={residual}")
    _compare(*_problem(m, c, x, residual))


def test_without_weight_eps_and_axes(gpu_lib):
    announce("rms norm options")
    _compare(*_problem(20, 96, "b", "f", weight=False, seed=1), eps=0.5)
    t, _ = _problem(24, 40, "f", "f", seed=2)
    flat, s = rms_norm(t["x"], t["weight"], residual=t["residual"])
    shaped = {k: v.view(2, 3, 4, 40) for k, v in t.items() if k != "weight"}
    y, s2 = rms_norm(shaped["x"], t["weight"], residual=shaped["residual"])
    assert torch.equal(y.view(24, 40), flat) and torch.equal(s2.view(24, 40), s)
    one = rms_norm(t["x"][0], t["weight"])
    assert one.output.shape == (40,) and one.sum.data_ptr() == t["x"].data_ptr()


def test_gradients_of_parts(gpu_lib):
    """Of the sum alone, of the output alone, of one input alone."""
    announce("rms norm parts")
    t, rng = _problem(30, 72, "b", "f", seed=3)
    t = {k: v.requires_grad_() for k, v in t.items()}
    y, s = rms_norm(t["x"], t["weight"], residual=t["residual"])
    d = torch.tensor(rng.normal(size=(30, 72)), device="cuda").float()
    gx, gr, gw = torch.autograd.grad(s, [t["x"], t["residual"], t["weight"]], d,
                                     retain_graph=True, allow_unused=True)
    assert torch.equal(gr, d) and torch.equal(gx, d.to(torch.bfloat16)) and (gw == 0).all()
    every = torch.autograd.grad(y, [t["x"], t["residual"], t["weight"]], d.to(y.dtype),
                                retain_graph=True)
    for i, name in enumerate(("x", "residual", "weight")):
        alone = {k: v.detach().requires_grad_(k == name) for k, v in t.items()}
        y2, _ = rms_norm(alone["x"], alone["weight"], residual=alone["residual"])
        g, = torch.autograd.grad(y2, [alone[name]], d.to(y.dtype))
        assert torch.equal(g, every[i]), name


@pytest.mark.parametrize("x,residual", [("f", ""), ("b", ""), ("b", "f"), ("f", "b"), ("b", "b")])
@pytest.mark.parametrize("m,c,block", [
    (1, 1, None), (5, 8, 32), (70, 100, 32), (33, 512, 64), (1000, 768, 128), (9, 1000, 256),
    (6, 1024, None), (4, 1032, 512), (40, 4096, 128), (3, 4096, None), (2, 8191, 32),
    (2, 12000, 512), (1, 32768, 32), (300, 40, 64), (7, 333, None), (3, 700, 64),
])
def test_8_bits(gpu_lib, m, c, block, x, residual):
    announce(f"rms norm e4m3 {m} x {c} block {block} x={x} residual={residual}")
    t, _ = _problem(m, c, x, residual, seed=4)
    q, scale, s = rms_norm_e4m3(t["x"], t["weight"], residual=t.get("residual"), block=block)
    want, total = _oracle(t, 1e-5)
    block = c if block is None or block > c else block
    blocks = -(-c // block)
    assert q.dtype == torch.float8_e4m3fn and q.shape == (m, c)
    assert scale.shape == (m, blocks) and scale.dtype == torch.float32
    assert (host(s.float()) == total).all()
    padded = np.zeros((m, blocks * block))
    padded[:, :c] = np.abs(want)
    most = padded.reshape(m, blocks, block).max(-1)
    np.testing.assert_allclose(host(scale), most / 448.0, rtol=F32)
    spread = np.repeat(host(scale), block, axis=1)[:, :c]
    error = np.abs(host(q.float()) * spread - want)
    limit = np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * spread) + 2 * F32 * np.abs(want)
    assert (error <= limit).all()
    # The rounding is to nearest of the value over the scale as they came out.
    y, _ = rms_norm(t["x"].float(), t["weight"], residual=None if "residual" not in t
                    else t["residual"]) if residual != "b" or x == "f" else (None, None)
    if y is not None:
        plain = (y.float() / torch.tensor(spread, device="cuda").float()).to(torch.float8_e4m3fn)
        same = (plain.float() == q.float()).float().mean().item()
        assert same > 1 - 1e-3 - 2.0 / (m * c)


def test_8_bits_of_zeros_and_bad_values(gpu_lib):
    announce("rms norm e4m3 zeros, NaN")
    x = torch.randn(6, 256, device="cuda")
    x[1] = 0.0
    x[2, 40] = float("nan")
    x[3, 200] = float("inf")
    x[4] *= 1e-30
    q, scale, _ = rms_norm_e4m3(x, block=64)
    assert (q[1].float() == 0).all() and (scale[1] == 2.0 ** -126).all()
    # (The statistics of a row with a NaN are NaN throughout.)
    assert torch.isnan(q[2].float()).all() and torch.isnan(scale[2]).all()
    # An infinite mean square leaves zeros, and a NaN in the infinity's own block.
    assert (q[3, :192].float() == 0).all() and torch.isnan(q[3, 192:].float()).all()
    good = torch.tensor([0, 4, 5], device="cuda")
    clean = rms_norm_e4m3(x[good], block=64)
    assert torch.equal(q[good].view(torch.uint8), clean.output.view(torch.uint8))
    assert torch.equal(scale[good], clean.scale)
    assert (q[good].float().abs().amax(-1) == 448).all()
    with pytest.raises(ValueError, match="no gradient"):
        rms_norm_e4m3(x.requires_grad_())


def test_a_rows_bits_do_not_depend_on_the_others(gpu_lib):
    announce("rms norm batch")
    for c in (40, 768, 2056, 999):
        t, _ = _problem(3000, c, "b", "f", seed=5)
        y, s = rms_norm(t["x"], t["weight"], residual=t["residual"])
        for n in (1, 3, 700):
            z, r = rms_norm(t["x"][:n], t["weight"], residual=t["residual"][:n])
            assert torch.equal(z, y[:n]) and torch.equal(r, s[:n])


def test_views_streams_and_repeats(gpu_lib):
    announce("rms norm views, streams")
    wide = torch.randn(500, 900, device="cuda").to(torch.bfloat16)
    weight = torch.randn(400, device="cuda")
    for x in (wide[:, 8:408], wide[:, 1:401], wide.t()[:, :400], wide[:1, :400].expand(500, 400)):
        y = rms_norm(x, weight).output
        assert torch.equal(y, rms_norm(x.contiguous(), weight).output)
    odd = torch.randn(40 * 64 + 1, device="cuda")[1:].view(40, 64)
    _check("unaligned", rms_norm(odd).output, oracle.rms(host(odd))[0], F32)
    t, rng = _problem(2000, 768, "b", "b", seed=6)
    d = torch.tensor(rng.normal(size=(2000, 768)), device="cuda").to(torch.bfloat16)

    def both():
        leaves = {k: v.detach().requires_grad_() for k, v in t.items()}
        y, s = rms_norm(leaves["x"], leaves["weight"], residual=leaves["residual"])
        return [y, s, *torch.autograd.grad([y, s], list(leaves.values()), [d, d])]

    want = both()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = both()
    stream.synchronize()
    for u, v, w in zip(want, both(), other):
        assert torch.equal(u, v) and torch.equal(u, w)


def test_other_types(gpu_lib):
    announce("rms norm types")
    x = torch.randn(10, 32, device="cuda")
    r = rms_norm(x.half(), residual=x.double())
    assert r.output.dtype == torch.float16 and r.sum.dtype == torch.float64
    want = rms_norm(x.half().float(), residual=x)
    assert torch.equal(r.output, want.output.half())


def test_gradients_against_differences(gpu_lib):
    """Central differences with a step of 2^-7 along a random direction: curvature about
    2^-14 of the terms, rounding 2^-24 2^7 of the loss's terms."""
    announce("rms norm differences")
    t, rng = _problem(6, 40, "f", "f", seed=7)
    t = {k: v.requires_grad_() for k, v in t.items()}
    d_y, d_s = rng.normal(size=(6, 40)), rng.normal(size=(6, 40))

    def loss(a):
        y, s = rms_norm(a["x"], a["weight"], residual=a["residual"])
        return y, s, (host(y) * d_y).sum() + (host(s) * d_s).sum()

    y, s, _ = loss(t)
    grads = torch.autograd.grad([y, s], list(t.values()), [
        torch.tensor(d, device="cuda").float() for d in (d_y, d_s)])
    step = 2.0 ** -7
    for name, g in zip(t, grads):
        direction = rng.normal(size=t[name].shape)
        move = torch.tensor(step * direction, device="cuda").float()
        up, down = (loss({**t, name: (t[name] + k * move).detach()})[2] for k in (1, -1))
        got, scale = (host(g) * direction).sum(), np.abs(host(g) * direction).sum()
        assert abs(got - (up - down) / (2 * step)) <= 2e-3 * scale, name


def test_graph_replays(gpu_lib):
    announce("rms norm graph")
    t, rng = _problem(300, 768, "b", "f", seed=8)
    t = {k: v.requires_grad_() for k, v in t.items()}
    d = torch.tensor(rng.normal(size=(300, 768)), device="cuda").to(torch.bfloat16)

    def both():
        y, s = rms_norm(t["x"], t["weight"], residual=t["residual"])
        with torch.no_grad():
            q = rms_norm_e4m3(t["x"], t["weight"], residual=t["residual"], block=128)
        return [y, s, q.scale, *torch.autograd.grad(y, list(t.values()), d)], q.output

    want, bits = both()
    want = [u.detach().clone() for u in want]
    bits = bits.view(torch.uint8).clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, q = both()
    for _ in range(3):
        for u in got:
            u.detach().fill_(float("nan"))
        q.view(torch.uint8).fill_(1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip(got, want):
            assert torch.equal(u, v)
        assert torch.equal(q.view(torch.uint8), bits)
    del graph, got, q


def test_empty(gpu_lib):
    announce("rms norm without rows")
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    y, s = rms_norm(x, w, residual=x.detach().to(torch.bfloat16))
    assert y.shape == (0, 16) and s.dtype == torch.bfloat16
    gx, gw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert gx.shape == (0, 16) and (gw == 0).all()
    q = rms_norm_e4m3(torch.zeros(2, 0, 16, device="cuda"), block=32)
    assert q.output.shape == (2, 0, 16) and q.scale.shape == (2, 0, 1)
