"""The selective scan on the GPU against the float64 oracle.

Tolerances, as max |difference| / max |expected|.  Float32: a decay is off by 2^-24
of itself and of its exponent, so that what survives k tokens is off by about
sqrt(k) 2^-24, k up to a few hundred here; results of a few such factors and sums of
up to 64 states or a few hundred channels: 2e-5.  Gradients of a, skip and the bias
sum signed terms over all tokens, up to a few times larger than their sum: 5e-5.
Bfloat16 results are rounded once, half a unit of 2^-8, of values to the same: 2^-8 +
2e-5.
"""

import numpy as np
import pytest
import torch

from mamba4_amd import selective_scan, selective_scan_step, selective_scan_step_
from oracle import selective as oracle
from tests.gpu_helpers import announce, host, normwise

pytestmark = pytest.mark.gpu

ROWS = ("x", "delta", "b", "c", "gate")
F32 = 2e-5
SUMS = 5e-5
BF16 = 2.0 ** -8 + F32


def _cast(x, bf16):
    t = torch.tensor(x, dtype=torch.float32)
    return (t.to(torch.bfloat16) if bf16 else t).double().numpy()


def _problem(b, t, d, g, n, bf16, softplus=True, gate=True, skip=True, initial=False, seed=0):
    rng = np.random.default_rng(seed)
    steps = np.exp(rng.uniform(np.log(1e-3), np.log(1e-1), d))
    x = dict(x=rng.normal(size=(b, t, d)), b=rng.normal(size=(b, t, g, n)),
             c=rng.normal(size=(b, t, g, n)))
    x["delta"] = rng.normal(0.0, 0.5, (b, t, d))
    x["a"] = -np.arange(1, n + 1) * rng.uniform(0.8, 1.2, (d, n))
    if softplus:
        x["bias"] = np.log(np.expm1(steps))
    else:
        x["delta"] = steps * np.exp(x["delta"])
    if skip:
        x["skip"] = rng.normal(1.0, 0.2, d)
    if gate:
        x["gate"] = rng.normal(size=(b, t, d))
    if initial:
        x["initial"] = rng.normal(size=(b, d, n))
    x = {k: _cast(v, bf16 and k in ROWS) for k, v in x.items()}
    d_out = _cast(rng.normal(size=(b, t, d)), bf16)
    d_state = _cast(rng.normal(size=(b, d, n)), False) if initial else None
    return x, d_out, d_state


def _tensors(x, bf16, grad):
    return {k: torch.tensor(v, device="cuda", dtype=torch.bfloat16 if bf16 and k in ROWS
                            else torch.float32).requires_grad_(grad) for k, v in x.items()}


def _call(t, softplus, lengths=None):
    lens = None if lengths is None else torch.tensor(lengths, device="cuda")
    return selective_scan(t["x"], t["delta"], t["a"], t["b"], t["c"], skip=t.get("skip"),
                          gate=t.get("gate"), delta_bias=t.get("bias"), softplus=softplus,
                          initial=t.get("initial"), lengths=lens)


def _check(label, got, want, limit):
    error = normwise(host(got.float()), want)
    assert error <= limit, f"{label}: {error:.3g} > {limit:.3g}"


def _grads(t, r, d_out, d_state):
    outs, cots = [r.output], [torch.tensor(d_out, device="cuda").to(r.output.dtype)]
    if d_state is not None:
        outs.append(r.state)
        cots.append(torch.tensor(d_state, device="cuda", dtype=torch.float32))
    return dict(zip(t, torch.autograd.grad(outs, list(t.values()), cots)))


def _compare(x, d_out, d_state, bf16, softplus, lengths=None):
    t = _tensors(x, bf16, True)
    r = _call(t, softplus, lengths)
    grads = _grads(t, r, d_out, d_state)
    torch.cuda.synchronize()
    out, state = oracle.scan(**x, softplus=softplus, lengths=lengths)
    want = oracle.scan_backward(**x, d_output=d_out, d_state=d_state, softplus=softplus,
                                lengths=lengths)
    rows = BF16 if bf16 else F32
    assert r.output.dtype == t["x"].dtype and r.state.dtype == torch.float32
    _check("output", r.output, out, rows)
    _check("state", r.state, state, F32)
    for name, g in grads.items():
        assert g.shape == t[name].shape and g.dtype == t[name].dtype
        limit = rows if name in ROWS else F32 if name == "initial" else SUMS
        _check("d_" + name, g, want[name], limit)
    with torch.no_grad():
        plain = _call(t, softplus, lengths)
    assert torch.equal(plain.output, r.output) and torch.equal(plain.state, r.state)
    return r, grads


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("b,t,d,g,n,softplus,initial", [
    (1, 1, 1, 1, 1, True, False),
    (2, 1, 70, 1, 16, True, True),
    (3, 15, 64, 1, 16, True, False),
    (2, 16, 16, 1, 16, False, True),
    (2, 17, 130, 2, 16, True, True),
    (1, 33, 5, 5, 4, True, False),
    (1, 300, 96, 1, 16, True, True),       # cut into segments
    (2, 131, 24, 3, 7, False, True),       # odd states
    (1, 95, 40, 1, 17, True, False),       # two sixteens of states
    (1, 64, 12, 4, 32, True, True),
    (2, 50, 66, 2, 40, True, True),        # four
    (1, 100, 20, 1, 64, False, True),
    (40, 70, 520, 1, 16, True, True),      # walked from end to end
    (1, 1000, 65, 1, 1, True, False),
])
def test_forward_and_gradients(gpu_lib, b, t, d, g, n, softplus, initial, bf16):
    announce(f"selective scan B{b} T{t} D{d} G{g} N{n} bf16={bf16}")
    _compare(*_problem(b, t, d, g, n, bf16, softplus, initial=initial), bf16, softplus)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("skip", [False, True])
@pytest.mark.parametrize("softplus", [False, True])
def test_options(gpu_lib, softplus, skip, gate, bf16):
    announce(f"selective scan softplus={softplus} skip={skip} gate={gate} bf16={bf16}")
    _compare(*_problem(2, 45, 36, 2, 16, bf16, softplus, gate, skip, seed=1), bf16, softplus)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("b,t,d,n,lengths", [
    (4, 40, 20, 16, [40, 0, 16, 17]),
    (3, 300, 64, 16, [300, 1, 129]),
    (3, 300, 64, 16, [5, 0, 40]),          # whole segments without a token
    (2, 100, 10, 20, [-3, 1000]),          # clamped
    (40, 64, 520, 16, [(7 * i) % 65 for i in range(40)]),
])
def test_lengths(gpu_lib, b, t, d, n, lengths, bf16):
    """Absent tokens hold NaN: they reach nothing, their outputs and gradients are zero."""
    announce(f"selective scan lengths B{b} T{t} D{d} N{n} bf16={bf16}")
    x, d_out, d_state = _problem(b, t, d, 1, n, bf16, initial=True, seed=2)
    absent = np.arange(t)[None] >= np.asarray(lengths)[:, None]
    for name in ROWS:
        x[name][absent] = np.nan
    d_out[absent] = np.nan
    r, grads = _compare(x, d_out, d_state, bf16, True, lengths)
    mask = torch.tensor(absent, device="cuda")
    assert (r.output[mask] == 0).all()
    for name in ROWS:
        assert (grads[name][mask] == 0).all(), name


def test_strided_rows(gpu_lib):
    """Parts of the rows of wider projections, b and c of [B,T,N], expanded rows."""
    announce("selective scan strides")
    b, t, d, n = 2, 37, 48, 16
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(b, t, 3 * d + 1, device="cuda").to(dtype)
        small = torch.randn(b, t, 2 * n + 3, device="cuda").to(dtype)
        a = -torch.rand(d, n, device="cuda")
        for shift in (0, 1):
            x, delta, gate = (wide[..., i * d + shift:(i + 1) * d + shift] for i in range(3))
            bb, cc = small[..., shift:n + shift], small[..., n + shift:2 * n + shift]
            got = selective_scan(x, delta, a, bb, cc, gate=gate, softplus=True)
            want = selective_scan(x.contiguous(), delta.contiguous(), a,
                                  bb[:, :, None].contiguous(), cc[:, :, None].contiguous(),
                                  gate=gate.contiguous(), softplus=True)
            assert torch.equal(got.output, want.output) and torch.equal(got.state, want.state)
        one = torch.randn(1, 1, d, device="cuda").to(dtype)
        got = selective_scan(x, one.expand(b, t, d), a, bb, cc, softplus=True)
        want = selective_scan(x, one.repeat(b, t, 1), a, bb, cc, softplus=True)
        assert torch.equal(got.output, want.output)
        turned = torch.randn(b, d, t, device="cuda").to(dtype).transpose(1, 2)
        got = selective_scan(turned, delta, a, bb, cc, softplus=True)
        want = selective_scan(turned.contiguous(), delta, a, bb, cc, softplus=True)
        assert torch.equal(got.output, want.output)


def test_mixed_and_other_types(gpu_lib):
    announce("selective scan types")
    x, _, _ = _problem(2, 20, 12, 1, 16, False, seed=3)
    t = _tensors(x, False, False)
    whole = _call(t, True)
    half = {k: v.half() if k == "x" else v for k, v in t.items()}
    r = _call(half, True)
    assert r.output.dtype == torch.float16 and r.state.dtype == torch.float32
    want = _call({**t, "x": half["x"].float()}, True)
    assert torch.equal(r.output, want.output.half()) and torch.equal(r.state, want.state)
    r = _call({**t, "x": t["x"].double()}, True)
    assert r.output.dtype == torch.float64 and torch.equal(r.output.float(), whole.output)


def test_two_runs_and_streams_give_the_same_bits(gpu_lib):
    announce("selective scan repeat, stream")
    for shape in ((1, 400, 72), (48, 64, 520)):
        x, d_out, d_state = _problem(*shape, 1, 16, True, initial=True, seed=4)

        def both():
            t = _tensors(x, True, True)
            r = _call(t, True)
            return [r.output, r.state, *_grads(t, r, d_out, d_state).values()]

        want = both()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            other = both()
        stream.synchronize()
        for u, v, w in zip(want, both(), other):
            assert torch.equal(u, v) and torch.equal(u, w)


def test_a_bad_value_reaches_later_tokens_of_its_channel_only(gpu_lib):
    announce("selective scan NaN")
    x, _, _ = _problem(1, 200, 40, 1, 16, False, seed=5)
    clean = _call(_tensors(x, False, False), True)
    for value in (np.nan, np.inf):
        y = dict(x, x=x["x"].copy())
        y["x"][0, 90, 7] = value
        r = _call(_tensors(y, False, False), True)
        bad = torch.zeros(r.output.shape, dtype=torch.bool, device="cuda")
        bad[0, 90:, 7] = True
        assert not torch.isfinite(r.output[bad]).any()
        assert torch.equal(r.output[~bad], clean.output[~bad])


def test_zero_and_dropping_decays(gpu_lib):
    """A rate of zero keeps the state; minus infinity drops it wherever the step is not
    zero (absent tokens, whose step is zero, keep it)."""
    announce("selective scan rates")
    b, t, d, n = 2, 40, 8, 4
    one = torch.ones(b, t, d, device="cuda")
    bc = torch.ones(b, t, n, device="cuda")
    a = torch.zeros(d, n, device="cuda")
    lens = torch.tensor([40, 7], device="cuda")
    r = selective_scan(one, one, a, bc, bc, lengths=lens)
    count = torch.arange(1, t + 1, device="cuda").float()
    assert torch.equal(r.output[0], (4 * count)[:, None].expand(t, d))
    assert (r.state[0] == 40).all() and (r.state[1] == 7).all()
    a = torch.full((d, n), -float("inf"), device="cuda")
    r = selective_scan(one, one, a, bc, bc, lengths=lens)
    assert (r.output[0] == 4).all() and (r.state == 1).all()


def test_large_steps(gpu_lib):
    """Softplus far from zero on both sides, against the definition."""
    announce("selective scan large steps")
    x, d_out, d_state = _problem(1, 48, 16, 1, 16, False, initial=True, seed=6)
    x["delta"] = _cast(np.linspace(-60.0, 60.0, 48 * 16).reshape(1, 48, 16), False)
    _compare(x, d_out, d_state, False, True)


def test_gradients_against_differences(gpu_lib):
    """Central differences with a step of 2^-6 along a random direction: curvature about
    2^-12 of the terms, rounding 2^-24 2^6 of the loss's terms."""
    announce("selective scan differences")
    x, d_out, d_state = _problem(2, 20, 8, 2, 4, False, initial=True, seed=7)
    t = _tensors(x, False, True)
    grads = _grads(t, _call(t, True), d_out, d_state)
    rng = np.random.default_rng(8)
    step = 2.0 ** -6
    for name, g in grads.items():
        direction = rng.normal(size=x[name].shape)
        values = []
        for s in (1, -1):
            r = _call(_tensors({**x, name: x[name] + s * step * direction}, False, False), True)
            values.append((host(r.output) * d_out).sum() + (host(r.state) * d_state).sum())
        got, scale = (host(g) * direction).sum(), np.abs(host(g) * direction).sum()
        assert abs(got - (values[0] - values[1]) / (2 * step)) <= 2e-3 * scale, name


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("b,d,g,n", [(1, 1, 1, 1), (4, 96, 1, 16), (3, 20, 4, 7), (2, 9, 3, 40),
                                     (300, 64, 1, 16), (5, 33, 1, 8), (2, 6, 1, 64)])
def test_step(gpu_lib, b, d, g, n, bf16):
    announce(f"selective scan step B{b} D{d} G{g} N{n} bf16={bf16}")
    x, _, _ = _problem(b, 1, d, g, n, bf16, initial=True, seed=9)
    t = _tensors(x, bf16, False)
    active = [i % 3 != 1 for i in range(b)]
    lengths = [int(v) for v in active]
    out, state = oracle.scan(**x, softplus=True, lengths=lengths)
    args = (t["x"][:, 0], t["delta"][:, 0], t["a"], t["b"][:, 0], t["c"][:, 0])
    more = dict(skip=t["skip"], gate=t["gate"][:, 0], delta_bias=t["bias"], softplus=True,
                active=torch.tensor(active, device="cuda"))
    before = t["initial"].clone()
    r = selective_scan_step(t["initial"], *args, **more)
    assert torch.equal(t["initial"], before)
    _check("output", r.output, out[:, 0], BF16 if bf16 else F32)
    _check("state", r.state, state, F32)
    idle = ~more["active"]
    assert (r.output[idle] == 0).all() and torch.equal(r.state[idle], before[idle])
    held = before.clone()
    version = held._version
    s = selective_scan_step_(held, *args, **more)
    assert s.state is held and held._version > version
    assert torch.equal(held, r.state) and torch.equal(s.output, r.output)


def test_steps_are_the_sequence(gpu_lib):
    announce("selective scan steps")
    x, _, _ = _problem(3, 40, 24, 2, 16, False, seed=10)
    t = _tensors(x, False, False)
    whole = _call(t, True)
    state = torch.zeros(3, 24, 16, device="cuda")
    for i in range(40):
        r = selective_scan_step_(state, t["x"][:, i], t["delta"][:, i], t["a"], t["b"][:, i],
                                 t["c"][:, i], skip=t["skip"], gate=t["gate"][:, i],
                                 delta_bias=t["bias"], softplus=True)
        _check("output", r.output, host(whole.output[:, i]), F32)
    _check("state", state, host(whole.state), F32)


def test_step_with_a_gradient_is_the_scan_of_one_token(gpu_lib):
    announce("selective scan step gradient")
    x, d_out, d_state = _problem(4, 1, 10, 1, 16, False, initial=True, seed=11)
    active = [True, False, True, True]
    t = _tensors(x, False, True)
    r = selective_scan_step(t["initial"], t["x"][:, 0], t["delta"][:, 0], t["a"], t["b"][:, 0],
                            t["c"][:, 0], skip=t["skip"], gate=t["gate"][:, 0],
                            delta_bias=t["bias"], softplus=True,
                            active=torch.tensor(active, device="cuda"))
    grads = _grads(t, r, d_out[:, 0], d_state)
    want = oracle.scan_backward(**x, d_output=d_out, d_state=d_state, softplus=True,
                                lengths=[int(v) for v in active])
    for name, g in grads.items():
        _check("d_" + name, g, want[name], SUMS)
    with pytest.raises(ValueError, match="no gradient"):
        selective_scan_step_(torch.zeros(4, 10, 16, device="cuda"), t["x"][:, 0],
                             t["delta"][:, 0], t["a"], t["b"][:, 0], t["c"][:, 0])


def test_some_gradients_only(gpu_lib):
    announce("selective scan some gradients")
    x, d_out, d_state = _problem(2, 50, 20, 1, 16, False, initial=True, seed=12)
    t = _tensors(x, False, True)
    every = _grads(t, _call(t, True), d_out, d_state)
    for names in (("x",), ("a", "gate"), ("initial",), ("bias",), ("b",)):
        t = {k: v.detach().requires_grad_(k in names) for k, v in t.items()}
        r = _call(t, True)
        got = torch.autograd.grad([r.output, r.state], [t[n] for n in names],
                                  [torch.tensor(d_out, device="cuda").float(),
                                   torch.tensor(d_state, device="cuda").float()])
        for n, g in zip(names, got):
            assert torch.equal(g, every[n]), n
    # A cotangent of the state alone.
    t = _tensors(x, False, True)
    got = torch.autograd.grad(_call(t, True).state, list(t.values()),
                              torch.tensor(d_state, device="cuda").float(), allow_unused=True)
    want = oracle.scan_backward(**x, d_output=np.zeros_like(d_out), d_state=d_state, softplus=True)
    for name, g in zip(t, got):
        if name in ("c", "gate", "skip"):
            assert (g == 0).all()
        else:
            _check("d_" + name, g, want[name], SUMS)


def test_graph_replays(gpu_lib):
    announce("selective scan graph")
    for shape in ((1, 300, 40), (40, 33, 520)):
        x, d_out, _ = _problem(*shape, 1, 16, True, seed=13)
        t = _tensors(x, True, True)
        cot = torch.tensor(d_out, device="cuda").to(torch.bfloat16)

        def both():
            r = _call(t, True)
            return [r.output, r.state, *torch.autograd.grad(r.output, list(t.values()), cot)]

        want = [u.detach().clone() for u in both()]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both()
        for _ in range(3):
            for u in got:
                u.detach().fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for u, v in zip(got, want):
                assert torch.equal(u, v)
            assert torch.equal(_call(t, True).output, want[0])
        del graph, got


def test_no_tokens(gpu_lib):
    announce("selective scan without tokens")
    a = -torch.ones(6, 4, device="cuda", requires_grad=True)
    for b, t in ((2, 0), (0, 5)):
        x = torch.randn(b, t, 6, device="cuda", requires_grad=True)
        bc = torch.randn(b, t, 1, 4, device="cuda")
        s0 = torch.randn(b, 6, 4, device="cuda", requires_grad=True)
        r = selective_scan(x, x, a, bc, bc, initial=s0)
        assert r.output.shape == (b, t, 6) and torch.equal(r.state, s0)
        gx, ga, gs = torch.autograd.grad([r.output, r.state], [x, a, s0],
                                         [torch.ones_like(r.output), torch.ones_like(r.state)])
        assert gx.shape == x.shape and (ga == 0).all() and (gs == 1).all()
    r = selective_scan_step(torch.zeros(0, 6, 4, device="cuda"), x[:, 0].detach(),
                            x[:, 0].detach(), a.detach(), bc[:, 0], bc[:, 0])
    assert r.output.shape == (0, 6)
