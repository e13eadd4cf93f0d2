"""The short causal convolution on the GPU against the float64 oracle.

Tolerances, as max |difference| / max |expected|.  Float32: sums of up to eight products
and one activation, a few roundings of 2^-24: 2e-6, and of the activation's
exponential 2^-24 of its argument (at most 16 here): 1e-5 in all.  Sums over tokens
(weight, bias) 2e-5.  Bfloat16 results are rounded once: 2^-8 + 1e-5.  The state holds
inputs: equal.
"""

import numpy as np
import pytest
import torch

from mamba4_amd import causal_conv, causal_conv_step, causal_conv_step_
from oracle import selective as oracle
from tests.gpu_helpers import announce, host, normwise

pytestmark = pytest.mark.gpu

F32 = 1e-5
SUMS = 2e-5
BF16 = 2.0 ** -8 + F32


def _cast(x, bf16):
    t = torch.tensor(x, dtype=torch.float32)
    return (t.to(torch.bfloat16) if bf16 else t).double().numpy()


def _problem(b, t, d, w, bf16, bias=True, initial=False, seed=0):
    rng = np.random.default_rng(seed)
    x = dict(x=_cast(rng.normal(size=(b, t, d)), bf16),
             weight=_cast(rng.normal(size=(d, w)) / np.sqrt(w), False))
    if bias:
        x["bias"] = _cast(rng.normal(size=d), False)
    if initial:
        x["initial"] = _cast(rng.normal(size=(b, w - 1, d)), bf16)
    d_out = _cast(rng.normal(size=(b, t, d)), bf16)
    d_state = _cast(rng.normal(size=(b, w - 1, d)), bf16) if initial else None
    return x, d_out, d_state


def _tensors(x, bf16, grad):
    return {k: torch.tensor(v, device="cuda", dtype=torch.bfloat16
                            if bf16 and k in ("x", "initial") else torch.float32)
            .requires_grad_(grad) for k, v in x.items()}


def _call(t, activation, lengths=None):
    lens = None if lengths is None else torch.tensor(lengths, device="cuda")
    return causal_conv(t["x"], t["weight"], t.get("bias"), activation=activation,
                       initial=t.get("initial"), lengths=lens)


def _check(label, got, want, limit):
    if want.size == 0:
        assert tuple(got.shape) == want.shape
        return
    error = normwise(host(got.float()), want)
    assert error <= limit, f"{label}: {error:.3g} > {limit:.3g}"


def _grads(t, r, d_out, d_state):
    outs, cots = [r.output], [torch.tensor(d_out, device="cuda").to(r.output.dtype)]
    if d_state is not None:
        outs.append(r.state)
        cots.append(torch.tensor(d_state, device="cuda").to(r.state.dtype))
    return dict(zip(t, torch.autograd.grad(outs, list(t.values()), cots)))


def _compare(x, d_out, d_state, bf16, activation, lengths=None):
    t = _tensors(x, bf16, True)
    r = _call(t, activation, lengths)
    grads = _grads(t, r, d_out, d_state)
    torch.cuda.synchronize()
    out, state = oracle.conv(**x, activation=activation, lengths=lengths)
    want = oracle.conv_backward(**x, d_output=d_out, d_state=d_state, activation=activation,
                                lengths=lengths)
    rows = BF16 if bf16 else F32
    assert r.output.dtype == t["x"].dtype == r.state.dtype
    _check("output", r.output, out, rows)
    assert (host(r.state.float()) == state).all()
    for name, g in grads.items():
        assert g.shape == t[name].shape and g.dtype == t[name].dtype
        _check("d_" + name, g, want[name], rows if name in ("x", "initial") else SUMS)
    with torch.no_grad():
        plain = _call(t, activation, lengths)
    assert torch.equal(plain.output, r.output) and torch.equal(plain.state, r.state)
    return r, grads


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("activation", ["none", "silu"])
@pytest.mark.parametrize("b,t,d,w,initial", [
    (1, 1, 1, 1, False), (2, 1, 8, 4, True), (2, 2, 16, 4, False), (3, 7, 24, 3, True),
    (2, 8, 64, 2, True), (1, 9, 5, 4, True), (2, 100, 96, 4, True), (1, 300, 33, 8, True),
    (4, 65, 520, 4, False), (2, 31, 40, 5, True), (2, 40, 8, 6, True), (3, 17, 16, 7, False),
    (2, 29, 48, 1, True), (70, 64, 768, 4, True), (2, 50, 1000, 3, True),
])
def test_forward_and_gradients(gpu_lib, b, t, d, w, initial, activation, bf16):
    announce(f"causal conv B{b} T{t} D{d} W{w} {activation} bf16={bf16}")
    _compare(*_problem(b, t, d, w, bf16, initial=initial), bf16, activation)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("b,t,d,w,lengths", [
    (4, 40, 16, 4, [40, 0, 1, 2]), (3, 20, 5, 8, [3, 20, 7]), (2, 30, 64, 2, [-5, 100]),
    (2, 9, 8, 1, [4, 0]),
])
def test_lengths(gpu_lib, b, t, d, w, lengths, bf16):
    """Absent tokens hold NaN: they reach nothing, their outputs and gradients are zero;
    the state of a short row begins with rows of the initial one."""
    announce(f"causal conv lengths B{b} T{t} D{d} W{w} bf16={bf16}")
    x, d_out, d_state = _problem(b, t, d, w, bf16, initial=True, seed=1)
    absent = np.arange(t)[None] >= np.asarray(lengths)[:, None]
    x["x"][absent] = np.nan
    d_out[absent] = np.nan
    r, grads = _compare(x, d_out, d_state, bf16, "silu", lengths)
    mask = torch.tensor(absent, device="cuda")
    assert (r.output[mask] == 0).all()
    # (The state's cotangent reaches tokens that are present only.)
    assert (grads["x"][mask] == 0).all()


def test_without_bias_and_initial(gpu_lib):
    announce("causal conv plain")
    _compare(*_problem(2, 21, 24, 4, False, bias=False, seed=2), False, "none")


def test_strided_and_unaligned_rows(gpu_lib):
    announce("causal conv strides")
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(3, 50, 100, device="cuda").to(dtype)
        weight = torch.randn(48, 4, device="cuda")
        for x in (wide[..., 4:52], wide[..., 8:56], wide[..., 1:49], wide[:, ::2, :48],
                  wide.transpose(1, 2)[:, :, :48], wide[:1, :1, :48].expand(3, 50, 48)):
            got = causal_conv(x, weight, activation="silu")
            want = causal_conv(x.contiguous(), weight, activation="silu")
            assert torch.equal(got.output, want.output) and torch.equal(got.state, want.state)
            assert torch.equal(want.state, x[:, -3:])


def test_other_types(gpu_lib):
    announce("causal conv types")
    x = torch.randn(2, 10, 8, device="cuda")
    w = torch.randn(8, 4, device="cuda")
    r = causal_conv(x.half(), w.to(torch.bfloat16))
    want = causal_conv(x.half().float(), w.to(torch.bfloat16).float())
    assert r.output.dtype == r.state.dtype == torch.float16
    assert torch.equal(r.output, want.output.half()) and torch.equal(r.state, x.half()[:, -3:])
    r = causal_conv(x.double(), w)
    assert r.output.dtype == torch.float64


def test_two_runs_and_streams_give_the_same_bits(gpu_lib):
    announce("causal conv repeat, stream")
    x, d_out, d_state = _problem(16, 200, 264, 4, True, initial=True, seed=3)

    def both():
        t = _tensors(x, True, True)
        r = _call(t, "silu")
        return [r.output, r.state, *_grads(t, r, d_out, d_state).values()]

    want = both()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = both()
    stream.synchronize()
    for u, v, w in zip(want, both(), other):
        assert torch.equal(u, v) and torch.equal(u, w)


def test_a_rows_bits_do_not_depend_on_the_batch(gpu_lib):
    announce("causal conv batch")
    x, _, _ = _problem(300, 90, 256, 4, False, seed=4)
    t = _tensors(x, False, False)
    whole = _call(t, "silu").output
    for n in (1, 7):
        assert torch.equal(_call({**t, "x": t["x"][:n]}, "silu").output, whole[:n])


def test_a_bad_value_reaches_the_next_taps_only(gpu_lib):
    announce("causal conv NaN")
    x, _, _ = _problem(1, 60, 16, 4, False, seed=5)
    clean = _call(_tensors(x, False, False), "silu")
    x["x"][0, 30, 5] = np.nan
    r = _call(_tensors(x, False, False), "silu")
    bad = torch.zeros(r.output.shape, dtype=torch.bool, device="cuda")
    bad[0, 30:34, 5] = True
    assert torch.isnan(r.output[bad]).all() and torch.equal(r.output[~bad], clean.output[~bad])


def test_gradients_against_differences(gpu_lib):
    """Central differences with a step of 2^-7 along a random direction: curvature about
    2^-14 of the terms, rounding 2^-24 2^7 of the loss's terms."""
    announce("causal conv differences")
    x, d_out, d_state = _problem(2, 20, 8, 4, False, initial=True, seed=6)
    t = _tensors(x, False, True)
    grads = _grads(t, _call(t, "silu"), d_out, d_state)
    rng = np.random.default_rng(7)
    step = 2.0 ** -7
    for name, g in grads.items():
        direction = rng.normal(size=x[name].shape)
        values = []
        for s in (1, -1):
            r = _call(_tensors({**x, name: x[name] + s * step * direction}, False, False), "silu")
            values.append((host(r.output) * d_out).sum() + (host(r.state) * d_state).sum())
        got, scale = (host(g) * direction).sum(), np.abs(host(g) * direction).sum()
        assert abs(got - (values[0] - values[1]) / (2 * step)) <= 2e-3 * scale, name


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("b,d,w", [(1, 1, 1), (5, 24, 4), (3, 33, 8), (300, 64, 2), (4, 16, 1)])
def test_step(gpu_lib, b, d, w, bf16):
    announce(f"causal conv step B{b} D{d} W{w} bf16={bf16}")
    x, _, _ = _problem(b, 1, d, w, bf16, initial=True, seed=8)
    t = _tensors(x, bf16, False)
    active = [i % 3 != 1 for i in range(b)]
    out, state = oracle.conv(**x, activation="silu", lengths=[int(v) for v in active])
    more = dict(activation="silu", active=torch.tensor(active, device="cuda"))
    before = t["initial"].clone()
    token = t["x"][:, 0].clone()
    token[~more["active"]] = float("nan")
    r = causal_conv_step(t["initial"], token, t["weight"], t["bias"], **more)
    assert torch.equal(t["initial"], before)
    _check("output", r.output, out[:, 0], BF16 if bf16 else F32)
    assert (host(r.state.float()) == state).all()
    held = before.clone()
    version = held._version
    s = causal_conv_step_(held, token, t["weight"], t["bias"], **more)
    assert s.state is held and (held._version > version)
    assert torch.equal(held, r.state) and torch.equal(s.output, r.output)


def test_steps_are_the_sequence_and_gradients_of_a_step(gpu_lib):
    announce("causal conv steps")
    x, d_out, d_state = _problem(3, 30, 24, 4, True, seed=9)
    t = _tensors(x, True, False)
    whole = _call(t, "silu")
    state = torch.zeros(3, 3, 24, dtype=torch.bfloat16, device="cuda")
    for i in range(30):
        r = causal_conv_step_(state, t["x"][:, i], t["weight"], t["bias"], activation="silu")
        assert torch.equal(r.output, whole.output[:, i])
    assert torch.equal(state, whole.state)
    x, d_out, d_state = _problem(4, 1, 10, 4, False, initial=True, seed=10)
    t = _tensors(x, False, True)
    r = causal_conv_step(t["initial"], t["x"][:, 0], t["weight"], t["bias"], activation="silu",
                         active=torch.tensor([True, False, True, True], device="cuda"))
    grads = _grads(t, r, d_out[:, 0], d_state)
    want = oracle.conv_backward(**x, d_output=d_out, d_state=d_state, activation="silu",
                                lengths=[1, 0, 1, 1])
    for name, g in grads.items():
        _check("d_" + name, g, want[name], SUMS)


def test_some_gradients_only(gpu_lib):
    announce("causal conv some gradients")
    x, d_out, d_state = _problem(2, 30, 20, 4, False, initial=True, seed=11)
    t = _tensors(x, False, True)
    every = _grads(t, _call(t, "silu"), d_out, d_state)
    for names in (("x",), ("weight",), ("bias", "initial")):
        t = {k: v.detach().requires_grad_(k in names) for k, v in t.items()}
        r = _call(t, "silu")
        outs, cots = [r.output], [torch.tensor(d_out, device="cuda").float()]
        if r.state.requires_grad:
            outs.append(r.state)
            cots.append(torch.tensor(d_state, device="cuda").float())
        for n, g in zip(names, torch.autograd.grad(outs, [t[n] for n in names], cots)):
            assert torch.equal(g, every[n]), n


def test_graph_replays(gpu_lib):
    announce("causal conv graph")
    x, d_out, _ = _problem(4, 70, 64, 4, True, seed=12)
    t = _tensors(x, True, True)
    cot = torch.tensor(d_out, device="cuda").to(torch.bfloat16)

    def both():
        r = _call(t, "silu")
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
        assert torch.equal(_call(t, "silu").output, want[0])
    del graph, got


def test_no_tokens(gpu_lib):
    announce("causal conv without tokens")
    w = torch.randn(6, 3, device="cuda", requires_grad=True)
    for b, t in ((2, 0), (0, 5)):
        x = torch.randn(b, t, 6, device="cuda", requires_grad=True)
        s0 = torch.randn(b, 2, 6, device="cuda", requires_grad=True)
        r = causal_conv(x, w, initial=s0)
        assert r.output.shape == (b, t, 6) and torch.equal(r.state, s0)
        gx, gw, gs = torch.autograd.grad([r.output, r.state], [x, w, s0],
                                         [torch.ones_like(r.output), torch.ones_like(r.state)])
        assert gx.shape == x.shape and (gw == 0).all() and (gs == 1).all()
        assert (causal_conv(x, w).state == 0).all()
    assert causal_conv_step(torch.zeros(0, 2, 6, device="cuda"), x.detach()[:, 0],
                            w.detach()).output.shape == (0, 6)
