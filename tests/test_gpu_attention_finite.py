"""Infinities and NaN in rows that are present: what the recurrence does not carry
them to keeps its bits.  A token's value reaches its column of the outputs from that
token on, its key all columns, its query its own output; in the gradients time runs
the other way."""

import pytest
import torch

from mamba4_amd import linear_attention
from tests.gpu_helpers import announce

pytestmark = pytest.mark.gpu

TIME, HEADS = 200, 2
PLACES = (0, 5, 17, 63, 64, 100, 130, 199)


def _inputs(dtype, n, p, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    x = dict(q=normal(2, TIME, HEADS, n).to(dtype), k=normal(2, TIME, HEADS, n).to(dtype),
             v=normal(2, TIME, HEADS, p).to(dtype), d=normal(2, TIME, HEADS, p).to(dtype))
    x["g"] = -0.2 * torch.rand(2, TIME, HEADS, device="cuda", generator=g)
    return x


def _forward(x):
    with torch.no_grad():
        r = linear_attention(x["q"], x["k"], x["v"], x["g"], scale=0.5)
    return r.output, r.state


def _gradients(x, decays):
    """dq, dk, dv from the cotangent alone (the outputs are not looked at)."""
    q, k, v = (x[n].clone().requires_grad_() for n in "qkv")
    r = linear_attention(q, k, v, x["g"].clone().requires_grad_(decays), scale=0.5)
    return torch.autograd.grad(r.output, (q, k, v), x["d"])


def _spoiled(x, name, time, column, bad):
    y = {n: t.clone() for n, t in x.items()}
    y[name][1, time, 1, column] = bad
    return y


CASES = [(torch.bfloat16, 64, 64), (torch.bfloat16, 128, 128), (torch.float32, 64, 64),
         (torch.float32, 100, 36), (torch.bfloat16, 33, 7)]


@pytest.mark.parametrize("dtype,n,p", CASES)
@pytest.mark.parametrize("bad", [torch.nan, torch.inf, -torch.inf])
@pytest.mark.parametrize("route", ["walk", "split"])
def test_outputs(gpu_lib, monkeypatch, dtype, n, p, bad, route):
    announce(f"not finite {dtype} N{n} P{p} {bad} {route}")
    monkeypatch.setenv("M4RT_ATTENTION", route)
    x = _inputs(dtype, n, p)
    out, state = _forward(x)
    for i, time in enumerate(PLACES):
        column = (7 * i) % min(n, p)
        # A value: its column, from its token on.
        got, after = _forward(_spoiled(x, "v", time, column, bad))
        reached = torch.zeros_like(out, dtype=torch.bool)
        reached[1, time:, 1, column] = True
        assert torch.equal(got[~reached], out[~reached]), time
        assert not torch.isfinite(got[reached]).any(), time
        in_state = torch.zeros_like(state, dtype=torch.bool)
        in_state[1, 1, :, column] = True
        assert torch.equal(after[~in_state], state[~in_state]), time
        assert not torch.isfinite(after[in_state]).any(), time
        # A key: every column, from its token on; its row of the state.
        got, after = _forward(_spoiled(x, "k", time, column, bad))
        reached[1, time:, 1] = True
        assert torch.equal(got[~reached], out[~reached]), time
        assert not torch.isfinite(got[reached]).any(), time
        in_state = torch.zeros_like(state, dtype=torch.bool)
        in_state[1, 1, column] = True
        assert torch.equal(after[~in_state], state[~in_state]), time
        assert not torch.isfinite(after[in_state]).any(), time
        # A query: its own output.
        got, after = _forward(_spoiled(x, "q", time, column, bad))
        reached[:] = False
        reached[1, time, 1] = True
        assert torch.equal(got[~reached], out[~reached]), time
        assert not torch.isfinite(got[reached]).any(), time
        assert torch.equal(after, state), time


@pytest.mark.parametrize("dtype,n,p", CASES)
@pytest.mark.parametrize("decays", [False, True])
@pytest.mark.parametrize("route", ["walk", "split"])
def test_gradients(gpu_lib, monkeypatch, dtype, n, p, decays, route):
    announce(f"not finite, gradients {dtype} N{n} P{p} decays={decays} {route}")
    monkeypatch.setenv("M4RT_ATTENTION", route)
    x = _inputs(dtype, n, p)
    clean = _gradients(x, decays)
    # Which tokens' dq, dk and dv something at `time` reaches: a range, or that token.
    own, later, earlier = "own", "later", "earlier"
    reach = dict(d=(own, earlier, earlier), q=(None, earlier, earlier), k=(later, None, own),
                 v=(later, own, None))
    for i, time in enumerate(PLACES):
        column = (7 * i) % min(n, p)
        for name, kinds in reach.items():
            got = _gradients(_spoiled(x, name, time, column, torch.nan), decays)
            for a, b, kind in zip(got, clean, kinds):
                reached = torch.zeros(a.shape[:3], dtype=torch.bool, device="cuda")
                at = {own: slice(time, time + 1), later: slice(time, None),
                      earlier: slice(0, time + 1), None: slice(0, 0)}[kind]
                reached[1, at, 1] = True
                assert torch.equal(a[~reached], b[~reached]), (name, time, kind)
                assert not torch.isfinite(a[reached]).all() or kind is None, (name, time, kind)
