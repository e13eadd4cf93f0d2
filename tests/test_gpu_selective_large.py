"""Arrays of more than 2^31 elements: what lies behind them is what a small call gives.

The scan's segments differ between the two calls, so that their float32 results differ by
roundings as its tests against the oracle allow; the others have the same bits.
"""

import pytest
import torch

from mamba4_amd import (
    causal_conv,
    causal_conv_step_,
    rms_norm,
    rms_norm_e4m3,
    selective_scan,
    selective_scan_step_,
)
from tests.gpu_helpers import announce

pytestmark = pytest.mark.gpu

T, D = 1_400_016, 1536  # 2.15e9 elements
LAST = 300
BF16 = torch.bfloat16


def _normal(*shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", dtype=dtype)


def _near(a, b, limit):
    a, b = a.double(), b.double()
    error = ((a - b).abs().max() / b.abs().max()).item()
    assert error <= limit, error


@pytest.fixture(scope="module")
def rows():
    torch.manual_seed(0)
    return _normal(1, T, D, dtype=BF16)


@pytest.mark.parametrize("dense", [False, True])
def test_scan(gpu_lib, rows, dense):
    # (Steps of one row for all tokens are read an element at a time, and so all rows.)
    announce(f"selective scan of 2^31 elements, dense steps {dense}")
    a = -torch.rand(D, 4, device="cuda")
    b, c = _normal(1, T, 4, dtype=BF16), _normal(1, T, 4, dtype=BF16)
    delta = torch.full((1, 1, D), 0.05, device="cuda", dtype=BF16).expand(1, T, D)
    if dense:
        delta = delta.contiguous()
    inputs = [rows.detach().requires_grad_(), b.requires_grad_(), c.requires_grad_()]
    d_out = torch.zeros_like(rows)
    d_out[:, -LAST:] = _normal(1, LAST, D, dtype=BF16)
    r = selective_scan(inputs[0], delta, a, *inputs[1:], gate=rows)
    grads = torch.autograd.grad(r.output, inputs, d_out)
    cut = T - LAST
    with torch.no_grad():
        before = selective_scan(rows[:, :cut], delta[:, :cut], a, b[:, :cut], c[:, :cut]).state
    some = [t.detach()[:, cut:].requires_grad_() for t in inputs]
    s = selective_scan(some[0], delta[:, cut:], a, *some[1:], gate=rows[:, cut:], initial=before)
    _near(s.output, r.output[:, cut:], 2.0 ** -8 + 2e-5)
    _near(s.state, r.state, 2e-5)
    for g, h in zip(torch.autograd.grad(s.output, some, d_out[:, cut:]), grads):
        _near(g, h[:, cut:], 2.0 ** -8 + 2e-5)
    del r, grads, d_out


@pytest.mark.parametrize("stride,segments", [(1 << 22, 10), (1 << 22, 1), (1 << 24, 10)])
def test_rows_far_apart(gpu_lib, monkeypatch, stride, segments):
    """Of a segment below 2^31 bytes, of one that has to be cut for that, and of none: the
    results of rows beside each other."""
    announce(f"selective scan of rows {stride} elements apart, {segments} segments")
    monkeypatch.setenv("M4SL_SEGMENTS", str(segments))
    time, d, n = 160 if stride == 1 << 22 else 80, 64, 16
    torch.manual_seed(1)
    wide = torch.zeros(time, stride, device="cuda", dtype=BF16)
    wide[:, :3 * d + 2 * n] = _normal(time, 3 * d + 2 * n, dtype=BF16)
    a = -torch.rand(d, n, device="cuda")
    d_out = _normal(1, time, d, dtype=BF16)

    def run(rows):
        x, delta, gate, b, c = (
            t.detach().requires_grad_() for t in rows[None].split([d, d, d, n, n], -1))
        r = selective_scan(x, delta, a, b, c, gate=gate, softplus=True)
        return [r.output, r.state,
                *torch.autograd.grad(r.output, [x, delta, gate, b, c], d_out)]

    near = run(wide[:, :3 * d + 2 * n].contiguous())
    far = run(wide[:, :3 * d + 2 * n])
    for x, y in zip(near, far):
        if segments == 10:
            assert torch.equal(x, y)
        else:
            _near(x, y, 2.0 ** -8 + 2e-5)


def test_conv_and_norm(gpu_lib, rows):
    announce("causal conv and rms norm of 2^31 elements")
    w = _normal(D, 4)
    cut = T - LAST
    r = causal_conv(rows, w, activation="silu")
    s = causal_conv(rows[:, cut:], w, activation="silu", initial=rows[:, cut - 3:cut])
    assert torch.equal(r.output[:, cut:], s.output) and torch.equal(r.state, s.state)
    del r
    x = rows.detach().requires_grad_()
    out = causal_conv(x, w).output
    d = torch.zeros_like(rows)
    d[:, -1] = 1.0
    g, = torch.autograd.grad(out, x, d)
    del out
    for j in range(4):
        assert torch.equal(g[0, T - 4 + j], w[:, j].to(BF16))
    assert (g[0, T - 5] == 0).all()
    del g, d
    weight = _normal(D)
    y, total = rms_norm(rows, weight, residual=rows)
    z, part = rms_norm(rows[:, cut:], weight, residual=rows[:, cut:])
    assert torch.equal(y[:, cut:], z) and torch.equal(total[:, cut:], part)
    del y, total
    q = rms_norm_e4m3(rows, weight, block=128)
    p = rms_norm_e4m3(rows[:, cut:], weight, block=128)
    assert torch.equal(q.output[:, cut:].view(torch.uint8), p.output.view(torch.uint8))
    assert torch.equal(q.scale[:, cut:], p.scale)


def test_steps(gpu_lib):
    announce("selective steps of 2^31 elements")
    batch, n = 87_500, 16  # 2.15e9 states
    state = torch.zeros(batch, D, n, device="cuda")
    state[-1] = _normal(D, n)
    x, bc = _normal(batch, D, dtype=BF16), _normal(batch, n, dtype=BF16)
    a = -torch.rand(D, n, device="cuda")
    small = state[-2:].clone()
    r = selective_scan_step_(state, x, x, a, bc, bc, softplus=True)
    s = selective_scan_step_(small, x[-2:], x[-2:], a, bc[-2:], bc[-2:], softplus=True)
    assert torch.equal(state[-2:], small) and torch.equal(r.output[-2:], s.output)
    del state, r
    batch = 470_000  # 2.17e9 elements
    rows = torch.zeros(batch, 3, D, device="cuda", dtype=BF16)
    rows[-1] = 1.0
    x = _normal(batch, D, dtype=BF16)
    w = _normal(D, 4)
    small = rows[-2:].clone()
    r = causal_conv_step_(rows, x, w)
    s = causal_conv_step_(small, x[-2:], w)
    assert torch.equal(rows[-2:], small) and torch.equal(r.output[-2:], s.output)
