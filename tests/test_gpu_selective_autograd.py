"""How the selective layer's operators stand in torch's automatic differentiation: what
has no derivative says so, what has one keeps its graph, and saved tensors that change are
noticed."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mamba4_amd import (
    causal_conv,
    causal_conv_step,
    causal_conv_step_,
    rms_norm,
    rms_norm_e4m3,
    selective_scan,
    selective_scan_step,
    selective_scan_step_,
)
from tests.gpu_helpers import announce

pytestmark = pytest.mark.gpu


def _normal(*shape):
    return torch.randn(*shape, device="cuda")


def _scan_arguments():
    return dict(x=_normal(2, 5, 8), delta=_normal(2, 5, 8), a=-torch.rand(8, 4, device="cuda"),
                b=_normal(2, 5, 4), c=_normal(2, 5, 4), skip=_normal(8), gate=_normal(2, 5, 8),
                delta_bias=_normal(8), initial=_normal(2, 8, 4))


def _calls():
    """Each operator as a function of one of its inputs, with that input."""
    full = _scan_arguments()
    calls = {}
    for name in full:
        calls["scan " + name] = (
            lambda t, name=name: selective_scan(**{**full, name: t}, softplus=True), full[name])
    one = {n: t[:, 0] if n in ("x", "delta", "b", "c", "gate") else t
           for n, t in full.items() if n != "initial"}
    calls["step state"] = (lambda t: selective_scan_step(t, **one), full["initial"])
    calls["step b"] = (lambda t: selective_scan_step(full["initial"], **{**one, "b": t}), one["b"])
    x, w, bias, rows = _normal(2, 5, 8), _normal(8, 4), _normal(8), _normal(2, 3, 8)
    calls["conv x"] = (lambda t: causal_conv(t, w, bias, initial=rows), x)
    calls["conv weight"] = (lambda t: causal_conv(x, t, bias), w)
    calls["conv bias"] = (lambda t: causal_conv(x, w, t), bias)
    calls["conv initial"] = (lambda t: causal_conv(x, w, initial=t), rows)
    calls["conv step state"] = (lambda t: causal_conv_step(t, x[:, 0], w, bias), rows)
    h, r, s = _normal(6, 8), _normal(6, 8), _normal(8)
    calls["norm x"] = (lambda t: rms_norm(t, s, residual=r), h)
    calls["norm residual"] = (lambda t: rms_norm(h, s, residual=t), r)
    calls["norm weight"] = (lambda t: rms_norm(h, t), s)
    return calls


NAMES = [*("scan " + n for n in ("x", "delta", "a", "b", "c", "skip", "gate", "delta_bias",
                                 "initial")),
         "step state", "step b", "conv x", "conv weight", "conv bias", "conv initial",
         "conv step state", "norm x", "norm residual", "norm weight"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(gpu_lib, name, grad):
    """A tangent that the call cannot carry on is no zero (no_grad does not stop forward
    mode)."""
    announce(f"forward mode {name} grad={grad}")
    call, x = _calls()[name]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="jvp"):
            call(dual)
        call(x)  # without a tangent nothing is refused


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_are_refused(gpu_lib, name):
    announce(f"second derivative {name}")
    call, x = _calls()[name]
    x.requires_grad_()
    out = sum((t * t).sum() for t in call(x) if t.requires_grad)
    g, = torch.autograd.grad(out, x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_calls_in_place_and_in_8_bits_have_no_gradient(gpu_lib):
    announce("selective in place")
    x = _normal(2, 8).requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        selective_scan_step_(torch.zeros(2, 8, 4, device="cuda"), x, x, -_normal(8, 4).abs(),
                             _normal(2, 4), _normal(2, 4))
    with pytest.raises(ValueError, match="no gradient"):
        causal_conv_step_(torch.zeros(2, 3, 8, device="cuda"), x, _normal(8, 4))
    with pytest.raises(ValueError, match="no gradient"):
        rms_norm_e4m3(x)
    for bad in (torch.zeros(2, 8, 4, device="cuda").half(),
                torch.zeros(2, 4, 8, device="cuda").transpose(1, 2)):
        with pytest.raises(ValueError, match="contiguous float32"):
            selective_scan_step_(bad, x.detach(), x.detach(), -_normal(8, 4).abs(), _normal(2, 4),
                                 _normal(2, 4))
    for bad in (torch.zeros(2, 3, 8, device="cuda").half(),
                torch.zeros(2, 8, 3, device="cuda").transpose(1, 2)):
        with pytest.raises(ValueError, match="contiguous state"):
            causal_conv_step_(bad, x.detach(), _normal(8, 4))


def test_states_may_be_stepped_before_the_backward(gpu_lib):
    """The final states are no saved tensors; a state that is saved (as an initial one) and
    then stepped in place is noticed."""
    announce("selective states before backward")
    full = _scan_arguments()
    full["x"].requires_grad_()
    r = selective_scan(**full)
    want, = torch.autograd.grad(r.output.sum(), full["x"], retain_graph=True)
    one = [full[n].detach()[:, 0] if n != "a" else full[n] for n in ("x", "delta", "a", "b", "c")]
    state = r.state.detach()
    selective_scan_step_(state, *one)
    got, = torch.autograd.grad(r.output.sum(), full["x"])
    assert torch.equal(got, want)
    rows = _normal(2, 3, 8)
    x, w = _normal(2, 5, 8), _normal(8, 4).requires_grad_()
    out = causal_conv(x, w, initial=rows).output
    causal_conv_step_(rows, x[:, 0], w.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_gradients_add_up_in_a_shared_input(gpu_lib):
    """One tensor as x, delta and gate: the sum of the three gradients."""
    announce("selective shared input")
    full = _scan_arguments()
    t = full["x"].detach()
    three = [t.clone().requires_grad_() for _ in range(3)]
    d = _normal(2, 5, 8)
    names = ("x", "delta", "gate")
    out = selective_scan(**{**full, **dict(zip(names, three))}, softplus=True).output
    parts = torch.autograd.grad(out, three, d)
    t.requires_grad_()
    out = selective_scan(**{**full, **dict.fromkeys(names, t)}, softplus=True).output
    whole, = torch.autograd.grad(out, t, d)
    assert torch.allclose(whole, sum(parts), rtol=1e-6, atol=1e-6)
