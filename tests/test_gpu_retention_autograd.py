"""How the retention operators stand in torch's automatic differentiation: what
has no derivative says so, what has one keeps its graph."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mamba4_amd import (
    embedding,
    group_norm,
    linear_attention,
    linear_attention_step,
    linear_attention_step_,
)
from tests.gpu_helpers import announce

pytestmark = pytest.mark.gpu


def _normal(*shape):
    return torch.randn(*shape, device="cuda")


def _calls():
    """Each operator as a function of one of its inputs, with that input."""
    q, k, v, s = _normal(2, 5, 2, 8), _normal(2, 5, 2, 8), _normal(2, 5, 2, 8), _normal(2, 2, 8, 8)
    g = -torch.rand(2, 5, 2, device="cuda")
    x, w, gate = _normal(6, 8), _normal(8), _normal(6, 8)
    ids = torch.tensor([1, 0, 3], device="cuda")
    return {
        "attention queries": (lambda t: linear_attention(t, k, v, g), q),
        "attention keys": (lambda t: linear_attention(q, t, v, g), k),
        "attention values": (lambda t: linear_attention(q, k, t, g), v),
        "attention decay": (lambda t: linear_attention(q, k, v, t), g),
        "attention initial": (lambda t: linear_attention(q, k, v, g, initial=t), s),
        "step state": (lambda t: linear_attention_step(t, q[:, 0], k[:, 0], v[:, 0], g[:, 0]), s),
        "step value": (lambda t: linear_attention_step(s, q[:, 0], k[:, 0], t, g[:, 0]), v[:, 0]),
        "norm": (lambda t: group_norm(t, 2, w, gate=gate, activation="silu"), x),
        "norm weight": (lambda t: group_norm(x, 2, t), w),
        "norm gate": (lambda t: group_norm(x, 2, gate=t, activation="silu"), gate),
        "embedding": (lambda t: embedding(ids, t), _normal(4, 8)),
    }


@pytest.mark.parametrize("name", [
    "attention queries", "attention keys", "attention values", "attention decay",
    "attention initial", "step state", "step value", "norm", "norm weight", "norm gate",
    "embedding"])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(gpu_lib, name, grad):
    """A tangent that the call cannot carry on is no zero (no_grad does not stop
    forward mode)."""
    announce(f"forward mode {name} grad={grad}")
    call, x = _calls()[name]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="jvp"):
            call(dual)
        call(x)  # without a tangent nothing is refused


def test_forward_mode_derivatives_of_the_step_in_place_are_refused(gpu_lib):
    announce("forward mode step in place")
    q, k, v, s = _normal(2, 2, 8), _normal(2, 2, 8), _normal(2, 2, 8), _normal(2, 2, 8, 8)
    g = -torch.rand(2, 2, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(v, torch.ones_like(v))
        before = s.clone()
        with pytest.raises(ValueError, match="no gradient"):
            linear_attention_step_(s, q, k, dual, g)
        assert torch.equal(s, before)
        linear_attention_step_(s, q, k, v, g)


def _prompt(decay_grad):
    q, k, v = (_normal(2, 70, 2, 8).requires_grad_() for _ in range(3))
    g = (-torch.rand(2, 70, 2, device="cuda")).requires_grad_(decay_grad)
    return q, k, v, g


def _advance(state):
    """One token more, in place, as a decode loop does after its prompt."""
    one = _normal(2, 2, 8)
    with torch.no_grad():
        linear_attention_step_(state, one, one, one, -torch.rand(2, 2, device="cuda"))


@pytest.mark.parametrize("decay_grad", [False, True])
def test_a_step_in_place_on_the_state_leaves_the_backward(gpu_lib, decay_grad):
    """The gradient from the output alone does not need the final state."""
    announce(f"step in place before the backward, decay_grad={decay_grad}")
    inputs = _prompt(decay_grad)
    wanted = [t for t in inputs if t.requires_grad]
    r = linear_attention(*inputs)
    d = _normal(*r.output.shape)
    want = torch.autograd.grad(r.output, wanted, d, retain_graph=True)
    _advance(r.state)
    got = torch.autograd.grad(r.output, wanted, d)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_a_modified_state_that_the_backward_needs_is_refused(gpu_lib):
    """The decays' gradient from a cotangent of the state is of the state that the
    forward gave; without the decays' it does not enter."""
    announce("step in place on a state the backward needs")
    for decay_grad in (True, False):
        inputs = _prompt(decay_grad)
        wanted = [t for t in inputs[1:] if t.requires_grad]
        r = linear_attention(*inputs)
        d = _normal(*r.state.shape)
        want = torch.autograd.grad(r.state, wanted, d, retain_graph=True)
        _advance(r.state.detach())
        if decay_grad:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(r.state, wanted, d)
        else:
            for a, b in zip(torch.autograd.grad(r.state, wanted, d), want):
                assert torch.equal(a, b)
