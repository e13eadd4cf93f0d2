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


@pytest.mark.parametrize("shape,groups", [((700, 96), 4), ((3, 200, 24), 3), ((2, 4000, 32), 2),
                                          ((5, 4096), 1)])
@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (3,), (0, 3), (1, 2)])
def test_norm_gradients_one_by_one(gpu_lib, shape, groups, wanted):
    """Any subset of the gradients has the bits of all of them."""
    announce(f"norm gradients {shape} G{groups} {wanted}")
    c = shape[-1]
    tensors = [_normal(*shape), _normal(c), _normal(c), _normal(*shape)]
    d = _normal(*shape)

    def gradients(of):
        x, w, b, gate = (t.clone().requires_grad_(i in of) for i, t in enumerate(tensors))
        y = group_norm(x, groups, w, b, gate=gate, activation="silu")
        return torch.autograd.grad(y, [(x, w, b, gate)[i] for i in of], d)

    every = gradients((0, 1, 2, 3))
    for i, got in zip(wanted, gradients(wanted)):
        assert torch.equal(got, every[i])


def test_norm_backward_takes_null_for_every_gradient(gpu_lib):
    """The C entry point: what is not wanted is neither refused nor written."""
    announce("norm backward with NULL gradients")
    from mamba4_amd import _lib

    m, c, groups = 70, 32, 2
    x, gate, d = _normal(m, c), _normal(m, c), _normal(m, c)
    stats = torch.empty(m, groups, 2, device="cuda")
    y, stream = torch.empty_like(x), torch.cuda.current_stream().cuda_stream
    lib = _lib.load()
    size = max(lib.m4rt_norm_workspace_bytes(m, 1, c, groups, 0, b) for b in (0, 1))
    work = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    _lib.check(lib.m4rt_norm_forward(
        x.data_ptr(), None, None, gate.data_ptr(), 0, m, 1, c, groups, 1, 1e-5, y.data_ptr(),
        stats.data_ptr(), work.data_ptr(), size, stream))

    def backward(d_x, d_weight, d_gate):
        at = [None if t is None else t.data_ptr() for t in (d_x, d_weight, d_gate)]
        _lib.check(lib.m4rt_norm_backward(
            x.data_ptr(), None, None, gate.data_ptr(), d.data_ptr(), stats.data_ptr(), 0, m, 1, c,
            groups, 1, 1e-5, at[0], at[1], None, at[2], work.data_ptr(), size, stream))

    every = [torch.empty_like(x), torch.empty(c, device="cuda"), torch.empty_like(x)]
    backward(*every)
    for i in range(3):
        got = [torch.empty_like(t) if i == j else None for j, t in enumerate(every)]
        backward(*got)
        assert torch.equal(got[i], every[i])
    backward(None, None, None)
