"""Arguments at the edges of what the retention operators take."""

import pytest
import torch

from mamba4_amd import group_norm, linear_attention, linear_attention_step
from tests.gpu_helpers import announce

pytestmark = pytest.mark.gpu


def _normal(*shape):
    return torch.randn(*shape, device="cuda")


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.uint16,
                                   torch.int32, torch.uint32, torch.int64])
def test_lengths_of_every_integer_type(gpu_lib, dtype):
    """Sequences longer than the type's largest value among them."""
    announce(f"lengths {dtype}")
    time = {torch.uint8: 300, torch.int8: 200, torch.int16: 33000}.get(dtype, 70)
    q, v = _normal(3, time, 1, 8), _normal(3, time, 1, 8)
    g = torch.full((1,), -0.1, device="cuda")
    values = [0, 7, 66]
    got = linear_attention(q, q, v, g, lengths=torch.tensor(values, dtype=dtype).cuda())
    want = linear_attention(q, q, v, g, lengths=torch.tensor(values, device="cuda"))
    assert torch.equal(got.output, want.output) and torch.equal(got.state, want.state)


@pytest.mark.parametrize("batch,time", [(0, 5), (2, 0), (0, 0)])
@pytest.mark.parametrize("initial", [None, torch.float32, torch.float64, torch.bfloat16])
@pytest.mark.parametrize("per_head", [False, True])
def test_no_tokens(gpu_lib, batch, time, initial, per_head):
    """The state is the initial one, in float32; every input has a gradient: zeros,
    and the state's cotangent for the initial one."""
    announce(f"no tokens B{batch} T{time} initial={initial} per_head={per_head}")
    q, k = (_normal(batch, time, 2, 8).requires_grad_() for _ in range(2))
    v = _normal(batch, time, 4, 6).to(torch.bfloat16).requires_grad_()
    g = (torch.full((4,), -torch.inf, device="cuda") if per_head
         else _normal(batch, time, 4)).requires_grad_()
    s0 = None
    if initial is not None:
        s0 = _normal(batch, 4, 8, 6).to(initial).requires_grad_()
    inputs = [t for t in (q, k, v, g, s0) if t is not None]
    r = linear_attention(q, k, v, g, initial=s0)
    assert r.output.shape == (batch, time, 4, 6) and r.output.dtype == torch.bfloat16
    assert r.state.shape == (batch, 4, 8, 6) and r.state.dtype == torch.float32
    want = torch.zeros(batch, 4, 8, 6, device="cuda") if s0 is None else s0.float()
    assert torch.equal(r.state, want)
    d_state = _normal(*r.state.shape)
    grads = torch.autograd.grad([r.output, r.state], inputs,
                                [torch.zeros_like(r.output), d_state])
    for t, d in zip(inputs, grads):
        assert d.shape == t.shape and d.dtype == t.dtype
    for d in grads[:4]:
        assert (d == 0).all()
    if s0 is not None:
        assert torch.equal(grads[4], d_state.to(initial))
    with torch.no_grad():
        again = linear_attention(q, k, v, g, initial=s0)
    assert torch.equal(again.state, want) and again.output.shape == r.output.shape


def test_no_tokens_from_the_output_alone(gpu_lib):
    announce("no tokens, output alone")
    x, s0 = _normal(2, 0, 2, 8).requires_grad_(), _normal(2, 2, 8, 8).requires_grad_()
    g = torch.zeros(2, device="cuda", requires_grad=True)
    r = linear_attention(x, x, x, g, initial=s0)
    grads = torch.autograd.grad(r.output, (x, g, s0), torch.zeros_like(r.output))
    assert grads[0].shape == x.shape and (grads[1] == 0).all() and (grads[2] == 0).all()


@pytest.mark.parametrize("dtype", [torch.int64, torch.bool, torch.complex64])
def test_results_of_no_floating_type_are_refused(gpu_lib, dtype):
    """Results come in the type of the values, or of x: whole numbers would cut
    them, complex ones are no inputs at all."""
    announce(f"results in {dtype}")
    x = torch.ones(2, 3, 1, 8, device="cuda")
    bad, g = x.to(dtype), torch.zeros(1, device="cuda")
    state = torch.zeros(2, 1, 8, 8, device="cuda")
    with pytest.raises(ValueError, match="floating"):
        linear_attention(x, x, bad, g)
    with pytest.raises(ValueError, match="floating"):
        linear_attention_step(state, x[:, 0], x[:, 0], bad[:, 0], g)
    with pytest.raises(ValueError, match="floating"):
        group_norm(bad, 1)


def test_complex_inputs_are_refused(gpu_lib):
    """Their imaginary parts would be dropped."""
    announce("complex inputs")
    x, g = torch.ones(2, 3, 1, 8, device="cuda"), torch.zeros(1, device="cuda")
    state, w = torch.zeros(2, 1, 8, 8, device="cuda"), torch.ones(8, device="cuda")

    def z(t):
        return t.to(torch.complex64)

    for args, initial in (((z(x), x, x, g), None), ((x, z(x), x, g), None), ((x, x, x, z(g)), None),
                          ((x, x, x, g), z(state))):
        with pytest.raises(ValueError, match="floating|real"):
            linear_attention(*args, initial=initial)
    with pytest.raises(ValueError, match="floating|real"):
        linear_attention_step(z(state), x[:, 0], x[:, 0], x[:, 0], g)
    for weight, bias, gate in ((z(w), None, None), (w, z(w), None), (w, w, z(x))):
        with pytest.raises(ValueError, match="floating|real"):
            group_norm(x, 1, weight, bias, gate=gate)


def test_whole_numbers_beside_floating_values(gpu_lib):
    """Queries, keys, decays and states of whole numbers are numbers like others."""
    announce("whole numbers")
    q, v = torch.randint(-2, 3, (1, 5, 1, 8), device="cuda"), _normal(1, 5, 1, 8)
    g, s = torch.tensor([-1], device="cuda"), torch.randint(-2, 3, (1, 1, 8, 8), device="cuda")
    got = linear_attention(q, q, v, g, initial=s)
    want = linear_attention(q.float(), q.float(), v, g.float(), initial=s.float())
    assert torch.equal(got.output, want.output) and torch.equal(got.state, want.state)
