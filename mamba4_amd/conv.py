"""The short causal convolution over each channel on MI355X.

    y_t = act(bias + sum over j < W of weight[d,j] x_{t-W+1+j})

``causal_conv`` runs whole sequences (prompts and training), ``causal_conv_step`` and
``causal_conv_step_`` one token from the last W - 1 rows.  Runs on the gfx950 HIP
library (``m4sl_conv_*``, include/mamba4_selective.h) on the current stream.  bfloat16
x is read and written as it is; any other dtype is computed in float32 and returned in
x's dtype.  Weights and sums are float32.
"""

from typing import NamedTuple

import torch

from mamba4_amd import _lib
from mamba4_amd.attention import _on, _same_device, _stream, _workspace
from mamba4_amd.memory import _differentiated, _ptr
from mamba4_amd.selective import _active, _as, _dense, _lengths, _new, _parameter, _rows, _unit

ACTIVATIONS = {"none": 0, "silu": 1}
MAX_TAPS = 8
_BF16 = torch.bfloat16


class CausalConvResult(NamedTuple):
    output: torch.Tensor
    state: torch.Tensor


def _forward(x, weight, bias, initial, activation, lengths):
    batch, time, channels = x.shape
    taps, device = weight.shape[1], x.device
    output = _new(x)
    if batch == 0 or time == 0:
        state = output.new_zeros((batch, taps - 1, channels)) if initial is None \
            else initial.clone()
        return output, state
    state = torch.empty((batch, taps - 1, channels), dtype=x.dtype, device=device)
    rc = _lib.load().m4sl_conv_forward(
        _lib.pack_rows(*_rows(x, 2)), weight.data_ptr(), _ptr(bias), _ptr(initial), _ptr(lengths),
        x.dtype == _BF16, batch, time, channels, taps, activation, output.data_ptr(),
        state.data_ptr(), _stream(device))
    if rc:
        _lib.check(rc)
    return output, state


class _CausalConv(torch.autograd.Function):
    """x and initial of one dtype, x's last axis dense; weight and bias float32, lengths
    int32; all but x contiguous."""

    @staticmethod
    def forward(ctx, x, weight, bias, initial, activation, lengths):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, initial, lengths)
        ctx.activation = activation
        return _forward(x, weight, bias, initial, activation, lengths)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_output, d_state):
        x, weight, bias, initial, lengths = ctx.saved_tensors
        batch, time, channels = x.shape
        taps, device = weight.shape[1], x.device
        inputs = (x, weight, bias, initial)
        if d_state is not None:
            d_state = _dense(d_state, x.dtype)
        if batch == 0 or time == 0:
            grads = [None if t is None else torch.zeros_like(t) for t in inputs]
            if initial is not None and d_state is not None:
                grads[3] = d_state
            return (*grads, None, None)
        if d_output is None:
            d_output = torch.zeros(x.shape, dtype=x.dtype, device=device)
        d_output = _dense(d_output, x.dtype)
        grads = [_new(t) if wanted else None for t, wanted in zip(inputs, ctx.needs_input_grad)]
        lib = _lib.load()
        sizes = (batch, time, channels, taps)
        bf16 = x.dtype == _BF16
        nbytes = lib.m4sl_conv_backward_workspace_bytes(*sizes)
        workspace = _workspace(nbytes, device)
        d_x, d_weight, d_bias, d_initial = grads
        rc = lib.m4sl_conv_backward(
            _lib.pack_rows(*_rows(x, 2)), weight.data_ptr(), _ptr(bias), _ptr(initial),
            _ptr(lengths), d_output.data_ptr(), _ptr(d_state), bf16, *sizes, ctx.activation,
            _ptr(d_x), _ptr(d_initial), _ptr(d_weight), _ptr(d_bias), _ptr(workspace), nbytes,
            _stream(device))
        if rc:
            _lib.check(rc)
        return (*grads, None, None)


def _inputs(name, lead, x, weight, bias, activation):
    """The checked x in a dtype of the kernels, the parameters float32."""
    layout = "[B,T,D]" if lead == 2 else "[B,D]"
    if activation not in ACTIVATIONS:
        raise ValueError(f"Unknown activation {activation}")
    if x.dim() != lead + 1 or not x.dtype.is_floating_point:
        raise ValueError(f"{name} needs a floating-point x {layout}")
    channels = x.shape[-1]
    if channels == 0:
        raise ValueError(f"{name} needs channels")
    if weight.dim() != 2 or weight.shape[0] != channels or not 1 <= weight.shape[1] <= MAX_TAPS:
        raise ValueError(f"{name} needs a weight [D,W] with W in 1..{MAX_TAPS}")
    if bias is not None and tuple(bias.shape) != (channels,):
        raise ValueError(f"{name} needs a bias [D]")
    rows = x if x.dtype == _BF16 else _as(x, torch.float32)
    return _unit(rows), _parameter(weight), _parameter(bias)


def _state(name, label, state, x, weight):
    """Rows [B,W-1,D] in the kernels' dtype."""
    if tuple(state.shape) != (x.shape[0], weight.shape[1] - 1, x.shape[-1]):
        raise ValueError(f"{name} needs {label} [B,W-1,D]")
    if state.dtype.is_complex:
        raise ValueError(f"{label} is complex; take its real part first")
    return _dense(state, x.dtype)


def causal_conv(x, weight, bias=None, *, activation="none", initial=None, lengths=None):
    """The causal convolution of x [B,T,D] with weight [D,W] (W <= 8; the last tap is of
    the token itself), plus bias [D], through the activation ("none" or "silu").
    Differentiable.

    initial [B,W-1,D] holds the rows before the first token, oldest first (zeros by
    default).  lengths [B] (integers): tokens from lengths[b] on are absent, whatever
    their rows hold; their outputs and gradients are zero.  x is read with its strides
    (a part of a projection's rows, say).

    Returns CausalConvResult(output [B,T,D], state [B,W-1,D], the last rows that are
    present, for the tokens that follow), in x's dtype.  A row's result does not depend on
    the batch size.
    """
    device = _same_device(x, weight, bias, initial, lengths)
    dtype = x.dtype
    x, weight, bias = _inputs("causal_conv", 2, x, weight, bias, activation)
    if initial is not None:
        initial = _state("causal_conv", "initial", initial, x, weight)
    lengths = _lengths("causal_conv", lengths, *x.shape[:2])
    args = (x, weight, bias, initial, ACTIVATIONS[activation], lengths)
    with _on(device):
        if _differentiated(*args[:4]):
            output, state = _CausalConv.apply(*args)
        else:
            output, state = _forward(*args)
    return CausalConvResult(_as(output, dtype), _as(state, dtype))


def _step(state, new_state, x, weight, bias, activation, active):
    batch, channels = x.shape
    output = _new(x)
    if batch:
        with _on(x.device):
            rc = _lib.load().m4sl_conv_step(
                _lib.pack_rows(*_rows(x, 1)), weight.data_ptr(), _ptr(bias), _ptr(active),
                x.dtype == _BF16, batch, channels, weight.shape[1], ACTIVATIONS[activation],
                _ptr(state), _ptr(new_state), output.data_ptr(), _stream(x.device))
        if rc:
            _lib.check(rc)
    return output


def causal_conv_step(state, x, weight, bias=None, *, activation="none", active=None):
    """One token of ``causal_conv``: x [B,D] after the rows of state [B,W-1,D].

    active [B] (bool): rows where it is false keep their state and give zeros, whatever
    their token holds.  Returns CausalConvResult(output [B,D], new state) in x's dtype;
    the state given is not modified.  Where a gradient is wanted the step is
    ``causal_conv`` over one token.
    """
    name = "causal_conv_step"
    _same_device(state, x, weight, bias, active)
    dtype = x.dtype
    x, weight, bias = _inputs(name, 1, x, weight, bias, activation)
    old = _state(name, "state", state, x, weight)
    active = _active(name, active, len(x))
    if _differentiated(state, x, weight, bias):
        one = causal_conv(x[:, None], weight, bias, activation=activation, initial=old,
                          lengths=None if active is None else active.to(torch.int32))
        return CausalConvResult(one.output[:, 0].to(dtype), one.state.to(dtype))
    new = torch.empty_like(old)
    output = _step(old, new, x, weight, bias, activation, active)
    return CausalConvResult(_as(output, dtype), _as(new, dtype))


def causal_conv_step_(state, x, weight, bias=None, *, activation="none", active=None):
    """In-place ``causal_conv_step``: shifts x into ``state``, which has to be contiguous
    and of the dtype that x is computed in (bfloat16 for bfloat16, else float32).  Not
    differentiable."""
    name = "causal_conv_step_"
    _same_device(state, x, weight, bias, active)
    dtype = x.dtype
    x, weight, bias = _inputs(name, 1, x, weight, bias, activation)
    if state.dtype != x.dtype or not state.is_contiguous():
        raise ValueError(f"{name} needs a contiguous state in the dtype of the computation")
    _state(name, "state", state, x, weight)
    active = _active(name, active, len(x))
    if _differentiated(state, x, weight, bias):
        raise ValueError(f"{name} has no gradient; use causal_conv_step")
    # The state may be saved for a backward: the write counts as one of torch's.
    torch.autograd.graph.increment_version(state)
    output = _step(state, state, x, weight, bias, activation, active)
    return CausalConvResult(_as(output, dtype), state)
