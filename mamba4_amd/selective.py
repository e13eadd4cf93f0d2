"""The selective scan on MI355X.

Per channel d with N states (its decays depend on the data through the step s):

    s_t = softplus(delta_t + delta_bias)    (or without the softplus)
    h_t[n] = exp(s_t a[d,n]) h_{t-1}[n] + s_t b_t[n] x_t
    y_t = sum_n c_t[n] h_t[n] + skip x_t,    out_t = y_t silu(gate_t)

``selective_scan`` runs whole sequences (prompts and training),
``selective_scan_step`` and ``selective_scan_step_`` one token from a cached state.

Runs on the gfx950 HIP library (``m4sl_*``, include/mamba4_selective.h) on the
current stream; there is no other implementation.  With x, delta, b, c and gate all
bfloat16 the kernels read them as they are and return bfloat16; any other mix is
computed in float32 and returned in x's dtype.  Steps, states and sums are float32.
"""

from typing import NamedTuple

import torch

from mamba4_amd import _lib
from mamba4_amd.attention import _f32, _on, _same_device, _stream, _workspace
from mamba4_amd.memory import _differentiated, _ptr

MAX_STATES = 64
_BF16 = torch.bfloat16
_F32 = torch.float32


class SelectiveScanResult(NamedTuple):
    output: torch.Tensor
    state: torch.Tensor


# (The checks before each conversion save its microsecond in the usual call.)


def _unit(t):
    """t, or a contiguous copy where its last axis is not dense."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _as(t, dtype):
    return t if t.dtype == dtype else t.to(dtype)


def _dense(t, dtype):
    """t in dtype, contiguous."""
    if t.dtype != dtype:
        t = t.to(dtype)
    return t if t.is_contiguous() else t.contiguous()


def _parameter(t):
    """t in float32, contiguous (None stays None)."""
    if t is None or (t.dtype == _F32 and t.is_contiguous()):
        return t
    return _f32(t)


def _new(t):
    """An empty contiguous tensor like t (torch.empty takes twice as long)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _rows(t, axes):
    """The m4sl_rows of t, with ``axes`` (batch, or batch and time) in front; strides of
    axes of one element are never used."""
    if t is None:
        return 0, 0, 0
    shape, stride = t.shape, t.stride()
    return (t.data_ptr(), stride[0] if shape[0] > 1 else 0,
            stride[1] if axes == 2 and shape[1] > 1 else 0)


def _scan(x, delta, a, b, c, skip, gate, bias, softplus):
    """The m4sl_scan of a call, packed into bytes."""
    axes = x.dim() - 1
    groups, states = b.shape[-2:]
    strides = (b.stride(-2), c.stride(-2)) if groups > 1 else (0, 0)
    return _lib.pack_scan(
        *_rows(x, axes), *_rows(delta, axes), *_rows(gate, axes), *_rows(b, axes),
        *_rows(c, axes), *strides, a.data_ptr(), 0 if skip is None else skip.data_ptr(),
        0 if bias is None else bias.data_ptr(), x.shape[0], x.shape[1] if axes == 2 else 1,
        x.shape[-1], groups, states, x.dtype == _BF16, softplus)


def _forward(x, delta, a, b, c, skip, gate, bias, initial, softplus, lengths, keep):
    """The output and final state, and with ``keep`` what the gradient needs."""
    batch, time, channels = x.shape
    states, device = a.shape[1], x.device
    output = _new(x)
    if batch == 0 or time == 0:
        state = torch.zeros((batch, channels, states), dtype=_F32, device=device) \
            if initial is None else initial.clone()
        return output, state, None
    lib = _lib.load()
    state = torch.empty((batch, channels, states), dtype=_F32, device=device)
    scan = _scan(x, delta, a, b, c, skip, gate, bias, softplus)
    kept = None
    if keep:
        kept = torch.empty(lib.m4sl_scan_kept_floats(scan), dtype=_F32, device=device)
    nbytes = lib.m4sl_scan_workspace_bytes(scan)
    workspace = _workspace(nbytes, device)
    rc = lib.m4sl_scan_forward(scan, _ptr(initial), _ptr(lengths), output.data_ptr(),
                               state.data_ptr(), _ptr(kept), _ptr(workspace), nbytes,
                               _stream(device))
    if rc:
        _lib.check(rc)
    return output, state, kept


class _SelectiveScan(torch.autograd.Function):
    """x, delta, b, c, gate of one dtype with dense last axes; the others float32 and
    contiguous, lengths int32."""

    @staticmethod
    def forward(ctx, x, delta, a, b, c, skip, gate, bias, initial, softplus, lengths):
        output, state, kept = _forward(x, delta, a, b, c, skip, gate, bias, initial, softplus,
                                       lengths, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, delta, a, b, c, skip, gate, bias, initial, lengths, kept)
        ctx.softplus = softplus
        return output, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_output, d_state):
        x, delta, a, b, c, skip, gate, bias, initial, lengths, kept = ctx.saved_tensors
        wanted = ctx.needs_input_grad
        inputs = (x, delta, a, b, c, skip, gate, bias, initial)
        d_state = _parameter(d_state)
        if kept is None:
            grads = [None if t is None else torch.zeros_like(t) for t in inputs]
            if initial is not None and d_state is not None:
                grads[-1] = d_state
            return (*grads, None, None)
        lib = _lib.load()
        device = x.device
        if d_output is None:
            d_output = torch.zeros(x.shape, dtype=x.dtype, device=device)
        d_output = _dense(d_output, x.dtype)
        # (The kernels form those of x, delta, b and c in any case.)
        grads = [_new(t) if t is not None and (wanted[i] or i in (0, 1, 3, 4)) else None
                 for i, t in enumerate(inputs)]
        d_x, d_delta, d_a, d_b, d_c, d_skip, d_gate, d_bias, d_initial = grads
        scan = _scan(x, delta, a, b, c, skip, gate, bias, ctx.softplus)
        nbytes = lib.m4sl_scan_backward_workspace_bytes(scan)
        workspace = _workspace(nbytes, device)
        out = _lib.pack_scan_grads(*(0 if t is None else t.data_ptr() for t in (
            d_x, d_delta, d_gate, d_b, d_c, d_a, d_skip, d_bias, d_initial)))
        rc = lib.m4sl_scan_backward(scan, _ptr(lengths), d_output.data_ptr(), _ptr(d_state),
                                    kept.data_ptr(), out, _ptr(workspace), nbytes,
                                    _stream(device))
        if rc:
            _lib.check(rc)
        return (*grads, None, None)


def _real(name, t):
    if t.dtype.is_complex:
        raise ValueError(f"{name} is complex; take its real part first")


def _scan_inputs(name, lead, x, delta, a, b, c, skip, gate, delta_bias):
    """The checked rows of a call in one dtype of the kernels, its parameters float32."""
    layout = "[B,T,D]" if lead == 2 else "[B,D]"
    if x.dim() != lead + 1 or not x.dtype.is_floating_point:
        raise ValueError(f"{name} needs a floating-point x {layout}")
    front, channels = x.shape[:-1], x.shape[-1]
    if channels == 0:
        raise ValueError(f"{name} needs channels")
    for label, t in (("delta", delta), ("gate", gate)):
        if t is not None:
            if t.shape != x.shape:
                raise ValueError(f"{name} needs {label} of x's shape")
            _real(label, t)
    if a.dim() != 2 or a.shape[0] != channels or not 1 <= a.shape[1] <= MAX_STATES:
        raise ValueError(f"{name} needs a [D,N] with N in 1..{MAX_STATES}")
    states = a.shape[1]
    if b.dim() == lead + 1:
        b = b.unsqueeze(-2)
    if c.dim() == lead + 1:
        c = c.unsqueeze(-2)
    if b.dim() != lead + 2 or b.shape[:-2] != front or b.shape[-1] != states \
            or b.shape[-2] == 0 or c.shape != b.shape:
        raise ValueError(f"{name} needs b and c {layout[:-2]}G,N] or {layout[:-2]}N]")
    if channels % b.shape[-2]:
        raise ValueError(f"{name}: the groups of b and c must divide the channels")
    for label, t in (("b", b), ("c", c), ("a", a)):
        _real(label, t)
    for label, t in (("skip", skip), ("delta_bias", delta_bias)):
        if t is not None and tuple(t.shape) != (channels,):
            raise ValueError(f"{name} needs {label} [D]")
    dtype = _F32
    if x.dtype == delta.dtype == b.dtype == c.dtype == _BF16 \
            and (gate is None or gate.dtype == _BF16):
        dtype = _BF16
    gate = None if gate is None else _unit(_as(gate, dtype))
    return (_unit(_as(x, dtype)), _unit(_as(delta, dtype)), _parameter(a), _unit(_as(b, dtype)),
            _unit(_as(c, dtype)), _parameter(skip), gate, _parameter(delta_bias))


def _lengths(name, lengths, batch, time):
    """lengths as int32, clamped where a narrower integer would wrap around (the kernels
    clamp the rest)."""
    if lengths is None:
        return None
    if tuple(lengths.shape) != (batch,) or lengths.dtype.is_floating_point \
            or lengths.dtype.is_complex or lengths.dtype == torch.bool:
        raise ValueError(f"{name} needs integer lengths [B]")
    if lengths.dtype != torch.int32:
        lengths = lengths.to(torch.int64).clamp(0, time).to(torch.int32)
    return lengths.contiguous()


def _active(name, active, batch):
    if active is None:
        return None
    if tuple(active.shape) != (batch,) or active.dtype != torch.bool:
        raise ValueError(f"{name} needs a boolean active [B]")
    return active.contiguous()


def selective_scan(x, delta, a, b, c, *, skip=None, gate=None, delta_bias=None, softplus=False,
                   initial=None, lengths=None):
    """The selective scan over sequences, differentiable.

    x, delta, gate [B,T,D]; a [D,N] (negative for decays; N <= 64); b, c [B,T,G,N], G
    groups of consecutive channels that share them, or [B,T,N]; skip, delta_bias [D].
    The step is delta + delta_bias, through ``softplus`` where that is set.  initial
    [B,D,N] is the state before the first token (zeros by default).  lengths [B]
    (integers): tokens from lengths[b] on are absent, whatever their rows hold; their
    outputs and gradients are zero.  Rows are read with their strides (parts of a
    projection's rows, say).

    Returns SelectiveScanResult(output [B,T,D] in x's dtype, state [B,D,N] float32
    after the last token).  A row's result may depend on the batch size, by rounding.
    """
    device = _same_device(x, delta, a, b, c, skip, gate, delta_bias, initial, lengths)
    dtype = x.dtype
    inputs = _scan_inputs("selective_scan", 2, x, delta, a, b, c, skip, gate, delta_bias)
    batch, time, channels = x.shape
    if initial is not None:
        if tuple(initial.shape) != (batch, channels, a.shape[1]):
            raise ValueError("selective_scan needs initial [B,D,N]")
        initial = _parameter(initial)
    lengths = _lengths("selective_scan", lengths, batch, time)
    with _on(device):
        if _differentiated(*inputs, initial):
            output, state = _SelectiveScan.apply(*inputs, initial, bool(softplus), lengths)
        else:
            output, state, _ = _forward(*inputs, initial, bool(softplus), lengths, False)
    return SelectiveScanResult(_as(output, dtype), state)


def _scan_step(state, new_state, inputs, softplus, active, dtype):
    x = inputs[0]
    output = _new(x)
    if len(x):
        with _on(x.device):
            rc = _lib.load().m4sl_scan_step(
                _scan(*inputs, softplus), _ptr(active), state.data_ptr(), new_state.data_ptr(),
                output.data_ptr(), _stream(x.device))
        if rc:
            _lib.check(rc)
    return SelectiveScanResult(_as(output, dtype), new_state)


def _step_checks(state, x, delta, a, b, c, skip, gate, delta_bias, active):
    _same_device(state, x, delta, a, b, c, skip, gate, delta_bias, active)
    inputs = _scan_inputs("selective_scan_step", 1, x, delta, a, b, c, skip, gate, delta_bias)
    if tuple(state.shape) != (*x.shape, a.shape[1]):
        raise ValueError("selective_scan_step needs state [B,D,N]")
    return inputs, _active("selective_scan_step", active, len(x))


def selective_scan_step(state, x, delta, a, b, c, *, skip=None, gate=None, delta_bias=None,
                        softplus=False, active=None):
    """One token of ``selective_scan`` from a cached state [B,D,N].

    x, delta, gate [B,D]; b, c [B,G,N] or [B,N]; the rest as there.  active [B] (bool):
    rows where it is false keep their state and give zeros, whatever their token holds.
    Returns SelectiveScanResult(output [B,D], new state); the state given is not
    modified.  Where a gradient is wanted the step is ``selective_scan`` over one token.
    """
    inputs, active = _step_checks(state, x, delta, a, b, c, skip, gate, delta_bias, active)
    if _differentiated(state, *inputs):
        x1, delta1, a1, b1, c1, skip1, gate1, bias1 = inputs
        one = selective_scan(
            x1[:, None], delta1[:, None], a1, b1[:, None], c1[:, None], skip=skip1,
            gate=None if gate1 is None else gate1[:, None], delta_bias=bias1, softplus=softplus,
            initial=state, lengths=None if active is None else active.to(torch.int32))
        return SelectiveScanResult(one.output[:, 0].to(x.dtype), one.state)
    old = _parameter(state)
    return _scan_step(old, torch.empty_like(old), inputs, bool(softplus), active, x.dtype)


def selective_scan_step_(state, x, delta, a, b, c, *, skip=None, gate=None, delta_bias=None,
                         softplus=False, active=None):
    """In-place ``selective_scan_step``: overwrites ``state``, which has to be float32 and
    contiguous, with the new state.  Not differentiable."""
    inputs, active = _step_checks(state, x, delta, a, b, c, skip, gate, delta_bias, active)
    if state.dtype != _F32 or not state.is_contiguous():
        raise ValueError("selective_scan_step_ needs a contiguous float32 state")
    if _differentiated(state, *inputs):
        raise ValueError("selective_scan_step_ has no gradient; use selective_scan_step")
    # The state may be saved for a backward: the write counts as one of torch's.
    torch.autograd.graph.increment_version(state)
    return _scan_step(state, state, inputs, bool(softplus), active, x.dtype)
