"""Group normalisation with an activation or a gate, channels last, on MI355X.

Over a sample's positions and the channels of a group

    n = (x - mean) / sqrt(variance + eps),    z = n * weight + bias,
    y = act(z),    or with a gate    y = z * act(gate).

The retention layer calls it on the heads of every token (one group a head,
``x`` [tokens, H * P]) under its gate; with positions ([M, L, C]) it is the
usual norm over space or time.  Runs on the gfx950 HIP library
(``m4rt_norm_*``, include/mamba4_retention.h) on the current stream.
"""

import torch

from mamba4_amd import _lib
from mamba4_amd.attention import _f32, _on, _same_device, _stream, _workspace
from mamba4_amd.memory import _differentiated, _ptr

ACTIVATIONS = {"none": 0, "silu": 1, "gelu": 2}


def _sizes(x):
    """M samples, L positions, C channels of [M, ..., C]."""
    channels = x.shape[-1]
    return x.shape[0], x.numel() // (x.shape[0] * channels), channels


def _forward(x, weight, bias, gate, groups, activation, eps, keep):
    """The result, and with ``keep`` the statistics that the gradient needs."""
    lib = _lib.load()
    samples, positions, channels = _sizes(x)
    bf16 = 1 if x.dtype == torch.bfloat16 else 0
    y = torch.empty_like(x)
    stats = None
    if keep:
        stats = torch.empty((samples, groups, 2), dtype=torch.float32, device=x.device)
    nbytes = lib.m4rt_norm_workspace_bytes(samples, positions, channels, groups, bf16, 0)
    workspace = _workspace(nbytes, x.device)
    rc = lib.m4rt_norm_forward(
        x.data_ptr(), _ptr(weight), _ptr(bias), _ptr(gate), bf16, samples, positions, channels,
        groups, activation, eps, y.data_ptr(), _ptr(stats), _ptr(workspace), nbytes,
        _stream(x.device),
    )
    if rc:
        _lib.check(rc)
    return y, stats


class _GroupNorm(torch.autograd.Function):
    """x, gate contiguous and of one dtype; weight and bias float32."""

    @staticmethod
    def forward(ctx, x, weight, bias, gate, groups, activation, eps):
        y, stats = _forward(x, weight, bias, gate, groups, activation, eps, True)
        ctx.save_for_backward(x, weight, bias, gate, stats)
        ctx.args = (groups, activation, eps)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y):
        lib = _lib.load()
        x, weight, bias, gate, stats = ctx.saved_tensors
        groups, activation, eps = ctx.args
        samples, positions, channels = _sizes(x)
        bf16 = int(x.dtype == torch.bfloat16)
        d_y = d_y.to(x.dtype).contiguous()
        d_x = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        d_weight = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        d_bias = torch.empty_like(bias) if ctx.needs_input_grad[2] else None
        d_gate = torch.empty_like(gate) if ctx.needs_input_grad[3] else None
        nbytes = lib.m4rt_norm_workspace_bytes(samples, positions, channels, groups, bf16, 1)
        workspace = _workspace(nbytes, x.device)
        _lib.check(
            lib.m4rt_norm_backward(
                _ptr(x), _ptr(weight), _ptr(bias), _ptr(gate), _ptr(d_y), _ptr(stats), bf16,
                samples, positions, channels, groups, activation, eps, _ptr(d_x), _ptr(d_weight),
                _ptr(d_bias), _ptr(d_gate), _ptr(workspace), nbytes, _stream(x.device),
            )
        )
        return d_x, d_weight, d_bias, d_gate, None, None, None


def group_norm(x, groups, weight=None, bias=None, *, gate=None, activation="none", eps=1e-5):
    """Normalises x [M, ..., C] over each group's positions and channels, then
    applies weight and bias [C] (optional, either alone too) and the activation
    ("none", "silu" or "gelu", by the error function): to the result, or to
    ``gate`` (of x's shape), which then multiplies the result.  Differentiable.

    bfloat16 x (with a bfloat16 gate) is read and written as bfloat16; any other
    dtype is computed in float32 and returned in x's dtype.  Statistics are
    float32 either way.  A sample's result does not depend on how many there are.
    """
    _same_device(x, weight, bias, gate)
    if activation not in ACTIVATIONS:
        raise ValueError(f"Unknown activation {activation}")
    if x.dim() < 2:
        raise ValueError("group_norm needs x [M, ..., C]")
    if not x.dtype.is_floating_point or (gate is not None and gate.dtype.is_complex):
        raise ValueError("group_norm needs a floating-point x, and a real gate")
    channels = x.shape[-1]
    if groups < 1 or channels == 0 or channels % groups:
        raise ValueError("the groups must divide the channels")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (channels,):
            raise ValueError(f"group_norm needs {name} [C]")
    if gate is not None and gate.shape != x.shape:
        raise ValueError("group_norm needs a gate of x's shape")
    if x.numel() == 0:
        return x * 1
    dtype = x.dtype
    rows = torch.float32
    if dtype == torch.bfloat16 and (gate is None or gate.dtype == torch.bfloat16):
        rows = torch.bfloat16
    x = x.to(rows).contiguous()
    gate = None if gate is None else gate.to(rows).contiguous()
    weight, bias = (None if t is None else _f32(t) for t in (weight, bias))
    args = (x, weight, bias, gate, int(groups), ACTIVATIONS[activation], float(eps))
    with _on(x.device):
        if _differentiated(*args[:4]):
            y = _GroupNorm.apply(*args)
        else:
            y = _forward(*args, False)[0]
    return y.to(dtype)
