"""Group normalisation with an activation or a gate, channels last, and the
root-mean-square norm with the residual's addition, on MI355X.

Over a sample's positions and the channels of a group

    n = (x - mean) / sqrt(variance + eps),    z = n * weight + bias,
    y = act(z),    or with a gate    y = z * act(gate).

The retention layer calls it on the heads of every token (one group a head,
``x`` [tokens, H * P]) under its gate; with positions ([M, L, C]) it is the
usual norm over space or time.

``rms_norm`` and ``rms_norm_e4m3`` are the norm before a layer of a residual stream:

    sum = x + residual,    y = sum / sqrt(mean(sum^2) + eps) * weight,

the latter with y in 8 bits and a scale for each row or block of channels, what a
product in 8 bits takes.  All run on the gfx950 HIP library (``m4rt_norm_*``,
include/mamba4_retention.h, and ``m4sl_rms_*``, include/mamba4_selective.h) on the
current stream.
"""

from typing import NamedTuple

import torch

from mamba4_amd import _lib
from mamba4_amd.attention import _f32, _on, _same_device, _stream, _workspace
from mamba4_amd.memory import _differentiated, _ptr
from mamba4_amd.selective import _as, _dense, _parameter

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


MAX_CHANNELS = 32768


class RmsNormResult(NamedTuple):
    output: torch.Tensor
    sum: torch.Tensor


class RmsNormE4M3Result(NamedTuple):
    output: torch.Tensor
    scale: torch.Tensor
    sum: torch.Tensor


def _rms_forward(x, residual, weight, eps, keep):
    """The result, the sum (x itself without a residual), and with ``keep`` the inverse
    roots that the gradient needs; x [M,C]."""
    rows, channels = x.shape
    y = torch.empty_like(x)
    total = x if residual is None else torch.empty_like(residual)
    inverse = torch.empty(rows, dtype=torch.float32, device=x.device) if keep else None
    rc = _lib.load().m4sl_rms_forward(
        x.data_ptr(), x.dtype == torch.bfloat16, _ptr(residual), total.dtype == torch.bfloat16,
        _ptr(weight), rows, channels, eps, y.data_ptr(),
        None if residual is None else total.data_ptr(), _ptr(inverse), _stream(x.device),
    )
    if rc:
        _lib.check(rc)
    return y, total, inverse


class _RmsNorm(torch.autograd.Function):
    """x, residual [M,C], contiguous, each float32 or bfloat16; weight float32."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, total, inverse = _rms_forward(x, residual, weight, eps, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(total, weight, inverse)
        ctx.dtype = x.dtype
        ctx.residual = residual is not None
        return (y, total) if ctx.residual else (y, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y, d_sum):
        total, weight, inverse = ctx.saved_tensors
        wanted, device = ctx.needs_input_grad, total.device
        rows, channels = total.shape
        if d_y is None:
            d_y = torch.zeros((rows, channels), dtype=ctx.dtype, device=device)
        d_y = _dense(d_y, ctx.dtype)
        d_sum = None if d_sum is None else _dense(d_sum, total.dtype)
        # (One array for both, where they have one type: they are the same numbers.)
        same = ctx.dtype == total.dtype
        d_x = d_residual = None
        if wanted[0] or (wanted[1] and same):
            d_x = torch.empty((rows, channels), dtype=ctx.dtype, device=device)
        if wanted[1] and not same:
            d_residual = torch.empty_like(total)
        d_weight = torch.empty_like(weight) if wanted[2] else None
        lib = _lib.load()
        nbytes = lib.m4sl_rms_backward_workspace_bytes(rows, channels)
        workspace = _workspace(nbytes, device)
        rc = lib.m4sl_rms_backward(
            total.data_ptr(), total.dtype == torch.bfloat16, _ptr(weight), inverse.data_ptr(),
            d_y.data_ptr(), ctx.dtype == torch.bfloat16, _ptr(d_sum), rows, channels, _ptr(d_x),
            _ptr(d_residual), _ptr(d_weight), _ptr(workspace), nbytes, _stream(device),
        )
        if rc:
            _lib.check(rc)
        if wanted[1] and same:
            d_residual = d_x
        return d_x if wanted[0] else None, d_residual, d_weight, None


def _rms_rows(t):
    """[M,C] in a dtype of the kernels."""
    t = _dense(t, torch.bfloat16 if t.dtype == torch.bfloat16 else torch.float32)
    return t if t.dim() == 2 else t.view(-1, t.shape[-1])


def _rms_inputs(name, x, weight, residual):
    if x.dim() < 1 or not x.dtype.is_floating_point:
        raise ValueError(f"{name} needs a floating-point x [..., C]")
    channels = x.shape[-1]
    if not 1 <= channels <= MAX_CHANNELS:
        raise ValueError(f"{name} needs 1..{MAX_CHANNELS} channels")
    if residual is not None:
        if residual.shape != x.shape or not residual.dtype.is_floating_point:
            raise ValueError(f"{name} needs a floating-point residual of x's shape")
    if weight is not None and tuple(weight.shape) != (channels,):
        raise ValueError(f"{name} needs a weight [C]")
    return (_rms_rows(x), None if residual is None else _rms_rows(residual),
            _parameter(weight))


def rms_norm(x, weight=None, *, residual=None, eps=1e-5):
    """The root-mean-square norm of x [..., C] plus the residual (of x's shape), times
    weight [C].  Differentiable.

    Returns RmsNormResult(output in x's dtype, sum in the residual's).  The sum is rounded
    to that dtype before it is normalised; without a residual it is x.  bfloat16 and
    float32 x and residuals, in any mix, are read and written as they are, other dtypes
    computed in float32; statistics are float32.  A row's result does not depend on how
    many there are.
    """
    _same_device(x, weight, residual)
    rows, other, scale = _rms_inputs("rms_norm", x, weight, residual)
    if x.numel() == 0:
        total = x if residual is None else (x + residual).to(residual.dtype)
        return RmsNormResult((total if weight is None else total * weight).to(x.dtype), total)
    with _on(x.device):
        if _differentiated(rows, other, scale):
            y, total = _RmsNorm.apply(rows, other, scale, float(eps))
        else:
            y, total, _ = _rms_forward(rows, other, scale, float(eps), False)
    if x.dim() != 2:
        y, total = y.view(x.shape), None if residual is None else total.view(x.shape)
    return RmsNormResult(_as(y, x.dtype),
                         x if residual is None else _as(total, residual.dtype))


def rms_norm_e4m3(x, weight=None, *, residual=None, eps=1e-5, block=None):
    """``rms_norm`` with its result in 8 bits (torch.float8_e4m3fn) and scales.

    Each ``block`` channels of a row (a power of two in 32..512; the last may be shorter;
    all of them by default) have a scale, the largest magnitude over 448 (at least 2^-126);
    the result is y / scale, rounded to nearest.  Returns RmsNormE4M3Result(output [..., C],
    scale [..., ceil(C / block)] float32, sum).  Not differentiable.
    """
    _same_device(x, weight, residual)
    rows, other, weights = _rms_inputs("rms_norm_e4m3", x, weight, residual)
    if _differentiated(rows, other, weights):
        raise ValueError("rms_norm_e4m3 has no gradient; use rms_norm")
    channels = x.shape[-1]
    block = channels if block is None else int(block)
    if block < 1 or (block < channels and block not in (32, 64, 128, 256, 512)):
        raise ValueError("a scale's block must be a power of two in 32..512, or all channels")
    blocks = -(-channels // block)
    y = torch.empty(rows.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty((len(rows), blocks), dtype=torch.float32, device=x.device)
    total = rows if other is None else torch.empty_like(other)
    if x.numel():
        with _on(x.device):
            rc = _lib.load().m4sl_rms_e4m3(
                rows.data_ptr(), rows.dtype == torch.bfloat16, _ptr(other),
                total.dtype == torch.bfloat16, _ptr(weights), len(rows), channels, float(eps),
                min(block, MAX_CHANNELS), y.data_ptr(), scale.data_ptr(),
                None if other is None else total.data_ptr(), _stream(x.device),
            )
        if rc:
            _lib.check(rc)
    total = x if other is None else total.view(x.shape).to(residual.dtype)
    return RmsNormE4M3Result(y.view(x.shape), scale.view(*x.shape[:-1], blocks), total)
