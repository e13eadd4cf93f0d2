"""Linear attention with a decay for each head on MI355X.

Per batch row and head, with a matrix state S [N, P]:

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,    o_t = scale * S_t^T q_t

``linear_attention`` runs whole sequences (chunked on the matrix cores, prompts
and training), ``linear_attention_step`` and ``linear_attention_step_`` one
token from a cached state.  The decays are data (a gate of every token and head)
or a constant of each head; queries, keys and values may have fewer heads than
the attention, each shared by as many consecutive heads.

Runs on the gfx950 HIP library (``m4rt_attention_*``,
include/mamba4_retention.h) on the current stream; there is no other
implementation.  With queries, keys and values all bfloat16 the kernels read
them as they are and return bfloat16; any other mix is computed in float32 and
returned in the values' dtype.  States, decays and sums are float32 or wider.
"""

import contextlib
from typing import NamedTuple

import torch

from mamba4_amd import _lib
from mamba4_amd.memory import _differentiated, _ptr

MAX_WIDTH = 128
_MAX_TOKEN_STRIDE = (2**31 - 1) // 256
_BF16 = torch.bfloat16
_F32 = torch.float32


class LinearAttentionResult(NamedTuple):
    output: torch.Tensor
    state: torch.Tensor


def _f32(t):
    if t.dtype.is_complex:
        raise ValueError("complex numbers are not floating-point ones; take their real part first")
    return t.to(_F32).contiguous()


_NOTHING = contextlib.nullcontext()


def _on(device):
    """Makes the device the current one (torch.cuda.device costs microseconds
    where it already is)."""
    return _NOTHING if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _same_device(*tensors):
    device = None
    for t in tensors:
        if t is not None and t.device != device:
            if device is not None or t.device.type != "cuda":
                devices = sorted({str(u.device) for u in tensors if u is not None})
                raise ValueError("all tensors must be ROCm device tensors on one device; got "
                                 + ", ".join(devices))
            device = t.device
    return device


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _strided(t):
    """t itself where the kernels can address it: unit stride along the width,
    tokens at least a row apart (views into a fused projection, say); else a
    contiguous copy."""
    if t.is_contiguous():
        return t
    unit = t.stride(-1) == 1 or t.shape[-1] == 1
    if unit and t.dim() == 4 and t.shape[1] > 1:
        unit = t.shape[-1] <= t.stride(1) <= _MAX_TOKEN_STRIDE
    return t if unit else t.contiguous()


def _row(t):
    """The m4rt_rows of [B,T,h,W] or [B,h,W]; strides of axes of one element are
    never used and given as zero (the token stride, as the width)."""
    shape, stride = t.shape, t.stride()
    width = shape[-1]
    if len(shape) == 4:
        token = stride[1] if shape[1] > 1 else width
    else:
        token = width
    return (t.data_ptr(), stride[0] if shape[0] > 1 else 0, token,
            stride[-2] if shape[-2] > 1 else 0, shape[-2], width)


def _qkv(q, k, v):
    return _lib.pack_qkv(*_row(q), *_row(k), *_row(v))


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _forward(q, k, v, log_decay, initial, lengths, scale):
    lib = _lib.load()
    batch, time, _, n = q.shape
    heads, p, device = log_decay.shape[-1], v.shape[-1], v.device
    bf16 = 1 if v.dtype == _BF16 else 0
    output = torch.empty((batch, time, heads, p), dtype=v.dtype, device=device)
    if batch == 0 or time == 0:
        return output, output.new_zeros((batch, heads, n, p), dtype=_F32) if initial is None \
            else initial.clone()
    state = torch.empty((batch, heads, n, p), dtype=_F32, device=device)
    rows = _qkv(q, k, v)
    nbytes = lib.m4rt_attention_workspace_bytes(rows, bf16, batch, time, heads)
    workspace = _workspace(nbytes, device)
    rc = lib.m4rt_attention_forward(
        rows, bf16, log_decay.data_ptr(), log_decay.dim() == 3, _ptr(lengths),
        _ptr(initial), scale, batch, time, heads, output.data_ptr(), state.data_ptr(),
        _ptr(workspace), nbytes, _stream(device),
    )
    if rc:
        _lib.check(rc)
    return output, state


class _Attention(torch.autograd.Function):
    """q, k, v all bfloat16 or all float32, strided as ``_strided`` leaves them;
    the other inputs float32 and contiguous, lengths int32."""

    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial, lengths, scale):
        output, state = _forward(q, k, v, log_decay, initial, lengths, scale)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, log_decay, initial, lengths)
        # The final state is needed for the decays' gradient from a cotangent of the
        # state alone, which only the backward knows: until then it may be stepped in
        # place, so it is no saved tensor but an alias with its version.
        ctx.state = state.detach() if ctx.needs_input_grad[3] else None
        ctx.version = state._version
        ctx.scale = scale
        return output, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_output, d_state):
        lib = _lib.load()
        q, k, v, log_decay, initial, lengths = ctx.saved_tensors
        batch, time, _, n = q.shape
        heads, p, device = log_decay.shape[-1], v.shape[-1], v.device
        bf16 = 1 if v.dtype == _BF16 else 0
        if batch == 0 or time == 0:
            d_initial = None
            if initial is not None:
                d_initial = torch.zeros_like(initial) if d_state is None else _f32(d_state)
            return (*(torch.zeros_like(t) for t in (q, k, v, log_decay)), d_initial, None, None)
        if d_output is None:
            d_output = torch.zeros((batch, time, heads, p), dtype=v.dtype, device=device)
        d_output = d_output.to(v.dtype).contiguous()
        d_state = None if d_state is None else _f32(d_state)
        d_q, d_k, d_v = (torch.empty(t.shape, dtype=t.dtype, device=device) for t in (q, k, v))
        d_decay = torch.empty_like(log_decay) if ctx.needs_input_grad[3] else None
        d_initial = torch.empty_like(initial) if ctx.needs_input_grad[4] else None
        state = None
        if d_state is not None and d_decay is not None:
            state = ctx.state
            if state._version != ctx.version:
                raise RuntimeError(
                    "one of the variables needed for gradient computation has been modified by "
                    "an inplace operation: the final state of linear_attention")
        rows = _qkv(q, k, v)
        nbytes = lib.m4rt_attention_backward_workspace_bytes(
            rows, d_output.data_ptr(), bf16, batch, time, heads, d_decay is not None)
        workspace = _workspace(nbytes, device)
        rc = lib.m4rt_attention_backward(
            rows, bf16, log_decay.data_ptr(), log_decay.dim() == 3, _ptr(lengths),
            _ptr(initial), ctx.scale, batch, time, heads, d_output.data_ptr(), _ptr(d_state),
            _ptr(state), d_q.data_ptr(), d_k.data_ptr(), d_v.data_ptr(), _ptr(d_decay),
            _ptr(d_initial), _ptr(workspace), nbytes, _stream(device),
        )
        if rc:
            _lib.check(rc)
        return d_q, d_k, d_v, d_decay, d_initial, None, None


def _model_rows(name, queries, keys, values, dims):
    """The heads of the call, and q, k, v in one dtype of the kernels."""
    qs, ks, vs = queries.shape, keys.shape, values.shape
    if len(qs) != dims or len(ks) != dims or len(vs) != dims:
        layout = "[B,T,h,W]" if dims == 4 else "[B,h,W]"
        raise ValueError(f"{name} needs queries, keys and values {layout}")
    lead = dims - 2
    if ks[:lead] != qs[:lead] or vs[:lead] != qs[:lead]:
        raise ValueError("queries, keys and values disagree")
    if qs[-1] != ks[-1]:
        raise ValueError("queries and keys disagree in width")
    hq, hk, hv = qs[-2], ks[-2], vs[-2]
    heads = max(hq, hk, hv)
    if min(hq, hk, hv) == 0 or heads % hq or heads % hk or heads % hv:
        raise ValueError("the heads of queries, keys and values must divide the largest of them")
    if queries.dtype.is_complex or keys.dtype.is_complex or not values.dtype.is_floating_point:
        raise ValueError(f"{name} needs floating-point values, and real queries and keys")
    if not (1 <= ks[-1] <= MAX_WIDTH and 1 <= vs[-1] <= MAX_WIDTH):
        raise ValueError(f"key and value widths must be 1..{MAX_WIDTH}")
    if queries.dtype != _BF16 or keys.dtype != _BF16 or values.dtype != _BF16:
        queries, keys, values = queries.to(_F32), keys.to(_F32), values.to(_F32)
    return heads, _strided(queries), _strided(keys), _strided(values)


def linear_attention(queries, keys, values, log_decay, *, initial=None, lengths=None, scale=1.0):
    """Decayed linear attention over sequences, differentiable.

    queries, keys [B,T,h,N], values [B,T,h,P] with N, P <= 128; the numbers of
    heads may differ if each divides the largest, H (consecutive heads share).
    log_decay [B,T,H], or [H] for one constant a head (log of the factor that the
    state keeps; -inf drops it).  initial [B,H,N,P] is the state before the first token
    (zeros by default).  lengths [B] (integers): tokens from lengths[b] on are
    absent, whatever their rows hold; their outputs and gradients are zero.  An infinity or
    NaN in a row that is present reaches its own and later outputs alone (possibly as NaN).

    Returns LinearAttentionResult(output [B,T,H,P] in the values' dtype, state
    [B,H,N,P] float32 after the last token).  A row's result does not depend on the
    batch size (nor, beyond rounding, on a longer T of the rows beside it).
    """
    device = _same_device(queries, keys, values, log_decay, initial, lengths)
    heads, q, k, v = _model_rows("linear_attention", queries, keys, values, 4)
    batch, time = queries.shape[:2]
    n, p = keys.shape[-1], values.shape[-1]
    if log_decay.shape not in ((batch, time, heads), (heads,)):
        raise ValueError("linear_attention needs log_decay [B,T,H] or [H]")
    if initial is not None and tuple(initial.shape) != (batch, heads, n, p):
        raise ValueError("linear_attention needs initial [B,H,N,P]")
    if lengths is not None:
        if tuple(lengths.shape) != (batch,) or lengths.dtype.is_floating_point \
                or lengths.dtype.is_complex or lengths.dtype == torch.bool:
            raise ValueError("linear_attention needs integer lengths [B]")
        # (The kernels clamp.  Other integers are clamped before they become int32, so
        # that none wraps around, in a type that holds the sequence's length.)
        if lengths.dtype != torch.int32:
            lengths = lengths.to(torch.int64).clamp(0, time).to(torch.int32)
        lengths = lengths.contiguous()
    g = _f32(log_decay)
    s0 = None if initial is None else _f32(initial)
    scale = float(scale)
    with _on(device):
        if _differentiated(q, k, v, g, s0):
            output, state = _Attention.apply(q, k, v, g, s0, lengths, scale)
        else:
            output, state = _forward(q, k, v, g, s0, lengths, scale)
    return LinearAttentionResult(output.to(values.dtype), state)


def _step_checks(state, query, key, value, log_decay, active):
    _same_device(state, query, key, value, log_decay, active)
    heads, q, k, v = _model_rows("linear_attention_step", query, key, value, 3)
    batch = query.shape[0]
    n, p = key.shape[-1], value.shape[-1]
    if state.shape != (batch, heads, n, p):
        raise ValueError("linear_attention_step needs state [B,H,N,P]")
    if log_decay.shape not in ((batch, heads), (heads,)):
        raise ValueError("linear_attention_step needs log_decay [B,H] or [H]")
    if active is not None and (tuple(active.shape) != (batch,) or active.dtype != torch.bool):
        raise ValueError("linear_attention_step needs a boolean active [B]")
    return heads, q, k, v


def _step(state, new_state, q, k, v, log_decay, active, scale, heads, dtype):
    batch, p, device = q.shape[0], v.shape[-1], v.device
    output = torch.empty((batch, heads, p), dtype=v.dtype, device=device)
    if batch:
        g = _f32(log_decay)
        active = None if active is None else active.contiguous()
        with _on(device):
            rc = _lib.load().m4rt_attention_step(
                _qkv(q, k, v), v.dtype == _BF16, g.data_ptr(), g.dim() == 2, _ptr(active),
                float(scale), batch, heads, state.data_ptr(), new_state.data_ptr(),
                output.data_ptr(), _stream(device),
            )
        if rc:
            _lib.check(rc)
    return LinearAttentionResult(output.to(dtype), new_state)


def linear_attention_step(state, query, key, value, log_decay, *, active=None, scale=1.0):
    """One token of ``linear_attention`` from a cached state.

    state [B,H,N,P]; query, key [B,h,N], value [B,h,P]; log_decay [B,H] or [H].
    active [B] (bool): rows where it is false keep their state and give zeros,
    whatever their token holds.  Returns LinearAttentionResult(output [B,H,P],
    new state); the state given is not modified.  Where a gradient is wanted the
    step is ``linear_attention`` over one token.
    """
    heads, q, k, v = _step_checks(state, query, key, value, log_decay, active)
    if _differentiated(state, query, key, value, log_decay):
        decay = log_decay if log_decay.dim() == 1 else log_decay[:, None]
        one = linear_attention(query[:, None], key[:, None], value[:, None], decay, initial=state,
                               lengths=None if active is None else active.to(torch.int32),
                               scale=scale)
        return LinearAttentionResult(one.output[:, 0], one.state)
    old = _f32(state)
    return _step(old, torch.empty_like(old), q, k, v, log_decay, active, scale, heads, value.dtype)


def linear_attention_step_(state, query, key, value, log_decay, *, active=None, scale=1.0):
    """In-place ``linear_attention_step``: overwrites ``state``, which has to be
    float32 and contiguous, with the new state.  Not differentiable."""
    heads, q, k, v = _step_checks(state, query, key, value, log_decay, active)
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError("linear_attention_step_ needs a contiguous float32 state")
    if _differentiated(state, query, key, value, log_decay):
        raise ValueError("linear_attention_step_ has no gradient; use linear_attention_step")
    # The state may be saved for a backward: the write counts as one of torch's.
    torch.autograd.graph.increment_version(state)
    return _step(state, state, q, k, v, log_decay, active, scale, heads, value.dtype)
