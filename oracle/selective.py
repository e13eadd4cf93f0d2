"""The selective layer's operators in float64, from their definitions.

The selective scan token by token in both directions (no tiles, no segments), the
causal convolution tap by tap, and the root-mean-square norm with the residual's
addition.  The forms share nothing with the kernels.
"""

import numpy as np


def _f64(a):
    return None if a is None else np.asarray(a, np.float64)


def sigmoid(z):
    return np.where(z >= 0, 1.0, np.exp(np.minimum(z, 0.0))) / (1.0 + np.exp(-np.abs(z)))


def silu(z):
    return z * sigmoid(z)


def silu_slope(z):
    s = sigmoid(z)
    return s + z * s * (1.0 - s)


def _here(lengths, batch, time):
    if lengths is None:
        return np.ones((batch, time), bool)
    return np.arange(time)[None] < np.asarray(lengths)[:, None]


class _Scan:
    """The operands of a scan with absent tokens cleared, b and c of every channel."""

    def __init__(self, x, delta, a, b, c, skip, gate, bias, softplus, lengths):
        x, delta, a, b, c = (_f64(t) for t in (x, delta, a, b, c))
        batch, time, d = x.shape
        self.groups = b.shape[2]
        self.here = _here(lengths, batch, time)
        on = self.here[..., None]
        raw = delta + (0.0 if bias is None else _f64(bias))
        self.raw = np.where(on, raw, 0.0)
        self.step = np.where(on, np.logaddexp(0.0, raw) if softplus else raw, 0.0)
        self.x = np.where(on, x, 0.0)
        self.a = a
        self.b, self.c = (np.where(on[..., None], np.repeat(t, d // self.groups, axis=2), 0.0)
                          for t in (b, c))
        self.skip = 0.0 if skip is None else _f64(skip)
        self.gate = None if gate is None else np.where(on, _f64(gate), 0.0)

    def keep(self, t):
        return np.where(self.here[:, t, None, None],
                        np.exp(self.step[:, t, :, None] * self.a), 1.0)

    def advance(self, h, t):
        return self.keep(t) * h + (self.step[:, t] * self.x[:, t])[..., None] * self.b[:, t]


def _start(initial, batch, d, n):
    return np.zeros((batch, d, n)) if initial is None else np.array(initial, np.float64)


def scan(x, delta, a, b, c, skip=None, gate=None, bias=None, softplus=False, initial=None,
         lengths=None):
    """output [B,T,D] and the final state [B,D,N]; b, c [B,T,G,N]."""
    s = _Scan(x, delta, a, b, c, skip, gate, bias, softplus, lengths)
    batch, time, d = s.x.shape
    h = _start(initial, batch, d, s.a.shape[1])
    y = np.zeros(s.x.shape)
    for t in range(time):
        h = s.advance(h, t)
        y[:, t] = (h * s.c[:, t]).sum(-1)
    y = y + s.skip * s.x
    out = y if s.gate is None else y * silu(s.gate)
    return np.where(s.here[..., None], out, 0.0), h


def scan_backward(x, delta, a, b, c, d_output, d_state=None, skip=None, gate=None, bias=None,
                  softplus=False, initial=None, lengths=None):
    """Gradients by name: x, delta, a, b, c, skip, gate, bias, initial."""
    s = _Scan(x, delta, a, b, c, skip, gate, bias, softplus, lengths)
    batch, time, d = s.x.shape
    n = s.a.shape[1]
    states = [_start(initial, batch, d, n)]
    for t in range(time):
        states.append(s.advance(states[-1], t))
    d_out = np.where(s.here[..., None], _f64(d_output), 0.0)
    dy = d_out if s.gate is None else d_out * silu(s.gate)
    g = np.zeros((batch, d, n)) if d_state is None else np.array(d_state, np.float64)
    d_x, d_step, y = np.zeros(s.x.shape), np.zeros(s.x.shape), np.zeros(s.x.shape)
    d_a = np.zeros(s.a.shape)
    d_b, d_c = np.zeros(s.b.shape), np.zeros(s.b.shape)
    for t in reversed(range(time)):
        y[:, t] = (states[t + 1] * s.c[:, t]).sum(-1)
        d_c[:, t] = states[t + 1] * dy[:, t, :, None]
        g = g + s.c[:, t] * dy[:, t, :, None]
        d_b[:, t] = g * (s.step[:, t] * s.x[:, t])[..., None]
        flow = (g * s.b[:, t]).sum(-1)
        g = g * s.keep(t)
        rate = np.where(s.here[:, t, None, None], g * states[t], 0.0)
        d_step[:, t] = flow * s.x[:, t] + (rate * s.a).sum(-1)
        d_x[:, t] = flow * s.step[:, t]
        d_a += (rate * s.step[:, t, :, None]).sum(0)
    shape = (batch, time, s.groups, d // s.groups, n)
    d_b, d_c = (np.where(s.here[..., None, None], t.reshape(shape).sum(3), 0.0)
                for t in (d_b, d_c))
    d_delta = d_step * sigmoid(s.raw) if softplus else d_step
    d_delta = np.where(s.here[..., None], d_delta, 0.0)
    y = y + s.skip * s.x
    return dict(x=d_x + s.skip * dy, delta=d_delta, a=d_a, b=d_b, c=d_c,
                skip=(dy * s.x).sum((0, 1)),
                gate=None if s.gate is None else d_out * y * silu_slope(s.gate),
                bias=d_delta.sum((0, 1)), initial=g)


def conv(x, weight, bias=None, activation="none", initial=None, lengths=None):
    """output [B,T,D] and the last W - 1 rows that are present [B,W-1,D]."""
    x, weight = _f64(x), _f64(weight)
    batch, time, d = x.shape
    taps = weight.shape[1]
    here = _here(lengths, batch, time)
    rows, z = _conv(x, weight, bias, initial, here)
    y = silu(z) if activation == "silu" else z
    ends = here.sum(1)
    state = np.stack([rows[i, e:e + taps - 1] for i, e in enumerate(ends)])
    return np.where(here[..., None], y, 0.0), state


def _conv(x, weight, bias, initial, here):
    batch, time, d = x.shape
    taps = weight.shape[1]
    start = np.zeros((batch, taps - 1, d)) if initial is None else _f64(initial)
    rows = np.concatenate([start, np.where(here[..., None], x, 0.0)], axis=1)
    z = np.zeros(x.shape) + (0.0 if bias is None else _f64(bias))
    for j in range(taps):
        z = z + rows[:, j:j + time] * weight[:, j]
    return rows, z


def conv_backward(x, weight, d_output, d_state=None, bias=None, activation="none", initial=None,
                  lengths=None):
    """Gradients by name: x, weight, bias, initial."""
    x, weight = _f64(x), _f64(weight)
    batch, time, d = x.shape
    taps = weight.shape[1]
    here = _here(lengths, batch, time)
    rows, z = _conv(x, weight, bias, initial, here)
    dz = np.where(here[..., None], _f64(d_output), 0.0)
    if activation == "silu":
        dz = np.where(here[..., None], dz * silu_slope(z), 0.0)
    d_rows = np.zeros(rows.shape)
    d_weight = np.zeros(weight.shape)
    for j in range(taps):
        d_rows[:, j:j + time] += dz * weight[:, j]
        d_weight[:, j] = (dz * rows[:, j:j + time]).sum((0, 1))
    if d_state is not None:
        for i, e in enumerate(here.sum(1)):
            d_rows[i, e:e + taps - 1] += _f64(d_state)[i]
    return dict(x=d_rows[:, taps - 1:], weight=d_weight, bias=dz.sum((0, 1)),
                initial=d_rows[:, :taps - 1])


def rms(x, weight=None, residual=None, eps=1e-5, rounded=lambda s: s):
    """The norm and the sum; ``rounded``: what the sum's type makes of it."""
    s = _f64(x) if residual is None else rounded(_f64(x) + _f64(residual))
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + eps)
    return (y if weight is None else y * _f64(weight)), s


def rms_backward(s, d_output, d_sum=None, weight=None, eps=1e-5):
    """Gradients of the sum s [M,C] (those of x and the residual) and of the weight."""
    s, d_output = _f64(s), _f64(d_output)
    inverse = 1.0 / np.sqrt((s * s).mean(-1, keepdims=True) + eps)
    n = s * inverse
    dn = d_output if weight is None else d_output * _f64(weight)
    d_s = inverse * (dn - n * (dn * n).mean(-1, keepdims=True))
    return (d_s if d_sum is None else d_s + _f64(d_sum)), (d_output * n).sum(0)
