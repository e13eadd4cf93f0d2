"""The retention layer's operators in float64, from their definitions.

Linear attention with a decay for each head, token by token in both directions
(no chunks, no products of decays), group normalisation over positions and the
channels of a group, and the embedding lookup with the sums of its rows.  The
forms share nothing with the kernels.
"""

import math

import numpy as np


def _spread(x, heads):
    """[..., h, W] -> [..., heads, W]: consecutive heads share a row."""
    return np.repeat(x, heads // x.shape[-2], axis=-2)


def _gather(d, own):
    """Gradient of ``_spread``: the sums over the heads that share."""
    shape = d.shape[:-2] + (own, d.shape[-2] // own, d.shape[-1])
    return d.reshape(shape).sum(axis=-2)


def _present(lengths, batch, time):
    if lengths is None:
        return np.ones((batch, time))
    return (np.arange(time)[None] < np.asarray(lengths)[:, None]).astype(np.float64)


def _operands(q, k, v, log_decay, initial, lengths):
    q, k, v, g = (np.asarray(a, np.float64) for a in (q, k, v, log_decay))
    batch, time = q.shape[:2]
    heads = max(a.shape[2] for a in (q, k, v))
    here = _present(lengths, batch, time)
    absent = here[:, :, None, None] == 0
    q, k, v = (np.where(absent, 0.0, _spread(a, heads)) for a in (q, k, v))
    lam = np.exp(np.broadcast_to(g, (batch, time, heads)))
    lam = np.where(absent[..., 0], 1.0, lam)
    n, p = q.shape[-1], v.shape[-1]
    state = np.zeros((batch, heads, n, p)) if initial is None else np.array(initial, np.float64)
    return q, k, v, lam, state, here


def attention(q, k, v, log_decay, initial=None, lengths=None, scale=1.0):
    """output [B,T,H,P] and the final state [B,H,N,P]."""
    q, k, v, lam, state, here = _operands(q, k, v, log_decay, initial, lengths)
    out = np.zeros(v.shape)
    for t in range(q.shape[1]):
        state = lam[:, t, :, None, None] * state + k[:, t, :, :, None] * v[:, t, :, None, :]
        out[:, t] = scale * (q[:, t, :, :, None] * state).sum(axis=-2)
    return out * here[:, :, None, None], state


def attention_backward(q, k, v, log_decay, d_output, d_state=None, initial=None, lengths=None,
                       scale=1.0):
    """Gradients of q, k, v, log_decay (in its shape) and the initial state."""
    shapes = [np.asarray(a).shape for a in (q, k, v)]
    per_head = np.asarray(log_decay).ndim == 1
    q, k, v, lam, state, here = _operands(q, k, v, log_decay, initial, lengths)
    time = q.shape[1]
    states = [state]
    for t in range(time):
        states.append(lam[:, t, :, None, None] * states[-1]
                      + k[:, t, :, :, None] * v[:, t, :, None, :])
    d_out = scale * np.asarray(d_output, np.float64) * here[:, :, None, None]
    r = np.zeros(state.shape) if d_state is None else np.array(d_state, np.float64)
    dq, dk, dv, dg = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape), np.zeros(lam.shape)
    for t in reversed(range(time)):
        dq[:, t] = (states[t + 1] * d_out[:, t, :, None, :]).sum(axis=-1)
        r = r + q[:, t, :, :, None] * d_out[:, t, :, None, :]
        dk[:, t] = (r * v[:, t, :, None, :]).sum(axis=-1)
        dv[:, t] = (r * k[:, t, :, :, None]).sum(axis=-2)
        dg[:, t] = lam[:, t] * (states[t] * r).sum(axis=(-2, -1))
        r = lam[:, t, :, None, None] * r
    mask = here[:, :, None, None]
    grads = [_gather(d * mask, s[2]) for d, s in zip((dq, dk, dv), shapes)]
    dg = dg * here[:, :, None]
    return (*grads, dg.sum(axis=(0, 1)) if per_head else dg, r)


def attention_step(state, q, k, v, log_decay, active=None, scale=1.0):
    """One token: output [B,H,P] and the new state."""
    state = np.asarray(state, np.float64)
    lengths = None if active is None else np.asarray(active).astype(int)
    out, new = attention(*(np.asarray(a)[:, None] for a in (q, k, v)),
                         log_decay if np.asarray(log_decay).ndim == 1
                         else np.asarray(log_decay)[:, None],
                         initial=state, lengths=lengths, scale=scale)
    return out[:, 0], new


_erf = np.vectorize(math.erf, otypes=[np.float64])


def _activation(z, name):
    """Its value and derivative."""
    if name == "silu":
        s = 0.5 * (1.0 + np.tanh(0.5 * z))
        return z * s, s * (1.0 + z * (1.0 - s))
    if name == "gelu":
        cdf = 0.5 * (1.0 + _erf(z / math.sqrt(2.0)))
        return z * cdf, cdf + z * np.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    return z, np.ones_like(z)


def _normalised(x, groups, eps):
    t = x.reshape(x.shape[0], -1, groups, x.shape[-1] // groups)
    mean = t.mean(axis=(1, 3), keepdims=True)
    var = ((t - mean) ** 2).mean(axis=(1, 3), keepdims=True)
    inv = 1.0 / np.sqrt(var + eps)
    return (t - mean) * inv, inv


def group_norm(x, groups, weight=None, bias=None, gate=None, activation="none", eps=1e-5):
    x = np.asarray(x, np.float64)
    z = _normalised(x, groups, eps)[0].reshape(x.shape)
    z = z * (1.0 if weight is None else np.asarray(weight, np.float64)) \
        + (0.0 if bias is None else np.asarray(bias, np.float64))
    if gate is None:
        return _activation(z, activation)[0]
    return z * _activation(np.asarray(gate, np.float64), activation)[0]


def group_norm_backward(x, groups, d_output, weight=None, bias=None, gate=None,
                        activation="none", eps=1e-5):
    """Gradients of x, weight, bias and gate (None without one)."""
    x, dy = np.asarray(x, np.float64), np.asarray(d_output, np.float64)
    unit, inv = _normalised(x, groups, eps)
    w = np.ones(x.shape[-1]) if weight is None else np.asarray(weight, np.float64)
    n = unit.reshape(x.shape)
    z = n * w + (0.0 if bias is None else np.asarray(bias, np.float64))
    d_gate = None
    if gate is None:
        dz = dy * _activation(z, activation)[1]
    else:
        a, da = _activation(np.asarray(gate, np.float64), activation)
        dz, d_gate = dy * a, dy * z * da
    axes = tuple(range(x.ndim - 1))
    dn = (dz * w).reshape(unit.shape)
    dx = inv * (dn - dn.mean(axis=(1, 3), keepdims=True)
                - unit * (dn * unit).mean(axis=(1, 3), keepdims=True))
    return dx.reshape(x.shape), (dz * n).sum(axis=axes), dz.sum(axis=axes), d_gate


def embedding(ids, table, scale=1.0):
    ids, table = np.asarray(ids), np.asarray(table, np.float64)
    known = (ids >= 0) & (ids < table.shape[0])
    return np.where(known[..., None], scale * table[np.where(known, ids, 0)], 0.0)


def embedding_backward(ids, rows, d_output, scale=1.0):
    """The table's gradient [rows, C]."""
    ids, d = np.asarray(ids).reshape(-1), np.asarray(d_output, np.float64)
    d = d.reshape(ids.size, -1)
    grad = np.zeros((rows, d.shape[-1]))
    known = (ids >= 0) & (ids < rows)
    np.add.at(grad, ids[known], scale * d[known])
    return grad
