"""The float64 oracle of the retention layer's operators against differences
and closed forms (CPU only)."""

import numpy as np
import pytest

from oracle import retention as oracle

STEP = 1e-6


def _difference(f, x, direction):
    """Central difference of the scalar f along a direction."""
    return (f(x + STEP * direction) - f(x - STEP * direction)) / (2 * STEP)


def _against_differences(f, arrays, grads, rng):
    """Central differences of order STEP^2 with cancellation about 1e-16 / STEP:
    both below 1e-9 of the values here."""
    for i, g in enumerate(grads):
        direction = rng.normal(size=arrays[i].shape)

        def along(x):
            return f(*(x if j == i else a for j, a in enumerate(arrays)))

        want = _difference(along, arrays[i], direction)
        assert np.isclose((g * direction).sum(), want, rtol=1e-7, atol=1e-7), i


@pytest.mark.parametrize("heads,per_head,lengths", [((2, 2, 2), False, None),
                                                    ((4, 2, 1), True, [5, 0, 3]),
                                                    ((1, 1, 3), False, [0, 5, 4])])
def test_attention_gradients(heads, per_head, lengths):
    rng = np.random.default_rng(1)
    b, t, n, p, h = 3, 5, 4, 3, max(heads)
    q, k = (rng.normal(size=(b, t, heads[i], n)) for i in (0, 1))
    v = rng.normal(size=(b, t, heads[2], p))
    g = -rng.uniform(0.1, 1.0, (h,) if per_head else (b, t, h))
    s0 = rng.normal(size=(b, h, n, p))
    d_out, d_state = rng.normal(size=(b, t, h, p)), rng.normal(size=(b, h, n, p))

    def loss(*a):
        out, state = oracle.attention(*a, lengths=lengths, scale=0.7)
        return (out * d_out).sum() + (state * d_state).sum()

    grads = oracle.attention_backward(q, k, v, g, d_out, d_state, s0, lengths, 0.7)
    _against_differences(loss, (q, k, v, g, s0), grads, rng)


def test_attention_without_decay_is_the_sum_over_pairs():
    rng = np.random.default_rng(2)
    q, k, v = (rng.normal(size=(2, 7, 3, 4)) for _ in range(3))
    out, state = oracle.attention(q, k, v, np.zeros(3))
    scores = np.einsum("bihn,bjhn->bhij", q, k) * np.tril(np.ones((7, 7)))
    np.testing.assert_allclose(out, np.einsum("bhij,bjhp->bihp", scores, v), rtol=1e-12,
                               atol=1e-12)
    np.testing.assert_allclose(state, np.einsum("bjhn,bjhp->bhnp", k, v), rtol=1e-12, atol=1e-12)


def test_attention_steps_are_the_sequence():
    rng = np.random.default_rng(3)
    q, k, v = (rng.normal(size=(2, 6, 3, 4)) for _ in range(3))
    g = -rng.uniform(0.1, 2.0, (2, 6, 3))
    g[:, 3] = -np.inf
    out, state = oracle.attention(q, k, v, g, scale=0.5)
    s = np.zeros((2, 3, 4, 4))
    for t in range(6):
        o, s = oracle.attention_step(s, q[:, t], k[:, t], v[:, t], g[:, t], scale=0.5)
        np.testing.assert_allclose(o, out[:, t], rtol=1e-13)
    np.testing.assert_allclose(s, state, rtol=1e-13)


@pytest.mark.parametrize("activation", ["none", "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
def test_norm_gradients(activation, gated):
    rng = np.random.default_rng(4)
    x, gate = rng.normal(size=(2, 3, 8)), rng.normal(size=(2, 3, 8))
    w, b, dy = rng.normal(size=8), rng.normal(size=8), rng.normal(size=(2, 3, 8))
    arrays = (x, w, b) + ((gate,) if gated else ())

    def loss(x, w, b, gate=None):
        return (oracle.group_norm(x, 4, w, b, gate, activation, 1e-3) * dy).sum()

    grads = oracle.group_norm_backward(x, 4, dy, w, b, gate if gated else None, activation, 1e-3)
    _against_differences(loss, arrays, grads[:len(arrays)], rng)


def test_norm_is_torchs():
    import torch

    rng = np.random.default_rng(5)
    x, w, b = rng.normal(size=(2, 6, 12)), rng.normal(size=12), rng.normal(size=12)
    got = oracle.group_norm(x, 3, w, b, eps=1e-4)
    want = torch.nn.functional.group_norm(torch.tensor(x).transpose(1, 2), 3, torch.tensor(w),
                                          torch.tensor(b), 1e-4).transpose(1, 2).numpy()
    np.testing.assert_allclose(got, want, rtol=1e-12, atol=1e-12)


def test_embedding_gradients():
    rng = np.random.default_rng(6)
    ids = np.array([[3, 0, -1, 3], [9, 5, 3, 12]])
    table, d = rng.normal(size=(10, 4)), rng.normal(size=(2, 4, 4))
    out = oracle.embedding(ids, table, 2.0)
    assert (out[0, 2] == 0).all() and (out[1, 3] == 0).all()
    np.testing.assert_array_equal(out[0, 0], 2.0 * table[3])

    def loss(t):
        return (oracle.embedding(ids, t, 2.0) * d).sum()

    _against_differences(loss, (table,), (oracle.embedding_backward(ids, 10, d, 2.0),), rng)
