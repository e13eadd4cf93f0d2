"""The float64 oracle of the selective layer's operators against differences and closed
forms (CPU only)."""

import numpy as np
import pytest

from oracle import selective as oracle

STEP = 1e-6


def _against_differences(f, arrays, grads, rng):
    """Central differences of order STEP^2, below 1e-9 of the values here, with
    cancellation: the two losses are off by a few 2^-53 of themselves, their difference
    over 2 STEP by a few times 1e-16 / STEP of a loss (1e11 where negative steps grow)."""
    for name, g in grads.items():
        if g is None:
            continue
        direction = rng.normal(size=g.shape)
        up, down = (f(**{**arrays, name: arrays[name] + s * STEP * direction}) for s in (1, -1))
        want = (up - down) / (2 * STEP)
        limit = 1e-7 + 1e-15 / STEP * abs(up)
        assert np.isclose((g * direction).sum(), want, rtol=1e-7, atol=limit), name


def _scan_arrays(rng, b, t, d, g, n):
    return dict(x=rng.normal(size=(b, t, d)), delta=rng.normal(-1.0, 1.0, (b, t, d)),
                a=-rng.uniform(0.2, 2.0, (d, n)), b=rng.normal(size=(b, t, g, n)),
                c=rng.normal(size=(b, t, g, n)), skip=rng.normal(size=d),
                gate=rng.normal(size=(b, t, d)), bias=rng.normal(size=d),
                initial=rng.normal(size=(b, d, n)))


@pytest.mark.parametrize("g,softplus,lengths", [(1, True, None), (3, False, [5, 0, 3]),
                                                (2, True, [0, 5, 4])])
def test_scan_gradients(g, softplus, lengths):
    rng = np.random.default_rng(1)
    arrays = _scan_arrays(rng, 3, 5, 6, g, 4)
    d_out, d_state = rng.normal(size=(3, 5, 6)), rng.normal(size=(3, 6, 4))

    def loss(**x):
        out, state = oracle.scan(**x, softplus=softplus, lengths=lengths)
        return (out * d_out).sum() + (state * d_state).sum()

    grads = oracle.scan_backward(**arrays, d_output=d_out, d_state=d_state, softplus=softplus,
                                 lengths=lengths)
    _against_differences(loss, arrays, grads, rng)


def test_scan_without_decay_is_a_running_sum():
    rng = np.random.default_rng(2)
    x, b, c = rng.normal(size=(2, 7, 3)), rng.normal(size=(2, 7, 1, 4)), rng.normal(size=(2, 7, 1, 4))
    out, state = oracle.scan(x, np.ones_like(x), np.zeros((3, 4)), b, c)
    flow = np.cumsum(x[..., None] * b, axis=1)
    np.testing.assert_allclose(out, (flow * c).sum(-1), rtol=1e-12, atol=1e-12)
    np.testing.assert_allclose(state, flow[:, -1], rtol=1e-12, atol=1e-12)


def test_scan_of_a_constant_decays_to_its_limit():
    """h <- e h + u has the limit u / (1 - e), reached to e^T."""
    out, _ = oracle.scan(np.full((1, 400, 1), 2.0), np.full((1, 400, 1), 0.5),
                         np.full((1, 1), -0.2), np.ones((1, 400, 1, 1)), np.ones((1, 400, 1, 1)))
    assert np.isclose(out[0, -1, 0], 1.0 / (1.0 - np.exp(-0.1)), rtol=1e-12)


def test_scan_in_two_parts_is_the_whole():
    rng = np.random.default_rng(3)
    x = _scan_arrays(rng, 2, 9, 4, 2, 3)
    out, state = oracle.scan(**x, softplus=True)
    timed = ("x", "delta", "b", "c", "gate")
    first, middle = oracle.scan(**{n: v[:, :4] if n in timed else v for n, v in x.items()},
                                softplus=True)
    rest = {n: v[:, 4:] if n in timed else v for n, v in x.items()}
    second, end = oracle.scan(**{**rest, "initial": middle}, softplus=True)
    np.testing.assert_allclose(np.concatenate([first, second], 1), out, rtol=1e-12, atol=1e-12)
    np.testing.assert_allclose(end, state, rtol=1e-12, atol=1e-12)


def test_absent_tokens_do_nothing():
    rng = np.random.default_rng(4)
    x = _scan_arrays(rng, 2, 6, 3, 1, 2)
    out, state = oracle.scan(**x, softplus=True, lengths=[4, 0])
    for n in ("x", "delta", "b", "c", "gate"):
        x[n][0, 4:] = np.nan
        x[n][1] = np.nan
    again, end = oracle.scan(**x, softplus=True, lengths=[4, 0])
    np.testing.assert_array_equal(out, again)
    np.testing.assert_array_equal(state, end)
    assert (out[1] == 0).all() and (state[1] == x["initial"][1]).all()


@pytest.mark.parametrize("taps,activation,lengths", [(4, "silu", None), (1, "none", [5, 0, 3]),
                                                     (3, "silu", [0, 1, 5])])
def test_conv_gradients(taps, activation, lengths):
    rng = np.random.default_rng(5)
    arrays = dict(x=rng.normal(size=(3, 5, 4)), weight=rng.normal(size=(4, taps)),
                  bias=rng.normal(size=4), initial=rng.normal(size=(3, taps - 1, 4)))
    d_out, d_state = rng.normal(size=(3, 5, 4)), rng.normal(size=(3, taps - 1, 4))

    def loss(**a):
        out, state = oracle.conv(**a, activation=activation, lengths=lengths)
        return (out * d_out).sum() + (state * d_state).sum()

    grads = oracle.conv_backward(**arrays, d_output=d_out, d_state=d_state,
                                 activation=activation, lengths=lengths)
    _against_differences(loss, arrays, grads, rng)


def test_conv_in_two_parts_and_its_state():
    rng = np.random.default_rng(6)
    x, w = rng.normal(size=(2, 9, 3)), rng.normal(size=(3, 4))
    out, state = oracle.conv(x, w)
    np.testing.assert_array_equal(state, x[:, -3:])
    first, middle = oracle.conv(x[:, :2], w)
    np.testing.assert_array_equal(middle, np.concatenate([np.zeros((2, 1, 3)), x[:, :2]], 1))
    second, _ = oracle.conv(x[:, 2:], w, initial=middle)
    np.testing.assert_allclose(np.concatenate([first, second], 1), out, rtol=1e-12, atol=1e-12)
    one, _ = oracle.conv(x, np.array([[0.0, 0.0, 1.0, 0.0]] * 3))
    np.testing.assert_array_equal(one[:, 1:], x[:, :-1])


def test_rms_gradients_and_norm():
    rng = np.random.default_rng(7)
    x, r, w = rng.normal(size=(4, 6)), rng.normal(size=(4, 6)), rng.normal(size=6)
    d_y, d_sum = rng.normal(size=(4, 6)), rng.normal(size=(4, 6))
    y, s = oracle.rms(x, None, r, eps=0.0)
    np.testing.assert_allclose((y * y).mean(-1), 1.0, rtol=1e-12)
    np.testing.assert_array_equal(s, x + r)

    def loss(**a):
        y, s = oracle.rms(**a, eps=1e-3)
        return (y * d_y).sum() + (s * d_sum).sum()

    d_s, d_w = oracle.rms_backward(s, d_y, d_sum, w, eps=1e-3)
    _against_differences(loss, dict(x=x, residual=r, weight=w),
                         dict(x=d_s, residual=d_s, weight=d_w), rng)
