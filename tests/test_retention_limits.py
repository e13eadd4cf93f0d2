"""Sizes that the retention entry points refuse, before any GPU work: M4MR_EINVAL with
nothing launched, not a launch that fails after others.  What is refused has no
workspace either."""

import pytest

from mamba4_amd import _lib

DATA = 1 << 20  # stands for device memory: never read, every call here is refused
HUGE = 1 << 60


def _qkv(heads, widths, token=None):
    """q, k, v of `heads` and `widths`, dense or with the token strides given."""
    rows = []
    for i, (h, w) in enumerate(zip(heads, widths)):
        rows += [DATA, 0, h * w if token is None else token[i], w, h, w]
    return _lib.pack_qkv(*rows)


def _sizes(rows, bf16, B, T, H):
    lib = _lib.load()
    return (lib.m4rt_attention_workspace_bytes(rows, bf16, B, T, H),
            lib.m4rt_attention_backward_workspace_bytes(rows, DATA, bf16, B, T, H, 1))


def _forward(rows, bf16, B, T, H):
    return _lib.load().m4rt_attention_forward(
        rows, bf16, DATA, 0, None, None, 1.0, B, T, H, DATA, DATA, DATA, HUGE, None)


def _backward(rows, bf16, B, T, H):
    return _lib.load().m4rt_attention_backward(
        rows, bf16, DATA, 0, None, None, 1.0, B, T, H, DATA, None, None, DATA, DATA, DATA, DATA,
        None, DATA, HUGE, None)


def _refused(rc, words):
    assert rc == _lib.EINVAL
    assert words in _lib.load().m4mr_last_error().decode()


@pytest.mark.parametrize("p,blocks", [(64, 1), (128, 2)])
def test_attention_forward_fits_a_launch(p, blocks):
    """2^32 threads along x: 512 a block of 64 value columns of a (b, h)."""
    most = 2**23 // blocks - 9
    rows = _qkv((1, 1, 1), (64, 64, p))
    _refused(_forward(rows, 1, most + 1, 5, 1), "too large")
    assert _sizes(rows, 1, most + 1, 5, 1)[0] == 0
    # (A call within the limits is not made here; it has a workspace where it needs one.)
    odd = _qkv((1, 1, 1), (63, 63, p))
    assert _sizes(odd, 1, most, 5, 1)[0] > 0 and _sizes(odd, 1, most + 1, 5, 1)[0] == 0


@pytest.mark.parametrize("n,p,blocks", [(64, 64, 3), (128, 64, 5), (64, 128, 4), (128, 128, 6)])
def test_attention_backward_fits_a_launch(n, p, blocks):
    most = 2**23 // blocks - 9
    rows = _qkv((1, 1, 1), (n, n, p))
    _refused(_backward(rows, 1, most + 2, 5, 1), "too large")
    assert _sizes(rows, 1, most, 5, 1)[1] > 0 and _sizes(rows, 1, most + 2, 5, 1)[1] == 0


def test_attention_step_fits_a_launch():
    """256 threads a (b, h)."""
    rc = _lib.load().m4rt_attention_step(_qkv((1, 1, 1), (1, 1, 1)), 0, DATA, 0, None, 1.0, 2**24,
                                         1, DATA, DATA, DATA, None)
    _refused(rc, "too large")


MOST = (2**31 - 1) // 256  # elements of a token stride: 64 of it in float32 below 2^31 bytes


@pytest.mark.parametrize("bf16", [0, 1])
def test_rows_that_are_copied_keep_to_the_strides(bf16):
    """Rows one element wide take a 16-byte piece in their copy."""
    piece = 8 if bf16 else 4
    most = MOST // piece
    for width in (1, piece - 1):
        ok, bad = (_qkv((1, 1, h), (8, 8, width), (8, 8, h * width)) for h in (most, most + 1))
        assert _sizes(ok, bf16, 1, 2, most)[0] > 0
        assert _sizes(bad, bf16, 1, 2, most + 1)[0] == 0
        _refused(_forward(bad, bf16, 1, 2, most + 1), "token stride")


@pytest.mark.parametrize("bf16", [0, 1])
def test_the_output_cotangent_keeps_to_the_strides(bf16):
    """[B,T,H,P], dense, where the values have fewer heads."""
    most = MOST // 128
    rows = _qkv((1, 1, 1), (8, 8, 128))
    assert _sizes(rows, bf16, 1, 2, most)[1] > 0
    assert _sizes(rows, bf16, 1, 2, most + 1)[1] == 0
    _refused(_backward(rows, bf16, 1, 2, most + 1), "token stride")


def _lookup(n, rows, width, out=DATA):
    return _lib.load().m4rt_embedding_forward(DATA, 0, DATA, 1, n, rows, width, 1.0, out, 1, None)


def _gradient(n, rows, width, table=DATA):
    return _lib.load().m4rt_embedding_backward(DATA, 0, DATA, 1, n, rows, width, 1.0, table, 1,
                                               DATA, HUGE, None)


@pytest.mark.parametrize("width,shift,pieces", [(1024, 0, 128), (1024, 8, 256), (1001, 0, 1001)])
def test_embedding_fits_a_launch(width, shift, pieces):
    """2^32 threads, four pieces each: of 16 bytes, of 8 at such an address, of one
    element in odd rows.  (The gradient's launch takes the table's rows so, beside the
    chunks of the tokens.)"""
    most = 4 * 2**32 // pieces
    for call in (_lookup, _gradient):
        n, rows = (most, 10) if call is _lookup else (10, most)
        _refused(call(n, rows, width, DATA + shift), "too large")


@pytest.mark.parametrize("bf16", [0, 1])
def test_one_token_has_no_stride(bf16):
    """However many heads: rows, copies and the cotangent of one token are within reach."""
    heads = MOST // 8 + 1
    for widths in ((8, 8, 128), (7, 7, 127)):
        rows = _qkv((1, 1, heads), widths, token=widths)
        assert _sizes(rows, bf16, 1, 1, heads)[1] > 0
        wide = _qkv((1, 1, heads), widths)
        assert _sizes(wide, bf16, 1, 2, heads)[1] == 0
