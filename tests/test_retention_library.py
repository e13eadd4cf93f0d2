"""The retention entry points' checks of arguments, before any GPU work."""

import ctypes

import pytest

from mamba4_amd import _lib

EINVAL = _lib.EINVAL
DATA = 1 << 20  # stands for device memory: never read, every call here is refused


def _qkv(heads=(2, 2, 2), n=64, p=64, q_data=DATA, token=None, q_width=None):
    rows = []
    for data, h, w in ((q_data, heads[0], q_width or n), (DATA, heads[1], n), (DATA, heads[2], p)):
        rows += [data, 0, h * w if token is None else token, w, h, w]
    return _lib.pack_qkv(*rows)


def _forward(rows=None, T=100, H=2, decay=DATA, output=DATA, workspace=DATA, nbytes=1 << 40):
    return _lib.load().m4rt_attention_forward(
        rows, 0, decay, 0, None, None, 1.0, 1, T, H, output, DATA, workspace, nbytes, None)


def _backward(rows, T=100, H=2, d_state=None, state=DATA, workspace=DATA, nbytes=1 << 40, d_q=DATA):
    return _lib.load().m4rt_attention_backward(
        rows, 0, DATA, 0, None, None, 1.0, 1, T, H, DATA, d_state, state, d_q, DATA, DATA, DATA,
        None, workspace, nbytes, None)


def _refused(rc, words):
    assert rc == EINVAL
    assert words in _lib.load().m4mr_last_error().decode()


@pytest.mark.parametrize("change,words", [
    (dict(rows=None), "NULL"),
    (dict(decay=None), "NULL"),
    (dict(output=None), "NULL"),
    (dict(T=0), "positive"),
    (dict(H=3), "divide H"),
    (dict(rows=_qkv(n=129)), "widths must be in"),
    (dict(rows=_qkv(p=0)), "widths must be in"),
    (dict(rows=_qkv(q_data=0)), "NULL"),
    (dict(rows=_qkv(q_data=DATA + 2)), "aligned to their elements"),
    (dict(rows=_qkv(token=32)), "token stride"),
    (dict(rows=_qkv(token=1 << 24)), "token stride"),
    (dict(rows=_qkv(q_width=32)), "disagree in width"),
    (dict(rows=_qkv(n=63), nbytes=256), "workspace too small"),
    (dict(rows=_qkv(n=63), workspace=None), "workspace too small"),
    (dict(rows=_qkv(n=63), workspace=DATA + 16), "256-byte aligned"),
])
def test_attention_forward_refuses(change, words):
    _refused(_forward(**{**dict(rows=_qkv()), **change}), words)


def test_attention_backward_refuses():
    _refused(_backward(None), "NULL")
    _refused(_backward(_qkv(), d_q=None), "NULL")
    _refused(_backward(_qkv(), d_state=DATA, state=None), "NULL")
    _refused(_backward(_qkv(), nbytes=0), "workspace too small")
    _refused(_backward(_qkv(n=129)), "widths must be in")


def test_attention_step_refuses():
    def step(rows, H=2, state=DATA, decay=DATA):
        return _lib.load().m4rt_attention_step(
            rows, 0, decay, 0, None, 1.0, 1, H, state, DATA, DATA, None)

    _refused(step(None), "NULL")
    _refused(step(_qkv(), state=None), "NULL")
    _refused(step(_qkv(), decay=None), "NULL")
    _refused(step(_qkv(), H=5), "divide H")
    _refused(step(_qkv(p=200)), "widths must be in")


def test_attention_workspaces():
    """Rows that are whole 16-byte pieces need no copies; what is refused has no
    size; a decay's gradient needs more."""
    lib = _lib.load()
    size = lib.m4rt_attention_workspace_bytes
    backward = lib.m4rt_attention_backward_workspace_bytes
    assert size(None, 0, 1, 100, 2) == 0
    assert size(_qkv(n=129), 0, 1, 100, 2) == 0
    assert size(_qkv(), 0, 1, 100, 3) == 0
    whole, odd = size(_qkv(), 0, 1, 100, 2), size(_qkv(n=63), 0, 1, 100, 2)
    assert odd - whole == 2 * 100 * 2 * 64 * 4
    moved = size(_qkv(q_data=DATA + 4), 0, 1, 100, 2)
    assert moved - whole == 100 * 2 * 64 * 4
    assert backward(None, DATA, 0, 1, 100, 2, 1) == 0
    assert backward(_qkv(), DATA, 0, 1, 100, 2, 1) > backward(_qkv(), DATA, 0, 1, 100, 2, 0)
    # 2^31 tokens' worth of heads are refused, not wrapped around.
    assert size(_qkv(), 0, 2**30, 100, 2**30) == 0


def _norm(x=DATA, M=4, L=1, C=64, G=4, activation=1, eps=1e-5, output=DATA, workspace=DATA,
          nbytes=1 << 40):
    return _lib.load().m4rt_norm_forward(x, None, None, None, 0, M, L, C, G, activation, eps,
                                         output, None, workspace, nbytes, None)


@pytest.mark.parametrize("change", [
    dict(x=None), dict(output=None), dict(M=0), dict(L=0), dict(C=0), dict(G=0), dict(G=5),
    dict(activation=3), dict(activation=-1),
    dict(x=DATA + 2), dict(M=64, L=100000, G=1, C=64, workspace=None),
])
def test_norm_refuses(change):
    assert _norm(**change) == EINVAL
    assert "m4rt_norm_forward: " in _lib.load().m4mr_last_error().decode()


def test_norm_backward_needs_the_statistics():
    rc = _lib.load().m4rt_norm_backward(DATA, None, None, None, DATA, None, 0, 4, 1, 64, 4, 0,
                                        1e-5, DATA, None, None, None, DATA, 1 << 40, None)
    _refused(rc, "m4rt_norm_backward: ")


def test_embedding_refuses():
    lib = _lib.load()

    def forward(ids=DATA, table=DATA, n=8, rows=10, width=64, output=DATA):
        return lib.m4rt_embedding_forward(ids, 0, table, 0, n, rows, width, 1.0, output, 0, None)

    def backward(ids=DATA, n=8, rows=10, width=64, d_table=DATA, workspace=DATA, nbytes=1 << 40):
        return lib.m4rt_embedding_backward(ids, 0, DATA, 0, n, rows, width, 1.0, d_table, 0,
                                           workspace, nbytes, None)

    for change in (dict(ids=None), dict(table=None), dict(output=None), dict(n=-1),
                   dict(rows=0), dict(width=0)):
        _refused(forward(**change), "m4rt_embedding_forward: ")
    for change in (dict(ids=None), dict(d_table=None), dict(n=-1), dict(rows=0), dict(width=0),
                   dict(workspace=None), dict(nbytes=16), dict(workspace=DATA + 4)):
        _refused(backward(**change), "m4rt_embedding_backward: ")
    need = lib.m4rt_embedding_workspace_bytes(1000, 50, 64)
    assert 0 < need <= lib.m4rt_embedding_workspace_bytes(2000, 50, 64)
    assert ctypes.c_size_t(need).value == need
