"""What the selective layer's functions and C entry points refuse, before any GPU work."""

import pytest
import torch

from mamba4_amd import _lib

EINVAL = _lib.EINVAL
DATA = 1 << 20  # stands for device memory: never read, every call here is refused
HUGE = 1 << 60


def _refused(rc, words):
    assert rc == EINVAL
    assert words in _lib.load().m4mr_last_error().decode()


def _scan(B=2, T=100, D=64, G=1, N=16, bf16=0, x=DATA, delta=DATA, gate=DATA, b=DATA, c=DATA,
          a=DATA):
    row = G * N
    return _lib.pack_scan(x, T * D, D, delta, T * D, D, gate, T * D, D, b, T * row, row, c, T * row,
                          row, N, N, a, DATA, DATA, B, T, D, G, N, bf16, 1)


def _scan_forward(scan, output=DATA, state=DATA, workspace=DATA, nbytes=HUGE):
    return _lib.load().m4sl_scan_forward(scan, None, None, output, state, None, workspace, nbytes,
                                         None)


def _scan_backward(scan, d_output=DATA, kept=DATA, x=DATA, workspace=DATA, nbytes=HUGE):
    grads = _lib.pack_scan_grads(x, *([DATA] * 8))
    return _lib.load().m4sl_scan_backward(scan, None, d_output, None, kept, grads, workspace,
                                          nbytes, None)


def _scan_step(scan, state=DATA, new_state=DATA, output=DATA):
    return _lib.load().m4sl_scan_step(scan, None, state, new_state, output, None)


@pytest.mark.parametrize("change,words", [
    (dict(B=0), "positive"), (dict(T=0), "positive"), (dict(D=0), "positive"),
    (dict(T=-1), "positive"),
    (dict(G=0), "G must divide D"), (dict(G=3), "G must divide D"),
    (dict(N=0), "states must be in"), (dict(N=65), "states must be in"),
    (dict(x=0), "NULL"), (dict(delta=0), "NULL"), (dict(b=0), "NULL"), (dict(c=0), "NULL"),
    (dict(a=0), "NULL"),
    (dict(x=DATA + 2), "aligned"), (dict(b=DATA + 1, bf16=1), "aligned"),
    (dict(gate=DATA + 2), "aligned"),
    (dict(B=2**24, D=1), "too large"), (dict(B=2**14, D=2**10, G=2**10), "too large"),
])
def test_scan_refuses_a_shape(change, words):
    scan = _scan(**change)
    lib = _lib.load()
    _refused(_scan_forward(scan), words)
    _refused(_scan_backward(scan), words)
    if "T" not in change:
        _refused(_scan_step(scan), words)
    assert lib.m4sl_scan_workspace_bytes(scan) == 0
    assert lib.m4sl_scan_backward_workspace_bytes(scan) == 0
    assert lib.m4sl_scan_kept_floats(scan) == 0


def test_scan_refuses_buffers():
    scan = _scan()
    for call in (_scan_forward, _scan_backward, _scan_step):
        _refused(call(None), "NULL")
    for change in (dict(output=None), dict(state=None)):
        _refused(_scan_forward(scan, **change), "NULL")
    _refused(_scan_forward(scan, output=DATA + 2), "aligned")
    for change in (dict(d_output=None), dict(kept=None), dict(x=0)):
        _refused(_scan_backward(scan, **change), "NULL")
    _refused(_scan_backward(scan, d_output=DATA + 2), "aligned")
    _refused(_scan_backward(scan, workspace=None), "workspace too small")
    _refused(_scan_backward(scan, nbytes=256), "workspace too small")
    _refused(_scan_backward(scan, workspace=DATA + 16), "256-byte aligned")
    for change in (dict(state=None), dict(new_state=None), dict(output=None)):
        _refused(_scan_step(scan, **change), "NULL")
    _refused(_scan_step(_scan(B=2**23, D=512), output=DATA), "too large")


def test_scan_sizes():
    """States before every sixteen tokens; segments of a small batch have a workspace, a
    large batch's walk none; the backward holds the sums of channel blocks."""
    lib = _lib.load()
    assert lib.m4sl_scan_kept_floats(_scan(B=3, T=33, D=20, N=7)) == 3 * 3 * 20 * 7
    assert lib.m4sl_scan_workspace_bytes(_scan(B=1, T=2000)) > 0
    assert lib.m4sl_scan_workspace_bytes(_scan(B=64, T=2000, D=2048)) == 0
    need = lib.m4sl_scan_backward_workspace_bytes(_scan(B=64, T=2000, D=2048))
    assert need >= 4 * 32 * 64 * 2000 * 2 * 16
    assert need % 256 == 0


def test_functions_refuse_other_devices():
    from mamba4_amd import selective_scan, selective_scan_step

    x = torch.zeros(2, 3, 8)
    a, bc = torch.zeros(8, 4), torch.zeros(2, 3, 4)
    with pytest.raises(ValueError, match="ROCm device"):
        selective_scan(x, x, a, bc, bc)
    with pytest.raises(ValueError, match="ROCm device"):
        selective_scan_step(torch.zeros(2, 8, 4), x[:, 0], x[:, 0], a, bc[:, 0], bc[:, 0])


def _checked(lead, **change):
    from mamba4_amd.selective import _scan_inputs

    front = (2, 3)[:lead]
    x = dict(x=torch.zeros(*front, 8), delta=torch.zeros(*front, 8), a=torch.zeros(8, 4),
             b=torch.zeros(*front, 4), c=torch.zeros(*front, 4), skip=None, gate=None,
             delta_bias=None)
    x.update(change)
    return _scan_inputs("scan", lead, **x)


@pytest.mark.parametrize("lead", [1, 2])
def test_scan_arguments(lead):
    """The checks of shapes and types, on host tensors."""
    front = (2, 3)[:lead]
    assert _checked(lead)[3].shape == (*front, 1, 4)
    for change, words in (
            (dict(x=torch.zeros(8)), "floating-point x"),
            (dict(x=torch.zeros(*front, 8, dtype=torch.int32)), "floating-point x"),
            (dict(x=torch.zeros(*front, 0)), "channels"),
            (dict(delta=torch.zeros(*front, 7)), "delta of x's shape"),
            (dict(gate=torch.zeros(*front, 9)), "gate of x's shape"),
            (dict(gate=torch.zeros(*front, 8, dtype=torch.complex64)), "complex"),
            (dict(a=torch.zeros(8)), "a \\[D,N\\]"),
            (dict(a=torch.zeros(7, 4)), "a \\[D,N\\]"),
            (dict(a=torch.zeros(8, 65)), "a \\[D,N\\]"),
            (dict(a=torch.zeros(8, 0)), "a \\[D,N\\]"),
            (dict(a=torch.zeros(8, 4, dtype=torch.complex64)), "complex"),
            (dict(b=torch.zeros(*front, 5)), "needs b and c"),
            (dict(b=torch.zeros(*front, 2, 4)), "needs b and c"),
            (dict(b=torch.zeros(*front, 3, 4), c=torch.zeros(*front, 3, 4)), "groups"),
            (dict(b=torch.zeros(*front, 0, 4), c=torch.zeros(*front, 0, 4)), "needs b and c"),
            (dict(skip=torch.zeros(7)), "skip"),
            (dict(delta_bias=torch.zeros(1, 8)), "delta_bias")):
        with pytest.raises(ValueError, match=words):
            _checked(lead, **change)


def test_lengths_and_active():
    from mamba4_amd.selective import _active, _lengths

    assert _lengths("f", None, 2, 5) is None
    wide = torch.tensor([2**40, -2**40])
    assert _lengths("f", wide, 2, 5).tolist() == [5, 0]
    assert _lengths("f", torch.tensor([300, 3], dtype=torch.int16), 2, 1000).tolist() == [300, 3]
    for bad in (torch.zeros(3, dtype=torch.int64), torch.zeros(2), torch.zeros(2, dtype=torch.bool)):
        with pytest.raises(ValueError, match="integer lengths"):
            _lengths("f", bad, 2, 5)
    for bad in (torch.ones(2), torch.ones(3, dtype=torch.bool)):
        with pytest.raises(ValueError, match="boolean active"):
            _active("f", bad, 2)
