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
    (dict(B=2**24, D=1), "too large"), (dict(B=1, T=16, D=2**29, N=1), "too large"), (dict(B=2**14, D=2**10, G=2**10), "too large"),
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


def _conv_forward(x=DATA, weight=DATA, initial=None, bf16=0, B=2, T=10, D=8, W=4, activation=1,
                  output=DATA, state=DATA):
    rows = _lib.pack_rows(x, T * D, D)
    return _lib.load().m4sl_conv_forward(rows, weight, None, initial, None, bf16, B, T, D, W,
                                         activation, output, state, None)


def _conv_backward(x=DATA, weight=DATA, bf16=0, B=2, T=10, D=8, W=4, activation=1, d_output=DATA,
                   d_x=DATA, workspace=DATA, nbytes=HUGE):
    rows = _lib.pack_rows(x, T * D, D)
    return _lib.load().m4sl_conv_backward(rows, weight, None, None, None, d_output, None, bf16, B,
                                          T, D, W, activation, d_x, None, DATA, DATA, workspace,
                                          nbytes, None)


def _conv_step(x=DATA, weight=DATA, bf16=0, B=2, D=8, W=4, activation=1, state=DATA,
               new_state=DATA, output=DATA):
    return _lib.load().m4sl_conv_step(_lib.pack_rows(x, D, 0), weight, None, None, bf16, B, D, W,
                                      activation, state, new_state, output, None)


@pytest.mark.parametrize("change,words", [
    (dict(B=0), "positive"), (dict(D=-1), "positive"), (dict(W=0), "taps must be in"),
    (dict(W=9), "taps must be in"), (dict(activation=2), "activation"),
    (dict(activation=-1), "activation"), (dict(x=0), "NULL"), (dict(weight=None), "NULL"),
    (dict(x=DATA + 2), "aligned"), (dict(x=DATA + 1, bf16=1), "aligned"),
    (dict(D=2**31 - 10), "too large"),
])
def test_conv_refuses(change, words):
    for call in (_conv_forward, _conv_backward, _conv_step):
        _refused(call(**change), words)


def test_conv_refuses_buffers():
    _refused(_conv_forward(T=0), "positive")
    _refused(_conv_forward(output=None), "NULL")
    _refused(_conv_forward(initial=DATA + 2), "aligned")
    _refused(_conv_forward(state=DATA + 2), "aligned")
    _refused(_conv_backward(d_output=None), "NULL")
    _refused(_conv_backward(d_x=DATA + 2), "aligned")
    _refused(_conv_backward(workspace=None), "workspace too small")
    _refused(_conv_backward(nbytes=64), "workspace too small")
    _refused(_conv_backward(workspace=DATA + 4), "256-byte aligned")
    for change in (dict(state=None), dict(new_state=None), dict(output=None)):
        _refused(_conv_step(**change), "NULL")
    # 2^32 threads of a piece each.
    _refused(_conv_step(B=2**30, D=2**6, x=DATA + 4), "too large")
    _refused(_conv_forward(B=2**20, T=2**17, D=2**6, x=DATA + 4), "too large")
    size = _lib.load().m4sl_conv_backward_workspace_bytes
    assert size(2, 0, 8, 4) == 0 and size(2, 10, 8, 9) == 0
    assert size(2, 10, 8, 4) >= 5 * 8 * 4
    assert size(16, 1024, 1536, 4) % 256 == 0


def test_conv_arguments():
    from mamba4_amd import causal_conv
    from mamba4_amd.conv import _inputs, _state

    x, w = torch.zeros(2, 5, 8), torch.zeros(8, 4)
    for args, words in (
            ((x[0], w, None, "none"), "floating-point x"), ((x.int(), w, None, "none"), "floating"),
            ((x[..., :0], w, None, "none"), "channels"), ((x, w[:7], None, "none"), "weight"),
            ((x, torch.zeros(8, 9), None, "none"), "weight"),
            ((x, w[:, :0], None, "none"), "weight"), ((x, w, w, "none"), "bias"),
            ((x, w, None, "gelu"), "activation"), ((x, w + 0j, None, "none"), "complex")):
        with pytest.raises(ValueError, match=words):
            _inputs("causal_conv", 2, *args)
    with pytest.raises(ValueError, match="initial"):
        _state("causal_conv", "initial", torch.zeros(2, 4, 8), x, w)
    with pytest.raises(ValueError, match="complex"):
        _state("causal_conv", "initial", torch.zeros(2, 3, 8) + 0j, x, w)
    with pytest.raises(ValueError, match="ROCm device"):
        causal_conv(x, w)


def _rms_forward(x=DATA, x_bf16=0, residual=DATA, residual_bf16=0, M=4, C=64, output=DATA,
                 sum=DATA):
    return _lib.load().m4sl_rms_forward(x, x_bf16, residual, residual_bf16, None, M, C, 1e-5,
                                        output, sum, None, None)


def _rms_e4m3(x=DATA, x_bf16=0, residual=DATA, residual_bf16=0, M=4, C=64, output=DATA, sum=DATA,
              block=32, scale=DATA):
    return _lib.load().m4sl_rms_e4m3(x, x_bf16, residual, residual_bf16, None, M, C, 1e-5, block,
                                     output, scale, sum, None)


@pytest.mark.parametrize("change,words", [
    (dict(M=0), "positive"), (dict(C=0), "positive"), (dict(C=32769), "at most"),
    (dict(M=2**50), "too large"), (dict(x=None), "NULL"), (dict(output=None), "NULL"),
    (dict(residual=None), "no sum"), (dict(x=DATA + 2), "aligned"),
    (dict(x=DATA + 1, x_bf16=1), "aligned"), (dict(residual=DATA + 2), "aligned"),
    (dict(sum=DATA + 1, residual_bf16=1), "aligned"),
])
def test_rms_refuses(change, words):
    _refused(_rms_forward(**change), words)
    _refused(_rms_e4m3(**change), words)


def test_rms_refuses_buffers():
    _refused(_rms_forward(output=DATA + 2), "aligned")
    _refused(_rms_e4m3(scale=None), "NULL")
    for block in (0, -32, 16, 48, 63):
        _refused(_rms_e4m3(block=block), "block")
    _refused(_rms_e4m3(C=2000, block=1024), "block")
    lib = _lib.load()

    def backward(sum=DATA, inverse=DATA, d_output=DATA, M=4, C=64, d_x=DATA, workspace=DATA,
                 nbytes=HUGE):
        return lib.m4sl_rms_backward(sum, 0, None, inverse, d_output, 0, None, M, C, d_x, None,
                                     DATA, workspace, nbytes, None)

    for change, words in ((dict(sum=None), "NULL"), (dict(inverse=None), "NULL"),
                          (dict(d_output=None), "NULL"), (dict(M=0), "positive"),
                          (dict(C=40000), "at most"), (dict(d_x=DATA + 2), "aligned"),
                          (dict(workspace=None), "workspace too small"),
                          (dict(nbytes=16), "workspace too small"),
                          (dict(workspace=DATA + 8), "256-byte aligned")):
        _refused(backward(**change), words)
    assert lib.m4sl_rms_backward_workspace_bytes(0, 64) == 0
    assert lib.m4sl_rms_backward_workspace_bytes(100, 64) >= 64 * 4


def test_rms_arguments():
    from mamba4_amd import rms_norm, rms_norm_e4m3
    from mamba4_amd.norm import _rms_inputs

    x = torch.zeros(3, 8)
    for args, words in (((x[0, 0], None, None), "floating-point x"),
                        ((x.int(), None, None), "floating-point x"),
                        ((x[:, :0], None, None), "channels"), ((x, x[0, :7], None), "weight"),
                        ((x, x, None), "weight"), ((x, None, x[:2]), "residual"),
                        ((x, None, x.int()), "residual"), ((x, x[0] + 0j, None), "complex"),
                        ((torch.zeros(1, 32769), None, None), "channels")):
        with pytest.raises(ValueError, match=words):
            _rms_inputs("rms_norm", *args)
    for call in (rms_norm, rms_norm_e4m3):
        with pytest.raises(ValueError, match="ROCm device"):
            call(x)
