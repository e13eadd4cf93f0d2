"""The memory read has no forward-mode derivative: inputs with a tangent are
refused, not computed without it."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mamba4_amd import SelectiveState, selective_decode, selective_gaussian_memory
from tests.gpu_helpers import announce

pytestmark = pytest.mark.gpu

NAMES = ["keys", "values", "queries", "beta", "log_decay", "floor", "evidence", "cross"]


def _inputs():
    g = torch.Generator().manual_seed(0)
    b, t, h, d, p = 2, 5, 2, 64, 64
    x = dict(keys=torch.randn(b, t, h, d, generator=g), values=torch.randn(b, t, h, p, generator=g),
             queries=torch.randn(b, t, h, d, generator=g), beta=torch.rand(b, t, h, generator=g),
             log_decay=-torch.rand(b, t, h, generator=g), floor=0.5 + torch.rand(h, d, generator=g),
             evidence=torch.eye(d).expand(b, h, d, d).clone(), cross=torch.randn(b, h, p, d,
                                                                                 generator=g))
    return {n: a.cuda() for n, a in x.items()}


def _read(x):
    return selective_gaussian_memory(x["keys"], x["values"], x["queries"], x["beta"],
                                     x["log_decay"], x["floor"],
                                     initial=SelectiveState(x["evidence"], x["cross"]))


def _decode(x):
    return selective_decode(SelectiveState(x["evidence"], x["cross"]), x["keys"][:, 0],
                            x["values"][:, 0], x["queries"][:, 0], x["beta"][:, 0],
                            x["log_decay"][:, 0], x["floor"])


@pytest.mark.parametrize("call", [_read, _decode])
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_derivatives_are_refused(gpu_lib, call, grad, name):
    announce(f"forward mode {call.__name__} {name} grad={grad}")
    x = _inputs()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        call(x)  # without a tangent nothing is refused
        x[name] = forward_ad.make_dual(x[name], torch.ones_like(x[name]))
        with pytest.raises(NotImplementedError, match="jvp"):
            call(x)
