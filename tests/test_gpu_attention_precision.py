"""How exact the linear attention's float32 results are, by the precision that its
operands are held in.

States and their gradients sum weighted keys (three bfloat16 planes, exact to 2^-24)
times values: the weights are off by 2^-23, each sum by 2^-24 of it a rounding, a few
a chunk.  Some ten units of 2^-24 at most: 1e-6 of the largest element.  (Two planes
would leave 2^-17 of a term, 2e-6 to 3e-6 of the largest element at these sizes.)  The
decays' gradient sums differences of some 256 float32 dots of 64 to 128 terms in
float64: each dot off by a unit or two of 2^-24 of its terms, which are a few times the
result, and 16 of those in the sum's square root: 5e-6."""

import numpy as np
import pytest
import torch

from mamba4_amd import linear_attention
from oracle import retention as oracle
from tests.gpu_helpers import announce, host, normwise

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("route", ["walk", "split"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("t,n,p", [(64, 64, 64), (300, 64, 128), (1000, 128, 64), (700, 63, 61)])
def test_float32_results(gpu_lib, monkeypatch, t, n, p, bf16, route):
    announce(f"linear attention precision T{t} N{n} P{p} bf16={bf16} {route}")
    monkeypatch.setenv("M4RT_ATTENTION", route)
    rng = np.random.default_rng(t)
    kind = torch.bfloat16 if bf16 else torch.float32

    def tensor(*shape, scale=1.0, dtype=torch.float32):
        return torch.tensor(scale * rng.normal(size=shape), dtype=torch.float32).to(dtype)

    q, k = (tensor(2, t, 2, n, scale=n**-0.5, dtype=kind) for _ in range(2))
    v, d = (tensor(2, t, 2, p, dtype=kind) for _ in range(2))
    s0, d_state = (tensor(2, 2, n, p) for _ in range(2))
    g = torch.nn.functional.logsigmoid(3.0 + 1.5 * tensor(2, t, 2))
    x = [a.cuda().requires_grad_() for a in (q, k, v, g, s0)]
    r = linear_attention(*x[:4], initial=x[4])
    grads = torch.autograd.grad((r.output, r.state), x, (d.cuda(), d_state.cuda()))
    exact = [a.double().numpy() for a in (q, k, v, g, s0)]
    _, state = oracle.attention(*exact)
    want = oracle.attention_backward(*exact[:4], d.double().numpy(), d_state.double().numpy(),
                                     exact[4])
    for name, got, e, limit in (("state", r.state, state, 1e-6),
                                ("d_initial", grads[4], want[4], 1e-6),
                                ("d_log_decay", grads[3], want[3], 5e-6)):
        error = normwise(host(got), e)
        assert error <= limit, f"{name}: {error:.3g} > {limit:.3g}"
