"""The embedding's gradient of so many tokens that a tile of its sort is longer than
its waves hold at once (more than 131,072), against the float64 oracle.

Float32 sums in the order of the tokens: one rounding of 2^-24 of the running sum a
term, sqrt(n) of them at random, n up to 300,000 for one row: 3e-5 of it, 1e-4 of the
largest sum with all of them equal; bfloat16 tables 2^-8."""

import numpy as np
import pytest
import torch

from mamba4_amd import embedding
from oracle import retention as oracle
from tests.gpu_helpers import announce, host, normwise

pytestmark = pytest.mark.gpu

WIDTH = 8


def _ids(kind, n, rows, rng):
    if kind == "random":
        ids = rng.integers(-1, rows + 1, n)  # one unknown id at either end
    elif kind == "equal":
        ids = np.full(n, rows - 1)
    else:  # frequencies as of text: the rank r about in proportion to 1 / r
        ids = np.minimum(np.exp(rng.uniform(0.0, np.log(rows + 1.0), n)).astype(np.int64), rows) - 1
        ids[rng.random(n) < 0.1] = -1
    return ids


@pytest.mark.parametrize("n", [131072, 131073, 300001])
@pytest.mark.parametrize("rows", [300, 50257, 300007])  # one, two and three passes
@pytest.mark.parametrize("kind", ["random", "equal", "text"])
@pytest.mark.parametrize("table_bf16", [False, True])
def test_gradient_of_many_tokens(gpu_lib, n, rows, kind, table_bf16):
    announce(f"embedding sort n={n} rows={rows} {kind} bf16={table_bf16}")
    rng = np.random.default_rng(n + rows)
    ids = _ids(kind, n, rows, rng)
    d = rng.normal(size=(n, WIDTH)).astype(np.float32)
    table = torch.zeros(rows, WIDTH, device="cuda",
                        dtype=torch.bfloat16 if table_bf16 else torch.float32, requires_grad=True)
    out = embedding(torch.tensor(ids, device="cuda"), table, scale=1.7, dtype=torch.float32)
    (grad,) = torch.autograd.grad(out, table, torch.tensor(d, device="cuda"))
    want = oracle.embedding_backward(ids, rows, d.astype(np.float64), 1.7)
    got = host(grad.float())
    assert normwise(got, want) <= (2.0 ** -8 if table_bf16 else 1e-4)
    assert (got[np.setdiff1d(np.arange(rows), ids)] == 0).all()


@pytest.mark.parametrize("n", [131073, 300001])
def test_order_of_the_sums(gpu_lib, n):
    """Equal tokens keep their order: the terms of a row that occurs in one chunk of the
    sorted tokens are added one after the other in float32, exactly."""
    announce(f"embedding order n={n}")
    rng = np.random.default_rng(n)
    rows = n // 3
    ids = rng.integers(0, rows, n)
    d = rng.normal(size=(n, WIDTH)).astype(np.float32) * np.float32(2.0) ** rng.integers(
        -12, 12, (n, 1)).astype(np.float32)
    table = torch.zeros(rows, WIDTH, device="cuda", requires_grad=True)
    out = embedding(torch.tensor(ids, device="cuda"), table)
    (grad,) = torch.autograd.grad(out, table, torch.tensor(d, device="cuda"))
    want = np.zeros((rows, WIDTH), np.float32)
    np.add.at(want, ids, d)  # one addition after the other, in the tokens' order
    order = np.argsort(ids, kind="stable")
    first = np.searchsorted(ids[order], np.arange(rows))
    last = np.searchsorted(ids[order], np.arange(rows), side="right") - 1
    inside = (last >= first) & (first // 64 == last // 64)
    assert inside.sum() > rows // 2
    np.testing.assert_array_equal(grad.cpu().numpy()[inside], want[inside])
