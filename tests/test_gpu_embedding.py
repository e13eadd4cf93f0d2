"""The embedding lookup and its gradient on the GPU against the float64 oracle.

The lookup is one product and one rounding: float32 results are within 2^-24 of
the element, bfloat16 ones within 2^-9 (max |difference| / max |expected|: 2e-7,
2^-8).  The gradient sums its terms in float32, one rounding of 2^-24 of the
running sum a term and sqrt(n) of them at random, n up to 10^5 for one row: 2e-5;
in bfloat16 2^-8.
"""

import numpy as np
import pytest
import torch

from mamba4_amd import embedding
from oracle import retention as oracle
from tests.gpu_helpers import announce, host, normwise

pytestmark = pytest.mark.gpu


def _compare(ids, rows, width, table_bf16, out_bf16, scale=1.7, seed=0, wide=True):
    g = torch.Generator().manual_seed(seed)
    kinds = {False: torch.float32, True: torch.bfloat16}
    table = torch.randn(rows, width, generator=g).to(kinds[table_bf16])
    d = torch.randn(*ids.shape, width, generator=g).to(kinds[out_bf16])
    t = table.cuda().requires_grad_()
    on = torch.tensor(ids, dtype=torch.int64 if wide else torch.int32, device="cuda")
    out = embedding(on, t, scale=scale, dtype=kinds[out_bf16])
    (grad,) = torch.autograd.grad(out, t, d.cuda())
    torch.cuda.synchronize()
    assert out.dtype == kinds[out_bf16] and grad.dtype == kinds[table_bf16]
    want = oracle.embedding(ids, table.double().numpy(), scale)
    assert normwise(host(out.float()), want) <= (2.0 ** -8 if out_bf16 else 2e-7)
    want = oracle.embedding_backward(ids, rows, d.double().numpy(), scale)
    assert normwise(host(grad.float()), want) <= (2.0 ** -8 if table_bf16 else 2e-5)
    known = np.unique(ids[(ids >= 0) & (ids < rows)])
    untouched = np.setdiff1d(np.arange(rows), known)
    assert (host(grad.float())[untouched] == 0).all()
    return out, grad


@pytest.mark.parametrize("table_bf16", [False, True])
@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("n,rows,width", [
    (1, 1, 1), (1, 300, 64), (15, 7, 33), (16, 511, 8), (17, 512, 6), (100, 40000, 36),
    (2047, 255, 100), (2048, 256, 48), (2049, 300000, 24), (5000, 1000, 130), (20000, 65536, 16)])
def test_lookup_and_gradient(gpu_lib, n, rows, width, table_bf16, out_bf16):
    announce(f"embedding n{n} rows {rows} width {width} {table_bf16} {out_bf16}")
    rng = np.random.default_rng(n)
    ids = rng.integers(-2, rows + 2, n)
    _compare(ids, rows, width, table_bf16, out_bf16, wide=n % 2 == 0)


@pytest.mark.parametrize("n", [1000, 70000])
def test_skewed_ids(gpu_lib, n):
    """One id for all, a few frequent ones, all of them padding, sorted and
    reversed ids: runs over many chunks, and none."""
    announce(f"embedding skewed n{n}")
    rng = np.random.default_rng(1)
    zipf = np.minimum(rng.zipf(1.3, n) - 1, 999)
    for i, ids in enumerate((np.full(n, 999), np.zeros(n, int), rng.integers(0, 3, n) * 400, zipf,
                             np.full(n, -1), np.sort(zipf), np.sort(zipf)[::-1].copy(),
                             np.arange(n) % 1000)):
        _compare(ids, 1000, 40, False, i % 2 == 1, seed=i)


def test_ids_far_outside_the_table(gpu_lib):
    announce("embedding far ids")
    ids = np.array([0, -1, 2**40, -2**40, 2**32, 2**31, 5, 9, 10, 2**63 - 1, -2**63])
    out, _ = _compare(ids, 10, 16, False, False)
    assert (out[[1, 2, 3, 4, 5, 8, 9, 10]] == 0).all()
    small = np.array([0, -1, 2**31 - 1, -2**31, 9, 10])
    _compare(small, 10, 16, False, False, wide=False)


def test_bad_rows_stay_apart(gpu_lib):
    """NaN in the rows of padding tokens and in rows of the table that no token
    has reach nothing."""
    announce("embedding NaN")
    ids = torch.tensor([3, -1, 1, 7, 3], device="cuda")
    table = torch.randn(8, 32, device="cuda")
    table[0] = float("nan")
    table.requires_grad_()
    out = embedding(ids, table)
    assert torch.isfinite(out).all()
    d = torch.randn(5, 32, device="cuda")
    d[1] = float("nan")
    assert torch.isfinite(torch.autograd.grad(out, table, d)[0]).all()


def test_gradient_is_the_same_on_every_run_and_stream(gpu_lib):
    announce("embedding repeat")
    ids = torch.randint(-1, 500, (8, 2000), device="cuda")
    table = torch.randn(500, 256, device="cuda", requires_grad=True)
    d = torch.randn(8, 2000, 256, device="cuda")

    def grad():
        return torch.autograd.grad(embedding(ids, table), table, d)[0]

    want = grad()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = grad()
    stream.synchronize()
    assert torch.equal(want, other)
    for _ in range(3):
        assert torch.equal(want, grad())
    # Views of ids and table.
    part = embedding(ids.t(), table.t().contiguous().t())
    assert torch.equal(part, embedding(ids, table).transpose(0, 1))
    odd = torch.randn(500 * 256 + 1, device="cuda").to(torch.bfloat16)[1:].view(500, 256)
    assert torch.equal(embedding(ids, odd), embedding(ids, odd.clone()))


def test_gradient_against_differences(gpu_lib):
    """The lookup is linear in the table: a step of one is exact but for the
    roundings of the two lookups (2^-24 of each term)."""
    announce("embedding differences")
    rng = np.random.default_rng(5)
    ids = torch.tensor(rng.integers(-1, 30, 400), device="cuda")
    table = torch.randn(30, 20, device="cuda", requires_grad=True)
    d = torch.randn(400, 20, device="cuda")
    g = torch.autograd.grad(embedding(ids, table, scale=3.0), table, d)[0]
    move = torch.randn(30, 20, device="cuda")
    with torch.no_grad():
        up, down = (host(embedding(ids, table + s * move, scale=3.0)) * host(d) for s in (1, -1))
    got = (host(g) * host(move)).sum()
    assert abs(got - (up.sum() - down.sum()) / 2) <= 1e-6 * np.abs(up).sum()


def test_graph_replays(gpu_lib):
    announce("embedding graph")
    ids = torch.randint(0, 300, (3000,), device="cuda")
    table = torch.randn(300, 64, device="cuda", requires_grad=True)
    d = torch.randn(3000, 64, device="cuda")
    want = torch.autograd.grad(embedding(ids, table), table, d)[0]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(embedding(ids, table), table, d)[0]
    for _ in range(3):
        got.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    del graph


def test_long_tables(gpu_lib):
    """Rows past 2^31 elements of the table and of the output."""
    announce("embedding offsets")
    rows, width = 2_200_000, 1024
    table = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    table[-1] = 3.0
    ids = torch.full((rows,), rows - 1, dtype=torch.int32, device="cuda")
    ids[0] = 0
    out = embedding(ids, table, scale=2.0)
    assert (out[-1] == 6.0).all() and (out[0] == 0).all() and (out[rows // 2] == 6.0).all()
    del out, table


def test_empty_and_refusals(gpu_lib):
    table = torch.randn(10, 8, device="cuda", requires_grad=True)
    ids = torch.zeros(0, 3, dtype=torch.int64, device="cuda")
    out = embedding(ids, table)
    assert out.shape == (0, 3, 8)
    assert (torch.autograd.grad(out, table, torch.zeros_like(out))[0] == 0).all()
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="ROCm device"):
        embedding(ids.cpu(), table)
    with pytest.raises(ValueError, match="ids"):
        embedding(ids.float(), table)
    with pytest.raises(ValueError, match="table"):
        embedding(ids, table[0])
    with pytest.raises(ValueError, match="float32 and bfloat16"):
        embedding(ids, table.double())
    with pytest.raises(ValueError, match="float32 and bfloat16"):
        embedding(ids, table, dtype=torch.float16)
