"""Linear attention on the GPU against the float64 oracle.

Tolerances, as max |difference| / max |expected|.  Float32 calls: operands are
exact to 2^-24 and sums of n terms off by about sqrt(n) 2^-24, n below a few
thousand here, gradients with operands that are results themselves: 2e-5
(d_log_decay sums differences over the sequence: 1e-4).  Bfloat16 calls: results
rounded to bfloat16, half a unit of 2^-8, twice that with what precedes: 2^-8.
Their float32 results come of operands exact to 2^-17 (two bfloat16 parts):
5e-5 for states, 2e-4 for the decays' gradient.
"""

import numpy as np
import pytest
import torch

from mamba4_amd import linear_attention, linear_attention_step, linear_attention_step_
from oracle import retention as oracle
from tests.gpu_helpers import announce, host, normwise

pytestmark = pytest.mark.gpu

NAMES = ("q", "k", "v", "log_decay", "initial")


def _limits(bf16):
    if bf16:
        return dict(rows=2.0 ** -8, state=5e-5, decay=2e-4)
    return dict(rows=2e-5, state=2e-5, decay=1e-4)


def _bf(x):
    return torch.tensor(x, dtype=torch.float32).to(torch.bfloat16).double().numpy()


def _problem(b, t, heads, n, p, bf16, per_head=False, initial=False, seed=0):
    rng = np.random.default_rng(seed)
    h = max(heads)
    q, k = (rng.normal(size=(b, t, heads[i], n)) / np.sqrt(n) for i in (0, 1))
    v = rng.normal(size=(b, t, heads[2], p))
    d_out = rng.normal(size=(b, t, h, p))
    cast = _bf if bf16 else (lambda a: a.astype(np.float32).astype(np.float64))
    q, k, v, d_out = (cast(a) for a in (q, k, v, d_out))
    shape = (h,) if per_head else (b, t, h)
    g = -np.log1p(np.exp(-rng.normal(3.0, 1.5, shape))).astype(np.float32).astype(np.float64)
    f32 = (lambda a: a.astype(np.float32).astype(np.float64))
    s0 = f32(rng.normal(size=(b, h, n, p))) if initial else None
    d_state = f32(rng.normal(size=(b, h, n, p))) if initial else None
    return [q, k, v, g, s0], d_out, d_state


def _device(a, dtype):
    return None if a is None else torch.tensor(a, dtype=dtype, device="cuda")


def _tensors(arrays, bf16, grad):
    rows = torch.bfloat16 if bf16 else torch.float32
    out = [_device(a, rows if i < 3 else torch.float32) for i, a in enumerate(arrays)]
    return [t if t is None else t.requires_grad_(grad) for t in out]


def _check(label, got, want, limit):
    error = normwise(host(got.float() if isinstance(got, torch.Tensor) else got), want)
    assert error <= limit, f"{label}: {error:.3g} > {limit:.3g}"


def _run(arrays, d_out, d_state, bf16, lengths=None, scale=1.0, train=True):
    q, k, v, g, s0 = _tensors(arrays, bf16, train)
    lens = None if lengths is None else torch.tensor(lengths, device="cuda")
    r = linear_attention(q, k, v, g, initial=s0, lengths=lens, scale=scale)
    if not train:
        return r, None
    outs, cots = [r.output], [_device(d_out, r.output.dtype)]
    if d_state is not None:
        outs, cots = outs + [r.state], cots + [_device(d_state, torch.float32)]
    inputs = [t for t in (q, k, v, g, s0) if t is not None]
    return r, torch.autograd.grad(outs, inputs, cots)


def _compare(arrays, d_out, d_state, bf16, lengths=None, scale=1.0):
    limits = _limits(bf16)
    r, grads = _run(arrays, d_out, d_state, bf16, lengths, scale)
    out, state = oracle.attention(*arrays, lengths=lengths, scale=scale)
    want = oracle.attention_backward(*arrays[:4], d_out, d_state, arrays[4], lengths, scale)
    torch.cuda.synchronize()
    _check("output", r.output, out, limits["rows"])
    _check("state", r.state, state, limits["state"])
    for name, got, expected in zip(NAMES, grads, want):
        kind = dict(log_decay="decay", initial="state").get(name, "rows")
        _check("d_" + name, got, expected, limits[kind])
    return r, grads


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("b,t,heads,n,p,per_head,initial", [
    (1, 1, (1, 1, 1), 64, 64, False, False),
    (2, 1, (3, 3, 3), 16, 32, True, True),
    (2, 63, (2, 2, 2), 64, 64, False, True),
    (1, 64, (2, 2, 2), 64, 128, True, False),
    (1, 65, (1, 1, 1), 128, 64, False, True),
    (2, 300, (3, 3, 3), 64, 64, False, False),
    (1, 513, (2, 2, 2), 128, 128, True, True),
    (2, 130, (4, 2, 2), 64, 64, False, True),     # keys and values shared
    (2, 130, (1, 1, 6), 128, 64, False, False),   # queries and keys shared
    (1, 70, (2, 4, 1), 33, 77, True, True),       # odd widths
    (1, 200, (2, 2, 2), 7, 1, False, True),
    (1, 96, (1, 1, 1), 1, 3, False, False),
    (1, 90, (2, 2, 2), 100, 66, False, True),     # widths of two or four
])
def test_forward_and_gradients(gpu_lib, b, t, heads, n, p, per_head, initial, bf16):
    announce(f"linear attention B{b} T{t} heads {heads} N{n} P{p} bf16={bf16}")
    _compare(*_problem(b, t, heads, n, p, bf16, per_head, initial), bf16, scale=0.5)


@pytest.mark.parametrize("bf16", [False, True])
def test_rows_of_every_length(gpu_lib, bf16):
    """Rows that end anywhere in a chunk or hold nothing; what the absent rows
    hold (NaN, infinities) reaches nothing, and their gradients are zero."""
    announce(f"linear attention lengths bf16={bf16}")
    lengths = [0, 1, 64, 65, 200, 129, 7, 500]
    arrays, d_out, d_state = _problem(8, 200, (2, 2, 2), 64, 64, bf16, initial=True, seed=3)
    for i, n in enumerate(lengths):
        for a, bad in zip(arrays[:4], (np.nan, np.inf, -np.inf, np.nan)):
            a[i, n:] = bad
        d_out[i, n:] = np.nan
    clean = [np.where(np.isfinite(a), a, 0.0) for a in arrays]
    limits = _limits(bf16)
    r, grads = _run(arrays, d_out, d_state, bf16, lengths)
    d_clean = np.where(np.isfinite(d_out), d_out, 0.0)
    out, state = oracle.attention(*clean, lengths=lengths)
    want = oracle.attention_backward(*clean[:4], d_clean, d_state, clean[4], lengths)
    _check("output", r.output, out, limits["rows"])
    _check("state", r.state, state, limits["state"])
    for name, got, expected in zip(NAMES, grads, want):
        _check("d_" + name, got, expected,
               limits[dict(log_decay="decay", initial="state").get(name, "rows")])
    for i, n in enumerate(lengths):
        for got in (r.output, *grads[:4]):
            assert (got[i, n:] == 0).all()


@pytest.mark.parametrize("bf16", [False, True])
def test_resets_and_steep_decays(gpu_lib, bf16):
    """Decays of zero (minus infinity, the type's lowest value) drop the past
    exactly; steep ones leave their neighbours' weights exact."""
    announce(f"linear attention resets bf16={bf16}")
    arrays, d_out, d_state = _problem(2, 260, (2, 2, 2), 64, 64, bf16, initial=True, seed=4)
    g = arrays[3]
    g[:, 10, 0] = -np.inf
    g[:, 64, 1] = np.finfo(np.float32).min
    g[0, 100:110] = -90.0
    g[1, 128:200:3] = -1000.0
    g[:, 150:230, 1] = 0.0
    r, grads = _compare(arrays, d_out, d_state, bf16)
    assert all(torch.isfinite(t.float()).all() for t in (r.output, r.state, *grads))
    assert (grads[3][:, 10, 0] == 0).all() and (grads[3][:, 64, 1] == 0).all()
    # Nothing from before a reset: other tokens there leave the rest bit for bit.
    other = [np.array(a) for a in arrays]
    other[1][:, :10] = 1.0
    s, _ = _run(other, None, None, bf16, train=False)
    s0, _ = _run(arrays, None, None, bf16, train=False)
    assert torch.equal(s.output[:, 10:, 0], s0.output[:, 10:, 0])


@pytest.mark.parametrize("bf16", [False, True])
def test_split_and_walked_sequences_have_the_same_bits(gpu_lib, monkeypatch, bf16):
    announce(f"linear attention split/walk bf16={bf16}")
    arrays, d_out, d_state = _problem(3, 1000, (2, 1, 2), 64, 100, bf16, initial=True, seed=5)
    lengths = [1000, 257, 700]
    results = []
    for mode in ("walk", "split"):
        monkeypatch.setenv("M4RT_ATTENTION", mode)
        r, grads = _run(arrays, d_out, d_state, bf16, lengths)
        results.append([r.output, r.state, *grads])
    for i, (a, b) in enumerate(zip(*results)):
        assert torch.equal(a, b), i


@pytest.mark.parametrize("bf16", [False, True])
def test_a_rows_bits_do_not_depend_on_the_batch(gpu_lib, bf16):
    announce(f"linear attention batch invariance bf16={bf16}")
    arrays, d_out, d_state = _problem(100, 600, (2, 2, 2), 64, 64, bf16, initial=True, seed=6)
    many, many_grads = _run(arrays, d_out, d_state, bf16)
    one, one_grads = _run([a[7:8] for a in arrays], d_out[7:8], d_state[7:8], bf16)
    for a, b in zip([many.output, many.state, *many_grads], [one.output, one.state, *one_grads]):
        assert torch.equal(a[7:8], b)


def test_views_of_a_fused_projection_and_other_strides(gpu_lib):
    """Rows strided along any axis, unaligned ones and transposed ones give the
    bits of their copies."""
    announce("linear attention strides")
    torch.manual_seed(0)
    b, t, h, n, p = 2, 150, 3, 64, 64
    fused = torch.randn(b, t, h * (2 * n + p) + 1, device="cuda").to(torch.bfloat16)
    g = -torch.rand(b, t, h, device="cuda")
    for first in (0, 1):
        rows = fused[..., first:first + h * (2 * n + p)]
        q, k, v = (x.unflatten(-1, (h, -1)) for x in rows.split([h * n, h * n, h * p], dim=-1))
        want = linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), g)
        got = linear_attention(q, k, v, g)
        assert torch.equal(got.output, want.output) and torch.equal(got.state, want.state)
        swapped = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
        got = linear_attention(*swapped, g)
        assert torch.equal(got.output, want.output)
        odd = [x.transpose(-1, -2).contiguous().transpose(-1, -2) for x in (q, k, v)]
        got = linear_attention(*odd, g.expand(b, t, h))
        assert torch.equal(got.output, want.output)
    one = torch.randn(1, 1, h, n, device="cuda").to(torch.bfloat16)
    same = one.expand(b, t, h, n)
    want = linear_attention(same.contiguous(), same.contiguous(), same.contiguous(), g)
    got = linear_attention(same, same, same, g)
    assert torch.equal(got.output, want.output)


def test_gradients_against_differences(gpu_lib):
    """Directional derivatives of a float32 call by central differences: with a step
    of 2^-6 the curvature leaves about 2^-12 and the sums' rounding 2^-24 * 2^6,
    both relative to the loss's scale."""
    announce("linear attention differences")
    arrays, d_out, d_state = _problem(2, 140, (2, 2, 2), 32, 48, False, initial=True, seed=8)
    _, grads = _run(arrays, d_out, d_state, False)
    rng = np.random.default_rng(9)
    step = 2.0 ** -6

    def loss(a):
        r, _ = _run(a, None, None, False, train=False)
        return float((host(r.output) * d_out).sum() + (host(r.state) * d_state).sum())

    for i, name in enumerate(NAMES):
        direction = rng.normal(size=arrays[i].shape) * (0.05 if name == "log_decay" else 1.0)
        moved = [[a if j != i else a + s * step * direction for j, a in enumerate(arrays)]
                 for s in (1, -1)]
        want = (loss(moved[0]) - loss(moved[1])) / (2 * step)
        got = float((host(grads[i]) * direction).sum())
        scale = float(np.abs(host(grads[i]) * direction).sum())
        assert abs(got - want) <= 2e-3 * scale, name


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("b,heads,n,p,per_head", [
    (1, (1, 1, 1), 64, 64, False), (3, (4, 2, 1), 64, 128, True), (2, (3, 3, 3), 128, 128, False),
    (5, (2, 2, 2), 33, 77, False), (2, (1, 1, 4), 1, 2, True), (300, (2, 2, 2), 64, 64, False)])
def test_step(gpu_lib, b, heads, n, p, per_head, bf16):
    announce(f"linear attention step B{b} heads {heads} N{n} P{p} bf16={bf16}")
    arrays, _, _ = _problem(b, 1, heads, n, p, bf16, per_head, True, seed=11)
    state = arrays[4]
    q, k, v = (a[:, 0] for a in arrays[:3])
    g = arrays[3] if per_head else arrays[3][:, 0]
    rows = torch.bfloat16 if bf16 else torch.float32
    args = [_device(a, rows) for a in (q, k, v)] + [_device(g, torch.float32)]
    for active in (None, np.arange(b) % 3 != 1):
        want, new = oracle.attention_step(state, q, k, v, g, active, 0.25)
        on = None if active is None else torch.tensor(active, device="cuda")
        s = _device(state, torch.float32)
        kept = s.clone()
        r = linear_attention_step(s, *args, active=on, scale=0.25)
        assert torch.equal(s, kept)
        # One product and a few roundings per state element; sums of N terms.
        _check("output", r.output, want, 2.0 ** -8 if bf16 else 2e-6)
        _check("state", r.state, new, 1e-6)
        into = linear_attention_step_(s, *args, active=on, scale=0.25)
        assert into.state is s
        assert torch.equal(s, r.state) and torch.equal(into.output, r.output)
        if active is not None:
            assert torch.equal(s[~on], kept[~on]) and (r.output[~on] == 0).all()


def test_steps_follow_a_prompt(gpu_lib):
    """A prompt's state taken on token by token is the whole sequence (float32,
    both near 1e-6 of the oracle)."""
    announce("linear attention prompt + steps")
    arrays, _, _ = _problem(2, 80, (2, 2, 2), 64, 64, False, seed=12)
    q, k, v, g, _ = _tensors(arrays, False, False)
    whole = linear_attention(q, k, v, g)
    part = linear_attention(q[:, :70], k[:, :70], v[:, :70], g[:, :70])
    state = part.state
    for t in range(70, 80):
        r = linear_attention_step(state, q[:, t], k[:, t], v[:, t], g[:, t])
        state = r.state
        _check("output", r.output, host(whole.output[:, t]), 1e-5)
    _check("state", state, host(whole.state), 1e-5)


def test_differentiable_step(gpu_lib):
    announce("linear attention step gradient")
    arrays, d_out, d_state = _problem(3, 1, (2, 2, 2), 64, 64, False, initial=True, seed=13)
    q, k, v, g, s0 = _tensors(arrays, False, True)
    on = torch.tensor([True, False, True], device="cuda")
    r = linear_attention_step(s0, q[:, 0], k[:, 0], v[:, 0], g[:, 0], active=on)
    grads = torch.autograd.grad([r.output, r.state], [q, k, v, g, s0],
                                [_device(d_out[:, 0], torch.float32),
                                 _device(d_state, torch.float32)])
    want = oracle.attention_backward(*arrays[:4], d_out, d_state, arrays[4], [1, 0, 1])
    for name, got, expected in zip(NAMES, grads, want):
        _check("d_" + name, got, expected, 2e-5)


def test_mixed_and_other_dtypes_are_float32_inside(gpu_lib):
    announce("linear attention dtypes")
    torch.manual_seed(1)
    q, k, v = (torch.randn(1, 70, 2, 32, device="cuda") for _ in range(3))
    g = -torch.rand(2, device="cuda")
    want = linear_attention(q.half().float(), k.half().float(), v.half().float(), g)
    got = linear_attention(q.half(), k.half(), v.half(), g.double())
    assert got.output.dtype == torch.float16
    assert torch.equal(got.output, want.output.half()) and torch.equal(got.state, want.state)
    mixed = linear_attention(q.bfloat16(), k, v, g)
    assert mixed.output.dtype == torch.float32


def test_no_tokens_and_no_rows(gpu_lib):
    announce("linear attention of nothing")
    z = torch.zeros(2, 0, 3, 16, device="cuda")
    s0 = torch.randn(2, 3, 16, 16, device="cuda")
    r = linear_attention(z, z, z, torch.zeros(3, device="cuda"), initial=s0)
    assert r.output.shape == (2, 0, 3, 16) and torch.equal(r.state, s0)
    r = linear_attention(z, z, z, torch.zeros(2, 0, 3, device="cuda"))
    assert (r.state == 0).all() and r.state.shape == (2, 3, 16, 16)
    e = torch.zeros(0, 5, 3, 16, device="cuda")
    assert linear_attention(e, e, e, torch.zeros(3, device="cuda")).state.shape == (0, 3, 16, 16)
    s = torch.zeros(0, 3, 16, 16, device="cuda")
    r = linear_attention_step(s, e[:, 0], e[:, 0], e[:, 0], torch.zeros(3, device="cuda"))
    assert r.output.shape == (0, 3, 16)


def test_other_streams_and_graph_replays(gpu_lib):
    """Work on a side stream, and a captured call replayed between eager work,
    has the bits of the plain call."""
    announce("linear attention streams and graph")
    arrays, d_out, d_state = _problem(2, 600, (2, 2, 2), 64, 64, True, initial=True, seed=14)
    q, k, v, g, s0 = _tensors(arrays, True, False)
    want = linear_attention(q, k, v, g, initial=s0)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = linear_attention(q, k, v, g, initial=s0)
        step = linear_attention_step(got.state, q[:, 0], k[:, 0], v[:, 0], g[:, 0])
    stream.synchronize()
    assert torch.equal(got.output, want.output) and torch.equal(got.state, want.state)
    assert torch.isfinite(step.state).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        caught = linear_attention(q, k, v, g, initial=s0)
    for _ in range(3):
        caught.output.fill_(float("nan"))
        caught.state.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(caught.output, want.output) and torch.equal(caught.state, want.state)
    del graph


def test_long_sequence_offsets(gpu_lib):
    """A strided sequence whose rows lie more than 2^31 elements apart."""
    announce("linear attention long strides")
    t, stride = 4100, 1 << 19
    big = torch.empty(t * stride + 64, dtype=torch.bfloat16, device="cuda")
    rows = big.as_strided((1, t, 1, 64), (t * stride, stride, 64, 1))
    torch.manual_seed(2)
    rows.copy_(torch.randn(1, t, 1, 64, device="cuda"))
    g = torch.full((1,), -0.01, device="cuda")
    dense = rows.contiguous()
    got, want = linear_attention(rows, rows, rows, g), linear_attention(dense, dense, dense, g)
    assert torch.equal(got.output, want.output) and torch.equal(got.state, want.state)
    del big


def test_refusals(gpu_lib):
    q = torch.zeros(2, 5, 2, 16, device="cuda")
    g = torch.zeros(2, device="cuda")
    with pytest.raises(ValueError, match="ROCm device"):
        linear_attention(q.cpu(), q, q, g)
    with pytest.raises(ValueError, match="disagree"):
        linear_attention(q, q[:, :4], q, g)
    with pytest.raises(ValueError, match="width"):
        linear_attention(q, q[..., :8], q, g)
    with pytest.raises(ValueError, match="widths must be"):
        linear_attention(q, q, torch.zeros(2, 5, 2, 129, device="cuda"), g)
    with pytest.raises(ValueError, match="divide"):
        linear_attention(q, q, torch.zeros(2, 5, 3, 16, device="cuda"), g)
    with pytest.raises(ValueError, match="log_decay"):
        linear_attention(q, q, q, torch.zeros(3, device="cuda"))
    with pytest.raises(ValueError, match="initial"):
        linear_attention(q, q, q, g, initial=torch.zeros(2, 2, 16, 8, device="cuda"))
    with pytest.raises(ValueError, match="lengths"):
        linear_attention(q, q, q, g, lengths=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError, match="lengths"):
        linear_attention(q, q, q, g, lengths=torch.zeros(3, dtype=torch.int32, device="cuda"))
    s = torch.zeros(2, 2, 16, 16, device="cuda")
    with pytest.raises(ValueError, match="state"):
        linear_attention_step(s[:1], q[:, 0], q[:, 0], q[:, 0], g)
    with pytest.raises(ValueError, match="contiguous"):
        linear_attention_step_(s.transpose(-1, -2), q[:, 0], q[:, 0], q[:, 0], g)
    with pytest.raises(ValueError, match="gradient"):
        linear_attention_step_(s, q[:, 0].clone().requires_grad_(), q[:, 0], q[:, 0], g)
    with pytest.raises(ValueError, match="active"):
        linear_attention_step(s, q[:, 0], q[:, 0], q[:, 0], g, active=g)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("t", [1, 65, 300])
def test_copied_rows_have_the_bits_of_whole_ones(gpu_lib, t, bf16):
    """Rows of odd widths are copied to padded ones: the same bits as whole rows
    with zeros in their place, whatever the absent tokens hold."""
    announce(f"linear attention copied rows T{t} bf16={bf16}")
    arrays, d_out, d_state = _problem(2, t, (4, 2, 1), 64, 128, bf16, initial=True, seed=11)
    q, k, v, g, s0 = arrays
    q[..., 63], k[..., 63], v[..., 125:] = 0, 0, 0
    s0[:, :, 63], s0[..., 125:] = 0, 0
    d_out[..., 125:], d_state[:, :, 63], d_state[..., 125:] = 0, 0, 0
    lengths = [t, t // 2]
    whole, whole_grads = _run(arrays, d_out, d_state, bf16, lengths)
    for a in (q, k, v, g, d_out):
        a[1, t // 2:] = np.nan
    odd, odd_grads = _run([q[..., :63], k[..., :63], v[..., :125], g, s0[:, :, :63, :125]],
                          d_out[..., :125], d_state[:, :, :63, :125], bf16, lengths)
    assert torch.equal(odd.output, whole.output[..., :125])
    assert torch.equal(odd.state, whole.state[:, :, :63, :125])
    cuts = (np.s_[..., :63], np.s_[..., :63], np.s_[..., :125], np.s_[...],
            np.s_[:, :, :63, :125])
    for name, got, want, cut in zip(NAMES, odd_grads, whole_grads, cuts):
        assert torch.equal(got, want[cut]), name
