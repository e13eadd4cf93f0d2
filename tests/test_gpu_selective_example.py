"""The selective language model of examples/, the operators as they are used together:
its logits and gradients are those of the same model of plain float64 operators, its
tokens one by one give what the whole sequence gives, and a decode step replays from a
graph.

Tolerances (2-norms of differences over those of the values): float32 products of up to
256 terms are off by about 16 2^-24 = 1e-6 of their terms; two layers with norms that
divide by a deviation and gates multiply that a few times over, and gradients pass
through both again: 1e-4.
"""

import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

from tests.gpu_helpers import announce

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "selective_lm.py")
LIMIT = 1e-4


def _load():
    spec = importlib.util.spec_from_file_location("selective_lm", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.fixture(scope="module")
def example():
    return _load()


def _plain_embedding(ids, table, scale=1.0, dtype=None):
    return table[ids] * scale


def _plain_rms_norm(x, weight, residual):
    s = x + residual
    return s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5) * weight, s


def _plain_conv(x, weight, bias, activation, lengths=None):
    taps = weight.shape[1]
    rows = torch.cat([x.new_zeros(x.shape[0], taps - 1, x.shape[2]), x], 1)
    z = bias + sum(rows[:, j:j + x.shape[1]] * weight[:, j] for j in range(taps))
    return F.silu(z), None


def _plain_scan(x, delta, a, b, c, skip, gate, delta_bias, softplus, lengths=None):
    each = x.shape[2] // b.shape[2]
    step = F.softplus(delta + delta_bias)
    h = x.new_zeros(x.shape[0], *a.shape)
    out = []
    for t in range(x.shape[1]):
        bt, ct = (m[:, t].repeat_interleave(each, 1) for m in (b, c))
        h = torch.exp(step[:, t, :, None] * a) * h + (step[:, t] * x[:, t])[..., None] * bt
        out.append((h * ct).sum(-1) + skip * x[:, t])
    return torch.stack(out, 1) * F.silu(gate), None


def _model(module, dtype=torch.float32, **kw):
    torch.manual_seed(1)
    sizes = dict(vocab=64, width=64, layers=2, states=16, groups=2)
    return module.SelectiveLM(dtype=dtype, **{**sizes, **kw})


def _error(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return ((a - b).norm() / b.norm()).item()


@pytest.mark.parametrize("states,groups", [(16, 2), (5, 1)])
def test_logits_and_gradients_are_the_plain_models(gpu_lib, example, states, groups):
    announce(f"selective example N{states} G{groups}")
    plain = _load()
    plain.embedding, plain.rms_norm = _plain_embedding, _plain_rms_norm
    plain.causal_conv, plain.selective_scan = _plain_conv, _plain_scan
    model = _model(example, states=states, groups=groups).to("cuda")
    twin = _model(plain, dtype=torch.float64, states=states, groups=groups).double()
    twin.load_state_dict({k: v.double().cpu() for k, v in model.state_dict().items()})
    ids, asked = example.pairs(3, 48, 64, 6, "cpu", torch.Generator().manual_seed(2))
    want = plain.SelectiveLM._logits
    plain.SelectiveLM._logits = lambda self, h, s: F.linear(
        _plain_rms_norm(h, self.norm, s)[0], self.table)
    try:
        logits, _ = twin(ids)
        loss = twin.loss(ids, asked)
    finally:
        plain.SelectiveLM._logits = want
    loss.backward()
    got, _ = model(ids.to("cuda"))
    mine = model.loss(ids.to("cuda"), asked.to("cuda"))
    mine.backward()
    assert _error(got, logits) <= LIMIT and abs(mine.item() - loss.item()) <= LIMIT * loss.item()
    for (name, p), q in zip(model.named_parameters(), twin.parameters()):
        assert _error(p.grad, q.grad) <= LIMIT, name


@pytest.mark.parametrize("dtype,limit", [(torch.float32, LIMIT), (torch.bfloat16, 4e-2)])
def test_tokens_one_by_one_are_the_sequence(gpu_lib, example, dtype, limit):
    """(bfloat16: about ten roundings of 2^-9 a layer, of values that both ways round at
    the same places but sum in other orders before.)"""
    announce(f"selective example steps {dtype}")
    model = _model(example, dtype=dtype).to("cuda")
    ids, _ = example.pairs(4, 60, 64, 6, "cuda", torch.Generator().manual_seed(3))
    with torch.no_grad():
        whole, last = model(ids)
        logits, states = model(ids[:, :37])
        assert _error(logits, whole[:, :37]) <= limit
        for t in range(37, 60):
            assert _error(model.step(ids[:, t], states), whole[:, t]) <= limit, t
    for (rows, state), (rows2, state2) in zip(states, last):
        assert _error(rows, rows2) <= limit and _error(state, state2) <= limit


def test_prompts_of_several_lengths(gpu_lib, example):
    """Padded prompts continue as each alone does, and rows that are not active keep
    their states."""
    announce("selective example lengths")
    model = _model(example).to("cuda")
    ids, _ = example.pairs(3, 40, 64, 6, "cuda", torch.Generator().manual_seed(4))
    lengths = torch.tensor([40, 11, 1], device="cuda")
    padded = torch.where(torch.arange(40, device="cuda") < lengths[:, None], ids, -1)
    together = model.generate(padded, 5, lengths)
    for i, n in enumerate(lengths.tolist()):
        assert torch.equal(together[i:i + 1], model.generate(ids[i:i + 1, :n], 5)), i
    with torch.no_grad():
        _, states = model(padded, lengths)
        before = [(r.clone(), s.clone()) for r, s in states]
        active = torch.tensor([True, False, True], device="cuda")
        model.step(ids[:, 0], states, active)
    for (r, s), (r0, s0) in zip(states, before):
        assert torch.equal(r[1], r0[1]) and torch.equal(s[1], s0[1])
        assert not torch.equal(r[0], r0[0]) and not torch.equal(s[2], s0[2])


def test_a_decode_step_replays(gpu_lib, example):
    announce("selective example graph")
    model = _model(example, dtype=torch.bfloat16).to("cuda")
    ids, _ = example.pairs(4, 24, 64, 6, "cuda", torch.Generator().manual_seed(5))
    with torch.no_grad():
        _, states = model(ids[:, :10])
        eager = [(r.clone(), s.clone()) for r, s in states]
        token = ids[:, 10].clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            model.step(token, [(r.clone(), s.clone()) for r, s in states])
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = model.step(token, states)
        for t in range(10, 24):
            token.copy_(ids[:, t])
            graph.replay()
            want = model.step(ids[:, t], eager)
            torch.cuda.synchronize()
            assert torch.equal(logits, want), t
    del graph


def test_a_training_step_replays_beside_an_eager_one(gpu_lib, example):
    """Forward and backward captured while no eager graph of the parameters lives, then
    replayed beside eager passes: the same gradients every time."""
    announce("selective example training graph")
    model = _model(example, dtype=torch.bfloat16).to("cuda")
    ids, asked = example.pairs(2, 33, 64, 6, "cuda", torch.Generator().manual_seed(6))
    parameters = list(model.parameters())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(model.loss(ids, asked), parameters)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, _ = model(ids[:, :-1])
        got = torch.autograd.grad(logits, parameters, torch.ones_like(logits))
        logits = logits.detach()
    for _ in range(3):
        graph.replay()
        logits2, _ = model(ids[:, :-1])
        want = torch.autograd.grad(logits2, parameters, torch.ones_like(logits2))
        torch.cuda.synchronize()
        assert torch.equal(logits, logits2)
        for (name, _), u, v in zip(model.named_parameters(), got, want):
            # (The library's own products may choose others in a capture.)
            assert _error(u, v) <= 1e-2, name
        del logits2, want
    del graph


def test_the_example_runs(gpu_lib, example):
    announce("selective example training")
    model = _model(example, dtype=torch.bfloat16).to("cuda")
    losses = example.train(model, 3, 4, 32, 64, 6)
    assert len(losses) == 3 and all(x == x and x < 100 for x in losses)
