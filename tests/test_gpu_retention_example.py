"""The example language model on the device: it learns, its gradient is the
differences', and its tokens one by one give what the whole sequence gives."""

import importlib.util
import os

import pytest
import torch

from tests.gpu_helpers import announce

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "retention_lm.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("retention_lm", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _model(example, **kw):
    torch.manual_seed(1)
    sizes = dict(vocab=97, width=96, heads=4, layers=2, key_heads=2)
    return example.RetentionLM(**{**sizes, **kw}).to("cuda")


def _error(a, b):
    return ((a - b).double().norm() / b.double().norm()).item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_lowers_the_loss(gpu_lib, example, dtype):
    """Sequences of 16 of the 97 tokens: learning which they are takes the loss
    from ln 97 = 4.6 (and more, of random weights) below ln 32 = 3.5."""
    announce(f"retention example training {dtype}")
    model = _model(example, dtype=dtype)
    losses = example.train(model, 80, 8, 100, 16)
    assert losses[0] > 4.0
    assert sum(losses[-5:]) / 5 < 3.5


def test_directional_derivative(gpu_lib, example):
    """Along the gradient, the loss of float32 weights rises by the squared norm:
    central differences over a step of 1e-2 / norm have an error of the third
    derivative's order (1e-4 of the step) and the loss's rounding, 1e-6 / 1e-2."""
    announce("retention example derivative")
    model = _model(example)
    ids = example.chains(3, 131, 97, "cuda", torch.Generator().manual_seed(2))
    parameters = list(model.parameters())
    grads = torch.autograd.grad(model.loss(ids), parameters)
    norm = torch.sqrt(sum((g.double()**2).sum() for g in grads)).item()
    values = []
    for sign in (1, -1):
        moved = {name: p.detach() + sign * 1e-2 / norm * g
                 for (name, p), g in zip(model.named_parameters(), grads)}
        original = [p.detach().clone() for p in parameters]
        with torch.no_grad():
            for name, p in model.named_parameters():
                p.copy_(moved[name])
            values.append(model.loss(ids).item())
            for p, o in zip(parameters, original):
                p.copy_(o)
    assert abs((values[0] - values[1]) / 2e-2 - norm) < 1e-2 * norm


def test_tokens_one_by_one(gpu_lib, example):
    """Float32 throughout: each operator is within 1e-5 of the exact result, some
    twenty of them follow each other."""
    announce("retention example steps")
    model = _model(example)
    ids = torch.randint(97, (5, 140), device="cuda")
    with torch.no_grad():
        whole, states = model(ids)
        lengths = torch.tensor([1, 64, 65, 100, 130], device="cuda")
        first, mine = model(ids, lengths)
    for row, length in enumerate(lengths.tolist()):
        assert _error(first[row, :length], whole[row, :length]) < 2e-4
    at = lengths.clone()
    rows = torch.arange(5, device="cuda")
    for _ in range(139):
        active = at < 140
        logits = model.step(ids[rows, at.clamp(max=139)], mine, active)
        for row in active.nonzero().flatten().tolist():
            assert _error(logits[row], whole[row, at[row]]) < 2e-4
        at += active.long()
    for a, b in zip(mine, states):
        assert _error(a, b) < 2e-4


def test_generation_of_ragged_prompts(gpu_lib, example):
    """A prompt's continuation does not depend on the rows beside it, nor on what
    its padding holds."""
    announce("retention example generation")
    model = _model(example)
    ids = torch.randint(97, (3, 90), device="cuda")
    lengths = torch.tensor([90, 33, 7], device="cuda")
    padded = ids.clone()
    for row, length in enumerate(lengths.tolist()):
        padded[row, length:] = -1
    a = model.generate(ids, 6, lengths)
    b = model.generate(padded, 6, lengths)
    assert torch.equal(a, b)
