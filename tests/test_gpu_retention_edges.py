"""Arguments at the edges of what the retention operators take."""

import pytest
import torch

from mamba4_amd import linear_attention
from tests.gpu_helpers import announce

pytestmark = pytest.mark.gpu


def _normal(*shape):
    return torch.randn(*shape, device="cuda")


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.uint16,
                                   torch.int32, torch.uint32, torch.int64])
def test_lengths_of_every_integer_type(gpu_lib, dtype):
    """Sequences longer than the type's largest value among them."""
    announce(f"lengths {dtype}")
    time = {torch.uint8: 300, torch.int8: 200, torch.int16: 33000}.get(dtype, 70)
    q, v = _normal(3, time, 1, 8), _normal(3, time, 1, 8)
    g = torch.full((1,), -0.1, device="cuda")
    values = [0, 7, 66]
    got = linear_attention(q, q, v, g, lengths=torch.tensor(values, dtype=dtype).cuda())
    want = linear_attention(q, q, v, g, lengths=torch.tensor(values, device="cuda"))
    assert torch.equal(got.output, want.output) and torch.equal(got.state, want.state)
