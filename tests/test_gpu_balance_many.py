"""The balance loss over very many tokens."""

import pytest
import torch

from titan_amd import ops

BF = torch.bfloat16
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1 << 20, (1 << 22) + 777])
@pytest.mark.parametrize("E", [60, 132, 200])
@pytest.mark.parametrize("masked", [False, True])
def test_equal_logits(dev, T, E, masked):
    """Equal probabilities all round to one side where they are added up: loss = E sum_e f_e / E = 1 however ids fall."""
    mask = torch.rand(T, device=dev, generator=torch.Generator(device=dev).manual_seed(1)) < 0.9 if masked else None
    ids = torch.arange(T, device=dev, dtype=torch.int32).reshape(T, 1) % 7
    loss, counts = ops.router_balance_loss(torch.zeros(T, E, dtype=BF, device=dev), ids, mask)
    live = torch.ones(T, device=dev) if mask is None else mask.float()
    assert torch.equal(counts[:7].double(), torch.stack([live[e::7].double().sum() for e in range(7)])) and not counts[7:].any()
    # in half steps of 2^-24: the division 2, its product with the exponential 1, sums of at most 16 rows of a lane 15, a
    # lane's sum 1, 16 lanes 4, 16 waves 15, the result 1.  Everything between is added in 64 bits.
    assert abs(loss.item() - 1.0) <= 39 * 2.0 ** -24, loss.item()
