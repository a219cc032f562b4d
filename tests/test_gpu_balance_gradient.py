"""The balance loss's gradient against differences of the loss in 64 bits, as near as its fp32 allows."""

import int8_oracle as o
import pytest
import torch

from titan_amd import ops

pytestmark = pytest.mark.gpu


def test_gradient_against_differences(dev):
    g = torch.Generator().manual_seed(7)
    logits = torch.randn(6, 10, generator=g)
    ids = torch.topk(logits + torch.randn(6, 10, generator=g), 2, -1).indices
    mask = torch.tensor([True, True, False, True, True, False])
    leaf = logits.to(dev).requires_grad_(True)
    ops.router_balance_loss(leaf, ids.to(dev), mask.to(dev))[0].backward()
    size = o.balance(logits, ids, mask)[3]
    h = 1e-5
    for t in range(6):
        for e in range(10):
            up, down = logits.double(), logits.double()
            up[t, e] += h
            down[t, e] -= h
            want = (o.balance(up, ids, mask)[0] - o.balance(down, ids, mask)[0]) / (2 * h)
            # differences: h^2 / 6 of the third derivative (at most 10, the largest loss: 1.7e-10) and 2 x 40 roundings to
            # 64 bits of a loss of at most 10 over 2 h (4.4e-9).  The gradient's fp32: p off by twice (2 * 10 + 28) half
            # steps of 2^-24 (logits within 10 of each other: two halves of that in the exponent, 28 for exponential, sum
            # and division), 40 more for f, the dot and the products, of E / n p (f + dot).
            tol = 5e-9 + size[t, e].item() * (2 * (2 * 10 + 28) + 40) * 2.0 ** -24
            assert abs(leaf.grad[t, e].item() - want) <= tol, (t, e)
