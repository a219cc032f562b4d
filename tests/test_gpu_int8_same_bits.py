"""Calls that share the work out differently and still give the same bits."""

import int8_oracle as o
import pytest
import torch

from titan_amd import ops
from titan_amd.switch_layers import QuantizedSwitchLinear, SwitchGLU

BF, HF, F4 = o.BF, o.HF, o.F4
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, HF, F4])
@pytest.mark.parametrize("D", [300, 1024, 2048, 5000])
def test_norm_of_a_row_alone_and_among_others(dev, D, dtype):
    """x and residual are multiples of 1/16 below 8, so that their sum is one below 16 and exact in every type (8 bits),
    its square a multiple of 2^-8 below 2^8, and the sum of up to 5000 of these below 2^21: exact in 64 bits in any
    order.  What follows goes element by element."""
    g = torch.Generator().manual_seed(D)
    x, r = (torch.randint(-127, 128, (3000, D), generator=g).float().div(16).to(dev, dtype) for _ in range(2))
    x[:, 0], r[:, 0] = 0.0, 0.0625
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(dev, dtype)
    got = ops.rms_norm_quantize(x, w, residual=r, norm=True)
    for rows in ([0], [1], [1500], [2999], list(range(40, 240)), list(range(1000, 2100))):
        one = ops.rms_norm_quantize(x[rows], w, residual=r[rows], norm=True)
        for a, b in zip(got, one):
            assert torch.equal(a[rows], b)
    alone = ops.rms_norm_quantize(x[7], w, residual=r[7], norm=True)  # one dimension
    assert all(torch.equal(a[7], b) for a, b in zip(got, alone))


@pytest.mark.parametrize("T,k", [(5, 4), (40, 4)])
def test_layer_whatever_its_ids_type(dev, T, k):
    E, H, I = 11, 144, 80
    g = torch.Generator().manual_seed(T)
    gate_up, down = (QuantizedSwitchLinear(*(t.to(dev) for t in o.quantize(torch.randn(s, generator=g) / s[-1] ** 0.5)), mode="int8")
                     for s in ((E, 2 * I, H), (E, H, I)))
    x, ids = torch.randn(T, H, generator=g).to(dev, BF), torch.randint(0, E, (T, k), generator=g).to(dev)
    glu = SwitchGLU(down, gate_up_proj=gate_up)
    want = glu(x, ids)
    assert torch.isfinite(want).all() and torch.equal(glu(x, ids.int()), want)
