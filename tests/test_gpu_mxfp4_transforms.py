"""Function transforms and tracing over the mxfp4 operators and the token sort on
the GPU: refused or served by the stock path, never lost."""

import pytest
import torch
from torch.autograd import forward_ad

from mx_helpers import codes
from titan_amd import ops
from titan_amd.ops import QmoeUnsupported

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def say(*a):
    print("[mxfp4 transforms]", *a, flush=True)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_gather_qqmm_refuses_forward_mode(dev, dtype):
    """Whichever way the rows reach the kernels."""
    say("forward mode", dtype)
    w, s = (t.to(dev) for t in codes(torch.Generator().manual_seed(1), 2, 8, 32))
    ids = torch.tensor([0, 0, 1], device=dev).to(dtype)
    tiles = ops.build_tiles(ids, 2)
    x = torch.ones(3, 1, 32, dtype=BF, device=dev)
    with forward_ad.dual_level():
        for v in (x, torch.ones(3, 2, 32, dtype=BF, device=dev), torch.ones(32, 1, 3, dtype=BF, device=dev).transpose(0, 2)):
            d = forward_ad.make_dual(v, torch.ones_like(v))
            for kw in ({}, {"sorted_indices": True}, {"lhs_indices": ids}) + (({"sorted_indices": True, "tiles": tiles},) if v.shape[1] == 1 else ()):
                for op in (ops.gather_qqmm, ops.gather_qmm):
                    with pytest.raises(NotImplementedError, match="forward"):
                        op(d, w, s, rhs_indices=ids, mode="mxfp4", **kw)


def test_gather_qqmm_refuses_a_gradient(dev):
    say("gradient")
    w, s = (t.to(dev) for t in codes(torch.Generator().manual_seed(1), 2, 8, 32))
    ids = torch.tensor([0, 0, 1], device=dev)
    x = torch.ones(3, 2, 32, dtype=BF, device=dev, requires_grad=True)
    with pytest.raises(QmoeUnsupported, match="gradient"):
        ops.gather_qqmm(x, w, s, rhs_indices=ids)
