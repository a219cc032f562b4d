"""What has to see an operation and cannot see a kernel's launch is refused by the
mxfp4 and token-sort binding, on the CPU: before it looks at the tensors."""

import pytest
import torch
from torch.autograd import forward_ad

from titan_amd import _lib
from titan_amd.ops import QmoeUnsupported

BF = torch.bfloat16


def _w(*shape):
    return torch.zeros(*shape[:-1], shape[-1] // 8, dtype=torch.int32), torch.zeros(*shape[:-1], shape[-1] // 32, dtype=torch.uint8)


def test_a_tangent_of_quantised_rows():
    """gather_qqmm's rows, as the Python path brings them: int64 indices, several rows a batch, a caller's table."""
    B = _lib.binding()
    w, s = _w(2, 8, 32)
    x = torch.ones(3, 32, dtype=BF)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for qq in (True, False):
            with pytest.raises(NotImplementedError, match="forward"):
                B.rows_product(d, w, s, None, 1, None, None, 3, True, qq)


def test_a_gradient_of_quantised_rows():
    B = _lib.binding()
    w, s = _w(2, 8, 32)
    x = torch.ones(3, 32, dtype=BF, requires_grad=True)
    with pytest.raises(QmoeUnsupported, match="gradient"):
        B.rows_product(x, w, s, None, 1, None, None, 3, True, True)
