"""Tensors wrapped by a function transform have no memory that a kernel could read:
the binding refuses them in those words, on the CPU before it looks at anything else."""

import pytest
import torch

from titan_amd import _lib
from titan_amd.ops import QmoeUnsupported

BF = torch.bfloat16


def _calls():
    """(call, a tensor to wrap): the operands that each function looks at first."""
    B = _lib.binding()
    x, w, od = torch.zeros(4, 64, dtype=BF), torch.zeros(5, 64, dtype=torch.int8), torch.zeros(4, dtype=torch.int32)
    q, s, sw, ids = x.to(torch.int8), torch.ones(4), torch.ones(5), torch.zeros(4, 2, dtype=torch.int32)
    return [(lambda v: B.int8_quantize(v, False), x), (lambda v: B.int8_dequantize(q, v, 0, False), s),
            (lambda v: B.rms_norm_quantize(v, None, 1e-6, None, False, False), x),
            (lambda v: B.int8_matmul(v, None, w, sw, -1, False), x),
            (lambda v: B.int8_gather(v, None, w[None], sw[None], None, od, True, -1, None), x),
            (lambda v: B.int8_rows_product(v, None, w[None], sw[None], None, 1, None, None, 4, -1), x),
            (lambda v: B.router_balance(v, ids, None, False), x),
            (lambda v: B.quantize(v, False), x), (lambda v: B.sort_tokens(v, od, od, False), x)]


@pytest.mark.parametrize("i", range(len(_calls())))
def test_transforms(i):
    call, t = _calls()[i]
    refused = []

    def f(v):
        with pytest.raises(QmoeUnsupported, match="vmap"):
            call(v)
        refused.append(i)
        return v.float().sum()

    torch.func.vmap(f)(t.unsqueeze(0))
    torch.func.grad(f)(t.float())
    assert refused == [i, i]


def test_calls_inside_a_transform():
    """What a transform does not wrap goes through as outside of it: here as far as the check for GPU memory."""
    call, t = _calls()[0]
    seen = []
    torch.func.vmap(lambda v: seen.append(call(t)) or v)(torch.zeros(2, 3))
    assert seen == [None]
