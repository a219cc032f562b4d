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


def _calls():
    B = _lib.binding()
    x, od, (w, s) = torch.zeros(4, 64, dtype=BF), torch.arange(4, dtype=torch.int32), _w(5, 64)
    return [lambda v: B.quantize(v, False), lambda v: B.dequantize(w, s, 0, False), lambda v: B.sort_tokens(v, od, od, False),
            lambda v: B.unsort_tokens(v, od, od, torch.ones(4, 1), False), lambda v: B.matmul(v, w, s, True, False, False),
            lambda v: B.gather(v, w[None], s[None], None, od, True, True, False),
            lambda v: B.rows_product(v, w[None], s[None], None, 1, None, None, 4, True, False)], x


@pytest.mark.parametrize("i", range(7))
def test_recorders(i):
    """A recorded call would hold the result's allocation and no kernel."""
    from torch.fx.experimental.proxy_tensor import make_fx

    calls, x = _calls()
    refusals = []

    def call(v):
        with pytest.raises(QmoeUnsupported, match="record"):
            calls[i](v)
        refusals.append(i)
        return v + 1

    torch.jit.trace(call, (x,), check_trace=False)
    make_fx(call)(x)
    assert refusals == [i, i]
