"""The 8-bit operators and the balance loss under vmap and torch.func: whichever
operand a transform has wrapped, the call is refused in words, and it computes
nothing from what the wrapper hides."""

import int8_oracle as o
import pytest
import torch

from titan_amd import ops

BF = o.BF
pytestmark = pytest.mark.gpu


def _calls(dev):
    """(call, the operand to wrap)"""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 64, generator=g).to(dev, BF)
    (w, sw), (q, s) = (tuple(t.to(dev) for t in o.quantize(torch.randn(n, 64, generator=g))) for n in (5, 4))
    e, se, ids = w[None].repeat(3, 1, 1), sw[None].repeat(3, 1), torch.zeros(4, dtype=torch.int32, device=dev)
    many = torch.zeros(80, dtype=torch.int32, device=dev)
    logits, top, mask = torch.randn(6, 8, generator=g).to(dev), torch.zeros(6, 2, dtype=torch.int32, device=dev), torch.ones(6, dtype=torch.bool, device=dev)
    gather = lambda v, i, rows=None, srt=False: ops.gather_qqmm(v, e, se, lhs_indices=rows, rhs_indices=i, mode="int8", sorted_indices=srt)  # noqa: E731
    return [(lambda v: ops.quantize(v, mode="int8"), x), (lambda v: ops.dequantize(v, s, mode="int8"), q),
            (lambda v: ops.dequantize(q, v, mode="int8"), s), (lambda v: ops.rms_norm_quantize(v, None), x),
            (lambda v: ops.rms_norm_quantize(x, v), x[0].clone()), (lambda v: ops.rms_norm_quantize(x, None, residual=v), x),
            (lambda v: ops.qqmm(v, w, sw, mode="int8"), x), (lambda v: ops.qqmm((v, s), w, sw, mode="int8"), q),
            (lambda v: ops.qqmm((q, v), w, sw, mode="int8"), s), (lambda v: ops.qqmm(x, v, sw, mode="int8"), w),
            (lambda v: ops.qqmm(x, w, v, mode="int8"), sw), (lambda v: gather(v, ids), x.unsqueeze(1)),
            (lambda v: gather(x.unsqueeze(1), v), ids), (lambda v: gather(x.unsqueeze(1), many, v, True), many),
            (lambda v: ops.router_balance_loss(v, top, mask), logits), (lambda v: ops.router_balance_loss(logits, v), top),
            (lambda v: ops.router_balance_loss(logits, top, v), mask)]


@pytest.mark.parametrize("i", range(17))
def test_transforms(dev, i):
    calls = _calls(dev)
    assert len(calls) == 17
    call, t = calls[i]
    call(t)
    refused = []

    def f(v):
        with pytest.raises(ops.QmoeUnsupported, match="vmap"):
            call(v)
        refused.append(i)
        return v.float().sum()

    torch.func.vmap(f)(t.unsqueeze(0))
    if t.is_floating_point():
        torch.func.grad(f)(t)
    assert refused == [i] * (2 if t.is_floating_point() else 1)


def test_calls_inside_a_transform(dev):
    """Operands that vmap has not wrapped: the results of the call outside of it."""
    for call, t in _calls(dev):
        want, seen = call(t), []
        torch.func.vmap(lambda v: seen.append(call(t)) or v)(torch.zeros(2, 3, device=dev))
        for a, b in zip(*(r if isinstance(r, tuple) else (r,) for r in (want, seen[0]))):
            assert (a is None and b is None) or torch.equal(a, b)
