"""Function transforms and tracing over the mxfp4 operators and the token sort on
the GPU: refused or served by the stock path, never lost."""

import pytest
import torch
from torch.autograd import forward_ad

from mx_helpers import check_sum, codes, dequantize_ref
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


def test_recorders(dev):
    """Under torch.jit.trace and make_fx the operators refuse; under the overlay the stock path is recorded."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from titan_amd import core, patches

    say("recorders")
    g = torch.Generator().manual_seed(2)
    w, s = (t.to(dev) for t in codes(g, 40, 64))
    ids, od = torch.zeros(5, dtype=torch.int32, device=dev), torch.arange(5, dtype=torch.int32, device=dev)
    x, other = torch.randn(2, 5, 64, generator=g).to(BF).to(dev)
    table = ops.build_tiles(ids, 1)
    for f in (lambda v: ops.quantized_matmul(v, w, s, mode="mxfp4"), lambda v: ops.qqmm(v, w, s),
              lambda v: ops.gather_qmm(v.unsqueeze(1), w[None], s[None], rhs_indices=ids, mode="mxfp4"),
              lambda v: ops.gather_qqmm(v.unsqueeze(1), w[None], s[None], rhs_indices=ids),
              lambda v: ops.gather_qqmm(v.unsqueeze(1), w[None], s[None], rhs_indices=ids, sorted_indices=True, tiles=table),
              lambda v: ops.quantize(v)[0], lambda v: ops.dequantize(w, s, mode="mxfp4") + v[0, 0],
              lambda v: ops.sort_tokens(v, od, od), lambda v: ops.unsort_tokens(v, od, od),
              lambda v: ops.unsort_tokens(v, od, od, torch.ones(5, 1, device=dev))):
        with pytest.raises(QmoeUnsupported, match="record"):
            torch.jit.trace(f, (x,), check_trace=False)
        with pytest.raises(QmoeUnsupported, match="record"):
            make_fx(f)(x)
    W, v = dequantize_ref(w, s).t(), other.cpu().double()
    want = v @ W, v.abs() @ W.abs()
    patches.install()
    try:
        for f in (lambda v: core.quantized_matmul(v, w, s, mode="mxfp4"),
                  lambda v: core.gather_qmm(v.unsqueeze(1), w[None], s[None], rhs_indices=ids, mode="mxfp4").squeeze(1)):
            traced = torch.jit.trace(f, (x,), check_trace=False)
            for got in (traced(other), f(other)):
                check_sum(got, *want, 64)
    finally:
        patches.uninstall()
