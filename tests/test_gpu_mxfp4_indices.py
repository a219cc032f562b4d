"""Indices outside their range in the mxfp4 gather calls, on the GPU: clamped, few
rows and many, forward and backward, whatever brings them."""

import pytest
import torch

from mx_helpers import check_sum, codes, dequantize_ref, quantize_ref
from titan_amd import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def say(*a):
    print("[mxfp4 indices]", *a, flush=True)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _by_expert(x, W, e):
    """x [n, M, C] times W[e] [C, O], and the sum of magnitudes, in 64 bits on the CPU."""
    x, V = x.detach().cpu().double(), W[e]
    return x @ V, x.abs() @ V.abs()


@pytest.mark.parametrize("is_sorted", [False, True])
@pytest.mark.parametrize("M,n", [(2, 5), (2, 50), (40, 7)])
def test_batches_of_several_rows(dev, M, n, is_sorted):
    say("batches", M, n, is_sorted)
    g = _gen(M + n)
    B, E, K, N = 6, 4, 64, 40
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s).transpose(1, 2)
    e = torch.randint(-2, E + 2, (n,), generator=g)
    e = torch.sort(e)[0] if is_sorted else e
    lhs = torch.randint(-3, B + 3, (n,), generator=g)
    lhs[:2] = torch.tensor([-1, B])
    x = torch.randn(B, M, K, generator=g).to(BF)
    xi, ei = lhs.clamp(0, B - 1), e.clamp(0, E - 1)
    xd = x.to(dev).requires_grad_(True)
    kw = {"lhs_indices": lhs.to(dev), "rhs_indices": e.to(dev), "sorted_indices": is_sorted}
    y = ops.gather_qmm(xd, w.to(dev), s.to(dev), mode="mxfp4", **kw)
    check_sum(y, *_by_expert(x[xi], W, ei), K)
    q = ops.gather_qqmm(xd.detach(), w.to(dev), s.to(dev), **kw)
    check_sum(q, *_by_expert(quantize_ref(x)[0][xi], W, ei), K)
    dy = torch.randn(n, M, N, generator=g).to(BF)
    (dx,) = torch.autograd.grad(y, xd, dy.to(dev))
    ref, mag = _by_expert(dy, W.transpose(1, 2), ei)
    zero = torch.zeros(B, M, K, dtype=torch.float64)
    check_sum(dx, zero.index_add(0, xi, ref), zero.index_add(0, xi, mag), N + n)


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32, torch.uint64])
@pytest.mark.parametrize("n", [5, 90])
def test_past_32_bits(dev, n, dtype):
    say("past 32 bits", n, dtype)
    g = _gen(n)
    E, K, N = 4, 64, 40
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s).transpose(1, 2)
    x = torch.randn(n, 1, K, generator=g).to(BF)
    far = (1 << 31) + 1 if dtype == torch.uint32 else (1 << 32) + 1
    e = torch.sort(torch.randint(0, E, (n,), generator=g))[0]
    lhs = torch.randint(0, n, (n,), generator=g)
    e[-2:] = far
    lhs[1] = far
    xi, ei = lhs.clamp(0, n - 1), e.clamp(0, E - 1)
    for is_sorted in (True, False):
        kw = {"lhs_indices": lhs.to(dtype).to(dev), "rhs_indices": e.to(dtype).to(dev), "sorted_indices": is_sorted}
        check_sum(ops.gather_qmm(x.to(dev), w.to(dev), s.to(dev), mode="mxfp4", **kw), *_by_expert(x[xi], W, ei), K)
        check_sum(ops.gather_qqmm(x.to(dev), w.to(dev), s.to(dev), **kw), *_by_expert(quantize_ref(x)[0][xi], W, ei), K)
