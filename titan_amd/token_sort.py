"""Tokens sorted by expert and back, with the router's scores applied, and the
gradients of both (titan/adapters/mlx/vendor/mlx_lm/models/switch_layers.py:13-25,
titan/kernels/moe_weighted_sum.py:44-98; the reference has no gradients).

Pair ``p = t * k + j`` is slot j of token t.  ``order`` (the pair of each sorted
row) and ``inv_order`` (the sorted row of each pair) are inverse permutations of
the T * k pairs, as :func:`titan_amd.ops.route` gives them.  Rows are bf16, fp16
or fp32, of any length; sums run in fp32 in slot order and are rounded once, so
results repeat bit for bit.
"""

from __future__ import annotations

import torch

from . import _lib, ops
from ._lib import QmoeUnsupported

__all__ = ["sort_tokens", "unsort_tokens"]


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    ops._dev(t, name)
    if t.dtype not in ops._DTYPES:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be [rows, D], got {tuple(t.shape)}")
    return ops._ready(t)


def _pairs(t: torch.Tensor, name: str, device, n: int | None = None) -> torch.Tensor:
    ops._dev(t, name)
    ops._same_device(t, name, device)
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    if n is not None and t.numel() != n:
        raise ValueError(f"{name} holds {t.numel()} pairs, not {n}")
    t = t if t.dtype == torch.int32 else t.to(torch.int32)
    return ops._ready(t if t.dim() == 1 else t.reshape(-1))


def unsort_sum(rows: torch.Tensor, inv: torch.Tensor | None, scores: torch.Tensor | None, T: int, k: int,
               first: torch.Tensor | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
    """sum_j scores[t, j] * rows[inv[t k + j]] (:func:`unsort_tokens` without its
    checks and gradient); ``first`` [T + 1] gives each output its own pairs."""
    y = torch.empty(T, rows.shape[1], dtype=dtype or rows.dtype, device=rows.device)
    ops._launch("qmoe_unsort_sum", rows, rows.data_ptr(), rows.shape[0], ops._DTYPES[rows.dtype], ops._ptr(inv), ops._ptr(scores),
            ops._ptr(first), T, k, rows.shape[1], ops._DTYPES[y.dtype], y.data_ptr())
    return y


def _sort_rows(x, order):
    n, (T, D) = order.numel(), x.shape
    xs = torch.empty(n, D, dtype=x.dtype, device=x.device)
    ops._launch("qmoe_sort_rows", x, x.data_ptr(), T, order.data_ptr(), n // T if T else 0, D, ops._DTYPES[x.dtype],
                xs.data_ptr())
    return xs


class _Sort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order, inv):
        ctx.save_for_backward(inv)
        ctx.T = x.shape[0]
        return _sort_rows(x, order)

    @staticmethod
    @ops._first_order
    def backward(ctx, dxs):
        (inv,), T = ctx.saved_tensors, ctx.T
        return unsort_sum(ops._ready(dxs), inv, None, T, dxs.shape[0] // T if T else 0), None, None


def _sort(x, order, inv):
    return _Sort.apply(x, order, inv) if ops._records(x) else _sort_rows(x, order)


class _Unsort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, xs, inv, scores):
        T, k = scores.shape
        ctx.save_for_backward(xs if ctx.needs_input_grad[2] else None, inv, scores)
        ctx.like = xs.shape, xs.dtype
        return unsort_sum(xs, inv, scores, T, k)

    @staticmethod
    @ops._first_order
    def backward(ctx, dy):
        xs, inv, scores = ctx.saved_tensors
        (n, D), dtype = ctx.like
        T, k = scores.shape
        dy = ops._ready(dy)
        dxs = torch.empty(n, D, dtype=dtype, device=dy.device) if ctx.needs_input_grad[0] else None
        ds = torch.empty(T, k, dtype=torch.float32, device=dy.device) if ctx.needs_input_grad[2] else None
        ops._launch("qmoe_unsort_grad", dy, dy.data_ptr(), ops._ptr(xs), n, ops._DTYPES[dtype], inv.data_ptr(), scores.data_ptr(),
                T, k, D, ops._ptr(dxs), ops._ptr(ds))
        return dxs, None, ds


def sort_tokens(x: torch.Tensor, order: torch.Tensor, inv_order: torch.Tensor) -> torch.Tensor:
    """x [T, D] -> [T * k, D], row i the token of pair ``order[i]``; the gradient
    of a token is the sum over its k rows, formed from ``inv_order``."""
    x = _rows(x, "x")
    order = _pairs(order, "order", x.device)
    n, T = order.numel(), x.shape[0]
    if n % T if T else n:
        raise ValueError(f"order holds {n} pairs, not a multiple of x's {T} rows")
    return _sort(x, order, _pairs(inv_order, "inv_order", x.device, n))


def unsort_tokens(xs: torch.Tensor, order: torch.Tensor, inv_order: torch.Tensor,
                  scores: torch.Tensor | None = None) -> torch.Tensor:
    """Sorted rows xs [T * k, D] back to their tokens: y [T, D] =
    sum_j scores[t, j] * xs[inv_order[t k + j]].  ``scores`` [T, k] are taken in
    fp32; None: the rows alone, [T * k, D] in pair order.  Gradients go to xs and
    scores."""
    xs = _rows(xs, "xs")
    n = xs.shape[0]
    inv = _pairs(inv_order, "inv_order", xs.device, n)
    order = _pairs(order, "order", xs.device, n)
    if scores is None:
        return _sort(xs, inv, order)
    ops._dev(scores, "scores")
    ops._same_device(scores, "scores", xs.device)
    if scores.dim() != 2 or scores.numel() != n:
        raise ValueError(f"scores must be [T, k] with T * k = {n}, got {tuple(scores.shape)}")
    scores = ops._ready(scores if scores.dtype == torch.float32 else scores.to(torch.float32))
    if ops._records(xs) or ops._records(scores):
        return _Unsort.apply(xs, inv, scores)
    return unsort_sum(xs, inv, scores, *scores.shape)
