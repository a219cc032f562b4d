"""Tokens sorted by expert and back, with the router's scores applied, and the
gradients of both (titan/adapters/mlx/vendor/mlx_lm/models/switch_layers.py:13-25,
titan/kernels/moe_weighted_sum.py:44-98; the reference has no gradients).

Pair ``p = t * k + j`` is slot j of token t.  ``order`` (the pair of each sorted
row) and ``inv_order`` (the sorted row of each pair) are inverse permutations of
the T * k pairs, as :func:`titan_amd.ops.route` gives them.  Rows are bf16, fp16
or fp32, of any length; sums run in fp32 in slot order and are rounded once, so
results repeat bit for bit.  Where they are not inverse permutations, rows that no
pair is sent to stay as their memory was; nothing is read or written out of bounds.
Forward-mode tangents, torch.jit.trace and make_fx are refused.

The calls and their autograd nodes are csrc/torch/binding.cpp's.  It takes what
the kernels can read as it is; the functions here check, convert or refuse the
rest.
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
    return ops._ready(t.reshape(-1).to(torch.int32))


def sort_tokens(x: torch.Tensor, order: torch.Tensor, inv_order: torch.Tensor) -> torch.Tensor:
    """x [T, D] -> [T * k, D], row i the token of pair ``order[i]``: each token's
    row is written to its k places ``inv_order``, and its gradient is the sum over
    them."""
    y = _lib.binding().sort_tokens(x, order, inv_order, False)
    if y is not None:
        return y
    x = _rows(x, "x")
    order = _pairs(order, "order", x.device)
    n, T = order.numel(), x.shape[0]
    if n % T if T else n:
        raise ValueError(f"order holds {n} pairs, not a multiple of x's {T} rows")
    return _lib.binding().sort_tokens(x, order, _pairs(inv_order, "inv_order", x.device, n), True)


def unsort_tokens(xs: torch.Tensor, order: torch.Tensor, inv_order: torch.Tensor,
                  scores: torch.Tensor | None = None) -> torch.Tensor:
    """Sorted rows xs [T * k, D] back to their tokens: y [T, D] =
    sum_j scores[t, j] * xs[inv_order[t k + j]].  ``scores`` [T, k] are taken in
    fp32; None: the rows alone, [T * k, D] in pair order.  Gradients go to xs and
    scores."""
    if scores is None:
        y = _lib.binding().sort_tokens(xs, inv_order, order, False)
    else:
        y = _lib.binding().unsort_tokens(xs, order, inv_order, scores, False)
    if y is not None and (scores is not None or y.shape == xs.shape):
        return y
    xs = _rows(xs, "xs")
    n = xs.shape[0]
    inv = _pairs(inv_order, "inv_order", xs.device, n)
    order = _pairs(order, "order", xs.device, n)
    if scores is None:
        return _lib.binding().sort_tokens(xs, inv, order, True)
    ops._dev(scores, "scores")
    ops._same_device(scores, "scores", xs.device)
    if scores.dim() != 2 or scores.numel() != n:
        raise ValueError(f"scores must be [T, k] with T * k = {n}, got {tuple(scores.shape)}")
    return _lib.binding().unsort_tokens(xs, order, inv, ops._ready(scores.to(torch.float32)), True)
