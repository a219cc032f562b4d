"""Both operands in 8-bit integers: the ``mode="int8"`` of quantize, dequantize,
qqmm and gather_qqmm, and the RMS norm that leaves its result in that form
(reached through :mod:`titan_amd.ops`; an extension, the reference has int8
activations against int4 weights only, titan/kernels/moe_gather_int8.py).

A row has codes int8 [.., K] and one float32 scale [..]: activations by token,
weights [N, K] or [E, N, K] by output channel.  scale = max|v| / 127, codes =
rint(v / scale), as :func:`titan_amd.ops.quantize_act_int8` has them; a row of
zeros has scale 0, a row with a NaN or an infinity scale NaN, so that all that
is computed from it is NaN.  Products are summed exactly in 32-bit integers
(K up to 131,056), scaled in fp32 and rounded once to the result's type.

Nothing here has a gradient: both operands are rounded.  The norm, the products
and dequantize refuse operands that ask for one; quantize takes them, and what it
returns asks for none, as if its operand had been detached.  Forward-mode
tangents, function transforms (vmap, torch.func), torch.jit.trace and make_fx are
refused.

The calls are csrc/torch/binding.cpp's.  It takes what the kernels can read as
it is; the functions here check, convert, arrange or refuse the rest.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib, mxfp4, ops
from ._lib import QmoeUnsupported

__all__ = ["Normed", "quantize", "dequantize", "rms_norm_quantize", "qqmm", "gather_qqmm"]

MAX_K = 131056


class Normed(NamedTuple):
    """What :func:`rms_norm_quantize` leaves; qqmm and gather_qqmm take it as their x."""

    codes: torch.Tensor        # int8 [.., D]
    scales: torch.Tensor       # float32 [..]
    sum: torch.Tensor | None   # x + residual; None without a residual
    norm: torch.Tensor | None  # the norm itself; None unless asked for


def _format(group_size: int | None, bits: int | None) -> None:
    if group_size is not None or bits not in (None, 8):
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"int8 has one scale per row and 8 bits, got group_size "
                                                    f"{group_size} and {bits} bits")


def _values(t: torch.Tensor, name: str) -> torch.Tensor:
    ops._dev(t, name)
    if t.dtype not in ops._DTYPES:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if t.dim() < 1:
        raise ValueError(f"{name} must have at least one dimension")
    return ops._ready(t.resolve_neg())


def _codes(t: torch.Tensor, name: str) -> torch.Tensor:
    ops._dev(t, name)
    if t.dtype != torch.int8:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"{name} must be int8, got {t.dtype}")
    if t.dim() < 1:
        raise ValueError(f"{name} must have at least one dimension")
    return ops._ready(t.resolve_neg())


def _row_scales(t: torch.Tensor, name: str, codes: torch.Tensor) -> torch.Tensor:
    ops._dev(t, name)
    ops._same_device(t, name, codes.device)
    if t.dtype != torch.float32:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"{name} must be float32, got {t.dtype}")
    if t.shape != codes.shape[:-1]:
        raise ValueError(f"codes {tuple(codes.shape)} and {name} {tuple(t.shape)} disagree")
    _no_grad(t, name)
    return t.resolve_neg().contiguous()


def _no_grad(t: torch.Tensor, name: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"what is rounded to 8 bits has no gradient: detach {name}")


# ------------------------------------------------------------ quantisation


def quantize(w: torch.Tensor, group_size: int | None = None, bits: int | None = None):
    """(codes int8 [.., K], scales float32 [..]) of bf16, fp16 or fp32 rows of any length."""
    _format(group_size, bits)
    q = _lib.binding().int8_quantize(w, False)
    return q if q is not None else _lib.binding().int8_quantize(_values(w, "w"), True)


def dequantize(w: torch.Tensor, scales: torch.Tensor, biases=None, group_size: int | None = None,
               bits: int | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [.., K] of codes and their rows' scales, rounded to ``dtype``."""
    _format(group_size, bits)
    if biases is not None:
        raise ValueError("int8 rows have no biases")
    if dtype not in ops._DTYPES:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"dtype={dtype}: bfloat16, float16 or float32")
    out = _lib.binding().int8_dequantize(w, scales, ops._DTYPES[dtype], False)
    if out is not None:
        return out
    w = _codes(w, "w")
    return _lib.binding().int8_dequantize(w, _row_scales(scales, "scales", w), ops._DTYPES[dtype], True)


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor | None, eps: float = 1e-6,
                      residual: torch.Tensor | None = None, norm: bool = False) -> Normed:
    """The RMS norm of h = x + residual over the last dimension, quantised:
    v = h / sqrt(mean(h^2) + eps) * weight in fp32, and the codes and scales of
    its rows.  x and residual are bf16, fp16 or fp32 [.., D], h is rounded to
    their type; weight [D] is of that type or fp32 (None: ones).  ``sum`` is h,
    the residual of the next layer; ``norm`` (asked for) v in x's type, for what
    reads the norm besides, such as a router."""
    eps = float(eps)
    if not 0.0 <= eps <= 1e30:
        raise ValueError(f"eps={eps}")
    norm = bool(norm)
    got = _lib.binding().rms_norm_quantize(x, weight, eps, residual, norm, False)
    if got is not None:
        return Normed(*got)
    x = _values(x, "x")
    _no_grad(x, "x")
    if weight is not None:
        _no_grad(weight, "weight")
        ops._same_device(weight, "weight", x.device)
        if weight.shape != x.shape[-1:]:
            raise ValueError(f"weight {tuple(weight.shape)} does not fit x {tuple(x.shape)}")
        weight = _values(weight, "weight")
        if weight.dtype != x.dtype:
            weight = weight.float()
    if residual is not None:
        _no_grad(residual, "residual")
        ops._same_device(residual, "residual", x.device)
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} is not x's {tuple(x.shape)} {x.dtype}")
        residual = _values(residual, "residual")
    return Normed(*_lib.binding().rms_norm_quantize(x, weight, eps, residual, norm, True))


# --------------------------------------------------------------- products


def _acts(x):
    """(values, None) or (codes, scales) of an x as the products take it."""
    if isinstance(x, torch.Tensor):
        return x, None
    if isinstance(x, Normed):
        x = x[:2]
    if isinstance(x, (tuple, list)) and len(x) == 2 and isinstance(x[0], torch.Tensor):
        return x
    raise TypeError("x must be a tensor, a pair of codes and scales, or what rms_norm_quantize returns")


def _checked(x, sx, w, scales, dims: int):
    """x, its scales, w and its scales as the kernels read them, K padded to their 16."""
    if sx is None:
        x = _values(x, "x")
        _no_grad(x, "x")
    else:
        x = _codes(x, "x")
        sx = _row_scales(sx, "x's scales", x)
    w = _codes(w, "w")
    ops._same_device(w, "w", x.device)
    if w.dim() != dims:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"w must have {dims} dimensions, got {tuple(w.shape)}")
    scales = _row_scales(scales, "scales", w)
    K = w.shape[-1]
    if x.shape[-1] != K:
        raise ValueError(f"x {tuple(x.shape)} does not fit w {tuple(w.shape)}")
    if K > MAX_K:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"K={K}: at most {MAX_K}")
    if K % 16:
        if sx is None:
            x, sx = quantize(x)
        x, w = (torch.nn.functional.pad(t, (0, -K % 16)) for t in (x, w))
    return x, sx, w, scales


def _type(dtype: torch.dtype | None) -> int:
    """The binding's number for a result's type: -1 for that of x (bf16 for codes)."""
    if dtype is None:
        return -1
    if dtype not in ops._DTYPES:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"dtype={dtype}: bfloat16, float16 or float32")
    return ops._DTYPES[dtype]


def qqmm(x, w: torch.Tensor, scales: torch.Tensor, group_size: int | None = None, bits: int | None = None,
         dtype: torch.dtype | None = None) -> torch.Tensor:
    """x [.., K] W^T for codes w [N, K] and their channels' scales [N].  x is a
    bf16, fp16 or fp32 tensor, quantised by row here as :func:`quantize` does, a
    pair of codes and scales, or a :class:`Normed`.  The result is of ``dtype``:
    by default x's own type, bf16 for codes.  Where K is no multiple of 16 both
    operands' codes are copied into rows that are, on every call."""
    _format(group_size, bits)
    x, sx = _acts(x)
    t = _type(dtype)
    y = _lib.binding().int8_matmul(x, sx, w, scales, t, False)
    if y is not None:
        return y
    own = x.dtype
    x, sx, w, scales = _checked(x, sx, w, scales, 2)
    return _lib.binding().int8_matmul(x, sx, w, scales, ops._DTYPES.get(own, 0) if t < 0 else t, True)


def gather_qqmm(x, w: torch.Tensor, scales: torch.Tensor, lhs_indices=None, rhs_indices=None,
                group_size: int | None = None, bits: int | None = None, sorted_indices: bool = False, tiles=None,
                dtype: torch.dtype | None = None) -> torch.Tensor:
    """:func:`titan_amd.ops.gather_qmm`'s gathered product, x [.., M, K] as in
    :func:`qqmm` (each activation row is quantised once however many experts take
    it) times W^T for codes w [E, N, K] and scales [E, N].  From 64 rows on the
    rows run through the grouped GEMM: as they are with ``sorted_indices``
    (ascending ``rhs_indices``), else sorted by expert first.  Indices outside
    their range are clamped into it.  ``tiles``: the table of sorted rows
    (:func:`titan_amd.ops.build_tiles` of ``rhs_indices``, or the routing's), which
    then says what expert a row takes."""
    _format(group_size, bits)
    x, sx = _acts(x)
    t = _type(dtype)
    table = None if tiles is None else (tiles.offsets, tiles.tile_row, tiles.tile_exp, tiles.ntiles, tiles.maxt)
    if tiles is None or (isinstance(rhs_indices, torch.Tensor) and tiles.rows == rhs_indices.numel() and
                         isinstance(w, torch.Tensor) and w.dim() == 3 and tiles.num_experts == w.shape[0] and
                         tiles.tile_rows == ops.tile_rows()):
        y = _lib.binding().int8_gather(x, sx, w, scales, lhs_indices, rhs_indices, bool(sorted_indices), t, table)
        if y is not None:
            return y
    own = x.dtype
    if x.dim() < 2:
        raise ValueError("x must be at least 2-D ([..., M, K])")
    x, sx, w, scales = _checked(x, sx, w, scales, 3)
    for name, i in (("lhs_indices", lhs_indices), ("rhs_indices", rhs_indices)):
        if i is not None and (not isinstance(i, torch.Tensor) or i.is_floating_point() or i.dtype == torch.bool):
            raise TypeError(f"{name} must be an integer tensor")
    batch, rows, order = mxfp4._gathered(x, w.shape[0], lhs_indices, rhs_indices, sorted_indices, tiles,
                                         mxfp4.SORTED_MIN_ROWS)
    r = rows.tiles
    table = None if r is None else (r.offsets, r.tile_row, r.tile_exp, r.ntiles, r.maxt)
    n_x = math.prod(x.shape[:-1])
    y = _lib.binding().int8_rows_product(x.reshape(n_x, x.shape[-1]), None if sx is None else sx.reshape(n_x), w, scales,
                                         rows.x_rows, rows.div, rows.experts, table, rows.n,
                                         ops._DTYPES.get(own, 0) if t < 0 else t)
    if order is not None:
        y = ops.sort_tokens(y, order[1], order[0])
    return y.reshape(batch + (x.shape[-2], w.shape[-2]))
