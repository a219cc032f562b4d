"""Microscaled 4-bit floating point: the ``mode="mxfp4"`` of the quantized
matmuls (mx.quantize, mx.dequantize, mx.quantized_matmul, mx.gather_qmm,
mx.qqmm; reached through :mod:`titan_amd.ops`).

Weights are codes [.., N, K/8] (int32 or uint32 words, eight e2m1 codes each,
low bits first) and scales uint8 [.., N, K/32], 2^(byte - 127) per block of 32
along K (OCP Microscaling Formats v1.0); there are no biases.  Activations are
bf16, products and sums fp32, results bf16.

The products are differentiable in x: with ``transpose`` (x W^T) dx = dy W, and
without (x W) dx = dy W^T, by the same kernels over the same codes.  The codes
and scales are constants of the graph.  ``qqmm`` and ``gather_qqmm`` quantise x
as well and have no gradient.  Forward-mode tangents, torch.jit.trace and
make_fx are refused.

The calls and their autograd nodes are csrc/torch/binding.cpp's.  It takes what
the kernels can read as it is; the functions here check, convert, arrange or
refuse the rest.
"""

from __future__ import annotations

import math

import torch

from . import _lib, ops
from ._lib import QmoeUnsupported

__all__ = ["BLOCK", "quantize", "dequantize", "quantized_matmul", "gather_qmm", "qqmm", "gather_qqmm"]

BLOCK = 32
# gathered rows from which the grouped GEMM runs, unsorted calls sorted for it (the binding has the same)
SORTED_MIN_ROWS = 64


def _format(group_size: int | None, bits: int, biases=None) -> None:
    if group_size not in (None, BLOCK) or bits != 4:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"mxfp4 has group_size 32 and 4 bits, got {group_size} and {bits}")
    if biases is not None:
        raise ValueError("mxfp4 weights have no biases")


def _scales(t: torch.Tensor, device) -> torch.Tensor:
    ops._dev(t, "scales")
    ops._same_device(t, "scales", device)
    if t.dtype != torch.uint8:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"mxfp4 scales must be uint8, got {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


def _weights(w: torch.Tensor, scales: torch.Tensor, device, dims: int):
    """Checked codes and scales, and their [(E,) N, K]."""
    w = ops._words(w, "w")
    ops._same_device(w, "w", device)
    scales = _scales(scales, device)
    if w.dim() != dims:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"w must have {dims} dimensions, got {tuple(w.shape)}")
    K = w.shape[-1] * 8
    if K % BLOCK or tuple(scales.shape) != (*w.shape[:-1], K // BLOCK):
        raise ValueError(f"codes {tuple(w.shape)} and scales {tuple(scales.shape)} disagree")
    return w, scales, w.shape[-2], K


# ------------------------------------------------------------ quantisation


def quantize(w: torch.Tensor, group_size: int | None = None, bits: int = 4, mode: str = "mxfp4"):
    """(codes int32 [.., K/8], scales uint8 [.., K/32]) of bf16, fp16 or fp32
    values [.., K], K a multiple of 32: scale 2^(floor(log2 max|w|) - 2) per
    block, elements to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the
    even code, larger ones to 6); a block with a NaN or an infinity reads back
    as NaN."""
    if mode != "mxfp4":
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"mode={mode!r}: quantize makes mxfp4")
    _format(group_size, bits)
    q = _lib.binding().quantize(w, False)
    if q is not None:
        return q
    ops._dev(w, "w")
    if w.dtype not in ops._DTYPES:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"w must be bfloat16, float16 or float32, got {w.dtype}")
    if w.dim() < 1 or w.shape[-1] % BLOCK:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"the last dimension must be a multiple of 32, got {tuple(w.shape)}")
    return _lib.binding().quantize(ops._ready(w), True)


def dequantize(w: torch.Tensor, scales: torch.Tensor, biases=None, group_size: int | None = None, bits: int = 4,
               dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [.., K] of codes [.., K/8], exact in bf16 and fp32 (but for
    magnitudes past the type's range, which become infinite), rounded in fp16."""
    _format(group_size, bits, biases)
    if dtype not in ops._DTYPES:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"dtype={dtype}: bfloat16, float16 or float32")
    out = _lib.binding().dequantize(w, scales, ops._DTYPES[dtype], False)
    if out is not None:
        return out
    w = ops._words(w, "w")
    scales = _scales(scales, w.device)
    K = w.shape[-1] * 8 if w.dim() else 0
    if w.dim() < 1 or K % BLOCK or tuple(scales.shape) != (*w.shape[:-1], K // BLOCK):
        raise ValueError(f"codes {tuple(w.shape)} and scales {tuple(scales.shape)} disagree")
    return _lib.binding().dequantize(w, scales, ops._DTYPES[dtype], True)


# --------------------------------------------------------------- products


class _Rows:
    """Which activation row and which expert each output row takes: ``x_rows``
    (or row i // div), ``experts``, and the tile table of sorted rows (None: not
    sorted).  With ``inv``, ``x_rows`` is the sorted form of row i // div, whose
    rows are at ``inv[i]``."""

    __slots__ = ("n", "x_rows", "div", "experts", "tiles", "inv")

    def __init__(self, n, x_rows=None, div=1, experts=None, tiles=None, inv=None):
        self.n, self.x_rows, self.div, self.experts, self.tiles, self.inv = n, x_rows, div, experts, tiles, inv


def _product(x, w, scales, transpose, rows: _Rows, qq: bool = False):
    """out[r] = x[row of r] W[expert of r]^T (transpose) or W, rows as ``rows``
    says, recorded where a gradient of x may be asked for; ``qq``: x in mxfp4."""
    t = rows.tiles
    table = None if t is None else (t.offsets, t.tile_row, t.tile_exp, t.ntiles, t.maxt)
    return _lib.binding().rows_product(x, w, scales, rows.x_rows, rows.div, rows.experts, table, rows.n, bool(transpose), qq,
                                        rows.inv)


def _x_rows(rows: _Rows, device):
    """The activation row of each row, None for row r itself."""
    if rows.x_rows is not None or rows.div == 1:
        return rows.x_rows
    return torch.div(torch.arange(rows.n, device=device, dtype=torch.int32), rows.div,
                     rounding_mode="floor").to(torch.int32)


def quantized_matmul(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases=None, transpose: bool = True,
                     group_size: int | None = None, bits: int = 4) -> torch.Tensor:
    """x [.., K] W^T (transpose) or x [.., N] W for codes w [N, K/8]."""
    _format(group_size, bits, biases)
    y = _lib.binding().matmul(x, w, scales, bool(transpose), False, False)
    if y is not None:
        return y
    x = ops._bf16(x, "x")
    w, scales, N, K = _weights(w, scales, x.device, 2)
    if x.dim() < 1 or x.shape[-1] != (K if transpose else N):
        raise ValueError(f"x {tuple(x.shape)} does not fit w [{N}, {K}] with transpose={transpose}")
    return _lib.binding().matmul(x, w, scales, bool(transpose), False, True)


def _broadcast(a, b) -> tuple:
    """torch.broadcast_shapes of two shapes, without its overhead."""
    a, b = tuple(a), tuple(b)
    a, b = (1,) * (len(b) - len(a)) + a, (1,) * (len(a) - len(b)) + b
    if any(i != j and i != 1 and j != 1 for i, j in zip(a, b)):
        raise ValueError(f"batches {a} and {b} do not broadcast")
    return tuple(j if i == 1 else i for i, j in zip(a, b))


def _flat(t, batch, n):
    """Indices into ``n`` over the batch as a contiguous int32 vector."""
    t = ops._narrow(t, n)
    if t.shape != batch:
        t = t.expand(batch)
    return ops._ready(t if t.dim() == 1 else t.reshape(-1))


def _gathered(x, E, lhs, rhs, sorted_indices, tiles, min_rows):
    """(batch, rows, order): the broadcast batch of a gather call over x
    [.., M, C], its output rows in the order they are computed in, and that
    order with its inverse (None: the batch's own).  ``min_rows`` rows or more
    are sorted and get a tile table."""
    dev = x.device
    M, xb = x.shape[-2], x.shape[:-2]
    if rhs is None:
        rhs = torch.arange(E, device=dev, dtype=torch.int32)
    else:
        ops._dev(rhs, "rhs_indices")
        ops._same_device(rhs, "rhs_indices", dev)
    x_rows, div = None, 1
    if lhs is None:
        batch = rhs.shape if xb == rhs.shape else torch.Size(_broadcast(xb, rhs.shape))
        nb = math.prod(batch)
        if xb != batch:
            nx = math.prod(xb)
            # batch index i reads x's batch index i // (nb / nx) where only x's last dimensions are broadcast
            lead = (1,) * (len(batch) - len(xb)) + tuple(xb)
            cut = len(batch)
            while cut and lead[cut - 1] == 1:
                cut -= 1
            if lead[:cut] == tuple(batch[:cut]):
                div = nb // nx if nx else 1
            else:
                x_rows = torch.arange(nx, device=dev, dtype=torch.int32).reshape(lead).expand(batch).reshape(-1)
    else:
        ops._dev(lhs, "lhs_indices")
        ops._same_device(lhs, "lhs_indices", dev)
        batch = lhs.shape if lhs.shape == rhs.shape else torch.Size(_broadcast(lhs.shape, rhs.shape))
        nb = math.prod(batch)
        x_rows = _flat(lhs, batch, math.prod(xb))
    experts = _flat(rhs, batch, E)
    if M != 1 and nb:  # rows of one batch index: M activation rows, one expert
        ar = torch.arange(M, device=dev, dtype=torch.int32)
        if lhs is not None:  # clamped here as a batch: the kernels clamp each of its rows
            x_rows = x_rows.clamp(0, max(math.prod(xb) - 1, 0))
        base = x_rows if x_rows is not None else None if div == 1 else _x_rows(_Rows(nb, None, div), dev)
        x_rows = None if base is None else (base[:, None] * M + ar).reshape(-1)
        div = 1
        experts = experts.repeat_interleave(M)
    n, order, known = nb * M, None, None
    if n and (E == 0 or math.prod(x.shape[:-1]) == 0):
        raise ValueError("rows are asked for, but there are no experts or no activation rows")
    if n >= min_rows:
        if sorted_indices:
            if tiles is None or tiles.rows != n:
                tiles = ops.build_tiles(experts, E)
            elif tiles.num_experts != E or tiles.tile_rows != ops.tile_rows():
                raise ValueError("tile table does not match this call")
        else:
            r = ops.route(experts, E)
            order, inv, tiles = r.order, r.inv_order, r.tiles
            experts = r.sorted_ids
            if x_rows is None:
                known = inv
                x_rows = order if div == 1 else torch.div(order, div, rounding_mode="floor")
            else:
                x_rows = x_rows[order.long()]
                div = 1
            order = order, inv
    else:
        tiles = None
    return batch, _Rows(n, x_rows, div, experts, tiles, known), order


def _check_gather(x, w, scales, transpose, lhs, rhs):
    w, scales, N, K = _weights(w, scales, x.device, 3)
    if x.dim() < 2:
        raise ValueError("x must be at least 2-D ([..., M, K])")
    if x.shape[-1] != (K if transpose else N):
        raise ValueError(f"x {tuple(x.shape)} does not fit w [{w.shape[0]}, {N}, {K}] with transpose={transpose}")
    for name, t in (("lhs_indices", lhs), ("rhs_indices", rhs)):
        if t is not None and (not isinstance(t, torch.Tensor) or t.is_floating_point() or t.dtype == torch.bool):
            raise TypeError(f"{name} must be an integer tensor")
    return w, scales, w.shape[0], N, K


def _rows_of(x):
    """x as [rows, C]."""
    return x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), x.shape[-1])


def gather_qmm(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases=None, lhs_indices=None,
               rhs_indices=None, transpose: bool = True, group_size: int | None = None, bits: int = 4,
               sorted_indices: bool = False, tiles=None) -> torch.Tensor:
    """:func:`titan_amd.ops.gather_qmm` for codes w [E, N, K/8]: x [.., M, K]
    times W^T, or x [.., M, N] times W without ``transpose``.  From 64 rows on
    the rows run through the grouped GEMM: as they are with ``sorted_indices``
    (ascending ``rhs_indices``), else sorted by expert first.  Indices outside
    their range are clamped into it.  ``tiles``: the table of sorted rows
    (:func:`titan_amd.ops.build_tiles` of ``rhs_indices``, or the routing's), which
    then says what expert a row takes."""
    _format(group_size, bits, biases)
    if tiles is None:
        y = _lib.binding().gather(x, w, scales, lhs_indices, rhs_indices, bool(transpose), bool(sorted_indices), False)
        if y is not None:
            return y
    x = ops._bf16(x, "x")
    w, scales, E, N, K = _check_gather(x, w, scales, transpose, lhs_indices, rhs_indices)
    batch, rows, order = _gathered(x, E, lhs_indices, rhs_indices, sorted_indices, tiles, SORTED_MIN_ROWS)
    y = _product(_rows_of(x), w, scales, transpose, rows)
    if order is not None:
        y = ops.sort_tokens(y, order[1], order[0])
    return y.reshape(batch + (x.shape[-2], y.shape[-1]))


def _no_grad(x: torch.Tensor) -> None:
    if x.requires_grad and torch.is_grad_enabled():
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, "the products of quantised activations have no gradient: "
                                                    "detach x, or use quantized_matmul / gather_qmm")


def qqmm(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, group_size: int | None = None, bits: int = 4,
         mode: str = "mxfp4") -> torch.Tensor:
    """x [.., K], quantised to mxfp4 as :func:`quantize` does, times W^T for
    codes w [N, K/8], both operands on the 4-bit matrix instructions (mx.qqmm)."""
    if mode != "mxfp4":
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"mode={mode!r}: only mxfp4")
    _format(group_size, bits)
    y = _lib.binding().matmul(x, w, scales, True, True, False)
    if y is not None:
        return y
    x = ops._bf16(x, "x")
    _no_grad(x)
    w, scales, N, K = _weights(w, scales, x.device, 2)
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"x {tuple(x.shape)} does not fit w [{N}, {K}]")
    return _lib.binding().matmul(x, w, scales, True, True, True)


def gather_qqmm(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, lhs_indices=None, rhs_indices=None,
                group_size: int | None = None, bits: int = 4, mode: str = "mxfp4", sorted_indices: bool = False,
                tiles=None) -> torch.Tensor:
    """:func:`gather_qmm` (transpose) with x quantised as in :func:`qqmm`, each
    activation row once however many experts take it.  Takes the grouped
    kernel's rows at any count: unsorted calls are sorted first."""
    if mode != "mxfp4":
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"mode={mode!r}: only mxfp4")
    _format(group_size, bits)
    if tiles is None:
        y = _lib.binding().gather(x, w, scales, lhs_indices, rhs_indices, True, bool(sorted_indices), True)
        if y is not None:
            return y
    x = ops._bf16(x, "x")
    _no_grad(x)
    w, scales, E, N, K = _check_gather(x, w, scales, True, lhs_indices, rhs_indices)
    batch, rows, order = _gathered(x, E, lhs_indices, rhs_indices, sorted_indices, tiles, 1)
    y = _product(_rows_of(x), w, scales, True, rows, qq=True)
    if order is not None:
        y = ops.sort_tokens(y, order[1], order[0])
    return y.reshape(batch + (x.shape[-2], N))
