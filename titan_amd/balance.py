"""The router's balance loss, with its gradient, and the experts' counts (reached
through :mod:`titan_amd.ops`; an extension, the reference only serves).

The call and its autograd node are csrc/torch/binding.cpp's.  It takes what the
kernels can read as it is; the function here checks, converts or refuses the
rest.
"""

from __future__ import annotations

import torch

from . import _lib, ops
from ._lib import QmoeUnsupported

__all__ = ["router_balance_loss"]


def router_balance_loss(logits: torch.Tensor, ids: torch.Tensor, mask: torch.Tensor | None = None):
    """(loss, counts) of router logits [.., E] (bf16, fp16 or fp32) and the chosen
    experts ids [.., k] (int32 or int64, clamped into range):

        loss = E * sum_e  counts[e] / (n k) * mean_t softmax(logits[t])[e]

    over the n tokens whose ``mask`` [..] (bool) is true, all of them without one;
    1 where the experts are used evenly, 0 where no token counts.  loss is
    float32, counts int32 [E] the pairs of those tokens routed to each expert, as
    a Routing's offsets have them.  A row of -inf counts as probabilities of zero.

    The gradient goes to the logits, the counts being constants; it is exactly 0
    for masked tokens, whatever they hold.  It is not differentiable again;
    forward-mode tangents, function transforms (vmap, torch.func), torch.jit.trace
    and make_fx are refused.  Sums over tokens go in a fixed order: results repeat
    bit for bit.  E is at most 1024.
    """
    got = _lib.binding().router_balance(logits, ids, mask, False)
    if got is not None:
        return got
    ops._dev(logits, "logits")
    if logits.dtype not in ops._DTYPES:
        raise QmoeUnsupported(_lib.ERR_UNSUPPORTED, f"logits must be bfloat16, float16 or float32, got {logits.dtype}")
    ops._dev(ids, "ids")
    ops._same_device(ids, "ids", logits.device)
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    if logits.dim() < 1 or ids.dim() != logits.dim() or ids.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"ids {tuple(ids.shape)} do not fit logits {tuple(logits.shape)}")
    if mask is not None:
        ops._dev(mask, "mask")
        ops._same_device(mask, "mask", logits.device)
        if mask.dtype != torch.bool or mask.shape != logits.shape[:-1]:
            raise ValueError(f"mask must be bool {tuple(logits.shape[:-1])}, got {mask.dtype} {tuple(mask.shape)}")
        mask = mask.contiguous()
    return _lib.binding().router_balance(ops._ready(logits.resolve_neg()), ops._ready(ids), mask, True)
