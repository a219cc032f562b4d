"""mxfp4 restated in 64 bits on the CPU, and the error bounds its tests use."""

import torch

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
BLOCK = 32
U32 = 2.0 ** -24  # half a step of fp32, relative
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# half a step between subnormals
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def quantize_ref(x):
    """(code magnitudes and signs as values / scale, bytes, values) of [.., K], float64."""
    v = x.detach().cpu().double().unflatten(-1, (-1, BLOCK))
    top = v.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(v).all(-1, keepdim=True)
    _, e = torch.frexp(torch.where(torch.isfinite(top), top, torch.ones_like(top)))
    e = torch.where(top > 0, e.double() - 3, torch.full_like(top, -127.0)).clamp(-127, 127)
    a = torch.where(bad, torch.zeros_like(v), v.abs()) / torch.pow(2.0, e)
    d = (a.unsqueeze(-1) - VALUES).abs()
    d = d * 16 + torch.arange(8, dtype=torch.float64) % 2 * 1e-9  # ties: the even code
    value = VALUES[d.argmin(-1)]
    out = torch.copysign(value, v) * torch.pow(2.0, e)
    out = torch.where(bad, torch.full_like(out, float("nan")), out)
    byte = torch.where(bad, torch.full_like(e, 255.0), e + 127).squeeze(-1).to(torch.uint8)
    return out.flatten(-2), byte


def dequantize_ref(w, s):
    q = (w.detach().cpu().to(torch.int64).unsqueeze(-1) >> torch.arange(0, 32, 4)) & 15
    v = VALUES[q & 7] * (1.0 - 2.0 * (q >> 3))
    s = s.detach().cpu().double()
    scale = torch.where(s == 255, torch.full_like(s, float("nan")), torch.pow(2.0, s - 127))
    return (v.flatten(-2).unflatten(-1, (-1, BLOCK)) * scale.unsqueeze(-1)).flatten(-2)


def codes(gen, *shape, lo=116, hi=124):
    """Random codes and scale bytes of weights [.., N, K], on the CPU."""
    K = shape[-1]
    w = torch.randint(-(1 << 31), 1 << 31, (*shape[:-1], K // 8), generator=gen, dtype=torch.int64).to(torch.int32)
    s = torch.randint(lo, hi, (*shape[:-1], K // BLOCK), generator=gen, dtype=torch.int64).to(torch.uint8)
    return w, s


def check_sum(got, ref, mag, terms, what=""):
    """``got`` is a sum of ``terms`` fp32 products rounded once to its type:
    |got - ref| <= half a step of the result + terms * 2^-24 * sum |products|
    (the fp32 roundings of a sum of that many terms in any order, first order;
    the 8 added to terms covers the rounding of the products and of ref's own)."""
    dt = got.dtype
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    err = (got - ref).abs()
    acc = (terms + 8) * U32 * mag
    tol = acc + (ref.abs() + acc) * HALF[dt] + TINY[dt]
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan), (what, "NaN elsewhere")
    bad = (err > tol) & ~nan
    assert not bad.any(), (what, int(bad.sum()), float((err / tol)[~nan].max()))
