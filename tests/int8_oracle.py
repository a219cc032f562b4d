"""The 8-bit rows, products and balance loss restated on the CPU, from their definitions."""

import torch

BF, HF, F4 = torch.bfloat16, torch.float16, torch.float32
UNIT = {BF: 2.0 ** -8, HF: 2.0 ** -11, F4: 2.0 ** -24}  # half a step, relative
TINY = {BF: 2.0 ** -134, HF: 2.0 ** -25, F4: 2.0 ** -150}  # half of the least value, where a result is subnormal


def quantize(v):
    """Codes int8 and scales float32 of float32 rows (CPU division is correctly rounded)."""
    s = v.abs().amax(-1) / torch.tensor(127.0) if v.shape[-1] else torch.zeros(v.shape[:-1])
    bad = ~torch.isfinite(v).all(-1)
    s = torch.where(bad, torch.tensor(float("nan")), s)
    q = torch.where((s > 0).unsqueeze(-1), torch.round(v / s.unsqueeze(-1)).clamp(-127, 127), torch.tensor(0.0))
    return q.to(torch.int8), s


def rms_norm(x, w, eps, r=None):
    """(h in x's type, the norm in 64 bits)."""
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    d = h.double()
    v = d / torch.sqrt(d.square().mean(-1, keepdim=True) + eps)
    return h, v if w is None else v * w.double()


def product(q, s, w, sw):
    """[rows, N] in 64 bits of codes and scales; the integer sums are exact there."""
    return (q.double() @ w.double().t()) * s.double().unsqueeze(-1) * sw.double()


def assert_rounded(got, want, roundings=3, what=""):
    """got within one rounding to its type and ``roundings`` to fp32 of want, NaN and infinities alike."""
    got64, want = got.detach().cpu().double(), want.cpu()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got64), nan), what
    tol = want.abs() * (UNIT[got.dtype] + roundings * 2.0 ** -24) * (1 + 2.0 ** -7) + TINY[got.dtype]
    top = torch.finfo(got.dtype).max
    over = want.abs() > top * (1 - UNIT[got.dtype])  # near or past the largest value: it or an infinity
    ok = (got64 - want).abs() <= tol
    ok |= nan | (over & (got64.sign() == want.sign()) & (got64.abs() >= top * (1 - 2 * UNIT[got.dtype])))
    assert bool(ok.all()), (what, got64[~ok][:4], want[~ok][:4])


def balance(logits, ids, mask=None, g=1.0):
    """(loss, counts, dlogits) in 64 bits, and sum_e f_e p_te with p for the gradient's bound."""
    E, k = logits.shape[-1], ids.shape[-1]
    x, i = logits.double().reshape(-1, E), ids.reshape(-1, k).long().clamp(0, E - 1)
    live = torch.ones(x.shape[0], dtype=torch.bool) if mask is None else mask.reshape(-1)
    n = int(live.sum())
    counts = torch.bincount(i[live].reshape(-1), minlength=E)
    d, size = torch.zeros_like(x), torch.zeros_like(x)
    if n == 0:
        return 0.0, counts, d.reshape(logits.shape), size.reshape(logits.shape)
    p = torch.softmax(x[live], -1)
    empty = (x[live] == -float("inf")).all(-1)
    p[empty] = 0.0
    f = counts.double() / (n * k)
    dot = (p * f).sum(-1, keepdim=True)
    d[live] = g * E / n * p * (f - dot)
    size[live] = abs(g) * E / n * p * (f + dot)
    return float(E * (f * p.sum(0) / n).sum()), counts, d.reshape(logits.shape), size.reshape(logits.shape)
