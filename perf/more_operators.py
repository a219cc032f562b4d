"""Timed cases of products in 8-bit integers (dense and by expert), their quantisation, the RMS norm that
writes 8 bits, and the router's balance loss.

``run`` computes each case either through this package (``own``) or in its
plain form: elementary torch operations in 32 bits, rounded once.  ``exact``
restates the definitions in 64 bits.

The format: a row v has one fp32 scale s = max|v| / 127 and codes
rint(v / s) in [-127, 127]; a row of zeros has scale 0.  8-bit results are
returned as the values they stand for, in bf16.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # one token between two layers: residual added, normed, in 8 bits for the next product; latency
        {"name": "norm_1_token", "op": "norm", "T": 1, "D": 2048, "dtype": "bf16", "residual": True, "norm": False},
        # a prefill chunk into a sparse layer: the router reads the norm itself too
        {"name": "norm_prefill", "op": "norm", "T": 4096, "D": 2048, "dtype": "bf16", "residual": True, "norm": True},
        # a first layer in float32, no residual yet, a ragged width
        {"name": "norm_ragged", "op": "norm", "T": 777, "D": 1999, "dtype": "fp32", "residual": False, "norm": False},
        # activations of a short chunk, hidden 2560
        {"name": "quantize_chunk", "op": "quantize", "rows": 61, "K": 2560, "dtype": "bf16"},
        # export of the float32 master weights of 64 experts' gate_up
        {"name": "quantize_weights", "op": "quantize", "rows": 65536, "K": 2048, "dtype": "fp32"},
        # one token through a dense projection: latency
        {"name": "product_1_token", "op": "product", "M": 1, "K": 2048, "N": 4096, "ready": False},
        # a batch of sequences decoding together, an odd number of them, ragged width
        {"name": "product_23_tokens", "op": "product", "M": 23, "K": 2080, "N": 4099, "ready": False},
        # a prefill through a projection whose input the norm has quantised
        {"name": "product_prefill", "op": "product", "M": 4096, "K": 4096, "N": 4096, "ready": True},
        # one token x top-10 of 256 experts, fused gate_up
        {"name": "experts_1_token", "op": "experts", "T": 1, "k": 10, "E": 256, "K": 2048, "N": 1024, "sorted": False},
        # a 4096-token prefill through gate_up, rows taken by index from the tokens
        {"name": "experts_prefill", "op": "experts", "T": 4096, "k": 10, "E": 256, "K": 2048, "N": 1024, "sorted": True},
        # a micro-batch of a small router, some of it padding, loss alone
        {"name": "balance_61_tokens", "op": "balance", "T": 61, "k": 4, "E": 60, "dtype": "fp32", "mask": True,
         "grad": False},
        # a training step's router with its gradient
        {"name": "balance_train", "op": "balance", "T": 32768, "k": 8, "E": 256, "dtype": "fp32", "mask": False,
         "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "product", "experts", "balance"])
    if op == "norm":
        return {"op": op, "T": _log(rng, 1, 4096), "D": _log(rng, 64, 4096), "dtype": rng.choice(list(DTYPES)),
                "residual": rng.random() < 0.7, "norm": rng.random() < 0.5}
    if op == "quantize":
        return {"op": op, "rows": _log(rng, 1, 32768), "K": _log(rng, 64, 4096), "dtype": rng.choice(list(DTYPES))}
    if op == "product":
        return {"op": op, "M": _log(rng, 1, 4096), "K": 16 * _log(rng, 8, 256), "N": _log(rng, 33, 4096),
                "ready": rng.random() < 0.5}
    if op == "experts":
        E = _log(rng, 4, 128)
        k = rng.randint(1, min(E, 10))
        is_sorted = rng.random() < 0.7
        T = _log(rng, 64, 2048) if is_sorted else rng.randint(1, max(1, 63 // k))
        return {"op": op, "T": T, "k": k, "E": E, "K": 16 * rng.randint(16, 128), "N": 8 * rng.randint(16, 128),
                "sorted": is_sorted}
    E = _log(rng, 4, 512)
    return {"op": op, "T": _log(rng, 1, 16384), "k": rng.randint(1, min(E, 10)), "E": E,
            "dtype": rng.choice(list(DTYPES)), "mask": rng.random() < 0.5, "grad": rng.random() < 0.6}


# ------------------------------------------------------------------ inputs


def _acts(g, rows, K, dtype=torch.bfloat16):
    """Normal activations, a few channels ten times the others, every row of its own size."""
    x = torch.randn(rows, K, device="cuda", generator=g)
    x *= 0.25 + torch.rand(rows, 1, device="cuda", generator=g)
    x[:, :: max(1, K // 7)] *= 10.0
    return x.to(dtype)


def _weights(g, *shape):
    """Codes [.., N, K] of normal weights about 1 / sqrt(K) in size, and their channels' scales."""
    w = (torch.randn(shape, device="cuda", generator=g, dtype=torch.bfloat16) * 32).round_().clamp_(-127, 127).to(torch.int8)
    s = (0.75 + 0.5 * torch.rand(shape[:-1], device="cuda", generator=g)) / (32 * math.sqrt(shape[-1]))
    return w, s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op == "norm":
        T, D, dt = case["T"], case["D"], DTYPES[case["dtype"]]
        s["x"] = _acts(g, T, D, dt)
        s["r"] = (2.0 * torch.randn(T, D, device="cuda", generator=g)).to(dt) if case["residual"] else None
        s["w"] = (1.0 + 0.1 * torch.randn(D, device="cuda", generator=g)).to(dt)
    elif op == "quantize":
        s["x"] = _acts(g, case["rows"], case["K"], DTYPES[case["dtype"]])
    elif op == "product":
        s["x"] = _acts(g, case["M"], case["K"])
        if case["ready"]:  # what the norm in front of it left
            s["x"] = _quantize(s["x"].float())
            s["x"] = (s["x"][0].to(torch.int8), s["x"][1].squeeze(-1).contiguous())
        s["w"], s["s"] = _weights(g, case["N"], case["K"])
    else:
        T, k, E = case["T"], case["k"], case["E"]
        # top-k of router logits in which some experts are liked better than others
        logits = torch.randn(T, E, device="cuda", generator=g) + 0.4 * torch.randn(1, E, device="cuda", generator=g)
        s["ids"] = torch.topk(logits, k, dim=-1).indices.to(torch.int32)
        if op == "balance":
            s["logits"] = logits.to(DTYPES[case["dtype"]])
            s["mask"] = torch.rand(T, device="cuda", generator=g) < 0.8 if case["mask"] else None
            if case["grad"]:
                s["logits"].requires_grad_(True)
                s["dloss"] = 0.01 + 0.01 * torch.rand((), device="cuda", generator=g)
                if case["dtype"] == "fp16":  # a loss scale that keeps the gradients above the type's smallest
                    s["dloss"] *= 16.0 * T
            return s
        s["x"] = _acts(g, T, case["K"])
        s["w"], s["s"] = _weights(g, E, case["N"], case["K"])
        if case["sorted"]:
            flat = s["ids"].reshape(-1)
            order = torch.argsort(flat, stable=True)
            s["sorted"] = flat[order]
            s["rows"] = torch.div(order, k, rounding_mode="floor").to(torch.int32)
            s["longest"] = int(torch.bincount(flat, minlength=E).max())
    return s


# -------------------------------------------------------------- plain form


def _quantize(v):
    """Codes (as float32) and scales [.., 1] of float32 rows."""
    s = v.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=v.device)
    return torch.where(s > 0, torch.round(v / s), 0.0).clamp(-127, 127), s


def _values(v):
    q, s = _quantize(v)
    return {"values": (q * s).to(torch.bfloat16), "scales": s.squeeze(-1)}


def _segments(ids, E):
    """Expert and place within the expert of each sorted pair."""
    start = torch.searchsorted(ids, torch.arange(E, device=ids.device, dtype=ids.dtype))
    return ids.long(), torch.arange(ids.numel(), device=ids.device) - start[ids.long()]


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "quantize":
        return _values(s["x"].float())
    if op == "norm":
        h = s["x"] if s["r"] is None else (s["x"].float() + s["r"].float()).to(s["x"].dtype)
        v = h.float()
        y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * s["w"].float()
        out = _values(y)
        if s["r"] is not None:
            out["sum"] = h
        if c["norm"]:
            out["norm"] = y.to(h.dtype)
        return out
    if op == "balance":
        T, k, E = c["T"], c["k"], c["E"]
        x = s["logits"].detach().float()
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        live = torch.ones(T, device=x.device) if s["mask"] is None else s["mask"].float()
        counts = torch.zeros(E, dtype=torch.int32, device=x.device)
        counts.index_add_(0, s["ids"].reshape(-1).long(), live.to(torch.int32).repeat_interleave(k))
        n = live.sum().clamp(min=1.0)
        f = counts.float() / (n * k)
        p = p * live.unsqueeze(-1)
        out = {"loss": E * (f * (p.double().sum(0).float() / n)).sum(), "counts": counts}
        if c["grad"]:
            d = p * (f - (p * f).sum(-1, keepdim=True)) * (s["dloss"] * E / n)
            out["dlogits"] = d.to(s["logits"].dtype)
        return out
    sw = s["s"]
    if op == "product":
        q, sx = (s["x"][0].float(), s["x"][1].unsqueeze(-1)) if c["ready"] else _quantize(s["x"].float())
        return ((q @ s["w"].float().t()) * sx * sw).to(torch.bfloat16)
    q, sx = _quantize(s["x"].float())
    if not c["sorted"]:
        e = s["ids"].long()
        y = torch.matmul(s["w"][e].float(), q.reshape(-1, 1, c["K"], 1)).squeeze(-1)
        return (y * sx.unsqueeze(1) * sw[e]).to(torch.bfloat16)
    rows, at = s["rows"].long(), _segments(s["sorted"], c["E"])
    pad = torch.zeros(c["E"], s["longest"], c["K"], device=q.device)
    pad[at] = q[rows]
    y = torch.bmm(pad, s["w"].float().transpose(1, 2).contiguous())[at]
    return (y * sx[rows] * sw[at[0]]).to(torch.bfloat16)


# -------------------------------------------------------- the package's own


def _own(s):
    from titan_amd import ops

    c = s["case"]
    op = c["op"]
    if op == "quantize":
        q, sc = ops.quantize(s["x"], mode="int8")
        return {"values": ops.dequantize(q, sc, mode="int8"), "scales": sc}
    if op == "norm":
        r = ops.rms_norm_quantize(s["x"], s["w"], EPS, residual=s["r"], norm=c["norm"])
        out = {"values": ops.dequantize(r.codes, r.scales, mode="int8"), "scales": r.scales}
        if s["r"] is not None:
            out["sum"] = r.sum
        if c["norm"]:
            out["norm"] = r.norm
        return out
    if op == "balance":
        loss, counts = ops.router_balance_loss(s["logits"], s["ids"], mask=s["mask"])
        out = {"loss": loss, "counts": counts}
        if c["grad"]:
            out["dlogits"] = torch.autograd.grad(loss, s["logits"], s["dloss"])[0]
        return out
    if op == "product":
        return ops.qqmm(s["x"], s["w"], s["s"], mode="int8")
    if not c["sorted"]:
        return ops.gather_qqmm(s["x"].reshape(-1, 1, 1, c["K"]), s["w"], s["s"], rhs_indices=s["ids"],
                               mode="int8").squeeze(2)
    return ops.gather_qqmm(s["x"].unsqueeze(1), s["w"], s["s"], lhs_indices=s["rows"], rhs_indices=s["sorted"],
                           mode="int8", sorted_indices=True).squeeze(1)


def run(state):
    return _own(state) if own else _plain(state)


# -------------------------------------------------------------------- work


def work(case):
    op = case["op"]
    if op == "norm":
        n, size = case["T"] * case["D"], DTYPES[case["dtype"]].itemsize
        moved = 1 + 2 * case["residual"] + case["norm"]  # x, the residual and the sum, the norm
        return {"bytes": n * (moved * size + 2) + 4 * case["T"] + size * case["D"], "flops": 4 * n}
    if op == "quantize":
        n = case["rows"] * case["K"]
        return {"bytes": n * (DTYPES[case["dtype"]].itemsize + 2) + 4 * case["rows"], "flops": 2 * n}
    if op == "balance":
        T, k, E, size = case["T"], case["k"], case["E"], DTYPES[case["dtype"]].itemsize
        logits = T * E * size
        return {"bytes": (3 if case["grad"] else 1) * logits + 4 * T * k + 4 * E + T * case["mask"], "flops": 8 * T * E}
    K, N = case["K"], case["N"]
    if op == "product":
        M = case["M"]
        return {"bytes": (1 if case["ready"] else 2) * M * K + N * K + 2 * M * N + 4 * N, "flops": 2.0 * M * N * K}
    T, k, E = case["T"], case["k"], case["E"]
    used = E * (1.0 - (1.0 - k / E) ** T)
    return {"bytes": 2 * T * K + used * N * (K + 4) + 2 * T * k * N, "flops": 2.0 * T * k * N * K}


# ------------------------------------------------------------------- exact


def _exact_quantize(v):
    """Codes and scales of rows in 64 bits; the scale is what 32 bits hold of it."""
    s = (v.abs().max(-1).values / 127.0).float().double()
    inv = s.unsqueeze(-1)
    q = torch.zeros_like(v)
    ok = s > 0
    q[ok] = torch.round(v[ok] / inv[ok])
    return q.clamp_(-127, 127), s


def _exact_values(v):
    parts = [_exact_quantize(p) for p in v.split(8192)]
    return {"values": torch.cat([q.mul_(sc.unsqueeze(-1)) for q, sc in parts]), "scales": torch.cat([sc for _, sc in parts])}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_values(s["x"].double())
    if op == "norm":
        h = s["x"].double()
        if s["r"] is not None:
            h = (h + s["r"].double()).to(s["x"].dtype).double()
        rms = (h.square().sum(-1, keepdim=True) / case["D"] + EPS).sqrt()
        y = h / rms * s["w"].double()
        out = _exact_values(y)
        if s["r"] is not None:
            out["sum"] = h
        if case["norm"]:
            out["norm"] = y
        return out
    if op == "balance":
        keep = torch.arange(case["T"], device="cuda") if s["mask"] is None else s["mask"].nonzero().flatten()
        x = s["logits"].detach().double().requires_grad_(True)
        counts = torch.bincount(s["ids"][keep].reshape(-1).long(), minlength=case["E"])
        n = max(1, keep.numel())
        mean = torch.softmax(x[keep], -1).sum(0) / n
        loss = case["E"] * torch.dot(counts.double() / (n * case["k"]), mean)
        out = {"loss": loss.detach(), "counts": counts}
        if case["grad"]:
            out["dlogits"] = torch.autograd.grad(loss * s["dloss"].double(), x)[0]
        return out
    K, N = case["K"], case["N"]
    if op == "product" and case["ready"]:
        q, sx = s["x"][0].double(), s["x"][1].double()
    else:
        q, sx = _exact_quantize(s["x"].double())
    if op == "product":
        return torch.matmul(q, s["w"].double().t()) * torch.outer(sx, s["s"].double())
    flat = s["sorted"].long() if case["sorted"] else s["ids"].reshape(-1).long()
    rows = s["rows"].long() if case["sorted"] else torch.arange(case["T"], device="cuda").repeat_interleave(case["k"])
    y = torch.empty(flat.numel(), N, dtype=torch.float64, device="cuda")
    for e in torch.unique(flat).tolist():
        i = (flat == e).nonzero().flatten()
        y[i] = torch.matmul(q[rows[i]], s["w"][e].double().t()) * torch.outer(sx[rows[i]], s["s"][e].double())
    return y if case["sorted"] else y.reshape(case["T"], case["k"], N)
