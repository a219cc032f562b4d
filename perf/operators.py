"""Timed cases of the microscaled 4-bit (mxfp4) operators and of the sort of tokens by expert.

``run`` computes each case either through this package (``own``) or in its
plain form: elementary torch operations in 32 bits, rounded once.  ``exact``
restates the definitions in 64 bits.

The format: blocks of 32 elements along the last axis share one scale, a power
of two held as the byte e + 127 (255: not a number); an element is a sign and
one of 0, 0.5, 1, 1.5, 2, 3, 4, 6, eight codes to a 32-bit word, low bits
first.  A block's scale is 2^(floor(log2 max|x|) - 2), an element is x / scale
rounded to the nearest value, ties to the even code, at most 6.
"""

import math

import torch

own = False

BLOCK = 32
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # activations of a short chunk on their way into a 4-bit product, hidden 2048
        {"name": "quantize_chunk", "op": "quantize", "rows": 61, "K": 2048, "dtype": "bf16"},
        # export of the float32 master weights of 64 experts' gate_up
        {"name": "quantize_weights", "op": "quantize", "rows": 65536, "K": 2048, "dtype": "fp32"},
        # one token through a dense projection: latency
        {"name": "matmul_1_token", "op": "matmul", "M": 1, "K": 2048, "N": 4096, "grad": False},
        # a batch of sequences decoding together, an odd number of them, ragged width
        {"name": "matmul_23_tokens", "op": "matmul", "M": 23, "K": 2080, "N": 4099, "grad": False},
        # a training step through a frozen projection: the product and its gradient
        {"name": "matmul_train", "op": "matmul", "M": 4096, "K": 2048, "N": 4096, "grad": True},
        # one token x top-10 of 256 experts, fused gate_up
        {"name": "experts_1_token", "op": "experts", "T": 1, "k": 10, "E": 256, "K": 2048, "N": 1024,
         "sorted": False, "grad": False},
        # a 4096-token prefill through gate_up, rows taken by index from the tokens
        {"name": "experts_prefill", "op": "experts", "T": 4096, "k": 10, "E": 256, "K": 2048, "N": 1024,
         "sorted": True, "grad": False},
        # a training step through 60 frozen experts of another width, ragged rows
        {"name": "experts_train", "op": "experts", "T": 2039, "k": 4, "E": 60, "K": 2048, "N": 1408,
         "sorted": True, "grad": True},
        # both operands in 4 bits: a dense prefill
        {"name": "qq_dense", "op": "qq", "T": 4096, "k": 0, "E": 1, "K": 4096, "N": 4096},
        # both operands in 4 bits: a chunk of tokens through the experts' gate_up
        {"name": "qq_experts", "op": "qq", "T": 1531, "k": 10, "E": 256, "K": 2048, "N": 1024},
        # a few tokens to their experts and back, with gradients, float32
        {"name": "sort_7_tokens", "op": "sort", "T": 7, "k": 3, "E": 16, "D": 1000, "dtype": "fp32"},
        # a training batch to its experts and back, with gradients
        {"name": "sort_train", "op": "sort", "T": 4096, "k": 10, "E": 256, "D": 2048, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "experts", "qq", "sort"])
    if op == "quantize":
        return {"op": op, "rows": _log(rng, 1, 32768), "K": BLOCK * _log(rng, 2, 128),
                "dtype": rng.choice(list(DTYPES))}
    if op == "matmul":
        return {"op": op, "M": _log(rng, 1, 4096), "K": BLOCK * _log(rng, 4, 64), "N": _log(rng, 33, 4096),
                "grad": rng.random() < 0.5}
    if op == "experts":
        E = _log(rng, 4, 128)
        k = rng.randint(1, min(E, 10))
        is_sorted = rng.random() < 0.7
        T = _log(rng, 64, 2048) if is_sorted else rng.randint(1, max(1, 63 // k))
        return {"op": op, "T": T, "k": k, "E": E, "K": BLOCK * rng.randint(8, 64), "N": 8 * rng.randint(16, 128),
                "sorted": is_sorted, "grad": is_sorted and rng.random() < 0.5}
    if op == "qq":
        k = rng.choice([0, 1, 2, 4, 8])
        return {"op": op, "T": _log(rng, 1, 2048), "k": k, "E": _log(rng, 8, 128) if k else 1,
                "K": BLOCK * rng.randint(8, 64), "N": 8 * rng.randint(16, 256)}
    E = _log(rng, 4, 256)
    return {"op": op, "T": _log(rng, 1, 4096), "k": rng.randint(1, min(E, 10)), "E": E, "D": rng.randint(64, 2048),
            "dtype": rng.choice(list(DTYPES))}


# ------------------------------------------------------------------ inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _acts(g, rows, K, dtype=torch.bfloat16):
    """Normal activations, a few channels ten times the others, every row of its own size."""
    x = torch.randn(rows, K, device="cuda", generator=g)
    x *= 0.25 + torch.rand(rows, 1, device="cuda", generator=g)
    x[:, :: max(1, K // 7)] *= 10.0
    return x.to(dtype)


def _codes(g, *shape):
    """Packed codes [.., N, K] of weights about 1 / sqrt(K) in size, and their scale bytes."""
    K = shape[-1]
    w = torch.randint(-(1 << 31), (1 << 31), (*shape[:-1], K // 8), device="cuda", generator=g, dtype=torch.int64)
    mid = 127 - 1 - int(0.5 * math.log2(K))
    s = torch.randint(mid - 2, mid + 1, (*shape[:-1], K // BLOCK), device="cuda", generator=g, dtype=torch.int64)
    return w.to(torch.int32), s.to(torch.uint8)


def _ids(g, T, k, E):
    """Top-k of router logits in which some experts are liked better than others: int32 [T, k]."""
    logits = torch.randn(T, E, device="cuda", generator=g) + 0.4 * torch.randn(1, E, device="cuda", generator=g)
    return torch.topk(logits, k, dim=-1).indices.to(torch.int32)


def _sort(ids, E):
    """order, its inverse and the sorted ids of the flattened pairs, int32; the longest segment's rows."""
    order = torch.argsort(ids.reshape(-1), stable=True)
    return (order.to(torch.int32), torch.argsort(order).to(torch.int32), ids.reshape(-1)[order].to(torch.int32),
            int(torch.bincount(ids.reshape(-1), minlength=E).max()))


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = {"case": case}
    if op == "quantize":
        s["x"] = _acts(g, case["rows"], case["K"], DTYPES[case["dtype"]])
    elif op == "matmul":
        s["x"] = _acts(g, case["M"], case["K"])
        s["w"], s["s"] = _codes(g, case["N"], case["K"])
        if case["grad"]:
            s["x"].requires_grad_(True)
            s["dy"] = torch.randn(case["M"], case["N"], device="cuda", generator=g).to(torch.bfloat16)
    elif op in ("experts", "qq"):
        T, k, E, K, N = (case[n] for n in ("T", "k", "E", "K", "N"))
        s["x"] = _acts(g, T, K)
        if k == 0:
            s["w"], s["s"] = _codes(g, N, K)
            return s
        s["w"], s["s"] = _codes(g, E, N, K)
        s["ids"] = _ids(g, T, k, E)
        if op == "qq" or case["sorted"]:
            order, _, s["sorted"], s["longest"] = _sort(s["ids"], E)
            s["rows"] = torch.div(order, k, rounding_mode="floor").to(torch.int32)
            if op == "experts" and case["grad"]:
                s["x"] = s["x"][s["rows"].long()].requires_grad_(True)
                s["dy"] = torch.randn(T * k, N, device="cuda", generator=g).to(torch.bfloat16)
    else:
        T, k, D, dt = case["T"], case["k"], case["D"], DTYPES[case["dtype"]]
        s["order"], s["inv"], _, _ = _sort(_ids(g, T, k, case["E"]), case["E"])
        s["x"] = _acts(g, T, D, dt).requires_grad_(True)
        s["ys"] = torch.randn(T * k, D, device="cuda", generator=g).to(dt).requires_grad_(True)
        s["scores"] = torch.softmax(torch.randn(T, k, device="cuda", generator=g), -1).requires_grad_(True)
        s["dxs"] = torch.randn(T * k, D, device="cuda", generator=g).to(dt)
        s["dy"] = torch.randn(T, D, device="cuda", generator=g).to(dt)
    return s


# -------------------------------------------------------------- plain form


def _quantize(x):
    """Values (in units of the scale) and exponents of blocks of 32, in 32 bits."""
    v = x.float().unflatten(-1, (-1, BLOCK))
    top = v.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 127)
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    a = torch.ldexp(torch.ldexp(v.abs(), -(e // 2)), -(e - e // 2))
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), v), e


def _weights(w, s):
    """Codes and scale bytes to float32 weights."""
    q = (w.unsqueeze(-1) >> torch.arange(0, 32, 4, device=w.device, dtype=torch.int32)) & 15
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=w.device)
    v = table[q.flatten(-2)].unflatten(-1, (-1, BLOCK))
    return (v * torch.exp2(s.float() - 127.0).unsqueeze(-1)).flatten(-2)


def _segments(ids, E, longest):
    """Row of each sorted pair in a table [E, longest]."""
    start = torch.searchsorted(ids, torch.arange(E, device=ids.device, dtype=ids.dtype))
    return ids.long(), torch.arange(ids.numel(), device=ids.device) - start[ids.long()]


def _grouped(x, w, ids, longest):
    """x [n, K] of sorted rows times w[expert] [N, K]^T, every expert padded to the longest."""
    at = _segments(ids, w.shape[0], longest)
    pad = torch.zeros(w.shape[0], longest, x.shape[-1], device=x.device)
    pad[at] = x
    return torch.bmm(pad, w.transpose(1, 2))[at]


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "quantize":
        v, e = _quantize(s["x"])
        return {"values": torch.ldexp(v, e).flatten(-2).to(s["x"].dtype), "scales": (e + 127).squeeze(-1).to(torch.uint8)}
    if op == "sort":
        x, ys, sc, dxs, dy = (s[n].detach().float() for n in ("x", "ys", "scores", "dxs", "dy"))
        order, inv, dt, k = s["order"].long(), s["inv"].long(), s["x"].dtype, c["k"]
        back = ys[inv].unflatten(0, (-1, k))
        return {"xs": x[order // k].to(dt), "y": (sc.unsqueeze(-1) * back).sum(1).to(dt),
                "dx": dxs[inv].unflatten(0, (-1, k)).sum(1).to(dt),
                "dys": (sc.reshape(-1)[order].unsqueeze(-1) * dy[order // k]).to(dt),
                "dscores": (dy.unsqueeze(1) * back).sum(-1)}
    x = s["x"].detach().float()
    if op == "qq":
        v, e = _quantize(x)
        x = torch.ldexp(v, e).flatten(-2)
    if op == "matmul" or c["k"] == 0:
        w = _weights(s["w"], s["s"])
        y = (x @ w.t()).to(torch.bfloat16)
        if not c.get("grad"):
            return y
        return {"y": y, "dx": (s["dy"].float() @ w).to(torch.bfloat16)}
    if op == "experts" and not c["sorted"]:
        e = s["ids"].long()
        w = _weights(s["w"][e], s["s"][e])
        return torch.matmul(w, x.reshape(-1, 1, c["K"], 1)).squeeze(-1).to(torch.bfloat16)
    w = _weights(s["w"], s["s"])
    if not c.get("grad"):
        return _grouped(x[s["rows"].long()], w, s["sorted"], s["longest"]).to(torch.bfloat16)
    return {"y": _grouped(x, w, s["sorted"], s["longest"]).to(torch.bfloat16),
            "dx": _grouped(s["dy"].float(), w.transpose(1, 2), s["sorted"], s["longest"]).to(torch.bfloat16)}


# -------------------------------------------------------- the package's own


def _own(s):
    from titan_amd import ops

    c = s["case"]
    op = c["op"]
    if op == "quantize":
        w, sc = ops.quantize(s["x"], mode="mxfp4")
        return {"values": ops.dequantize(w, sc, mode="mxfp4", dtype=s["x"].dtype), "scales": sc}
    if op == "sort":
        xs = ops.sort_tokens(s["x"], s["order"], s["inv"])
        y = ops.unsort_tokens(s["ys"], s["order"], s["inv"], s["scores"])
        dx, dys, dsc = torch.autograd.grad((xs, y), (s["x"], s["ys"], s["scores"]), (s["dxs"], s["dy"]))
        return {"xs": xs, "y": y, "dx": dx, "dys": dys, "dscores": dsc}
    if op == "matmul":
        y = ops.quantized_matmul(s["x"], s["w"], s["s"], mode="mxfp4")
        if not c["grad"]:
            return y
        return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    if op == "qq":
        if c["k"] == 0:
            return ops.qqmm(s["x"], s["w"], s["s"], mode="mxfp4")
        return ops.gather_qqmm(s["x"].unsqueeze(1), s["w"], s["s"], lhs_indices=s["rows"], rhs_indices=s["sorted"],
                               mode="mxfp4", sorted_indices=True).squeeze(1)
    if not c["sorted"]:
        return ops.gather_qmm(s["x"].reshape(-1, 1, 1, c["K"]), s["w"], s["s"], rhs_indices=s["ids"],
                              mode="mxfp4").squeeze(2)
    if not c["grad"]:
        return ops.gather_qmm(s["x"].unsqueeze(1), s["w"], s["s"], lhs_indices=s["rows"], rhs_indices=s["sorted"],
                              mode="mxfp4", sorted_indices=True).squeeze(1)
    y = ops.gather_qmm(s["x"].unsqueeze(1), s["w"], s["s"], rhs_indices=s["sorted"], mode="mxfp4",
                       sorted_indices=True).squeeze(1)
    return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}


def run(state):
    return _own(state) if own else _plain(state)


# -------------------------------------------------------------------- work


def work(case):
    op = case["op"]
    packed = 0.5 + 1.0 / BLOCK  # bytes of a weight in 4 bits with its share of the scale
    if op == "quantize":
        n, size = case["rows"] * case["K"], DTYPES[case["dtype"]].itemsize
        return {"bytes": n * (2 * size + 1.0 / BLOCK), "flops": 0}
    if op == "sort":
        T, k, D, size = case["T"], case["k"], case["D"], DTYPES[case["dtype"]].itemsize
        rows = T * D * size
        # in: x, ys, dxs, dy, scores, order and its inverse; out: xs, y, dx, dys, dscores
        return {"bytes": 4 * rows + 4 * k * rows + 16 * T * k, "flops": 5 * T * k * D}
    K, N = case["K"], case["N"]
    if op == "matmul" or case["k"] == 0:
        tokens, rows, used = (case["M"] if op == "matmul" else case["T"],) * 2 + (1.0,)
    else:
        tokens, rows = case["T"], case["T"] * case["k"]
        used = case["E"] * (1.0 - (1.0 - case["k"] / case["E"]) ** case["T"])
    if case.get("grad"):
        return {"bytes": 4 * rows * (K + N) + used * N * K * packed, "flops": 4.0 * rows * N * K}
    return {"bytes": 2 * tokens * K + 2 * rows * N + used * N * K * packed, "flops": 2.0 * rows * N * K}


# ------------------------------------------------------------------- exact


def _exact_quantize(x):
    """Nearest of the eight magnitudes by comparing distances in 64 bits, ties to the even one."""
    v = x.detach().double().reshape(-1, BLOCK)
    top = v.abs().amax(1)
    e = torch.floor(torch.log2(top))
    e = torch.where(torch.exp2(e) > top, e - 1, e)  # a logarithm rounded up to a whole number
    e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)
    e = torch.where(top > 0, e - 2, torch.full_like(e, -127)).clamp(-127, 127)
    a = v.abs() / torch.exp2(e).unsqueeze(1)
    best, dist = torch.zeros_like(a), a.clone()
    for i, m in enumerate(VALUES[1:], 1):
        d = (a - m).abs()
        take = (d < dist) | ((d == dist) & (i % 2 == 0))
        best, dist = torch.where(take, m, best), torch.where(take, d, dist)
    return (torch.sign(v) * best * torch.exp2(e).unsqueeze(1)).reshape(x.shape), e


def _exact_weights(w, s):
    b = torch.stack([(w >> (8 * i)) & 255 for i in range(4)], -1).flatten(-2).long()  # bytes, low first
    pair = [(c & 7, -1.0 if c & 8 else 1.0) for c in range(16)]
    value = torch.tensor([[sg * VALUES[m] for m, sg in (pair[c & 15], pair[c >> 4])] for c in range(256)],
                         dtype=torch.float64, device=w.device)
    return value[b].flatten(-2) * torch.pow(2.0, s.double() - 127).repeat_interleave(BLOCK, -1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        parts = [_exact_quantize(p) for p in s["x"].split(8192)]
        v, e = (torch.cat(p) for p in zip(*parts))
        return {"values": v, "scales": (e + 127).to(torch.int64).reshape(case["rows"], -1)}
    if op == "sort":
        x, ys, sc, dxs, dy = (s[n].detach().double() for n in ("x", "ys", "scores", "dxs", "dy"))
        k, T = case["k"], case["T"]
        order, inv = s["order"].long(), s["inv"].long().reshape(T, k)
        y, dx, dsc = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(sc)
        for j in range(k):
            y += sc[:, j: j + 1] * ys[inv[:, j]]
            dx += dxs[inv[:, j]]
            dsc[:, j] = (dy * ys[inv[:, j]]).sum(1)
        dys = torch.empty_like(ys)
        for j in range(k):
            dys[inv[:, j]] = sc[:, j: j + 1] * dy
        return {"xs": x[torch.div(order, k, rounding_mode="floor")], "y": y, "dx": dx, "dys": dys, "dscores": dsc}
    x = _exact_quantize(s["x"])[0] if op == "qq" else s["x"].detach().double()
    if op == "matmul" or case["k"] == 0:
        w = _exact_weights(s["w"], s["s"])
        y = torch.matmul(x, w.t())
        return {"y": y, "dx": torch.matmul(s["dy"].double(), w)} if case.get("grad") else y
    N = case["N"]
    flat = s["ids"].reshape(-1).long() if op == "experts" and not case["sorted"] else s["sorted"].long()
    if op == "experts" and not case["sorted"]:
        x = x.repeat_interleave(case["k"], 0)
    elif not case.get("grad"):
        x = x[s["rows"].long()]
    y = torch.empty(flat.numel(), N, dtype=torch.float64, device="cuda")
    dx = torch.empty_like(x)
    for e in torch.unique(flat).tolist():
        rows = (flat == e).nonzero().flatten()
        w = _exact_weights(s["w"][e], s["s"][e])
        y[rows] = torch.matmul(x[rows], w.t())
        if case.get("grad"):
            dx[rows] = torch.matmul(s["dy"][rows].double(), w)
    if case.get("grad"):
        return {"y": y, "dx": dx}
    return y.reshape(*s["ids"].shape, N) if op == "experts" and not case["sorted"] else y
