"""A sparse layer as a serving program runs it in 8 bits (residual and norm, the
router, its experts' products, the way back) and a router's training step beside
it, each against the same steps restated on the CPU."""

import int8_oracle as o
import pytest
import torch

from titan_amd import ops

BF, F4 = o.BF, o.F4
pytestmark = pytest.mark.gpu


def _layer(H, I, E, seed):
    g = torch.Generator().manual_seed(seed)
    gu = torch.randn(E, 2 * I, H, generator=g) / H ** 0.5
    dn = torch.randn(E, H, I, generator=g) / I ** 0.5
    return {"norm": 1 + 0.1 * torch.randn(H, generator=g), "router": (torch.randn(E, H, generator=g) / H ** 0.5).to(BF),
            "gu": o.quantize(gu), "dn": o.quantize(dn)}


def _run(p, x, res, k, dev):
    """The layer through the framework; every stage's result, for the oracle to start the next one from."""
    T = x.shape[0]
    n = ops.rms_norm_quantize(x, p["norm"], 1e-6, residual=res, norm=True)
    logits = ops.router_logits(n.norm, p["router"])
    ids, scores = ops.router_topk(logits, k)
    if T * k < 64:
        gu = ops.gather_qqmm((n.codes.reshape(T, 1, 1, -1), n.scales.reshape(T, 1, 1)), *p["gu"], rhs_indices=ids, mode="int8")
        h = ops.swiglu(gu)
        yd = ops.gather_qqmm(h, *p["dn"], rhs_indices=ids, mode="int8").squeeze(2)
        y = ops.moe_weighted_sum(yd, None, scores, x.shape, "fast")
        order = torch.arange(T * k, device=dev)
    else:
        r = ops.route(ids, p["router"].shape[0])
        rows = torch.div(r.order, k, rounding_mode="floor").to(torch.int32)
        gu = ops.gather_qqmm((n.codes.unsqueeze(1), n.scales.unsqueeze(1)), *p["gu"], lhs_indices=rows, rhs_indices=r.sorted_ids,
                             mode="int8", sorted_indices=True, tiles=r.tiles)
        h = ops.swiglu(gu)
        yd = ops.gather_qqmm(h, *p["dn"], rhs_indices=r.sorted_ids, mode="int8", sorted_indices=True, tiles=r.tiles)
        y = ops.moe_weighted_sum(yd, r.inv_order, scores, x.shape, "fast")
        order = r.order
    return n, logits, ids, scores, order, gu, h, yd, y


@pytest.mark.parametrize("T", [1, 5, 40, 333])
def test_serving_layer(dev, T):
    H, I, E, k = 256, 128, 16, 4
    p = _layer(H, I, E, 1)
    g = torch.Generator().manual_seed(T)
    x, res = torch.randn(T, H, generator=g).to(BF), (2 * torch.randn(T, H, generator=g)).to(BF)
    d = {a: tuple(t.to(dev) for t in b) if isinstance(b, tuple) else b.to(dev) for a, b in p.items()}
    got = _run(d, x.to(dev), res.to(dev), k, dev)
    n, logits, ids, scores, order, gu, h, yd, y = (t if isinstance(t, tuple) else t.cpu() for t in got)
    total, v = o.rms_norm(x, p["norm"], 1e-6, res)
    assert torch.equal(n.sum.cpu(), total)
    o.assert_rounded(n.norm, v)
    order = order.long()
    flat, tok = ids.flatten().long()[order], torch.div(order, k, rounding_mode="floor")
    gu, h, yd = (t.reshape(T * k, -1) for t in (gu, h, yd))
    qh, sh = o.quantize(h.float())
    for e in range(E):
        i = (flat == e).nonzero().flatten()
        o.assert_rounded(gu[i], o.product(n.codes.cpu()[tok[i]], n.scales.cpu()[tok[i]], p["gu"][0][e], p["gu"][1][e]))
        o.assert_rounded(yd[i], o.product(qh[i], sh[i], p["dn"][0][e], p["dn"][1][e]))
    back = torch.empty(T * k, H, dtype=torch.float64)
    back[order] = yd.double()
    want = (back.reshape(T, k, H) * scores.double().unsqueeze(-1)).sum(1)
    size = (back.reshape(T, k, H).abs() * scores.double().unsqueeze(-1)).sum(1)
    # k products and additions in fp32, rounded once
    assert bool(((y.double() - want).abs() <= want.abs() * 2.0 ** -8 + size * 2 * k * 2.0 ** -24).all())


def test_serving_layer_in_a_graph(dev):
    H, I, E, k, T = 256, 128, 16, 4, 70
    d = {a: tuple(t.to(dev) for t in b) if isinstance(b, tuple) else b.to(dev) for a, b in _layer(H, I, E, 2).items()}
    x, res = torch.randn(T, H, device=dev).to(BF), torch.randn(T, H, device=dev).to(BF)
    _run(d, x, res, k, dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(d, x, res, k, dev)
    for i in range(3):
        x.copy_(torch.randn(T, H, generator=torch.Generator().manual_seed(i)).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        kept = out[-1].clone(), out[0].sum.clone()
        again = _run(d, x, res, k, dev)
        assert torch.equal(kept[0], again[-1]) and torch.equal(kept[1], again[0].sum)


def test_router_training_step(dev):
    """Logits that are leaves of both the experts' scores and the balance loss: the gradients add up."""
    T, E, k, H = 90, 16, 2, 64
    g = torch.Generator().manual_seed(3)
    logits, yd, dy = torch.randn(T, E, generator=g), torch.randn(T * k, H, generator=g), torch.randn(T, H, generator=g)
    mask = torch.rand(T, generator=g) < 0.8
    leaf = logits.to(dev).requires_grad_(True)
    ids, _ = ops.router_topk(leaf.detach(), k)
    r = ops.route(ids, E)
    scores = torch.softmax(leaf.gather(1, ids.long()), -1)
    y = ops.unsort_tokens(yd.to(dev), r.order, r.inv_order, scores)
    loss, counts = ops.router_balance_loss(leaf, ids, mask.to(dev))
    ((y * dy.to(dev)).sum() + 0.5 * loss).backward()
    x = logits.double().requires_grad_(True)
    i = ids.cpu().long()
    back = yd.double()[r.inv_order.cpu().long()].reshape(T, k, H)
    ((torch.softmax(x.gather(1, i), -1).unsqueeze(-1) * back).sum(1) * dy.double()).sum().backward()
    wl, wc, wd, _ = o.balance(logits, i, mask, 0.5)
    want = x.grad + wd
    assert torch.equal(counts.cpu().long(), wc)
    # sums of H products of size 1 in fp32 through a softmax, and the loss's part
    assert bool(((leaf.grad.cpu().double() - want).abs() <= 1e-5 * (1 + want.abs())).all())
