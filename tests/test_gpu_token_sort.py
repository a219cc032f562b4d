"""Tokens sorted by expert and back, and the gradients, against the formulas in
64 bits: moved rows bit for bit, sums within fp32 and one rounding."""

import pytest
import torch

from mx_helpers import check_sum, codes, dequantize_ref
from titan_amd import ops

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _setup(dev, T, k, E, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + T + k + D)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]) if T else torch.empty(0, k, dtype=torch.int64)
    order = torch.argsort(ids.reshape(-1), stable=True)
    inv = torch.argsort(order)
    x = torch.randn(T, D, generator=g).to(dtype)
    ys = torch.randn(T * k, D, generator=g).to(dtype)
    scores = torch.rand(T, k, generator=g)
    if T > 1:
        scores[1] = 0
    return g, ids, order, inv, x, ys, scores


CASES = [(1, 1, 1, 8), (7, 3, 16, 1000), (5, 2, 4, 1), (3, 9, 20, 33), (65, 10, 32, 2048), (130, 4, 4, 515),
         (2, 17, 20, 4104), (33, 1, 8, 64), (4, 8, 8, 2049)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,E,D", CASES)
def test_there_and_back(dev, T, k, E, D, dtype):
    print("[sort]", T, k, E, D, dtype, flush=True)
    g, ids, order, inv, x, ys, scores = _setup(dev, T, k, E, D, dtype)
    od, iv = order.to(torch.int32).to(dev), inv.to(torch.int32).to(dev)
    xd, yd, sd = (t.to(dev).requires_grad_(True) for t in (x, ys, scores))
    xs = ops.sort_tokens(xd, od, iv)
    assert torch.equal(xs.cpu(), x[order // k])
    y = ops.unsort_tokens(yd, od, iv, sd)
    back = ys.double()[inv].reshape(T, k, D)
    s = scores.double().unsqueeze(-1)
    check_sum(y, (s * back).sum(1), (s * back).abs().sum(1), k)
    dxs, dy = torch.randn(T * k, D, generator=g).to(dtype), torch.randn(T, D, generator=g).to(dtype)
    dx, dys, ds = torch.autograd.grad((xs, y), (xd, yd, sd), (dxs.to(dev), dy.to(dev)))
    r = dxs.double()[inv].reshape(T, k, D)
    check_sum(dx, r.sum(1), r.abs().sum(1), k)
    ref = scores.double().reshape(-1)[order].unsqueeze(-1) * dy.double()[order // k]
    check_sum(dys, ref, ref.abs(), 1)
    prod = dy.double().unsqueeze(1) * back
    check_sum(ds, prod.sum(-1), prod.abs().sum(-1), D)
    # without scores: every pair's row, in pair order
    flat = ops.unsort_tokens(yd, od, iv)
    assert torch.equal(flat.cpu(), ys[inv])
    (dflat,) = torch.autograd.grad(flat, yd, dxs.to(dev))
    assert torch.equal(dflat.cpu(), dxs[order])


def test_routing_and_the_sum_agree_with_the_block_ops(dev):
    g, ids, _, _, x, _, scores = _setup(dev, 50, 4, 8, 256, torch.bfloat16)
    r = ops.route(ids.to(dev), 8)
    xs = ops.sort_tokens(x.to(dev), r.order, r.inv_order)
    assert torch.equal(xs, ops.gather_rows(x.to(dev), r.order, 4))
    y = ops.unsort_tokens(xs, r.order, r.inv_order, scores.to(dev))
    want = scores.double().sum(1, keepdim=True) * x.double()
    check_sum(y, want, (scores.double().unsqueeze(-1) * x.double().unsqueeze(1)).abs().sum(1), 4)


def test_only_one_gradient_is_asked_for(dev):
    g, ids, order, inv, x, ys, scores = _setup(dev, 6, 3, 5, 40, torch.float32)
    od, iv = order.to(dev), inv.to(dev)
    dy = torch.randn(6, 40, generator=g)
    yd = ys.to(dev).requires_grad_(True)
    (a,) = torch.autograd.grad(ops.unsort_tokens(yd, od, iv, scores.to(dev)), yd, dy.to(dev))
    sd = scores.to(dev).requires_grad_(True)
    (b,) = torch.autograd.grad(ops.unsort_tokens(ys.to(dev), od, iv, sd), sd, dy.to(dev))
    yd2, sd2 = ys.to(dev).requires_grad_(True), scores.to(dev).requires_grad_(True)
    both = torch.autograd.grad(ops.unsort_tokens(yd2, od, iv, sd2), (yd2, sd2), dy.to(dev))
    assert torch.equal(a, both[0]) and torch.equal(b, both[1])


def test_views_and_expanded_gradients(dev):
    g, ids, order, inv, x, ys, scores = _setup(dev, 9, 2, 4, 48, torch.bfloat16)
    od, iv = order.to(dev), inv.to(dev)
    wide = torch.randn(9, 100, generator=g).to(torch.bfloat16).to(dev)
    for v in (wide[:, 3:51], wide[:, ::2][:, :48], wide[:, :48]):
        leaf = v.detach().requires_grad_(True)
        xs = ops.sort_tokens(leaf, od, iv)
        assert torch.equal(xs, v[order.to(dev) // 2])
        (dx,) = torch.autograd.grad(xs.sum(), leaf)
        assert torch.equal(dx, torch.full_like(dx, 2.0))
    half = scores.to(torch.bfloat16).to(dev).requires_grad_(True)  # scores of another type are taken in fp32
    y = ops.unsort_tokens(ys.to(dev), od, iv, half)
    (ds,) = torch.autograd.grad(y.sum(), half)
    assert ds.dtype == torch.bfloat16 and ds.shape == (9, 2)


def test_no_tokens(dev):
    e = torch.empty(0, dtype=torch.int32, device=dev)
    x = torch.empty(0, 16, device=dev, requires_grad=True)
    assert ops.sort_tokens(x, e, e).shape == (0, 16)
    y = ops.unsort_tokens(x, e, e, torch.empty(0, 4, device=dev))
    assert y.shape == (0, 16)
    y.sum().backward()
    assert x.grad.shape == (0, 16)


def test_rows_without_elements(dev):
    """D = 0: the scores' gradients are empty sums."""
    ids = torch.arange(6, dtype=torch.int32, device=dev)
    xs = torch.empty(6, 0, device=dev, requires_grad=True)
    scores = torch.ones(3, 2, device=dev, requires_grad=True)
    y = ops.unsort_tokens(xs, ids, ids, scores)
    assert y.shape == (3, 0) and ops.sort_tokens(y.detach(), ids, ids).shape == (6, 0)
    y.sum().backward()
    assert xs.grad.shape == (6, 0) and torch.equal(scores.grad, torch.zeros(3, 2, device=dev))


def test_gradients_against_differences(dev):
    """In fp32 the sums are linear in xs and in scores."""
    g, ids, order, inv, x, ys, scores = _setup(dev, 5, 3, 6, 37, torch.float32)
    od, iv = order.to(dev), inv.to(dev)
    yd, sd = ys.to(dev).requires_grad_(True), scores.to(dev).requires_grad_(True)
    dy = torch.randn(5, 37, generator=g)
    dys, ds = torch.autograd.grad(ops.unsort_tokens(yd, od, iv, sd), (yd, sd), dy.to(dev))
    back = ys.double()[inv].reshape(5, 3, 37)
    for j in range(3):  # d loss / d scores[:, j] as a central difference in 64 bits
        h = 0.25
        loss = lambda sc: ((sc.unsqueeze(-1) * back).sum(1) * dy.double()).sum(1)  # noqa: E731
        up, dn = scores.double().clone(), scores.double().clone()
        up[:, j] += h
        dn[:, j] -= h
        diff = (loss(up) - loss(dn)) / (2 * h)
        bound = (37 + 16) * 2.0 ** -24 * (back[:, j] * dy.double()).abs().sum(1) + 2.0 ** -20 * 1e-6
        assert ((ds[:, j].cpu().double() - diff).abs() <= bound).all()


def test_layer_of_mxfp4_experts(dev):
    """Sort, two expert products, SwiGLU between and the weighted sum, with the
    gradient of the tokens and the scores, against the same layer in 64 bits.
    Each of the three bf16 roundings on the way is 2^-8 of its value; with sums
    of products that do not cancel on average, the whole stays within 2% of the
    result's norm (4 * 3 * 2^-8 = 4.7% is the bound asserted)."""
    T, k, E, H, I = 40, 4, 8, 256, 96
    g, ids, _, _, x, _, scores = _setup(dev, T, k, E, H, torch.bfloat16)
    w1, s1 = codes(g, E, 2 * I, H)
    w2, s2 = codes(g, E, H, I)
    r = ops.route(ids.to(dev), E)
    xd, sd = x.to(dev).requires_grad_(True), scores.to(dev).requires_grad_(True)

    def layer(x_, sc, up, down, sort, unsort):
        gu = up(sort(x_))
        a, b = gu.chunk(2, -1)
        return unsort(down(torch.nn.functional.silu(a) * b), sc)

    mx = lambda w, s: (lambda v: ops.gather_qmm(v.unsqueeze(1), w.to(dev), s.to(dev), rhs_indices=r.sorted_ids,  # noqa: E731
                                                mode="mxfp4", sorted_indices=True, tiles=r.tiles).squeeze(1))
    y = layer(xd, sd, mx(w1, s1), mx(w2, s2), lambda v: ops.sort_tokens(v, r.order, r.inv_order),
              lambda v, sc: ops.unsort_tokens(v, r.order, r.inv_order, sc))
    order, inv, e = r.order.cpu().long(), r.inv_order.cpu().long(), r.sorted_ids.cpu().long()
    x64, s64 = x.double().requires_grad_(True), scores.double().requires_grad_(True)
    ref = lambda w, s: (lambda v: torch.bmm(dequantize_ref(w, s)[e], v.unsqueeze(-1)).squeeze(-1))  # noqa: E731
    y64 = layer(x64, s64, ref(w1, s1), ref(w2, s2), lambda v: v[order // k],
                lambda v, sc: (sc.unsqueeze(-1) * v[inv].reshape(T, k, H)).sum(1))
    dy = torch.randn(T, H, generator=g).to(torch.bfloat16)
    got = (y, *torch.autograd.grad(y, (xd, sd), dy.to(dev)))
    want = (y64, *torch.autograd.grad(y64, (x64, s64), dy.double()))
    for a, b in zip(got, want):
        rel = float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
        print("[layer]", rel, flush=True)
        assert rel <= 12 * 2.0 ** -8


def test_graph_replays(dev):
    g, ids, order, inv, x, ys, scores = _setup(dev, 20, 4, 8, 96, torch.bfloat16)
    od, iv = order.to(torch.int32).to(dev), inv.to(torch.int32).to(dev)
    xd, yd, sd = x.to(dev), ys.to(dev), scores.to(dev)
    step = lambda: (ops.sort_tokens(xd, od, iv), ops.unsort_tokens(yd, od, iv, sd))  # noqa: E731
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        xd.copy_(torch.randn(20, 96, generator=g))
        sd.copy_(torch.rand(20, 4, generator=g))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_second_derivatives_are_refused(dev):
    """The gradients are not differentiable themselves, and say so instead of being constants."""
    g, ids, order, inv, x, ys, scores = _setup(dev, 4, 2, 4, 16, torch.float32)
    xd = x.to(dev).requires_grad_(True)
    (dx,) = torch.autograd.grad(ops.sort_tokens(xd, order.to(dev), inv.to(dev)).square().sum(), xd, create_graph=True)
    assert torch.equal(dx.cpu(), 2 * 2 * x)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


def test_rows_past_four_gigabytes(dev):
    """Sorted rows of 5 GB, there and back and their gradients, with a weight of one on each slot."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("less than 40 GiB of GPU memory free")
    T, k, D = 150_000, 8, 2048
    g = torch.Generator(device=dev).manual_seed(3)
    ids = torch.randint(0, 64, (T, k), generator=g, device=dev, dtype=torch.int32)
    r = ops.route(ids, 64)
    x = torch.randn(T, D, generator=g, device=dev).to(torch.bfloat16)
    xs = ops.sort_tokens(x, r.order, r.inv_order)
    assert xs.numel() * 2 > 1 << 32
    some = torch.tensor([0, 1, T * k // 2, T * k - 2, T * k - 1], device=dev)
    assert torch.equal(xs[some], x[r.order.long()[some] // k])
    scores = torch.zeros(T, k, device=dev)
    scores[:, k - 1] = 2.0
    xs.requires_grad_(True)
    scores.requires_grad_(True)
    y = ops.unsort_tokens(xs, r.order, r.inv_order, scores)
    assert torch.equal(y, 2 * x)
    dxs, ds = torch.autograd.grad(y, (xs, scores), x)
    last = r.order.long() % k == k - 1
    assert torch.equal(dxs[some], torch.where(last[some, None], 2 * x[r.order.long()[some] // k], 0))
    # each slot's row is the token's: the same dot product, D fp32 terms that are all positive
    want = x[-3:].double().square().sum(-1)
    assert ((ds[-3:].double() - want[:, None]).abs() <= (D + 8) * 2.0 ** -24 * want[:, None]).all()
    assert torch.equal(ds, ds[:, :1].expand(T, k))
    del xs, dxs, y
    torch.cuda.empty_cache()
