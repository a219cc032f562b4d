"""The router's balance loss, its gradient and the experts' counts, against the
definition in 64 bits."""

import int8_oracle as o
import pytest
import torch

from titan_amd import ops

BF, HF, F4 = o.BF, o.HF, o.F4
pytestmark = pytest.mark.gpu


def _case(T, E, k, dtype, seed, masked):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(T, E, generator=g) + 0.5 * torch.randn(1, E, generator=g)).to(dtype)
    ids = torch.topk(logits.float() + torch.randn(T, E, generator=g), k, -1).indices
    return logits, ids, (torch.rand(T, generator=g) < 0.7) if masked else None


def _check(dev, logits, ids, mask, g=0.37, spread=40.0, long=64):
    """spread: the largest difference of a row's logits; long: the most terms that one sum adds in a row."""
    leaf = logits.to(dev).requires_grad_(True)
    loss, counts = ops.router_balance_loss(leaf, ids.to(dev), None if mask is None else mask.to(dev))
    assert loss.dtype == F4 and loss.shape == () and counts.dtype == torch.int32
    d, = torch.autograd.grad(loss, leaf, torch.tensor(g, device=dev))
    wl, wc, wd, size = o.balance(logits, ids, mask, float(torch.tensor(g, dtype=F4)))
    assert torch.equal(counts.cpu().long(), wc)
    # p: the difference and its product with log2 e (each half a step of up to `spread`), the exponential (2 half
    # steps), the sum of up to 16 + 6 additions, the division and the product; then the sum over tokens.
    u = 2.0 ** -24
    p_err = (2 * spread + 2 + 22 + 4) * u
    assert abs(loss.item() - wl) <= wl * (p_err + (long + 6) * u), (loss.item(), wl)
    assert d.dtype == logits.dtype and d.shape == logits.shape
    # a probability below fp32's least normal value may be lost whole: it stands in p (f - dot), f and dot at most 1
    n = max(1, logits[..., 0].numel() if mask is None else int(mask.sum()))
    lost = abs(g) * logits.shape[-1] / n * 2 * 2.0 ** -126
    tol = lost + size * (2 * p_err + 40 * u) + wd.abs() * o.UNIT[logits.dtype] + o.TINY[logits.dtype]
    err = (d.cpu().double() - wd).abs()
    assert bool((err <= tol).all()), (err - tol).max()
    if mask is not None:
        assert not d.cpu()[~mask].any()
    return loss, counts, d


@pytest.mark.parametrize("dtype", [BF, HF, F4])
@pytest.mark.parametrize("E,k", [(1, 1), (2, 1), (3, 2), (8, 2), (17, 5), (60, 4), (64, 8), (100, 10), (128, 1), (256, 8),
                                 (500, 10), (512, 64), (1000, 7), (1024, 70)])
@pytest.mark.parametrize("masked", [False, True])
def test_experts(dev, E, k, dtype, masked):
    _check(dev, *_case(77, E, k, dtype, E, masked))


@pytest.mark.parametrize("T", [1, 2, 5, 16, 17, 255, 1025, 4100, 30000])
def test_tokens(dev, T):
    _check(dev, *_case(T, 60, 4, F4, T, True))
    _check(dev, *_case(T, 256, 8, BF, T, False))


def test_dimensions_types_and_layouts(dev):
    logits, ids, mask = _case(60, 32, 3, F4, 1, True)
    loss, counts, d = _check(dev, logits, ids, mask)
    for l, i, m in ((logits.reshape(3, 20, 32), ids.reshape(3, 20, 3).int(), mask.reshape(3, 20)),
                    (torch.cat([logits, logits], -1)[:, 32:], ids.t().contiguous().t(), torch.stack([mask, mask], 1)[:, 1])):
        a, b, c = _check(dev, l, i, m)
        assert torch.equal(a, loss) and torch.equal(b, counts) and torch.equal(c.reshape(60, 32), d)
    one, n = ops.router_balance_loss(logits[0].to(dev), ids[0].to(dev))
    assert n.sum().item() == 3 and abs(one.item() - o.balance(logits[:1], ids[:1])[0]) < 1e-5


def test_counts_are_the_routings(dev):
    logits, ids, _ = _case(700, 40, 4, F4, 2, False)
    idx, _ = ops.router_topk(logits.to(dev), 4)
    _, counts = ops.router_balance_loss(logits.to(dev), idx)
    offsets = ops.route(idx, 40).tiles.offsets
    assert torch.equal(counts, offsets[1:] - offsets[:-1])


def test_even_use_is_one(dev):
    for E, k in ((8, 2), (256, 8)):
        ids = torch.arange(E * k).reshape(E, k) % E
        loss, counts = ops.router_balance_loss(torch.zeros(E, E, device=dev), ids.to(dev))
        assert abs(loss.item() - 1.0) < 1e-6 and bool((counts == k).all())


def test_ids_out_of_range_and_repeated(dev):
    logits, _, mask = _case(50, 12, 3, F4, 3, True)
    ids = torch.randint(-5, 20, (50, 3), generator=torch.Generator().manual_seed(3))
    ids[4] = 7  # the same expert three times
    ids[5, 0] = 1 << 40
    _check(dev, logits, ids, mask)


def test_masks_and_rows_that_leave_nothing(dev):
    logits, ids, _ = _case(9, 20, 2, F4, 4, False)
    none = torch.zeros(9, dtype=torch.bool)
    loss, counts, d = _check(dev, logits, ids, none)
    assert loss.item() == 0.0 and not counts.any() and not d.any()
    one = none.clone()
    one[6] = True
    _check(dev, logits, ids, one)
    # what masked tokens hold does not matter
    spoilt = logits.clone()
    spoilt[0], spoilt[1], spoilt[2] = float("nan"), float("inf"), -float("inf")
    mask = torch.arange(9) > 2
    a, b = _check(dev, logits, ids, mask), _check(dev, spoilt, ids, mask)
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    # experts that a mask of -inf or of the type's lowest value takes out; a row in which it takes all
    for low in (-float("inf"), torch.finfo(F4).min):
        cut = logits.clone()
        cut[:, 3:9] = low
        _check(dev, cut, ids, None)
    cut[4] = -float("inf")
    _check(dev, cut, ids, None)
    empty = ops.router_balance_loss(torch.zeros(0, 20, device=dev), torch.zeros(0, 2, dtype=torch.int32, device=dev))
    assert empty[0].item() == 0.0 and not empty[1].any()
    leaf = torch.zeros(0, 20, device=dev, requires_grad=True)
    ops.router_balance_loss(leaf, torch.zeros(0, 2, dtype=torch.int32, device=dev))[0].backward()
    assert leaf.grad.shape == (0, 20)


def test_nan_and_infinite_logits(dev):
    logits, ids, _ = _case(5, 16, 2, F4, 5, False)
    for v in (float("nan"), float("inf")):
        bad = logits.clone()
        bad[2, 3] = v
        leaf = bad.to(dev).requires_grad_(True)
        loss, counts = ops.router_balance_loss(leaf, ids.to(dev))
        loss.backward()
        assert torch.isnan(loss) and torch.isnan(leaf.grad[2]).all() and torch.isfinite(leaf.grad[[0, 1, 3, 4]]).all()
        assert counts.sum().item() == 10


def test_extreme_logits(dev):
    logits, ids, _ = _case(40, 30, 3, F4, 6, False)
    _check(dev, logits * 30, ids, None, spread=400.0)
    _check(dev, logits + 1e4, ids, None)


def test_gradient_against_differences(dev):
    logits, ids, mask = _case(6, 10, 2, F4, 7, True)
    leaf = logits.to(dev).requires_grad_(True)
    ops.router_balance_loss(leaf, ids.to(dev), mask.to(dev))[0].backward()
    h = 1e-5
    for t in range(6):
        for e in range(10):
            up, down = logits.double(), logits.double()
            up[t, e] += h
            down[t, e] -= h
            want = (o.balance(up, ids, mask)[0] - o.balance(down, ids, mask)[0]) / (2 * h)
            # differences: h^2 of the third derivative (at most 6 losses) and 2 roundings of 64 bits over h
            assert abs(leaf.grad[t, e].item() - want) < 1e-8 + 2e-5 * 10 / 6


def test_autograd_surface(dev):
    logits, ids, mask = (None if t is None else t.to(dev) for t in _case(33, 24, 3, F4, 8, True))
    leaf = logits.clone().requires_grad_(True)
    loss, counts = ops.router_balance_loss(leaf, ids, mask)
    assert loss.requires_grad and not counts.requires_grad
    (3 * loss + (leaf ** 2).sum()).backward()
    first = leaf.grad.clone()
    d, = torch.autograd.grad(ops.router_balance_loss(leaf, ids, mask)[0], leaf)
    assert torch.allclose(first, 3 * d + 2 * leaf.detach(), rtol=1e-6, atol=1e-7)
    again, = torch.autograd.grad(ops.router_balance_loss(leaf, ids, mask)[0], leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        again.sum().backward()
    with torch.no_grad():
        assert not ops.router_balance_loss(leaf, ids, mask)[0].requires_grad
    import torch.autograd.forward_ad as fw

    with fw.dual_level(), pytest.raises(NotImplementedError):
        ops.router_balance_loss(fw.make_dual(logits, logits), ids, mask)
    with pytest.raises(ops.QmoeUnsupported, match="trace"):
        torch.jit.trace(lambda t: ops.router_balance_loss(t, ids)[0], (logits,))


def test_streams_graph_and_repeats(dev):
    logits, ids, mask = (t.to(dev) for t in _case(3000, 64, 4, F4, 9, True))
    static = logits.clone().requires_grad_(True)
    g0 = torch.tensor(0.01, device=dev)

    def run(x):
        loss, counts = ops.router_balance_loss(x, ids, mask)
        return loss.detach(), counts, torch.autograd.grad(loss, x, g0)[0]

    want = run(logits.clone().requires_grad_(True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(logits.clone().requires_grad_(True))
        warm = run(static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other)) and all(torch.equal(a, b) for a, b in zip(want, warm))
    del warm, other
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run(static)
    for i in range(4):
        with torch.no_grad():
            static.copy_(torch.randn(3000, 64, generator=torch.Generator().manual_seed(i)))
        g.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(kept, run(static.detach().clone().requires_grad_(True))))
