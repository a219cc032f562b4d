"""Indices outside their range in the mxfp4 gather calls, on the GPU: clamped, few
rows and many, forward and backward, whatever brings them."""

import pytest
import torch

from mx_helpers import check_sum, codes, dequantize_ref, quantize_ref
from titan_amd import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def say(*a):
    print("[mxfp4 indices]", *a, flush=True)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _by_expert(x, W, e):
    """x [n, M, C] times W[e] [C, O], and the sum of magnitudes, in 64 bits on the CPU."""
    x, V = x.detach().cpu().double(), W[e]
    return x @ V, x.abs() @ V.abs()


@pytest.mark.parametrize("is_sorted", [False, True])
@pytest.mark.parametrize("M,n", [(2, 5), (2, 50), (40, 7)])
def test_batches_of_several_rows(dev, M, n, is_sorted):
    say("batches", M, n, is_sorted)
    g = _gen(M + n)
    B, E, K, N = 6, 4, 64, 40
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s).transpose(1, 2)
    e = torch.randint(-2, E + 2, (n,), generator=g)
    e = torch.sort(e)[0] if is_sorted else e
    lhs = torch.randint(-3, B + 3, (n,), generator=g)
    lhs[:2] = torch.tensor([-1, B])
    x = torch.randn(B, M, K, generator=g).to(BF)
    xi, ei = lhs.clamp(0, B - 1), e.clamp(0, E - 1)
    xd = x.to(dev).requires_grad_(True)
    kw = {"lhs_indices": lhs.to(dev), "rhs_indices": e.to(dev), "sorted_indices": is_sorted}
    y = ops.gather_qmm(xd, w.to(dev), s.to(dev), mode="mxfp4", **kw)
    check_sum(y, *_by_expert(x[xi], W, ei), K)
    q = ops.gather_qqmm(xd.detach(), w.to(dev), s.to(dev), **kw)
    check_sum(q, *_by_expert(quantize_ref(x)[0][xi], W, ei), K)
    dy = torch.randn(n, M, N, generator=g).to(BF)
    (dx,) = torch.autograd.grad(y, xd, dy.to(dev))
    ref, mag = _by_expert(dy, W.transpose(1, 2), ei)
    zero = torch.zeros(B, M, K, dtype=torch.float64)
    check_sum(dx, zero.index_add(0, xi, ref), zero.index_add(0, xi, mag), N + n)


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32, torch.uint64])
@pytest.mark.parametrize("n", [5, 90])
def test_past_32_bits(dev, n, dtype):
    say("past 32 bits", n, dtype)
    g = _gen(n)
    E, K, N = 4, 64, 40
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s).transpose(1, 2)
    x = torch.randn(n, 1, K, generator=g).to(BF)
    far = (1 << 31) + 1 if dtype == torch.uint32 else (1 << 32) + 1
    e = torch.sort(torch.randint(0, E, (n,), generator=g))[0]
    lhs = torch.randint(0, n, (n,), generator=g)
    e[-2:] = far
    lhs[1] = far
    xi, ei = lhs.clamp(0, n - 1), e.clamp(0, E - 1)
    for is_sorted in (True, False):
        kw = {"lhs_indices": lhs.to(dtype).to(dev), "rhs_indices": e.to(dtype).to(dev), "sorted_indices": is_sorted}
        check_sum(ops.gather_qmm(x.to(dev), w.to(dev), s.to(dev), mode="mxfp4", **kw), *_by_expert(x[xi], W, ei), K)
        check_sum(ops.gather_qqmm(x.to(dev), w.to(dev), s.to(dev), **kw), *_by_expert(quantize_ref(x)[0][xi], W, ei), K)


@pytest.mark.parametrize("n", [64, 300])
def test_with_a_table_of_the_callers(dev, n):
    """Rows whose ids are out of range are in the table too: computed, none left as its memory was."""
    say("table", n)
    g = _gen(n)
    E, K, N = 4, 64, 40
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s).transpose(1, 2)
    x, dy = torch.randn(n, 1, K, generator=g).to(BF), torch.randn(n, 1, N, generator=g).to(BF)
    for e in (torch.sort(torch.randint(-3, E + 3, (n,), generator=g))[0], torch.full((n,), -1), torch.full((n,), E),
              torch.cat([torch.zeros(n - 2, dtype=torch.int64), torch.tensor([1 << 31, (1 << 32) + 1])])):
        ei = e.clamp(0, E - 1)
        for ids in (e, e.clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32)):
            tiles = ops.build_tiles(ids.to(dev), E)
            for width in (N, K):  # what the results' memory held before
                torch.full((n, width), float("nan"), dtype=BF, device=dev)
            xd = x.to(dev).requires_grad_(True)
            y = ops.gather_qmm(xd, w.to(dev), s.to(dev), rhs_indices=ids.to(dev), mode="mxfp4", sorted_indices=True, tiles=tiles)
            check_sum(y, *_by_expert(x, W, ei), K)
            (dx,) = torch.autograd.grad(y, xd, dy.to(dev))
            check_sum(dx, *_by_expert(dy, W.transpose(1, 2), ei), N)
            q = ops.gather_qqmm(x.to(dev), w.to(dev), s.to(dev), rhs_indices=ids.to(dev), sorted_indices=True, tiles=tiles)
            check_sum(q, *_by_expert(quantize_ref(x)[0], W, ei), K)


def test_a_table_covers_every_row(dev):
    say("tables")
    for ids, E in (([-5, -1, 0, 2, 2, 3, 9], 4), ([7] * 130, 3), ([-1] * 130, 3), ([], 3), ([1, 1], 1)):
        t = ops.build_tiles(torch.tensor(ids, dtype=torch.int32, device=dev), E)
        inside = torch.tensor(ids, dtype=torch.int64).clamp(0, E - 1)
        want = torch.searchsorted(inside, torch.arange(E + 1))
        assert t.offsets.tolist() == want.tolist()
        k = int(t.ntiles)
        rows = [(int(r) + i, int(x)) for r, x in zip(t.tile_row[:k], t.tile_exp[:k])
                for i in range(min(t.tile_rows, int(want[int(x) + 1]) - int(r)))]
        assert rows == list(enumerate(inside.tolist()))


@pytest.mark.parametrize("count", [0, 1, 255, 256, 5000])
def test_narrowed_ids(dev, count):
    """int64 ids in memory of every order: as they are, strided, expanded, of several dimensions."""
    say("narrow", count)
    g = _gen(count)
    v = torch.randint(-(1 << 62), 1 << 62, (count,), generator=g) >> torch.randint(0, 63, (count,), generator=g)
    for n in (0, 1, 7, 1 << 20, (1 << 31) - 1, 1 << 31):
        t = v.to(dev)
        for s in (t, torch.stack([t, t], 1)[:, 1], t[None].expand(2, -1), t.reshape(1, -1, 1)):
            got = ops._narrow(s, n)
            assert got.dtype == torch.int32 and got.shape == s.shape
            assert torch.equal(got.cpu().long(), s.cpu().clamp(0, min(max(n - 1, 0), (1 << 31) - 1)))


def test_int64_ids_in_a_graph(dev):
    say("graph")
    g = _gen(1)
    E, K, N = 6, 64, 40
    w, s = (t.to(dev) for t in codes(g, E, N, K))
    W = dequantize_ref(w, s).transpose(1, 2)
    x, ids = torch.randn(9, 1, K, generator=g).to(BF).to(dev), torch.zeros(9, dtype=torch.int64, device=dev)

    def step():
        return ops.gather_qmm(x, w, s, rhs_indices=ids, mode="mxfp4"), ops.gather_qqmm(x, w, s, rhs_indices=ids)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        new = torch.randint(-2, E + 2, (9,), generator=_gen(seed))
        new[seed] = (1 << 32) + 1
        ids.copy_(new)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed
        check_sum(want[0], *_by_expert(x, W, new.clamp(0, E - 1)), K)
