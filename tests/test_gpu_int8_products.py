"""Products of 8-bit integers with scales by token and channel, dense and by
expert, against the definition in 64 bits."""

import int8_oracle as o
import pytest
import torch

from titan_amd import ops

BF, HF, F4 = o.BF, o.HF, o.F4
pytestmark = pytest.mark.gpu


def _codes(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-128, 128, shape, generator=g).to(torch.int8),
            0.001 + 0.01 * torch.rand(shape[:-1], generator=g))


def _dense(dev, M, K, N, out=BF, seed=0):
    x, sx = _codes((M, K), seed)
    w, sw = _codes((N, K), seed + 1)
    y = ops.qqmm((x.to(dev), sx.to(dev)), w.to(dev), sw.to(dev), mode="int8", dtype=out)
    assert y.shape == (M, N) and y.dtype == out
    o.assert_rounded(y, o.product(x, sx, w, sw), what=(M, K, N))


@pytest.mark.parametrize("out", [BF, HF, F4])
@pytest.mark.parametrize("M", [1, 2, 4, 5, 16, 17, 33, 64, 65, 97, 128, 129, 300])
def test_dense_rows(dev, M, out):
    _dense(dev, M, 272, 301, out, M)


@pytest.mark.parametrize("M", [1, 3, 20, 70, 200])
@pytest.mark.parametrize("N,K", [(1, 16), (7, 32), (16, 48), (31, 2048), (33, 128), (64, 1040), (130, 144), (256, 64),
                                 (257, 4096), (520, 96), (1000, 256)])
def test_dense_shapes(dev, M, N, K):
    _dense(dev, M, K, N, BF, M + N)
    if N % 2:
        _dense(dev, M, K, N, F4, M + N)


@pytest.mark.parametrize("M,N,K", [(1024, 1024, 512), (700, 2100, 384), (2048, 640, 2048), (4096, 4096, 256), (520, 8192, 1152)])
def test_dense_large(dev, M, N, K):
    x, sx = _codes((M, K), 3)
    w, sw = _codes((N, K), 4)
    for out in (BF, F4):
        y = ops.qqmm((x.to(dev), sx.to(dev)), w.to(dev), sw.to(dev), mode="int8", dtype=out)
        o.assert_rounded(y, o.product(x, sx, w, sw), what=(M, K, N))


@pytest.mark.parametrize("K", [1, 15, 50, 1001])
def test_ragged_contractions(dev, K):
    for M in (1, 40, 130):
        _dense(dev, M, K, 65, BF, K)


def test_largest_sums(dev):
    """The longest contraction of the largest codes: 2^31 is just not reached."""
    K = 131056
    for M in (1, 5, 70):
        x = torch.full((M, K), -128, dtype=torch.int8)
        w = torch.full((3, K), -128, dtype=torch.int8)
        w[1] = 127
        s = torch.ones(M), torch.ones(3)
        y = ops.qqmm((x.to(dev), s[0].to(dev)), w.to(dev), s[1].to(dev), mode="int8", dtype=F4)
        assert torch.equal(y.cpu(), torch.tensor([K * 16384.0, -K * 128.0 * 127, K * 16384.0]).expand(M, 3).float())
    with pytest.raises(ops.QmoeUnsupported):
        ops.qqmm((torch.zeros(1, 131072, dtype=torch.int8, device=dev), torch.ones(1, device=dev)),
                 torch.zeros(1, 131072, dtype=torch.int8, device=dev), torch.ones(1, device=dev), mode="int8")


@pytest.mark.parametrize("M", [1, 30, 200])
def test_scales(dev, M):
    """Scales of zero, of either sign, far apart in size, infinite and NaN: each row and column by itself."""
    x, _ = _codes((M, 64), 5)
    w, _ = _codes((9, 64), 6)
    sx = torch.ones(M)
    sw = torch.tensor([1.0, 0.0, -2.0, 1e30, 1e-30, float("nan"), float("inf"), 1e-38, 3e38])
    for v in (1.0, 1e-32, 1e25, -1.0, 0.0, float("nan")):
        sx[0] = v
        y = ops.qqmm((x.to(dev), sx.to(dev)), w.to(dev), sw.to(dev), mode="int8", dtype=F4)
        acc = x.double() @ w.double().t()
        want = acc * torch.outer(sx.double(), sw.double())
        o.assert_rounded(y, want, what=(M, v))


@pytest.mark.parametrize("dtype", [BF, HF, F4])
def test_values_are_quantised_by_row(dev, dtype):
    x = torch.randn(2, 23, 128, generator=torch.Generator().manual_seed(7)).to(dtype)
    x[0, 3, 5] = float("nan")
    w, sw = _codes((70, 128), 8)
    q, s = o.quantize(x.float())
    y = ops.qqmm(x.to(dev), w.to(dev), sw.to(dev), mode="int8")
    assert y.dtype == dtype and y.shape == (2, 23, 70)
    o.assert_rounded(y.reshape(46, 70), o.product(q.reshape(46, 128), s.reshape(46), w, sw))
    assert torch.isnan(y[0, 3]).all() and torch.isfinite(y[0, :3]).all()
    pair = ops.quantize(x.to(dev), mode="int8")
    assert torch.equal(ops.qqmm(pair, w.to(dev), sw.to(dev), mode="int8", dtype=dtype).nan_to_num(7), y.nan_to_num(7))
    assert ops.qqmm(x.to(dev), w.to(dev), sw.to(dev), mode="int8", dtype=F4).dtype == F4


def test_empty_and_layouts(dev):
    w, sw = (t.to(dev) for t in _codes((40, 64), 9))
    x, sx = (t.to(dev) for t in _codes((6, 64), 10))
    want = ops.qqmm((x, sx), w, sw, mode="int8")
    assert ops.qqmm((x[:0], sx[:0]), w, sw, mode="int8").shape == (0, 40)
    assert ops.qqmm((x, sx), w[:0], sw[:0], mode="int8").shape == (6, 0)
    assert not ops.qqmm((x[:, :0], sx), w[:, :0], sw, mode="int8").any()
    assert torch.equal(ops.qqmm((x[0], sx[0]), w, sw, mode="int8"), want[0])
    wide = torch.cat([x, x], -1)
    assert torch.equal(ops.qqmm((wide[:, 64:], sx), w.t().contiguous().t(), sw, mode="int8"), want)
    off = torch.cat([x.new_zeros(1), x.flatten()])[1:].reshape(x.shape)
    assert torch.equal(ops.qqmm((off, torch.stack([sx, sx], 1)[:, 0]), w, sw, mode="int8"), want)
    assert torch.equal(ops.qqmm((x.reshape(2, 3, 64), sx.reshape(2, 3)), w, sw, mode="int8").reshape(6, 40), want)


# ------------------------------------------------------------------- experts


def _gather_oracle(x, sx, w, sw, rows, ids):
    out = torch.empty(ids.numel(), w.shape[1], dtype=torch.float64)
    for e in range(w.shape[0]):
        i = (ids == e).nonzero().flatten()
        out[i] = o.product(x[rows[i]], sx[rows[i]], w[e], sw[e])
    return out


@pytest.mark.parametrize("T,k,E,K,N", [(1, 1, 1, 16, 5), (1, 10, 16, 256, 100), (6, 4, 9, 144, 65), (7, 9, 30, 64, 8),
                                       (20, 4, 3, 272, 257), (64, 4, 60, 96, 96), (300, 3, 7, 128, 300), (500, 2, 200, 64, 40),
                                       (1200, 2, 8, 320, 264)])
@pytest.mark.parametrize("out", [BF, F4])
def test_experts(dev, T, k, E, K, N, out):
    """Unsorted, sorted with rows by index, and sorted with the routing's table."""
    g = torch.Generator().manual_seed(T)
    x, sx = _codes((T, K), 11)
    w, sw = _codes((E, N, K), 12)
    ids = torch.multinomial(torch.rand(E, generator=g).square() + 0.01, T * k, replacement=True, generator=g).reshape(T, k)
    want = _gather_oracle(x, sx, w, sw, torch.arange(T).repeat_interleave(k), ids.flatten())
    xd, sxd, wd, swd, idd = (t.to(dev) for t in (x, sx, w, sw, ids.int()))
    for i in (idd, idd.long()):
        y = ops.gather_qqmm((xd.reshape(T, 1, 1, K), sxd.reshape(T, 1, 1)), wd, swd, rhs_indices=i, mode="int8", dtype=out)
        assert y.shape == (T, k, 1, N) and y.dtype == out
        o.assert_rounded(y.reshape(T * k, N), want, what="unsorted")
    r = ops.route(idd, E)
    rows = torch.div(r.order, k, rounding_mode="floor").int()
    sorted_want = want[r.order.long().cpu()]
    for tiles in (None, r.tiles):
        y = ops.gather_qqmm((xd.unsqueeze(1), sxd.unsqueeze(1)), wd, swd, lhs_indices=rows, rhs_indices=r.sorted_ids,
                            mode="int8", sorted_indices=True, tiles=tiles, dtype=out)
        assert y.shape == (T * k, 1, N)
        o.assert_rounded(y.squeeze(1), sorted_want, what="sorted")
    xs = ops.sort_tokens(x.to(dev).float(), r.order, r.inv_order).to(torch.int8)  # a row of its own for every pair
    y = ops.gather_qqmm((xs.unsqueeze(1), sxd[rows.long()].unsqueeze(1)), wd, swd, rhs_indices=r.sorted_ids, mode="int8",
                        sorted_indices=True, dtype=out)
    o.assert_rounded(y.squeeze(1), sorted_want, what="rows of their own")


def test_experts_values_and_broadcasts(dev):
    """x quantised once per row; several rows per batch index; batches that broadcast; padding rows past the last."""
    g = torch.Generator().manual_seed(13)
    x = torch.randn(3, 2, 5, 64, generator=g).to(BF)
    w, sw = _codes((4, 24, 64), 14)
    ids = torch.randint(0, 4, (3, 2), generator=g)
    q, s = o.quantize(x.float())
    want = torch.stack([o.product(q[i, j], s[i, j], w[ids[i, j]], sw[ids[i, j]]) for i in range(3) for j in range(2)])
    y = ops.gather_qqmm(x.to(dev), w.to(dev), sw.to(dev), rhs_indices=ids.to(dev), mode="int8")
    assert y.shape == (3, 2, 5, 24) and y.dtype == BF
    o.assert_rounded(y.reshape(6, 5, 24), want)
    lhs = torch.tensor([[5, 0, 3], [1, 1, 4]])
    y = ops.gather_qqmm(x.reshape(6, 5, 64).to(dev), w.to(dev), sw.to(dev), lhs_indices=lhs.to(dev),
                        rhs_indices=torch.tensor([2, 0, 1]).to(dev), mode="int8")
    assert y.shape == (2, 3, 5, 24)
    q6, s6 = q.reshape(6, 5, 64), s.reshape(6, 5)
    for i in range(2):
        for j, e in enumerate((2, 0, 1)):
            o.assert_rounded(y[i, j], o.product(q6[lhs[i, j]], s6[lhs[i, j]], w[e], sw[e]))
    every = ops.gather_qqmm(x[0, :1].to(dev), w.to(dev), sw.to(dev), mode="int8")  # no indices: one expert after another
    assert every.shape == (4, 5, 24)
    for e in range(4):
        o.assert_rounded(every[e], o.product(q[0, 0], s[0, 0], w[e], sw[e]))


@pytest.mark.parametrize("n", [5, 80])
def test_indices_out_of_range_are_clamped(dev, n):
    x, sx = _codes((6, 1, 32), 15)
    w, sw = _codes((3, 20, 32), 16)
    g = torch.Generator().manual_seed(n)
    ids, rows = torch.randint(-3, 6, (n,), generator=g), torch.randint(-4, 12, (n,), generator=g)
    want = _gather_oracle(x[:, 0], sx[:, 0], w, sw, rows.clamp(0, 5), ids.clamp(0, 2))
    for t in (torch.int32, torch.int64):
        y = ops.gather_qqmm((x.to(dev), sx.to(dev)), w.to(dev), sw.to(dev), lhs_indices=rows.to(dev, t),
                            rhs_indices=ids.to(dev, t), mode="int8")
        o.assert_rounded(y.squeeze(1), want)
    order = torch.argsort(ids, stable=True)
    y = ops.gather_qqmm((x.to(dev), sx.to(dev)), w.to(dev), sw.to(dev), lhs_indices=rows[order].to(dev),
                        rhs_indices=ids[order].to(dev), mode="int8", sorted_indices=True)
    o.assert_rounded(y.squeeze(1), want[order])


def test_no_rows_and_no_experts(dev):
    w, sw = (t.to(dev) for t in _codes((3, 20, 32), 17))
    x = torch.zeros(4, 1, 32, dtype=BF, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    assert ops.gather_qqmm(x, w, sw, lhs_indices=none, rhs_indices=none, mode="int8").shape == (0, 1, 20)
    with pytest.raises(ValueError):
        ops.gather_qqmm(x, w[:0], sw[:0], rhs_indices=torch.zeros(4, dtype=torch.int32, device=dev), mode="int8")


def test_rows_behind_the_last_tile_stay(dev):
    """A table of fewer rows than the buffer: the C entry writes what the table holds and nothing behind it."""
    from titan_amd import _lib

    x, sx = (t.to(dev) for t in _codes((200, 64), 18))
    w, sw = (t.to(dev) for t in _codes((4, 48, 64), 19))
    ids = torch.sort(torch.randint(0, 4, (150,), generator=torch.Generator().manual_seed(1))).values.int().to(dev)
    t = ops.build_tiles(ids, 4)
    out = torch.full((200, 48), 7.0, dtype=BF, device=dev)
    _lib.call("qmoe_int8_gather_qqmm", x.data_ptr(), sx.data_ptr(), 200, None, 150, w.data_ptr(), sw.data_ptr(), 4, 48, 64,
              t.offsets.data_ptr(), t.tile_row.data_ptr(), t.tile_exp.data_ptr(), t.ntiles.data_ptr(), t.maxt, 0,
              out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert bool((out[150:] == 7).all())
    o.assert_rounded(out[:150], _gather_oracle(x.cpu(), sx.cpu(), w.cpu(), sw.cpu(), torch.arange(150), ids.cpu().long()))


def test_weights_past_4_gb(dev):
    E, N, K = 70, 4096, 16384  # 4.7 GB
    w = torch.zeros(E, N, K, dtype=torch.int8, device=dev)
    sw = torch.ones(E, N, device=dev)
    g = torch.Generator(device=dev).manual_seed(20)
    for e in (0, 69):
        w[e] = torch.randint(-127, 128, (N, K), generator=g, device=dev, dtype=torch.int8)
    x, sx = _codes((100, K), 21)
    xd, sxd = x.to(dev).unsqueeze(1), sx.to(dev).unsqueeze(1)
    for n in (3, 100):
        ids = torch.tensor([0] * (n // 3) + [69] * (n - n // 3), dtype=torch.int32, device=dev)
        y = ops.gather_qqmm((xd[:n], sxd[:n]), w, sw, rhs_indices=ids, mode="int8", sorted_indices=True, dtype=F4).squeeze(1)
        i = torch.cat([torch.arange(5), torch.arange(4091, 4096)])
        for r in (0, n - 1):
            e = int(ids[r])
            o.assert_rounded(y[r:r + 1, i.to(dev)], o.product(x[r:r + 1], sx[r:r + 1], w[e, i.to(dev)].cpu(), torch.ones(10)))


def test_results_past_4_g_elements(dev):
    M, N, K = 70000, 65600, 16
    x, sx = _codes((M, K), 22)
    w, sw = _codes((N, K), 23)
    y = ops.qqmm((x.to(dev), sx.to(dev)), w.to(dev), sw.to(dev), mode="int8")
    for r in (0, 65535, 65537, M - 1):
        o.assert_rounded(y[r:r + 1], o.product(x[r:r + 1], sx[r:r + 1], w, sw))


def test_streams_graph_and_repeats(dev):
    """A captured layer's products, replayed with the program's own work between, and the same bits on every run."""
    x, sx = (t.to(dev) for t in _codes((300, 512), 24))
    w, sw = (t.to(dev) for t in _codes((8, 256, 512), 25))
    ids = torch.sort(torch.randint(0, 8, (300,), generator=torch.Generator().manual_seed(2))).values.int().to(dev)
    v = torch.randn(300, 512, device=dev).to(BF)

    def run():
        return (ops.gather_qqmm((x.unsqueeze(1), sx.unsqueeze(1)), w, sw, rhs_indices=ids, mode="int8", sorted_indices=True),
                ops.gather_qqmm(v[:9].unsqueeze(1), w, sw, rhs_indices=ids[:9], mode="int8"),
                ops.qqmm(v, w[0], sw[0], mode="int8"), ops.qqmm(v[:20], w[1], sw[1], mode="int8"),
                ops.qqmm(v[:1], w[1], sw[1], mode="int8"))

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for i in range(4):
        v.copy_(torch.randn(300, 512, generator=torch.Generator().manual_seed(30 + i)).to(BF))
        g.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(kept, run()))


def test_gradients_and_recorders_are_refused(dev):
    x = torch.randn(4, 64, device=dev).to(BF).requires_grad_(True)
    w, sw = (t.to(dev) for t in _codes((16, 64), 26))
    for call in (lambda t, s: ops.qqmm(t, w, s, mode="int8"),
                 lambda t, s: ops.gather_qqmm(t.unsqueeze(1), w.unsqueeze(0), s.unsqueeze(0), mode="int8",
                                              rhs_indices=torch.zeros(4, dtype=torch.int32, device=dev))):
        with pytest.raises(ops.QmoeUnsupported, match="gradient"):
            call(x, sw)
        with pytest.raises(ops.QmoeUnsupported, match="gradient"):
            call(x.detach(), sw.clone().requires_grad_(True))
        with torch.no_grad():
            assert call(x, sw).shape[-1] == 16
    with pytest.raises(ops.QmoeUnsupported, match="trace"):
        torch.jit.trace(lambda t: ops.qqmm(t, w, sw, mode="int8"), (x.detach(),))
    import torch.autograd.forward_ad as fw

    with fw.dual_level(), pytest.raises(NotImplementedError):
        ops.qqmm(fw.make_dual(x.detach(), x.detach()), w, sw, mode="int8")


@pytest.mark.parametrize("dtype", [BF, HF, F4])
@pytest.mark.parametrize("K", [16, 112, 1024, 2048, 4096, 6160, 16384, 20480])
def test_values_quantised_in_the_product(dev, K, dtype):
    """Few rows of values: the codes, and so the bits, of the product of rows quantised before."""
    g = torch.Generator().manual_seed(K)
    x = (torch.randn(4, K, generator=g) * torch.tensor([1.0, 30.0, 1e-3, 0.0]).unsqueeze(-1)).to(dtype)
    x[1, K // 2] = float("inf")
    w, sw = (t.to(dev) for t in _codes((3, 21, K), 27))
    pair = ops.quantize(x.to(dev), mode="int8")
    for m in (1, 4):
        a = ops.qqmm(x[:m].to(dev), w[0], sw[0], mode="int8", dtype=F4)
        b = ops.qqmm((pair[0][:m], pair[1][:m]), w[0], sw[0], mode="int8", dtype=F4)
        assert torch.equal(a.nan_to_num(7), b.nan_to_num(7)) and torch.equal(torch.isnan(a), torch.isnan(b))
    ids = torch.tensor([[0, 2], [1, 1], [2, 0], [0, 1]], dtype=torch.int32, device=dev)
    a = ops.gather_qqmm(x.reshape(4, 1, 1, K).to(dev), w, sw, rhs_indices=ids, mode="int8")
    b = ops.gather_qqmm((pair[0].reshape(4, 1, 1, K), pair[1].reshape(4, 1, 1)), w, sw, rhs_indices=ids, mode="int8", dtype=dtype)
    assert a.dtype == dtype and torch.equal(a.nan_to_num(7), b.nan_to_num(7))
    assert torch.isnan(a[1]).all() and not a[3].any()


@pytest.mark.parametrize("E,n,N,K", [(1100, 1500, 40, 32),   # more tiles than are ranked
                                     (300, 2000, 1030, 64),  # four rounds of units and more: every second XCD's order reversed
                                     (2, 3000, 333, 144)])   # pairs of tiles
@pytest.mark.parametrize("out", [BF, HF, F4])
def test_orders_of_units(dev, E, n, N, K, out):
    g = torch.Generator().manual_seed(n)
    x, sx = _codes((90, K), 28)
    w, sw = _codes((E, N, K), 29)
    ids, rows = torch.randint(0, E, (n,), generator=g).sort().values, torch.randint(0, 90, (n,), generator=g)
    y = ops.gather_qqmm((x.to(dev).unsqueeze(1), sx.to(dev).unsqueeze(1)), w.to(dev), sw.to(dev), lhs_indices=rows.to(dev),
                        rhs_indices=ids.to(dev), mode="int8", sorted_indices=True, dtype=out)
    o.assert_rounded(y.squeeze(1), _gather_oracle(x, sx, w, sw, rows, ids))


@pytest.mark.parametrize("M,N,K", [(96, 5700, 48),    # blocks of few rows, the most of them
                                   (100, 9001, 80),   # 64 x 128
                                   (520, 4100, 400),  # 128 x 128
                                   (1030, 4098, 272), # 128 x 256
                                   (4000, 4091, 144)])  # 256 x 256
def test_dense_forms(dev, M, N, K):
    """Each form of a unit with odd rows and columns, in every type."""
    for out in (BF, HF, F4):
        _dense(dev, M, K, N, out, M)


def test_a_table_larger_than_its_buffers(dev):
    """More tiles than there is room for: those that fit are computed, nothing is read behind them."""
    from titan_amd import _lib

    x, sx = (t.to(dev) for t in _codes((256, 64), 31))
    w, sw = (t.to(dev) for t in _codes((2, 48, 64), 32))
    t = ops.build_tiles(torch.tensor([0] * 128 + [1] * 128, dtype=torch.int32, device=dev), 2)
    out = torch.full((256, 48), 7.0, dtype=BF, device=dev)
    _lib.call("qmoe_int8_gather_qqmm", x.data_ptr(), sx.data_ptr(), 256, None, 256, w.data_ptr(), sw.data_ptr(), 2, 48, 64,
              t.offsets.data_ptr(), t.tile_row.data_ptr(), t.tile_exp.data_ptr(), t.ntiles.data_ptr(), 1, 0,
              out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    ids = torch.tensor([0] * 128)
    o.assert_rounded(out[:128], _gather_oracle(x.cpu(), sx.cpu(), w.cpu(), sw.cpu(), torch.arange(128), ids))
    assert bool((out[128:] == 7).all())


def test_calls_of_two_threads(dev):
    """Each on a stream of its own: no state is shared."""
    import threading

    w, sw = (t.to(dev) for t in _codes((8, 256, 512), 33))
    v = [torch.randn(200, 512, generator=torch.Generator().manual_seed(40 + i)).to(dev, BF) for i in range(2)]
    ids = [torch.randint(0, 8, (200,), generator=torch.Generator().manual_seed(50 + i)).sort().values.to(dev) for i in range(2)]
    logits = [torch.randn(5000, 64, generator=torch.Generator().manual_seed(60 + i)).to(dev) for i in range(2)]

    def run(i):
        n = ops.rms_norm_quantize(v[i], None, residual=v[i])
        return (ops.qqmm(n, w[i], sw[i], mode="int8"), ops.qqmm(v[i][:3], w[i], sw[i], mode="int8"),
                ops.gather_qqmm(v[i].unsqueeze(1), w, sw, rhs_indices=ids[i], mode="int8", sorted_indices=True),
                *ops.router_balance_loss(logits[i], ids[i][:100].repeat(50).reshape(5000, 1)))

    want = [run(i) for i in range(2)]
    got, streams = [None, None], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(30):
                got[i] = run(i)
            streams[i].synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(want[i], got[i]))


def test_more_rounds_of_units_than_are_planned_at_once(dev):
    """80 rounds of a table's units on 256 CUs."""
    E, n, N, K = 1000, 1300, 5120, 16
    g = torch.Generator().manual_seed(34)
    x, sx = _codes((50, K), 35)
    w, sw = _codes((E, N, K), 36)
    ids, rows = torch.cat([torch.arange(E), torch.randint(0, E, (n - E,), generator=g)]).sort().values, torch.randint(0, 50, (n,), generator=g)
    y = ops.gather_qqmm((x.to(dev).unsqueeze(1), sx.to(dev).unsqueeze(1)), w.to(dev), sw.to(dev), lhs_indices=rows.to(dev),
                        rhs_indices=ids.to(dev), mode="int8", sorted_indices=True, dtype=F4)
    o.assert_rounded(y.squeeze(1), _gather_oracle(x, sx, w, sw, rows, ids))


@pytest.mark.parametrize("E,n,N,K", [(6, 700, 300, 272),    # half tiles by 128 columns
                                     (5, 6000, 333, 144),   # tiles by 128
                                     (3, 9000, 500, 64),    # tiles by 256
                                     (3, 20000, 600, 48)])  # pairs of tiles by 256
def test_units_of_tables(dev, E, n, N, K):
    """Each shape of a table's units, with experts of every share of rows and one without, in every type."""
    g = torch.Generator().manual_seed(n)
    x, sx = _codes((900, K), 37)
    w, sw = _codes((E, N, K), 38)
    p = torch.linspace(0, 1, E)  # expert 0: no rows
    ids, rows = torch.multinomial(p, n, replacement=True, generator=g).sort().values, torch.randint(0, 900, (n,), generator=g)
    want = _gather_oracle(x, sx, w, sw, rows, ids)
    for out in (BF, HF, F4):
        y = ops.gather_qqmm((x.to(dev).unsqueeze(1), sx.to(dev).unsqueeze(1)), w.to(dev), sw.to(dev), lhs_indices=rows.to(dev),
                            rhs_indices=ids.to(dev), mode="int8", sorted_indices=True, dtype=out)
        o.assert_rounded(y.squeeze(1), want, what=out)


def test_tables_that_do_not_fit(dev):
    """A table for other rows is made anew; one whose tensors are too short, of another type or of another device is refused."""
    import dataclasses

    x, sx = (t.to(dev) for t in _codes((100, 1, 64), 39))
    w, sw = (t.to(dev) for t in _codes((4, 48, 64), 40))
    ids = torch.randint(0, 4, (100,), generator=torch.Generator().manual_seed(3)).sort().values.int().to(dev)

    def call(t, i=ids):
        return ops.gather_qqmm((x[:i.numel()], sx[:i.numel()]), w, sw, rhs_indices=i, mode="int8", sorted_indices=True, tiles=t)

    want, table = call(None), ops.build_tiles(ids, 4)
    assert torch.equal(call(table), want) and torch.equal(call(table, ids[:70]), want[:70])
    assert torch.equal(call(table, ids.long()), want) and torch.equal(call(table, ids[:9]), want[:9])
    for change in ({"tile_row": table.tile_row[:1]}, {"tile_exp": table.tile_exp.long()}, {"offsets": table.offsets[:4]},
                   {"ntiles": table.ntiles[:0]}, {"maxt": 0}, {"tile_row": table.tile_row.cpu()}):
        with pytest.raises(RuntimeError, match="tile table"):
            call(dataclasses.replace(table, **change))
    with pytest.raises(ValueError, match="tile table"):
        call(dataclasses.replace(table, num_experts=5))
    with pytest.raises(ValueError, match="tile table"):
        call(dataclasses.replace(table, tile_rows=64))


@pytest.mark.parametrize("M", [2, 3, 5, 8, 16, 17])
@pytest.mark.parametrize("N,K", [(301, 272), (4099, 2080), (9, 16384), (2000, 1040), (70, 16400)])
def test_few_rows_of_values(dev, M, N, K):
    """However few rows of values are taken, the bits of the product of the rows quantised before."""
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dev, BF)
    w, sw = (t.to(dev) for t in _codes((N, K), 41))
    q, s = ops.quantize(x, mode="int8")
    y = ops.qqmm(x, w, sw, mode="int8")
    assert torch.equal(y, ops.qqmm((q, s), w, sw, mode="int8"))
    i = torch.tensor([0, N // 2, N - 1])
    o.assert_rounded(y[:, i.to(dev)], o.product(q.cpu(), s.cpu(), w[i.to(dev)].cpu(), sw[i.to(dev)].cpu()))
