"""Rows in 8 bits with one scale each, the values back, and the RMS norm that
leaves its result in that form, against the definitions on the CPU."""

import int8_oracle as o
import pytest
import torch

from titan_amd import ops

BF, HF, F4 = o.BF, o.HF, o.F4
pytestmark = pytest.mark.gpu

# one element to rows past what a block keeps in registers, odd ones, whole and ragged vectors
SHAPES = [(1, 1), (3, 7), (2, 15), (5, 64), (130, 96), (1, 2048), (9, 1999), (4, 2560), (3, 4096), (33, 1000), (2, 8200),
          (1, 16384), (2, 20001), (1, 70000)]


def _rows(shape, dtype, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * (0.1 + torch.rand(shape[:-1], generator=g)).unsqueeze(-1) * size
    x[..., :: max(1, shape[-1] // 5)] *= 8
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF, HF, F4])
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize(dev, shape, dtype):
    x = _rows(shape, dtype, 1)
    q, s = ops.quantize(x.to(dev), mode="int8")
    wq, ws = o.quantize(x.float())
    assert q.dtype == torch.int8 and s.dtype == F4 and q.shape == x.shape and s.shape == x.shape[:-1]
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(q.cpu(), wq)
    for out in (BF, HF, F4):
        v = ops.dequantize(q, s, mode="int8", dtype=out)
        assert torch.equal(v.cpu(), (wq.float() * ws.unsqueeze(-1)).to(out))


def test_quantize_is_the_token_quantiser(dev):
    x = _rows((37, 1536), BF, 2).to(dev)
    for a, b in zip(ops.quantize(x, mode="int8"), ops.quantize_act_int8(x)):
        assert torch.equal(a, b)


def test_every_rounding_border(dev):
    """Values on, next to and between the borders of two codes."""
    for top in (127.0, 1.0, 3.7, 1e-30, 2e37):
        s = torch.tensor(top) / torch.tensor(127.0)
        half = (torch.arange(-126, 127).float() + 0.5) * s
        up = torch.nextafter(half, torch.tensor(float("inf")))
        down = torch.nextafter(half, torch.tensor(-float("inf")))
        x = torch.cat([torch.tensor([top]), half, up, down, -half, torch.tensor([0.0, -0.0, -top])]).unsqueeze(0)
        q, sc = ops.quantize(x.to(dev), mode="int8")
        wq, ws = o.quantize(x)
        assert torch.equal(sc.cpu(), ws) and torch.equal(q.cpu(), wq)


@pytest.mark.parametrize("dtype", [BF, HF, F4])
def test_odd_rows(dev, dtype):
    """Rows of zeros, of the least and the largest values, and with NaN and infinities: those alone are NaN."""
    x = _rows((9, 200), dtype, 3)
    info = torch.finfo(dtype)
    x[0] = 0.0
    x[1, 5] = float("nan")
    x[2, 199] = float("inf")
    x[3, 0] = -float("inf")
    x[4] = info.max
    x[5] = info.smallest_normal
    x[6] = -0.0
    x[7] = 0.0
    x[7, 3] = info.smallest_normal * info.eps  # the least subnormal: its scale vanishes or is the least
    q, s = ops.quantize(x.to(dev), mode="int8")
    wq, ws = o.quantize(x.float())
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(ws)) and torch.equal(s.cpu().nan_to_num(-1), ws.nan_to_num(-1))
    assert torch.equal(q.cpu(), wq)
    v = ops.dequantize(q, s, mode="int8", dtype=F4).cpu()
    assert torch.isnan(v[1:4]).all() and torch.isfinite(v[[0, 5, 6, 7, 8]]).all()
    # in fp32 the largest value M = 2^128 (1 - 2^-24) may read back as infinite: its scale, M / 127 rounded up by as much
    # as 2^-24 of itself, times 127 can be 2^128 (1 - 2^-25) or more
    assert torch.equal(v[4], wq[4].float() * ws[4]) and (dtype == F4 or torch.isfinite(v[4]).all())


def _check_norm(got, x, w, eps, r, dtype):
    h, v = o.rms_norm(x, w, eps, r)
    codes, scales, total, norm = (None if t is None else t.cpu() for t in got)
    if r is None:
        assert total is None
    else:
        assert total.dtype == dtype and torch.equal(total, h)
    top = v.abs().amax(-1)
    # v: 1 / rms and two products rounded to fp32; the scale: one division more.  Its squares are summed in 64 bits.
    assert bool(((scales.double() * 127 - top).abs() <= top * 4.1 * 2.0 ** -24 + 127 * 2.0 ** -149).all())
    exact = v / scales.double().unsqueeze(-1)
    exact[scales == 0] = 0.0
    assert bool(((codes.double() - exact).abs() <= 0.5 + 127.5 * 5 * 2.0 ** -24).all())
    if norm is not None:
        o.assert_rounded(norm, v)


@pytest.mark.parametrize("dtype", [BF, HF, F4])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm(dev, shape, dtype):
    x, r = _rows(shape, dtype, 4), _rows(shape, dtype, 5, 2.0)
    w = (1 + 0.2 * torch.randn(shape[-1], generator=torch.Generator().manual_seed(6))).to(dtype)
    for res, norm, weight in ((r, True, w), (r, False, w.float()), (None, True, None), (None, False, w)):
        got = ops.rms_norm_quantize(x.to(dev), None if weight is None else weight.to(dev), 1e-5,
                                    residual=None if res is None else res.to(dev), norm=norm)
        assert got.codes.dtype == torch.int8 and got.codes.shape == x.shape and got.scales.shape == x.shape[:-1]
        assert (got.norm is not None) == norm
        _check_norm(got, x, weight, 1e-5, res, dtype)


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 1000, 4097])
def test_norm_row_counts(dev, rows):
    """Each way of sharing rows out gives a row the same bits."""
    x, r = _rows((rows, 1024), BF, 7).to(dev), _rows((rows, 1024), BF, 8).to(dev)
    w = _rows((1024,), BF, 9).to(dev)
    all_ = ops.rms_norm_quantize(x, w, residual=r, norm=True)
    _check_norm(all_, x.cpu(), w.cpu(), 1e-6, r.cpu(), BF)
    for i in (0, rows // 2, rows - 1):
        one = ops.rms_norm_quantize(x[i], w, residual=r[i], norm=True)
        assert torch.equal(one.sum, all_.sum[i])
        _check_norm([t.unsqueeze(0) for t in one], x[i:i + 1].cpu(), w.cpu(), 1e-6, r[i:i + 1].cpu(), BF)


def test_norm_extremes(dev):
    """Values whose squares 32 bits do not hold, rows of zeros, and rows that hold no number."""
    x = _rows((8, 512), F4, 10)
    x[0] = 0.0
    x[1] *= 1e25
    x[2] *= 1e-25
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    x[5] = 0.0
    x[5, 100] = 1e30
    got = ops.rms_norm_quantize(x.to(dev), None, 0.0, norm=True)
    bad = [0, 3, 4]  # 0 / 0 with no eps, and what holds none
    assert torch.isnan(got.scales[bad].cpu()).all() and not got.codes[bad].any()
    good = [1, 2, 5, 6, 7]
    _check_norm([got.codes[good], got.scales[good], None, got.norm[good]], x[good], None, 0.0, None, F4)
    zero = ops.rms_norm_quantize(x[:1].to(dev), None, 1e-6, norm=True)
    assert not zero.codes.any() and not zero.scales.any() and not zero.norm.any()


@pytest.mark.parametrize("shape", [(2, 300), (2, 2048), (1, 70000)])
def test_norm_factors_past_32_bits(dev, shape):
    """Rows whose factor 1 / rms, or the precision of it, 32 bits do not hold; the norm itself is ordinary."""
    x = _rows(shape, F4, 15).clamp(-8, 8)
    for size in (2.0 ** -145, 2.0 ** -130, 2.0 ** -99, 2.0 ** 99, 2.0 ** 124):
        for dtype in (BF, F4) if size > 2.0 ** -133 else (F4,):  # bf16's least value
            v = (x * size).to(dtype)
            got = ops.rms_norm_quantize(v.to(dev), None, 0.0, norm=True)
            _check_norm(got, v, None, 0.0, None, dtype)


def test_layouts_types_and_empty(dev):
    x = _rows((4, 6, 130), BF, 11).to(dev)
    want = ops.quantize(x.contiguous(), mode="int8")
    for y in (x.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([x, x], -1)[..., :130],
              torch.cat([x.flatten().new_zeros(1), x.flatten()])[1:].reshape(x.shape)):
        got = ops.quantize(y, mode="int8")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        a, b = (ops.rms_norm_quantize(t, None, residual=t, norm=True) for t in (y, x))
        assert all(torch.equal(i, j) for i, j in zip(a, b))
    for shape in ((0, 64), (3, 0, 8)):
        q, s = ops.quantize(torch.zeros(shape, dtype=BF, device=dev), mode="int8")
        assert q.shape == shape and s.shape == shape[:-1]
        assert ops.dequantize(q, s, mode="int8").shape == shape
        n = ops.rms_norm_quantize(torch.zeros(shape, dtype=BF, device=dev), None, norm=True)
        assert n.codes.shape == shape and n.norm.shape == shape
    q, s = ops.quantize(torch.zeros(3, 0, dtype=BF, device=dev), mode="int8")
    assert q.shape == (3, 0) and s.tolist() == [0, 0, 0]
    with pytest.raises(ops.QmoeError):
        ops.rms_norm_quantize(torch.zeros(3, 0, dtype=BF, device=dev), None)


def test_rows_past_32_bits(dev):
    x = torch.zeros(2, 3, dtype=BF, device=dev)
    rows, K = 1 << 20, 4112  # 4.3 G elements
    big = torch.zeros(rows, K, dtype=BF, device=dev)
    big[-1] = torch.arange(K, device=dev) % 255 - 127
    q, s = ops.quantize(big, mode="int8")
    assert torch.equal(q[-1].cpu().float(), (torch.arange(K) % 255 - 127).float()) and s[-1].item() == 1.0
    assert not q[: rows // 2].any() and not s[:-1].any()
    del big
    v = ops.dequantize(q, s, mode="int8")
    assert torch.equal(v[-1].cpu().float(), (torch.arange(K) % 255 - 127).float())
    assert x.shape == (2, 3)


def test_streams_and_graph(dev):
    x, r, w = (_rows(s, BF, i).to(dev) for i, s in ((12, (64, 2048)), (13, (64, 2048)), (14, (2048,))))

    def run():
        n = ops.rms_norm_quantize(x, w, residual=r, norm=True)
        q, s = ops.quantize(n.sum, mode="int8")
        return (*n, q, s, ops.dequantize(q, s, mode="int8"))

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
        x.copy_(_rows((64, 2048), BF, 20 + i))
        g.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(kept, run()))


def test_refusals_on_the_gpu(dev):
    x = torch.zeros(2, 32, dtype=BF, device=dev)
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(ops.QmoeUnsupported, match="gradient"):
        ops.rms_norm_quantize(leaf, None)
    with pytest.raises(ops.QmoeUnsupported, match="gradient"):
        ops.rms_norm_quantize(x, None, residual=leaf)
    with pytest.raises(ops.QmoeUnsupported, match="gradient"):
        ops.rms_norm_quantize(x, leaf[0].detach().requires_grad_(True))
    q, s = ops.quantize(leaf, mode="int8")  # the codes of a layer's weight, say
    assert not q.requires_grad and not s.requires_grad
    with pytest.raises(ops.QmoeUnsupported, match="gradient"):
        ops.dequantize(q, s.requires_grad_(True), mode="int8")
    import torch.autograd.forward_ad as fw

    with fw.dual_level():
        for call in (lambda t: ops.quantize(t, mode="int8"), lambda t: ops.rms_norm_quantize(t, None)):
            with pytest.raises(NotImplementedError):
                call(fw.make_dual(x, x))
    with torch.no_grad():
        assert ops.rms_norm_quantize(leaf, None, residual=leaf).sum.shape == x.shape
    with pytest.raises(ops.QmoeUnsupported):
        ops.quantize(x.cpu(), mode="int8")
    with pytest.raises(ValueError):
        ops.rms_norm_quantize(x, None, float("nan"))


@pytest.mark.parametrize("rows,K,dtype", [(1, 5, BF), (700, 2048, BF), (3000, 1000, HF), (40, 4096, F4), (5, 20000, F4), (9, 0, BF), (0, 64, BF)])
@pytest.mark.parametrize("n,E", [(0, 3), (64, 1), (1000, 60), (5000, 256), (300, 700)])
def test_quantize_with_the_table_of_sorted_ids(dev, rows, K, dtype, n, E):
    """One launch for both: the bits of the two."""
    from titan_amd import _lib

    x = _rows((rows, K), dtype, 16).to(dev) if K else torch.zeros(rows, 0, dtype=dtype, device=dev)
    ids = torch.randint(-1, E + 1, (n,), generator=torch.Generator().manual_seed(n)).sort().values.int().to(dev)
    q, s = ops.quantize(x, mode="int8")
    t = ops.build_tiles(ids, E)
    codes, scales = torch.full_like(q, 99), torch.full_like(s, -1.0)
    tables = [torch.full_like(i, -7) for i in (t.offsets, t.tile_row, t.tile_exp, t.ntiles)]
    _lib.call("qmoe_int8_quantize_sorted", x.data_ptr(), ops._DTYPES[dtype], rows, K, codes.data_ptr(), scales.data_ptr(),
              ids.data_ptr(), n, E, ops.tile_rows(), *(i.data_ptr() for i in tables), t.maxt,
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(codes, q) and torch.equal(scales, s)
    assert all(torch.equal(a, b) for a, b in zip(tables, (t.offsets, t.tile_row, t.tile_exp, t.ntiles)))
