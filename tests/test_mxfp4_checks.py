"""What the mxfp4 operators and the token sort refuse, before any launch: CPU
tensors with the device check taken out, a launch counted as a failure."""

import pytest
import torch

from titan_amd import _lib, mxfp4, ops
from titan_amd.ops import QmoeUnsupported

BF = torch.bfloat16
_lib_binding = _lib.binding


class Binding:
    """Declines every call that may be declined, and counts the others as launches."""

    def __getattr__(self, name):
        def call(*args):
            if args[-1] is False and name != "rows_product" or name == "gather":
                return None
            raise AssertionError(f"{name} launched")

        return call


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    def launch(name, *args):
        raise AssertionError(f"{name} launched")

    monkeypatch.setattr(ops, "_dev", lambda t, name: None)
    monkeypatch.setattr(ops, "_stream", lambda t: 0)
    monkeypatch.setattr(ops, "tile_rows", lambda: 128)
    monkeypatch.setattr(_lib, "call", launch)
    monkeypatch.setattr(_lib, "binding", lambda: Binding())


def _w(*shape):
    return torch.zeros(*shape[:-1], shape[-1] // 8, dtype=torch.int32), torch.zeros(*shape[:-1], shape[-1] // 32, dtype=torch.uint8)


def test_quantize():
    x = torch.zeros(2, 64)
    for bad in (x.double(), x.int(), torch.zeros(2, 63), torch.zeros(2, 48), torch.tensor(1.0)):
        with pytest.raises(QmoeUnsupported):
            ops.quantize(bad)
    for kw in ({"mode": "affine"}, {"group_size": 64}, {"bits": 8}):
        with pytest.raises(QmoeUnsupported):
            ops.quantize(x, **kw)
    with pytest.raises(AssertionError, match="launched"):
        ops.quantize(x, 32, 4, "mxfp4")


def test_dequantize():
    w, s = _w(3, 64)
    with pytest.raises(ValueError, match="biases"):
        ops.dequantize(w, s, s, mode="mxfp4")
    with pytest.raises(ValueError, match="disagree"):
        ops.dequantize(w, s[:, :1], mode="mxfp4")
    with pytest.raises(ValueError, match="disagree"):
        ops.dequantize(w[:, :6], s, mode="mxfp4")
    with pytest.raises(QmoeUnsupported):
        ops.dequantize(w, s.to(torch.int8), mode="mxfp4")
    with pytest.raises(QmoeUnsupported):
        ops.dequantize(w, s, mode="mxfp4", dtype=torch.float64)
    with pytest.raises(QmoeUnsupported):
        ops.dequantize(w, s, mode="mxfp4", group_size=64)
    with pytest.raises(QmoeUnsupported):
        ops.dequantize(w, s, mode="nvfp4")
    with pytest.raises(AssertionError, match="launched"):
        ops.dequantize(w, s, mode="mxfp4", group_size=32)


@pytest.mark.parametrize("op", [ops.quantized_matmul, ops.qqmm])
def test_dense(op):
    w, s = _w(5, 64)
    x = torch.zeros(3, 64, dtype=BF)
    kw = {"mode": "mxfp4"}
    for bad in (x.float(), x.half()):
        with pytest.raises(QmoeUnsupported, match="bfloat16"):
            op(bad, w, s, **kw)
    for bad in (x[:, :32], torch.zeros(3, 96, dtype=BF), torch.tensor(0.0, dtype=BF)):
        with pytest.raises(ValueError, match="fit"):
            op(bad, w, s, **kw)
    with pytest.raises(QmoeUnsupported):
        op(x, w.float(), s, **kw)
    with pytest.raises(QmoeUnsupported):
        op(x, w[None], s[None], **kw)
    with pytest.raises(ValueError, match="disagree"):
        op(x, w, s[:4], **kw)
    for more in ({"group_size": 64}, {"bits": 8}):
        with pytest.raises(QmoeUnsupported):
            op(x, w, s, **kw, **more)
    with pytest.raises(QmoeUnsupported):
        op(x, w, s, mode="mxfp8")
    with pytest.raises(AssertionError, match="launched"):
        op(x, w, s, **kw)


def test_dense_transposed():
    w, s = _w(5, 64)
    with pytest.raises(ValueError, match="fit"):
        ops.quantized_matmul(torch.zeros(3, 64, dtype=BF), w, s, transpose=False, mode="mxfp4")
    with pytest.raises(ValueError, match="biases"):
        ops.quantized_matmul(torch.zeros(3, 64, dtype=BF), w, s, s, mode="mxfp4")
    with pytest.raises(AssertionError, match="launched"):
        ops.quantized_matmul(torch.zeros(3, 5, dtype=BF), w, s, transpose=False, mode="mxfp4")


def test_affine_calls_are_refused_as_before():
    w, s = _w(5, 64)
    x = torch.zeros(3, 64, dtype=BF)
    for call in (lambda **k: ops.quantized_matmul(x, w, s, **k), lambda **k: ops.gather_qmm(x, w[None], s[None], **k),
                 lambda **k: ops.dequantize(w, s, **k)):
        with pytest.raises(QmoeUnsupported, match="biases"):
            call()
        with pytest.raises(QmoeUnsupported, match="mode"):
            call(mode="mxfp8")


@pytest.mark.parametrize("op", [ops.gather_qmm, ops.gather_qqmm])
def test_gather(op):
    w, s = _w(4, 5, 64)
    x = torch.zeros(3, 1, 64, dtype=BF)
    ids = torch.zeros(3, dtype=torch.int32)
    kw = {"mode": "mxfp4"}
    with pytest.raises(QmoeUnsupported):
        op(x, w[0], s[0], rhs_indices=ids, **kw)
    with pytest.raises(ValueError, match="fit"):
        op(x[..., :32], w, s, rhs_indices=ids, **kw)
    with pytest.raises(ValueError, match="2-D"):
        op(x[0, 0], w, s, rhs_indices=ids, **kw)
    for bad in (ids.float(), ids.bool(), [0, 0, 0]):
        with pytest.raises(TypeError, match="rhs_indices"):
            op(x, w, s, rhs_indices=bad, **kw)
        with pytest.raises(TypeError, match="lhs_indices"):
            op(x, w, s, lhs_indices=bad, rhs_indices=ids, **kw)
    with pytest.raises(ValueError, match="broadcast"):
        op(x, w, s, rhs_indices=ids[:2], **kw)
    with pytest.raises(ValueError, match="no activation rows"):
        op(x[:0], w, s, lhs_indices=ids, rhs_indices=ids, **kw)
    with pytest.raises(ValueError, match="no experts"):
        op(x, w[:0], s[:0], rhs_indices=ids, **kw)
    with pytest.raises(QmoeUnsupported):
        op(x, w, s, rhs_indices=ids, group_size=64, **kw)
    n = 70
    i32 = torch.zeros(6, dtype=torch.int32)
    table = ops.TileTable(i32, i32, i32, i32[:1], 6, 128, 5, n)  # of five experts
    with pytest.raises(ValueError, match="tile table"):
        op(torch.zeros(n, 1, 64, dtype=BF), w, s, rhs_indices=torch.zeros(n, dtype=torch.int32), sorted_indices=True,
           tiles=table, **kw)
    with pytest.raises(AssertionError, match="launched"):
        op(x, w, s, rhs_indices=ids, **kw)


def test_sort_tokens():
    x, od = torch.zeros(3, 8), torch.arange(6, dtype=torch.int32)
    for bad in (x.double(), x.int()):
        with pytest.raises(QmoeUnsupported):
            ops.sort_tokens(bad, od, od)
    for args in ((x[0], od, od), (x, od[:5], od[:5]), (x, od, od[:3]), (x[:0], od, od)):
        with pytest.raises(ValueError):
            ops.sort_tokens(*args)
    with pytest.raises(TypeError):
        ops.sort_tokens(x, od.float(), od)
    with pytest.raises(AssertionError, match="launched"):
        ops.sort_tokens(x, od, od)


def test_unsort_tokens():
    xs, od, sc = torch.zeros(6, 8), torch.arange(6, dtype=torch.int32), torch.zeros(3, 2)
    for args in ((xs[:5], od, od, sc), (xs, od[:5], od, sc), (xs, od, od[:5], sc), (xs, od, od, sc[:2]),
                 (xs, od, od, sc.reshape(-1))):
        with pytest.raises(ValueError):
            ops.unsort_tokens(*args)
    with pytest.raises(QmoeUnsupported):
        ops.unsort_tokens(xs.double(), od, od, sc)
    with pytest.raises(AssertionError, match="launched"):
        ops.unsort_tokens(xs, od, od, sc)


def test_bad_arguments_at_the_entry_points():
    """Wrong sizes and pointers are errors at the C boundary too, before any device call."""
    L = _lib.load()
    one = 4096  # any aligned address: nothing is read
    INV, UNS = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED
    assert L.qmoe_mxfp4_quantize(None, 0, 2, 64, one, one, None) == INV
    assert L.qmoe_mxfp4_quantize(one, 3, 2, 64, one, one, None) == UNS
    assert L.qmoe_mxfp4_quantize(one, 0, 2, 48, one, one, None) == UNS
    assert L.qmoe_mxfp4_quantize(one + 2, 0, 2, 64, one, one, None) == UNS
    assert L.qmoe_mxfp4_quantize(one, 0, -1, 64, one, one, None) == INV
    assert L.qmoe_mxfp4_quantize(one, 0, 1 << 60, 64, one, one, None) == UNS
    assert L.qmoe_mxfp4_quantize(None, 0, 0, 64, None, None, None) == _lib.OK
    assert L.qmoe_mxfp4_dequantize(one, None, 2, 64, 0, one, None) == INV

    def qmv(x=one, n_x=4, ldx=64, div=1, n=4, E=1, N=8, K=64, tr=1, dt=0, out=one):
        return L.qmoe_mxfp4_gather_qmv(x, n_x, ldx, None, div, None, n, one, one, E, N, K, tr, dt, out, None)

    assert qmv(x=None) == INV and qmv(n_x=0) == INV and qmv(ldx=32) == INV and qmv(div=0) == INV and qmv(E=0) == INV
    assert qmv(K=40) == UNS and qmv(dt=1) == UNS and qmv(n=70000) == UNS and qmv(x=one + 2) == UNS
    assert qmv(tr=0, ldx=7) == INV and qmv(n=0) == _lib.OK and qmv(N=0) == _lib.OK and qmv(K=0) == INV

    def qmm(x=one, n_x=4, ldx=64, n=4, E=1, N=8, K=64, tr=1, tab=(None,) * 4, mt=0, dt=0):
        return L.qmoe_mxfp4_gather_qmm(x, n_x, ldx, None, n, one, one, E, N, K, tr, *tab, mt, dt, one, None)

    assert qmm(x=None) == INV and qmm(E=2) == INV and qmm(n=5) == INV and qmm(tab=(one, None, one, one), mt=3) == INV
    assert qmm(tab=(one,) * 4) == INV and qmm(ldx=68) == UNS and qmm(ldx=32) == UNS and qmm(K=48) == UNS
    assert qmm(tr=0, N=72) == UNS and qmm(n=0) == _lib.OK and qmm(dt=1) == UNS

    def qq(xq=one, n_x=4, n=4, E=1, K=64, lines=None):
        return L.qmoe_mxfp4_gather_qqmm(xq, one, n_x, None, n, one, one, E, 8, K, None, None, None, None, 0, lines, one, None)

    assert qq(xq=None) == INV and qq(E=3) == INV and qq(n=5) == INV and qq(K=16) == UNS and qq(xq=one + 4) == UNS
    assert qq(lines=one + 2) == UNS

    def lines(x=one, n_x=4, K=64, xq=one, s=one, E=2, N=8, at=one, words=20):
        return L.qmoe_mxfp4_quantize_lines(x, n_x, K, xq, s, E, N, at, words, None)

    assert lines(x=None) == INV and lines(at=None) == INV and lines(N=-1) == INV and lines(K=48) == UNS
    assert lines(words=19) == _lib.ERR_WORKSPACE and lines(x=one + 2) == UNS and lines(n_x=0) == _lib.OK
    assert L.qmoe_sort_rows(one, 3, None, 2, 8, 0, one, None) == INV
    assert L.qmoe_sort_rows(one, 3, one, 2, 8, 7, one, None) == UNS
    assert L.qmoe_sort_rows(one, 1 << 30, one, 4, 8, 0, one, None) == UNS
    assert L.qmoe_unsort_sum(one, 6, 0, one, one, None, 3, 3, 8, 0, one, None) == INV
    assert L.qmoe_unsort_sum(one, 6, 0, one, one, None, 3, 2, 8, 2, one, None) == UNS
    assert L.qmoe_unsort_sum(one, 6, 0, one, one, None, 3, 2, 8, 0, None, None) == INV
    assert L.qmoe_unsort_grad(one, one, 6, 0, one, one, 3, 3, 8, one, one, None) == INV
    assert L.qmoe_unsort_grad(one, None, 6, 0, one, one, 3, 2, 8, one, one, None) == INV
    assert L.qmoe_unsort_grad(one, one, 6, 0, one, None, 3, 2, 8, one, one, None) == INV


def test_more_than_one_launch_holds():
    """A grid of 2^32 threads or more is refused, not cut off."""
    L = _lib.load()
    one, UNS = 4096, _lib.ERR_UNSUPPORTED
    many = 1 << 31
    assert L.qmoe_mxfp4_quantize(one, 0, many, 32, one, one, None) == UNS
    assert L.qmoe_mxfp4_dequantize(one, one, many // 4, 32, 2, one, None) == UNS
    assert L.qmoe_mxfp4_quantize_lines(one, 1 << 29, 32, one, one, 1, 8, one, 1 << 40, None) == UNS
    assert L.qmoe_mxfp4_gather_qmv(one, 4, 64, None, 1, None, 65535, one, one, 1, 1 << 20, 64, 1, 0, one, None) == UNS
    assert L.qmoe_mxfp4_gather_qmv(one, 4, 64, None, 1, None, 65535, one, one, 1, 64, 1 << 20, 0, 0, one, None) == UNS
    assert L.qmoe_mxfp4_gather_qmm(one, 9, 64, None, 9, one, one, 1, many - 1, 64, 1, *(None,) * 4, 0, 0, one, None) == UNS
    assert L.qmoe_sort_rows(one, 1 << 25, one, 2, 4096, 0, one, None) == UNS
    assert L.qmoe_unsort_sum(one, 1 << 25, 0, one, one, None, 1 << 25, 1, 4096, 0, one, None) == UNS
    assert L.qmoe_unsort_grad(one, one, 1 << 25, 0, one, one, 1 << 25, 1, 4096, one, one, None) == UNS


def test_the_binding_declines_what_is_not_on_the_gpu():
    """Without a GPU tensor every function answers None, and says so where it must not."""
    B = _lib_binding()
    x, od, (w, s) = torch.zeros(4, 64, dtype=BF), torch.arange(4, dtype=torch.int32), _w(5, 64)
    for call in (lambda m: B.quantize(x, m), lambda m: B.dequantize(w, s, 0, m), lambda m: B.sort_tokens(x, od, od, m),
                 lambda m: B.unsort_tokens(x, od, od, torch.ones(4, 1), m), lambda m: B.matmul(x, w, s, True, False, m),
                 lambda m: B.quantize(None, m), lambda m: B.matmul("x", w, s, True, True, m)):
        assert call(False) is None
        with pytest.raises(RuntimeError, match="not what the kernels read"):
            call(True)
    assert B.gather(x, w, s, None, od, True, True, False) is None
    with pytest.raises(RuntimeError, match="not what the kernels read"):
        B.rows_product(x, w[None], s[None], None, 1, None, None, 4, True, False)


def test_one_width_of_sorting():
    assert mxfp4.SORTED_MIN_ROWS == ops.SORTED_MIN_ROWS == 64
