"""What the 8-bit operators and the balance loss refuse, before any launch: CPU
tensors with the device check taken out, a launch counted as a failure; and the
C entries' own checks."""

import ctypes

import pytest
import torch

from titan_amd import _lib, ops
from titan_amd.int8 import Normed
from titan_amd.ops import QmoeUnsupported

BF = torch.bfloat16
real_binding = _lib.binding


class Binding:
    """Declines every call that may be declined, and counts the others as launches."""

    def __getattr__(self, name):
        def call(*args):
            if args[-1] is False or name == "int8_gather":
                return None
            raise AssertionError(f"{name} launched")

        return call


@pytest.fixture
def no_launch(monkeypatch):
    def launch(name, *args):
        raise AssertionError(f"{name} launched")

    monkeypatch.setattr(ops, "_dev", lambda t, name: None)
    monkeypatch.setattr(ops, "tile_rows", lambda: 128)
    monkeypatch.setattr(_lib, "call", launch)
    monkeypatch.setattr(_lib, "binding", lambda: Binding())


def _w(*shape):
    return torch.zeros(shape, dtype=torch.int8), torch.ones(shape[:-1])


launched = pytest.raises(AssertionError, match="launched")


def test_quantize(no_launch):
    x = torch.zeros(2, 63)
    for bad in (x.double(), x.int()):
        with pytest.raises(QmoeUnsupported):
            ops.quantize(bad, mode="int8")
    with pytest.raises(ValueError):
        ops.quantize(torch.tensor(1.0), mode="int8")
    for kw in ({"group_size": 64}, {"bits": 4}):
        with pytest.raises(QmoeUnsupported):
            ops.quantize(x, mode="int8", **kw)
    for kw in ({}, {"bits": 8}):
        with launched:
            ops.quantize(x, mode="int8", **kw)


def test_dequantize(no_launch):
    w, s = _w(3, 64)
    with pytest.raises(ValueError, match="biases"):
        ops.dequantize(w, s, s, mode="int8")
    for bad in (s[:2], s.unsqueeze(-1)):
        with pytest.raises(ValueError, match="disagree"):
            ops.dequantize(w, bad, mode="int8")
    for a, b, kw in ((w.int(), s, {}), (w, s.to(BF), {}), (w, s, {"dtype": torch.float64}), (w, s, {"bits": 4}),
                     (w, s, {"group_size": 32})):
        with pytest.raises(QmoeUnsupported):
            ops.dequantize(a, b, mode="int8", **kw)
    with launched:
        ops.dequantize(w, s, mode="int8", dtype=torch.float16)


def test_rms_norm_quantize(no_launch):
    x, w = torch.zeros(2, 5, 64, dtype=BF), torch.zeros(64, dtype=BF)
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            ops.rms_norm_quantize(x, w, eps)
    for kw in ({"residual": x[:1]}, {"residual": x.float()}):
        with pytest.raises(ValueError, match="residual"):
            ops.rms_norm_quantize(x, w, **kw)
    for bad in (w[:63], w.unsqueeze(0)):
        with pytest.raises(ValueError, match="weight"):
            ops.rms_norm_quantize(x, bad)
    with pytest.raises(QmoeUnsupported):
        ops.rms_norm_quantize(x.double(), None)
    with pytest.raises(QmoeUnsupported):
        ops.rms_norm_quantize(x, w.double())
    leaf = x.clone().requires_grad_(True)
    for args, kw in (((leaf, w), {}), ((x, w.clone().requires_grad_(True)), {}), ((x, w), {"residual": leaf})):
        with pytest.raises(QmoeUnsupported, match="gradient"):
            ops.rms_norm_quantize(*args, **kw)
    for weight in (None, w, w.float(), w.half()):
        with launched:
            ops.rms_norm_quantize(x, weight, residual=x, norm=True)


def test_qqmm(no_launch):
    x, (w, s) = torch.zeros(3, 64, dtype=BF), _w(16, 64)
    with pytest.raises(ValueError, match="fit"):
        ops.qqmm(x[:, :32], w, s, mode="int8")
    with pytest.raises(ValueError, match="disagree"):
        ops.qqmm(x, w, s[:8], mode="int8")
    with pytest.raises(ValueError, match="disagree"):
        ops.qqmm(_w(3, 64)[0:1] + (torch.ones(2),), w, s, mode="int8")
    for args, kw in (((x.double(), w, s), {}), ((x, w.int(), s), {}), ((x, w, s.half()), {}), ((x, *_w(2, 16, 64)), {}),
                     ((x, w, s), {"bits": 4}), ((x, w, s), {"group_size": 64}), ((x, w, s), {"dtype": torch.float64}),
                     ((torch.zeros(1, 131072), *_w(1, 131072)), {}), (((x, torch.ones(3)), w, s), {})):
        with pytest.raises(QmoeUnsupported):
            ops.qqmm(*args, mode="int8", **kw)
    for bad in (None, (w,), (w, s, s), "x"):
        with pytest.raises(TypeError):
            ops.qqmm(bad, w, s, mode="int8")
    with pytest.raises(QmoeUnsupported, match="gradient"):
        ops.qqmm(x.clone().requires_grad_(True), w, s, mode="int8")
    with pytest.raises(QmoeUnsupported, match="gradient"):
        ops.qqmm(x, w, s.clone().requires_grad_(True), mode="int8")
    for good in (x, _w(3, 64), list(_w(3, 64)), Normed(*_w(3, 64), None, None)):
        with launched:
            ops.qqmm(good, w, s, mode="int8")
    with pytest.raises(QmoeUnsupported, match="bfloat16"):
        ops.qqmm(x, w, s, dtype=torch.float16)


def test_gather_qqmm(no_launch):
    x, (w, s) = torch.zeros(3, 1, 64, dtype=BF), _w(4, 16, 64)
    ids = torch.zeros(3, dtype=torch.int32)
    for bad in (ids.float(), ids.bool(), [0, 1, 2]):
        with pytest.raises(TypeError):
            ops.gather_qqmm(x, w, s, rhs_indices=bad, mode="int8")
        with pytest.raises(TypeError):
            ops.gather_qqmm(x, w, s, lhs_indices=bad, rhs_indices=ids, mode="int8")
    with pytest.raises(ValueError, match="broadcast"):
        ops.gather_qqmm(x, w, s, rhs_indices=torch.zeros(2, dtype=torch.int32), mode="int8")
    with pytest.raises(ValueError, match="2-D"):
        ops.gather_qqmm(x[0, 0], w, s, rhs_indices=ids, mode="int8")
    with pytest.raises(ValueError, match="no experts"):
        ops.gather_qqmm(x, w[:0], s[:0], rhs_indices=ids, mode="int8")
    with pytest.raises(QmoeUnsupported):
        ops.gather_qqmm(x, w[0], s[0], rhs_indices=ids, mode="int8")
    with pytest.raises(QmoeUnsupported, match="gradient"):
        ops.gather_qqmm(x.clone().requires_grad_(True), w, s, rhs_indices=ids, mode="int8")
    big = torch.zeros(80, 1, 64, dtype=BF)
    many = torch.zeros(80, dtype=torch.int32)
    table = ops.TileTable(*[torch.zeros(9, dtype=torch.int32)] * 4, 4, 128, 3, 80)
    with pytest.raises(ValueError, match="tile table"):
        ops.gather_qqmm(big, w, s, rhs_indices=many, mode="int8", sorted_indices=True, tiles=table)
    for i in (ids, ids.long()):
        with launched:
            ops.gather_qqmm(x, w, s, rhs_indices=i, mode="int8")
    with pytest.raises(QmoeUnsupported, match="bfloat16"):
        ops.gather_qqmm(x, w, s, rhs_indices=ids, dtype=torch.float32)


def test_router_balance_loss(no_launch):
    logits, ids = torch.zeros(5, 8), torch.zeros(5, 2, dtype=torch.int64)
    with pytest.raises(QmoeUnsupported):
        ops.router_balance_loss(logits.double(), ids)
    for bad in (ids.float(), ids.to(torch.int16), ids.bool()):
        with pytest.raises(TypeError):
            ops.router_balance_loss(logits, bad)
    for bad in (ids[:4], ids[0], ids.unsqueeze(0)):
        with pytest.raises(ValueError, match="fit"):
            ops.router_balance_loss(logits, bad)
    for bad in (torch.ones(4, dtype=torch.bool), torch.ones(5), torch.ones(5, 1, dtype=torch.bool)):
        with pytest.raises(ValueError, match="mask"):
            ops.router_balance_loss(logits, ids, bad)
    with launched:
        ops.router_balance_loss(logits, ids, torch.ones(5, dtype=torch.bool))


def test_cpu_tensors_are_refused():
    x, (w, s) = torch.zeros(3, 64, dtype=BF), _w(4, 64)
    for call in (lambda: ops.quantize(x, mode="int8"), lambda: ops.dequantize(w, s, mode="int8"),
                 lambda: ops.rms_norm_quantize(x, None), lambda: ops.qqmm(x, w, s, mode="int8"),
                 lambda: ops.gather_qqmm(x.unsqueeze(1), w.unsqueeze(0), s.unsqueeze(0), mode="int8"),
                 lambda: ops.router_balance_loss(torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int32))):
        with pytest.raises(QmoeUnsupported):
            call()


# ------------------------------------------------------------- the C entries

P = ctypes.c_void_p(256)  # never read: refused on the host, or nothing to do
ODD = ctypes.c_void_p(264)


def _rc(name, *args):
    return getattr(_lib.load(), name)(*args)


def test_rows_entries():
    for bad, rc in (((P, 3, 2, 8, P, P, None), _lib.ERR_UNSUPPORTED), ((P, 0, -1, 8, P, P, None), _lib.ERR_INVALID),
                    ((None, 0, 2, 8, P, P, None), _lib.ERR_INVALID), ((P, 0, 2, 8, None, P, None), _lib.ERR_INVALID),
                    ((P, 0, 2, 8, P, None, None), _lib.ERR_INVALID), ((ODD, 0, 2, 8, P, P, None), _lib.ERR_UNSUPPORTED),
                    ((P, 0, 2, 8, ODD, P, None), _lib.ERR_UNSUPPORTED), ((P, 0, 1 << 33, 8, P, P, None), _lib.ERR_UNSUPPORTED),
                    ((P, 0, 2, 1 << 31, P, P, None), _lib.ERR_UNSUPPORTED), ((None, 0, 0, 8, None, None, None), _lib.OK)):
        assert _rc("qmoe_int8_quantize", *bad) == rc, bad
    both = dict(x=P, dt=0, rows=2, K=8, q=P, s=P, ids=P, n=4, E=2, tr=128, off=P, row=P, exp=P, nt=P, maxt=3)
    for change, rc in (({"dt": 3}, _lib.ERR_UNSUPPORTED), ({"x": None}, _lib.ERR_INVALID), ({"q": ODD}, _lib.ERR_UNSUPPORTED),
                       ({"n": -1}, _lib.ERR_INVALID), ({"E": 0}, _lib.ERR_INVALID), ({"tr": 0}, _lib.ERR_INVALID),
                       ({"ids": None}, _lib.ERR_INVALID), ({"off": None}, _lib.ERR_INVALID), ({"nt": None}, _lib.ERR_INVALID),
                       ({"n": 1 << 31}, _lib.ERR_UNSUPPORTED), ({"maxt": -1}, _lib.ERR_INVALID)):
        assert _rc("qmoe_int8_quantize_sorted", *{**both, **change}.values(), None) == rc, change
    for bad, rc in (((P, P, 2, 8, 3, P, None), _lib.ERR_UNSUPPORTED), ((P, None, 2, 8, 0, P, None), _lib.ERR_INVALID),
                    ((P, P, 2, 8, 0, ODD, None), _lib.ERR_UNSUPPORTED), ((P, P, 2, 0, 0, P, None), _lib.OK)):
        assert _rc("qmoe_int8_dequantize", *bad) == rc, bad
    norm = dict(x=P, r=None, w=None, wd=0, dt=0, rows=2, D=8, eps=1e-6, q=P, s=P, sum=None, norm=None)
    for change, rc in (({"dt": 7}, _lib.ERR_UNSUPPORTED), ({"w": P, "wd": 1}, _lib.ERR_UNSUPPORTED), ({"D": 0}, _lib.ERR_INVALID),
                       ({"eps": -1.0}, _lib.ERR_INVALID), ({"eps": float("nan")}, _lib.ERR_INVALID), ({"q": None}, _lib.ERR_INVALID),
                       ({"r": ODD}, _lib.ERR_UNSUPPORTED), ({"sum": ODD}, _lib.ERR_UNSUPPORTED), ({"w": ODD}, _lib.ERR_UNSUPPORTED),
                       ({"rows": 0}, _lib.OK)):
        assert _rc("qmoe_int8_rms_norm", *{**norm, **change}.values(), None) == rc, change


def test_product_entries():
    few = dict(x=P, sx=P, n_x=2, rows=None, div=1, ex=None, n=2, w=P, sw=P, E=1, N=8, K=32, dt=0, out=P)
    for change, rc in (({"n": -1}, _lib.ERR_INVALID), ({"div": 0}, _lib.ERR_INVALID), ({"dt": 5}, _lib.ERR_UNSUPPORTED),
                       ({"K": 24}, _lib.ERR_UNSUPPORTED), ({"K": 131072}, _lib.ERR_UNSUPPORTED), ({"K": 0}, _lib.ERR_INVALID),
                       ({"n_x": 0}, _lib.ERR_INVALID), ({"E": 0}, _lib.ERR_INVALID), ({"w": None}, _lib.ERR_INVALID),
                       ({"x": ODD}, _lib.ERR_UNSUPPORTED), ({"out": ODD}, _lib.ERR_UNSUPPORTED), ({"n": 65536}, _lib.ERR_UNSUPPORTED),
                       ({"N": 1 << 31}, _lib.ERR_UNSUPPORTED), ({"n": 0}, _lib.OK), ({"N": 0}, _lib.OK)):
        assert _rc("qmoe_int8_gather_qqmv", *{**few, **change}.values(), None) == rc, change
    val = dict(x=P, xdt=0, **{k: v for k, v in few.items() if k not in ("x", "sx")})
    for change, rc in (({"xdt": 3}, _lib.ERR_UNSUPPORTED), ({"K": 16400}, _lib.ERR_UNSUPPORTED), ({"x": None}, _lib.ERR_INVALID),
                       ({"n": 65536}, _lib.ERR_UNSUPPORTED), ({"x": ODD}, _lib.ERR_UNSUPPORTED), ({"n": 0}, _lib.OK)):
        assert _rc("qmoe_int8_gather_qmv", *{**val, **change}.values(), None) == rc, change
    many = dict(x=P, sx=P, n_x=2, rows=None, n=2, w=P, sw=P, E=1, N=8, K=32, off=None, tr=None, te=None, nt=None, maxt=0, dt=0,
                out=P)
    for change, rc in (({"E": 2}, _lib.ERR_INVALID), ({"off": P}, _lib.ERR_INVALID), ({"n": 3}, _lib.ERR_INVALID),
                       ({"off": P, "tr": P, "te": P, "nt": P}, _lib.ERR_INVALID), ({"K": 8}, _lib.ERR_UNSUPPORTED),
                       ({"sx": None}, _lib.ERR_INVALID), ({"n": 0}, _lib.OK)):
        assert _rc("qmoe_int8_gather_qqmm", *{**many, **change}.values(), None) == rc, change


def test_balance_entries():
    L = _lib.load()
    size = L.qmoe_router_balance_workspace_size(100, 64)
    assert size > 0 and L.qmoe_router_balance_workspace_size(-1, 64) == 0
    assert L.qmoe_router_balance_workspace_size(100, 2000) == 0
    call = dict(x=P, dt=2, T=100, E=64, ids=P, w=0, k=2, mask=None, loss=P, counts=P, n=P, ws=P, size=size)
    for change, rc in (({"E": 1025}, _lib.ERR_UNSUPPORTED), ({"E": 0}, _lib.ERR_INVALID), ({"k": 0}, _lib.ERR_INVALID),
                       ({"T": -1}, _lib.ERR_INVALID), ({"dt": 4}, _lib.ERR_UNSUPPORTED), ({"ids": None}, _lib.ERR_INVALID),
                       ({"x": None}, _lib.ERR_INVALID), ({"x": ODD}, _lib.ERR_UNSUPPORTED), ({"loss": None}, _lib.ERR_INVALID),
                       ({"ws": None}, _lib.ERR_WORKSPACE), ({"size": size - 1}, _lib.ERR_WORKSPACE),
                       ({"T": 1 << 30, "k": 4}, _lib.ERR_UNSUPPORTED)):
        assert _rc("qmoe_router_balance", *{**call, **change}.values(), None) == rc, change
    grad = dict(x=P, dt=2, T=100, E=64, k=2, mask=None, counts=P, n=P, g=P, d=P)
    for change, rc in (({"counts": None}, _lib.ERR_INVALID), ({"d": None}, _lib.ERR_INVALID), ({"g": None}, _lib.ERR_INVALID),
                       ({"d": ODD}, _lib.ERR_UNSUPPORTED), ({"T": 0}, _lib.OK)):
        assert _rc("qmoe_router_balance_grad", *{**grad, **change}.values(), None) == rc, change
