"""mxfp4 on the stock path (CPU tensors) against its definition in 64 bits, and
what the decode overlay routes of the mode."""

import types

import pytest
import torch

from mx_helpers import check_sum, codes, dequantize_ref
from titan_amd import core, ops, stock
from titan_amd.patches import gather_qmv
from titan_amd.switch_layers import QuantizedSwitchLinear, SwitchGLU


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def test_stock_dequantize():
    w, s = codes(_gen(1), 3, 5, 96, lo=0, hi=250)
    s[0, 0, 0], s[0, 1, 1] = 255, 0
    got = stock.dequantize(w, s, None, mode="mxfp4")
    want = dequantize_ref(w, s).to(torch.bfloat16)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(0), want.nan_to_num(0))
    for bad in ({"group_size": 64}, {"bits": 8}, {"biases": s}):
        kw = {"biases": None, "mode": "mxfp4", **bad}
        with pytest.raises(ValueError):
            stock.dequantize(w, s, **kw)
    with pytest.raises(ValueError, match="disagree"):
        stock.dequantize(w, s[..., :2], None, mode="mxfp4")
    with pytest.raises(ValueError, match="mode"):
        stock.dequantize(w, s, None, mode="nvfp4")


@pytest.mark.parametrize("transpose", [True, False])
def test_stock_products(transpose):
    g = _gen(2)
    w, s = codes(g, 4, 24, 64)
    W = dequantize_ref(w, s)
    x = torch.randn(7, 64 if transpose else 24, generator=g).to(torch.bfloat16)
    e = torch.tensor([0, 1, 1, 3, 3, 3, 0])
    got = core.gather_qmm(x.unsqueeze(1), w, s, rhs_indices=e, transpose=transpose, mode="mxfp4").squeeze(1)
    mats = W[e] if not transpose else W[e].transpose(1, 2)
    ref, mag = (torch.bmm(v.unsqueeze(1), m).squeeze(1) for v, m in ((x.double(), mats), (x.double().abs(), mats.abs())))
    check_sum(got, ref, mag, x.shape[1])
    one = core.quantized_matmul(x, w[1], s[1], transpose=transpose, group_size=32, mode="mxfp4")
    m = W[1].t() if transpose else W[1]
    check_sum(one, x.double() @ m, x.double().abs() @ m.abs(), x.shape[1])


def test_layers_take_the_mode():
    """A SwitchGLU of mxfp4 layers on the CPU, sorted and not, and its gradient by torch."""
    g = _gen(3)
    E, H, I = 4, 64, 32
    up, down = QuantizedSwitchLinear(*codes(g, E, 2 * I, H), mode="mxfp4"), QuantizedSwitchLinear(*codes(g, E, H, I), mode="mxfp4")
    assert (up.group_size, up.input_dims, up.output_dims, up.num_experts) == (32, H, 2 * I, E)
    glu = SwitchGLU(down, gate_up_proj=up)
    x = torch.randn(40, H, generator=g).to(torch.bfloat16).requires_grad_(True)
    ids = torch.stack([torch.randperm(E, generator=g)[:2] for _ in range(40)])
    y = glu(x, ids)
    narrow = torch.cat([glu(x[i:i + 8], ids[i:i + 8]) for i in range(0, 40, 8)])
    assert y.shape == (40, 2, H) and torch.allclose(y.float(), narrow.float(), rtol=2.0 ** -6, atol=1e-2)
    y.float().sum().backward()
    assert x.grad.isfinite().all() and x.grad.abs().sum() > 0


def test_overlay_routes_every_mxfp4_call(monkeypatch):
    seen = []
    base = lambda *a, **kw: seen.append("base") or "base"  # noqa: E731
    ns = types.SimpleNamespace(gather_qmm=base, quantized_matmul=base)
    monkeypatch.setattr(gather_qmv, "_gpu_bf16", lambda x: True)
    monkeypatch.setattr(ops, "gather_qmm", lambda *a, **kw: seen.append(("gather", len(a), sorted(kw))) or 1)
    monkeypatch.setattr(ops, "quantized_matmul", lambda *a, **kw: seen.append(("qmm", len(a), sorted(kw))) or 1)
    monkeypatch.setattr(gather_qmv._OV, "self_check", None)
    assert gather_qmv.install(ns)
    try:
        x, w, s = torch.zeros(2, 1, 32), torch.zeros(1), torch.zeros(1)
        ns.gather_qmm(x, w, s, rhs_indices=0, mode="mxfp4", sorted_indices=True)
        ns.gather_qmm(x, w, s, None, None, 0, False, 32, 4, "mxfp4")
        ns.quantized_matmul(x, w, s, mode="mxfp4", transpose=False)
        ns.quantized_matmul(x, w, s, None, True, 32, 4, "mxfp4")
        assert seen == [("gather", 3, ["mode", "rhs_indices", "sorted_indices"]), ("gather", 10, []),
                        ("qmm", 3, ["mode", "transpose"]), ("qmm", 8, [])]
        monkeypatch.setenv("TITAN_AMD_MOE_DECODE", "0")
        ns.gather_qmm(x, w, s, mode="mxfp4")
        ns.gather_qmm(x, w, s, torch.zeros(1), sorted_indices=True)
        assert seen[-2:] == ["base", "base"]
    finally:
        gather_qmv.uninstall()
        gather_qmv._OV.reset_stats()
