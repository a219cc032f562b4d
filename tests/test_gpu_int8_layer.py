"""SwitchGLU over experts in 8-bit integers: the products of its projections, bit for
bit, whether the pairs are sorted or not."""

import int8_oracle as o
import pytest
import torch

from titan_amd import ops
from titan_amd.switch_layers import QuantizedSwitchLinear, SwitchGLU, swiglu

BF, HF, F4 = o.BF, o.HF, o.F4
pytestmark = pytest.mark.gpu
E, H, I = 11, 144, 80


def _weights(dev, seed, *shape):
    w = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) / shape[-1] ** 0.5
    return tuple(t.to(dev) for t in o.quantize(w))


def _pairs(x, ids, lin):
    """The projection of every pair by itself: x [T, k, K]."""
    T, k = ids.shape
    q, s = o.quantize(x.float().cpu())
    out = torch.empty(T, k, lin.output_dims, dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            e = int(ids[t, j])
            out[t, j] = o.product(q[t, j][None], s[t, j][None], lin.weight[e].cpu(), lin.scales[e].cpu())[0]
    return out


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF, F4])
@pytest.mark.parametrize("T,k", [(1, 1), (5, 4), (21, 3), (40, 4)])
def test_layer(dev, T, k, dtype, split):
    gate, up, down = _weights(dev, 1, E, I, H), _weights(dev, 2, E, I, H), _weights(dev, 3, E, H, I)
    lin = lambda t: QuantizedSwitchLinear(*t, mode="int8")  # noqa: E731
    both = lin(tuple(torch.cat(p, 1) for p in zip(gate, up)))
    glu = SwitchGLU(lin(down), gate_proj=lin(gate), up_proj=lin(up)) if split else SwitchGLU(lin(down), gate_up_proj=both)
    assert (both.input_dims, both.output_dims, both.num_experts) == (H, 2 * I, E)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, H, generator=g).to(dtype)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    for i in (ids, ids.int()):
        y = glu(x.to(dev), i.to(dev))
        assert y.shape == (T, k, H) and y.dtype == dtype
    # the layer restated from its products: gathered one by one, checked against 64 bits, then the activation
    flat = ids.reshape(-1).to(dev)
    xr = x.to(dev).repeat_interleave(k, 0).unsqueeze(1)

    def one_by_one(v, w):  # few rows at a time: no sort
        return torch.cat([ops.gather_qqmm(v[j:j + 20], *w, rhs_indices=flat[j:j + 20], mode="int8") for j in range(0, T * k, 20)])

    gu = one_by_one(xr, (both.weight, both.scales))
    o.assert_rounded(gu.reshape(T, k, 2 * I), _pairs(x.unsqueeze(1).expand(T, k, H), ids, both))
    h = swiglu(gu[..., :I], gu[..., I:]) if split or dtype != BF else ops.swiglu(gu)
    want = one_by_one(h, down).reshape(T, k, H)
    o.assert_rounded(want, _pairs(h.reshape(T, k, I), ids, glu.down_proj))
    assert torch.equal(y, want)


def test_bias_batches_and_refusals(dev):
    w = _weights(dev, 4, E, I, H)
    bias = torch.randn(E, I, generator=torch.Generator().manual_seed(5)).to(dev, BF)
    lin, plain = QuantizedSwitchLinear(*w, mode="int8", bias=bias), QuantizedSwitchLinear(*w, mode="int8")
    x = torch.randn(2, 3, H, generator=torch.Generator().manual_seed(6)).to(dev, BF)
    ids = torch.randint(0, E, (2, 3, 4), generator=torch.Generator().manual_seed(7)).to(dev)
    v = x.unsqueeze(-2).unsqueeze(-2)
    assert torch.equal(lin(v, ids), plain(v, ids) + bias[ids].unsqueeze(-2))
    down = QuantizedSwitchLinear(*_weights(dev, 8, E, H, I // 2), mode="int8")
    glu = SwitchGLU(down, gate_up_proj=plain)
    wide = x.repeat(1, 8, 1)
    a, b = glu(wide, ids.repeat(1, 8, 1)), glu(x, ids)  # 192 pairs, sorted; 24
    assert a.shape == (2, 24, 4, H) and torch.equal(a[:, :3], b) and torch.equal(a[:, 21:], b)
    for t in (x, wide):
        with pytest.raises(ops.QmoeUnsupported, match="gradient"):
            glu(t.clone().requires_grad_(True), ids.repeat(1, t.shape[1] // 3, 1))
    with pytest.raises(IndexError):
        glu(wide[:1], ids.repeat(1, 8, 1))
    with pytest.raises(ops.QmoeUnsupported):
        glu(x.cpu(), ids.cpu())
    with pytest.raises(ValueError, match="no biases"):
        QuantizedSwitchLinear(*w, w[1], mode="int8")
    with pytest.raises(ValueError, match="one scale"):
        QuantizedSwitchLinear(*w, group_size=64, mode="int8")


def test_layer_in_a_graph(dev):
    glu = SwitchGLU(QuantizedSwitchLinear(*_weights(dev, 9, E, H, I), mode="int8"),
                    gate_up_proj=QuantizedSwitchLinear(*_weights(dev, 10, E, 2 * I, H), mode="int8"))
    for T in (3, 50):
        x = torch.randn(T, H, device=dev).to(BF)
        ids = torch.randint(0, E, (T, 4), dtype=torch.int32, device=dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            glu(x, ids)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = glu(x, ids)
        for i in range(4):
            gen = torch.Generator().manual_seed(i)
            x.copy_(torch.randn(T, H, generator=gen).to(BF))
            ids.copy_(torch.randint(0, E, (T, 4), generator=gen, dtype=torch.int32))
            g.replay()
            torch.cuda.synchronize()
            kept = y.clone()
            assert torch.equal(kept, glu(x, ids))


def test_projections_of_other_kinds(dev):
    """A projection that is no QuantizedSwitchLinear stands beside one in 8-bit integers."""
    w = _weights(dev, 11, E, 2 * I, H)
    plain = QuantizedSwitchLinear(*w, mode="int8")
    calls = []

    def gate_up(x, indices, sorted_indices=False, tiles=None):
        calls.append(sorted_indices)
        return plain(x, indices, sorted_indices=sorted_indices, tiles=tiles)

    down = QuantizedSwitchLinear(*_weights(dev, 12, E, H, I), mode="int8")
    g = torch.Generator().manual_seed(8)
    for T in (5, 40):
        x, ids = torch.randn(T, H, generator=g).to(dev, BF), torch.randint(0, E, (T, 4), generator=g).to(dev)
        assert torch.equal(SwitchGLU(down, gate_up_proj=gate_up)(x, ids), SwitchGLU(down, gate_up_proj=plain)(x, ids))
    assert calls == [False, True]
