"""mxfp4 through the framework's layers on the GPU: SwitchGLU over the stock path
and over the kernels, served and trained through."""

import pytest
import torch

from mx_helpers import codes, dequantize_ref
from titan_amd import core, patches, stock
from titan_amd.patches import gather_qmv
from titan_amd.switch_layers import QuantizedSwitchLinear, SwitchGLU

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
E, H, I = 8, 256, 96


@pytest.fixture
def installed():
    patches.install()
    yield
    patches.uninstall()


def _glu(dev, gen, split=False):
    """The layer, and the same in 64 bits on the CPU."""
    up, down = codes(gen, E, 2 * I, H), codes(gen, E, H, I)
    on = lambda t: tuple(v.to(dev) for v in t)  # noqa: E731
    lin = lambda t: QuantizedSwitchLinear(*on(t), mode="mxfp4")  # noqa: E731
    if split:
        halves = [tuple(v[:, i * I:(i + 1) * I].contiguous() for v in up) for i in (0, 1)]
        glu = SwitchGLU(lin(down), gate_proj=lin(halves[0]), up_proj=lin(halves[1]))
    else:
        glu = SwitchGLU(lin(down), gate_up_proj=lin(up))
    U, D = dequantize_ref(*up), dequantize_ref(*down)

    def ref(x, ids):
        gu = torch.einsum("th,tkoh->tko", x, U[ids])
        h = torch.nn.functional.silu(gu[..., :I]) * gu[..., I:]
        return torch.einsum("tki,tkhi->tkh", h, D[ids])

    return glu, ref


def _ids(gen, T, k):
    return torch.stack([torch.randperm(E, generator=gen)[:k] for _ in range(T)])


def _rel(a, b):
    return float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())


# three bf16 roundings (gate_up, activation, down) of 2^-8 each, amplified by at most about 4 through SwiGLU's
# derivative: 12 * 2^-8 of the result's norm bounds them
BOUND = 12 * 2.0 ** -8


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("T,k", [(1, 1), (1, 8), (7, 4), (16, 4), (65, 3), (130, 8)])
def test_layer_through_the_overlay(dev, installed, T, k, split):
    print("[layer]", T, k, split, flush=True)
    g = torch.Generator().manual_seed(T + k)
    glu, ref = _glu(dev, g, split)
    x = torch.randn(T, H, generator=g).to(BF)
    ids = _ids(g, T, k)
    r0 = gather_qmv.stats()["routed"]
    y = glu(x.to(dev), ids.to(dev))
    assert gather_qmv.stats()["routed"] - r0 == (3 if split else 2)
    assert y.shape == (T, k, H) and _rel(y, ref(x.double(), ids)) <= BOUND


@pytest.mark.parametrize("T,k", [(5, 2), (65, 3)])
def test_layer_on_the_stock_path(dev, T, k):
    g = torch.Generator().manual_seed(T)
    glu, ref = _glu(dev, g)
    assert core.gather_qmm is stock.gather_qmm
    x, ids = torch.randn(T, H, generator=g).to(BF), _ids(g, T, k)
    assert _rel(glu(x.to(dev), ids.to(dev)), ref(x.double(), ids)) <= BOUND


@pytest.mark.parametrize("T,k", [(5, 2), (40, 4), (130, 8)])
def test_layer_is_trained_through(dev, installed, T, k):
    print("[layer grad]", T, k, flush=True)
    g = torch.Generator().manual_seed(T * k)
    glu, ref = _glu(dev, g)
    x, ids = torch.randn(T, H, generator=g).to(BF), _ids(g, T, k)
    dy = torch.randn(T, k, H, generator=g).to(BF)
    xd = x.to(dev).requires_grad_(True)
    y = glu(xd, ids.to(dev))
    y.backward(dy.to(dev))
    x64 = x.double().requires_grad_(True)
    y64 = ref(x64, ids)
    y64.backward(dy.double())
    assert _rel(y, y64) <= BOUND and _rel(xd.grad, x64.grad) <= BOUND
    # twice gives the same bits
    xd2 = x.to(dev).requires_grad_(True)
    glu(xd2, ids.to(dev)).backward(dy.to(dev))
    assert torch.equal(xd2.grad, xd.grad)
