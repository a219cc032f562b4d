"""The mxfp4 GEMMs where there are enough units for their wide forms (160 units of
128 rows x 256 outputs, 96 with both operands in 4 bits): every form by rows,
both layouts of the scales, contractions of one group to many and ragged ones,
every output against a product in 64 bits."""

import pytest
import torch

from mx_helpers import check_sum, codes, dequantize_ref, quantize_ref
from titan_amd import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
TILE, COLS = 128, 256


def say(*a):
    print("[mxfp4 wide]", *a, flush=True)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _acts(gen, rows, K):
    x = torch.randn(rows, K, generator=gen)
    return (x * (0.25 + torch.rand(rows, 1, generator=gen))).to(BF)


def _units(n, outputs, E=0):
    return (-(-n // TILE) + E) * -(-outputs // COLS)


def _product(x, W):
    """x W and the sum of magnitudes in 64 bits, formed on the GPU."""
    x, W = x.double(), W.double()
    return (x @ W).cpu(), (x.abs() @ W.abs()).cpu()


# rows that end in a tile of 128, 97 to 128, 65 to 96, 33 to 64 and 1 to 32
@pytest.mark.parametrize("M", [2688, 2597 + 64, 2640, 2597, 2561])
@pytest.mark.parametrize("K,N", [(2048, 2100), (1056, 2060)])
def test_forward_by_rows(dev, M, K, N):
    say("forward rows", M, K, N)
    assert _units(M, N) >= 160
    g = _gen(M + K)
    w, s = codes(g, N, K)
    x = _acts(g, M, K)
    x[M // 2] = float("nan")  # in a row of its own, whatever shares its tile
    got = ops.quantized_matmul(x.to(dev), w.to(dev), s.to(dev), mode="mxfp4")
    check_sum(got, *_product(x.to(dev), dequantize_ref(w, s).t().to(dev)), K, (M, K, N))


# groups of 64 columns: 1 (half and whole), 2, 2, 3, 4, 5, 6, 8, 9, 33
@pytest.mark.parametrize("K", [32, 64, 96, 128, 160, 256, 288, 384, 512, 544, 2080])
def test_forward_by_groups(dev, K):
    say("forward groups", K)
    M, N = 2592, 2049
    assert _units(M, N) >= 160
    g = _gen(K)
    w, s = codes(g, N, K)
    x = _acts(g, M, K)
    got = ops.quantized_matmul(x.to(dev), w.to(dev), s.to(dev), mode="mxfp4")
    check_sum(got, *_product(x.to(dev), dequantize_ref(w, s).t().to(dev)), K, K)


@pytest.mark.parametrize("M", [2688, 2597 + 64, 2640, 2597, 2561])
@pytest.mark.parametrize("K,N", [(2176, 1024), (2080, 531)])
def test_transposed_by_rows(dev, M, K, N):
    say("transposed rows", M, K, N)
    assert _units(M, K) >= 160
    g = _gen(M + N)
    w, s = codes(g, N, K)
    x = _acts(g, M, N)
    x[M // 2] = float("nan")
    got = ops.quantized_matmul(x.to(dev), w.to(dev), s.to(dev), transpose=False, mode="mxfp4")
    check_sum(got, *_product(x.to(dev), dequantize_ref(w, s).to(dev)), N, (M, K, N))


# groups of 64 rows: 1 (in part and whole), 2, 3, 3, 4, 5, 6, 9, 17
@pytest.mark.parametrize("N", [1, 33, 64, 100, 129, 192, 256, 300, 381, 520, 1061])
@pytest.mark.parametrize("K", [2304, 2080])
def test_transposed_by_groups(dev, K, N):
    say("transposed groups", K, N)
    M = 2592
    assert _units(M, K) >= 160
    g = _gen(N)
    w, s = codes(g, N, K)
    x = _acts(g, M, N)
    got = ops.quantized_matmul(x.to(dev), w.to(dev), s.to(dev), transpose=False, mode="mxfp4")
    check_sum(got, *_product(x.to(dev), dequantize_ref(w, s).to(dev)), N, (K, N))


@pytest.mark.parametrize("M,K,N", [(2688, 2048, 2100), (2597, 1056, 2060), (2561, 32, 2049), (2592, 128, 2049),
                                   (2592, 160, 2049), (2592, 256, 2049), (2592, 288, 2049), (2592, 384, 2049),
                                   (2592, 512, 2049), (2640, 544, 2049)])
def test_both_in_four_bits(dev, M, K, N):
    """Many rows of one matrix: the scales in lines."""
    say("qqmm", M, K, N)
    assert _units(M, N) >= 96
    g = _gen(M + K + N)
    w, s = codes(g, N, K)
    x = _acts(g, M, K)
    got = ops.qqmm(x.to(dev), w.to(dev), s.to(dev))
    check_sum(got, *_product(quantize_ref(x)[0].to(dev), dequantize_ref(w, s).t().to(dev)), K, (M, K, N))


# ---------------------------------------------------------------- experts

COUNTS = [200, 128, 97, 96, 65, 64, 33, 32, 1, 0, 127, 129, 300, 31, 0, 256, 80, 112, 385, 5, 48, 66, 98, 2]


def _ids(counts):
    return torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))


def _experts(x, W, e):
    """Rows of x times the matrix of each one's expert, and the sum of magnitudes, 64 bits on the GPU; e ascending."""
    out = torch.zeros(len(e), W.shape[2], dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(out)
    x = x.double()
    for i in torch.unique(e).tolist():
        at = (e == i).nonzero().flatten().to(x.device)
        V = W[i].to(x.device)
        out[at], mag[at] = x[at] @ V, x[at].abs() @ V.abs()
    return out, mag


@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("K,N", [(1152, 1028), (1184, 1061)])
def test_experts_with_gradient(dev, K, N, transpose):
    """Experts of every number of rows, rows taken by index and shared, results in 16 bits and gradients summed in 32."""
    say("experts", K, N, transpose)
    e = _ids(COUNTS)
    n, E, T = len(e), len(COUNTS), 700
    C, O = (K, N) if transpose else (N, K)
    assert _units(n, C, E) >= 160 and _units(n, O, E) >= 160
    g = _gen(K)
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s)
    lhs = torch.randint(0, T, (n,), generator=g)
    x = _acts(g, T, C).to(dev)
    xd = x.unsqueeze(1).requires_grad_(True)
    y = ops.gather_qmm(xd, w.to(dev), s.to(dev), lhs_indices=lhs.to(dev), rhs_indices=e.to(dev), transpose=transpose,
                       mode="mxfp4", sorted_indices=True).squeeze(1)
    ref, mag = _experts(x[lhs.to(dev)], W.transpose(1, 2) if transpose else W, e)
    check_sum(y, ref.cpu(), mag.cpu(), C)
    dy = _acts(g, n, O).to(dev)
    (dx,) = torch.autograd.grad(y, xd, dy)
    ref, mag = _experts(dy, W if transpose else W.transpose(1, 2), e)
    zero = torch.zeros(T, C, dtype=torch.float64)
    check_sum(dx.squeeze(1), zero.index_add(0, lhs, ref.cpu()), zero.index_add(0, lhs, mag.cpu()), O + n)
    # rows in hand, their gradients rounded as they are
    xs = x[lhs.to(dev)].unsqueeze(1).requires_grad_(True)
    again = ops.gather_qmm(xs, w.to(dev), s.to(dev), rhs_indices=e.to(dev), transpose=transpose, mode="mxfp4",
                           sorted_indices=True).squeeze(1)
    assert torch.equal(again, y)
    check_sum(torch.autograd.grad(again, xs, dy)[0].squeeze(1), ref.cpu(), mag.cpu(), O)


@pytest.mark.parametrize("K,N", [(512, 1028), (544, 1061)])
def test_experts_both_in_four_bits(dev, K, N):
    """Enough rows per expert for the scales in lines, and too few of them: read from the rows, by words or bytes."""
    say("experts qq", K, N)
    for counts in (COUNTS, [3, 0, 17, 20] * 30 + [500, 70, 129]):
        e = _ids(counts)
        n, E = len(e), len(counts)
        assert _units(n, N, E) >= 96 and (n >= 32 * E) == (counts is COUNTS)
        g = _gen(n)
        w, s = codes(g, E, N, K)
        x = _acts(g, n, K)
        got = ops.gather_qqmm(x.to(dev).unsqueeze(1), w.to(dev), s.to(dev), rhs_indices=e.to(dev), sorted_indices=True)
        ref, mag = _experts(quantize_ref(x)[0].to(dev), dequantize_ref(w, s).transpose(1, 2), e)
        check_sum(got.squeeze(1), ref.cpu(), mag.cpu(), K, n)


@pytest.mark.parametrize("transpose", [True, False])
def test_more_tiles_than_are_ranked(dev, transpose):
    say("many tiles", transpose)
    counts = [2, 0, 3, 130] * 180
    e = _ids(counts)
    n, E, K, N = len(e), len(counts), 96, 40
    assert sum(-(-c // TILE) for c in counts) > 512
    C, O = (K, N) if transpose else (N, K)
    g = _gen(3)
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s)
    x, dy = _acts(g, n, C).to(dev), _acts(g, n, O).to(dev)
    xd = x.unsqueeze(1).requires_grad_(True)
    y = ops.gather_qmm(xd, w.to(dev), s.to(dev), rhs_indices=e.to(dev), transpose=transpose, mode="mxfp4",
                       sorted_indices=True).squeeze(1)
    ref, mag = _experts(x, W.transpose(1, 2) if transpose else W, e)
    check_sum(y, ref.cpu(), mag.cpu(), C)
    (dx,) = torch.autograd.grad(y, xd, dy)
    ref, mag = _experts(dy, W if transpose else W.transpose(1, 2), e)
    check_sum(dx.squeeze(1), ref.cpu(), mag.cpu(), O)


def test_repeats_in_graphs(dev):
    """Bit-equal in replayed graphs with new inputs, forward and gradient."""
    say("graph")
    M, K, N = 2597, 2080, 2100
    g = _gen(5)
    w, s = (t.to(dev) for t in codes(g, N, K))
    x, dy = _acts(g, M, K).to(dev), _acts(g, M, N).to(dev)

    def step():
        xd = x.detach().requires_grad_(True)
        y = ops.quantized_matmul(xd, w, s, mode="mxfp4")
        return y.detach(), ops.qqmm(x, w, s), torch.autograd.grad(y, xd, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        x.copy_(_acts(_gen(seed), M, K))
        dy.copy_(_acts(_gen(seed + 10), M, N))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_more_rows_than_one_launch_lays_out_in_lines(dev):
    """Rows that are quantised in one launch but whose scales fill more than one in lines."""
    say("rows past the lines")
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("less than 60 GiB of GPU memory free")
    M, K, N = (1 << 28) + 77, 32, 8
    g = _gen(7)
    w, s = codes(g, N, K)
    some = torch.tensor([0, 127, 1 << 27, (1 << 28) - 1, 1 << 28, M - 1])
    few = _acts(g, len(some), K)
    x = torch.zeros(M, K, dtype=BF, device=dev)
    x[some.to(dev)] = few.to(dev)
    y = ops.qqmm(x, w.to(dev), s.to(dev))
    del x
    check_sum(y[some.to(dev)], *_product(quantize_ref(few)[0].to(dev), dequantize_ref(w, s).t().to(dev)), K)
    assert not y[1:127].any() and not y[(1 << 27) + 1:(1 << 27) + 5000].any()
    del y
    torch.cuda.empty_cache()
