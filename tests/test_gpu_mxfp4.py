"""The mxfp4 operators against their definition in 64 bits: quantisation both
ways bit for bit, products within the bound of one rounding and fp32 sums,
gradients against the formula and against differences."""

import pytest
import torch

from mx_helpers import check_sum, codes, dequantize_ref, quantize_ref
from titan_amd import ops
from titan_amd.ops import QmoeUnsupported

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def say(*a):
    print("[mxfp4]", *a, flush=True)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------ quantisation


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 32), (3, 64), (5, 7, 96), (1, 2080), (33, 2048), (0, 64), (4, 0)])
def test_quantize_both_ways(dev, shape, dtype):
    say("quantize", shape, dtype)
    x = (torch.randn(shape, generator=_gen(1)) * torch.exp2(torch.randint(-6, 7, (*shape[:-1], 1), generator=_gen(2)).float())).to(dtype)
    w, s = ops.quantize(x.to(dev), mode="mxfp4")
    assert w.dtype == torch.int32 and s.dtype == torch.uint8
    if not x.numel():
        assert w.numel() == s.numel() == 0
        return
    ref, byte = quantize_ref(x)
    assert torch.equal(s.cpu(), byte)
    assert torch.equal(dequantize_ref(w, s), ref)
    for out in (BF, torch.float16, torch.float32):
        got = ops.dequantize(w, s, mode="mxfp4", dtype=out)
        assert got.dtype == out and torch.equal(got.cpu(), ref.to(out)), out


@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
def test_quantize_borders(dev, dtype):
    say("quantize borders", dtype)
    # every midpoint and its neighbours, both signs, over scales the type has; the block's largest is set apart
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.5], dtype=torch.float64)
    rows = []
    for e in (-10, -3, 0, 5, 11):
        near = torch.cat([mids, mids * (1 + 2.0 ** -7), mids * (1 - 2.0 ** -8)])
        rows.append(torch.cat([near, torch.tensor([4.0, -0.0])]) * 2.0 ** e)
        rows.append(-rows[-1])
    x = torch.stack(rows).to(dtype)
    ref, byte = quantize_ref(x)
    w, s = ops.quantize(x.to(dev))
    assert torch.equal(s.cpu(), byte) and torch.equal(dequantize_ref(w, s), ref)


def test_quantize_zeros_subnormals_and_what_is_not_finite(dev):
    say("quantize edges")
    x = torch.zeros(9, 64)
    x[1, 3] = -0.0
    x[2, 5], x[2, 40] = 2.0 ** -149, 2.0 ** -130      # subnormal blocks
    x[3, :32] = torch.linspace(-1, 1, 32) * 2.0 ** -126
    x[4, 0], x[4, 33] = 3.4e38, -2.0 ** 127           # the largest scale
    x[5, 1] = float("inf")
    x[6, 35] = float("nan")
    x[7, 2], x[7, 3] = -float("inf"), 1.0
    x[8] = torch.arange(64) * 2.0 ** -133
    ref, byte = quantize_ref(x)
    w, s = ops.quantize(x.to(dev))
    assert torch.equal(s.cpu(), byte)
    got = dequantize_ref(w, s)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got.nan_to_num(0), ref.nan_to_num(0))
    back = ops.dequantize(w, s, mode="mxfp4", dtype=torch.float32).cpu()
    assert torch.equal(torch.isnan(back), torch.isnan(ref))
    assert torch.equal(back.double().nan_to_num(0), ref.float().double().nan_to_num(0))
    assert torch.signbit(back[1, 3])


def test_dequantize_every_code_and_scale(dev):
    say("dequantize all")
    w = torch.tensor([0x76543210, 0xFEDCBA98 - (1 << 32), 0, 0], dtype=torch.int64).to(torch.int32).repeat(256, 1)
    s = torch.arange(256, dtype=torch.int64).to(torch.uint8).reshape(256, 1)
    ref = dequantize_ref(w, s)
    for dt in (BF, torch.float32, torch.float16):
        got = ops.dequantize(w.to(dev), s.to(dev), mode="mxfp4", dtype=dt).cpu()
        want = ref.to(dt)
        assert torch.equal(torch.isnan(got), torch.isnan(want)), dt
        assert torch.equal(got.nan_to_num(0, 1, -1), want.nan_to_num(0, 1, -1)), dt


def test_quantize_takes_views(dev):
    say("quantize views")
    x = torch.randn(6, 200, generator=_gen(3)).to(BF).to(dev)
    for v in (x[:, 8:72], x[::2, 1:129], x[:, :64].t().contiguous().t()):
        w, s = ops.quantize(v)
        assert torch.equal(dequantize_ref(w, s), quantize_ref(v)[0])


# ----------------------------------------------------------------- dense


def _acts(gen, rows, K):
    x = torch.randn(rows, K, generator=gen)
    return (x * (0.25 + torch.rand(rows, 1, generator=gen))).to(BF)


def _dense(x, W, transpose):
    """Reference and sum of magnitudes."""
    W = W.t() if transpose else W
    x = x.detach().cpu().double()
    return x @ W, x.abs() @ W.abs()


DENSE = [(1, 32, 1), (1, 64, 33), (2, 2048, 96), (3, 96, 257), (4, 4096, 64), (5, 32, 7), (7, 160, 65), (16, 2048, 128),
         (23, 2080, 515), (33, 512, 300), (64, 96, 256), (100, 1056, 129), (128, 64, 256), (129, 2048, 512),
         (300, 544, 777), (1, 1056, 5), (1, 8192, 40)]


@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("M,K,N", DENSE)
def test_quantized_matmul(dev, M, K, N, transpose):
    say("matmul", M, K, N, transpose)
    g = _gen(M * 7 + K + N)
    w, s = codes(g, N, K)
    x = _acts(g, M, K if transpose else N)
    got = ops.quantized_matmul(x.to(dev), w.to(dev), s.to(dev), transpose=transpose, group_size=32, mode="mxfp4")
    ref, mag = _dense(x, dequantize_ref(w, s), transpose)
    check_sum(got, ref, mag, x.shape[1], (M, K, N, transpose))


@pytest.mark.parametrize("K", [1056, 2080, 2176, 2560, 3200, 4128, 6144])
@pytest.mark.parametrize("M", [5, 23, 40, 64])
def test_few_rows_past_whole_rounds(dev, M, K):
    """Contractions that end in every part of a round of the waves' batches, both kinds of activations."""
    say("few rows", M, K)
    g = _gen(67)
    w, s = codes(g, 35, K)
    x = _acts(g, M, K)
    W = dequantize_ref(w, s)
    check_sum(ops.quantized_matmul(x.to(dev), w.to(dev), s.to(dev), mode="mxfp4"), *_dense(x, W, True), K)
    check_sum(ops.qqmm(x.to(dev), w.to(dev), s.to(dev)), *_dense(quantize_ref(x)[0], W, True), K)


@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("shape", [(0,), (3, 0), (2, 5), (1, 1, 70)])
def test_quantized_matmul_batch_shapes(dev, shape, transpose):
    say("matmul shape", shape, transpose)
    g = _gen(4)
    w, s = codes(g, 40, 64)
    x = torch.randn(*shape, 64 if transpose else 40, generator=g).to(BF)
    got = ops.quantized_matmul(x.to(dev), w.to(dev), s.to(dev), transpose=transpose, mode="mxfp4")
    assert got.shape == (*shape, 40 if transpose else 64)
    if x.numel():
        W = dequantize_ref(w, s)
        W = W.t() if transpose else W
        check_sum(got, x.double() @ W, x.double().abs() @ W.abs(), x.shape[-1])


@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("M", [1, 6, 70, 200])
def test_quantized_matmul_takes_views(dev, M, transpose):
    say("matmul views", M, transpose)
    g = _gen(5)
    w, s = codes(g, 72, 96)
    C = 96 if transpose else 72
    big = torch.randn(M + 2, C + 24, generator=g).to(BF).to(dev)
    W = dequantize_ref(w, s)
    ws = torch.stack([w, w], 1).to(dev)[:, 1], torch.stack([s, s], 1).to(dev)[:, 1]
    assert not ws[0].is_contiguous()
    for x in (big[1:-1, 8:8 + C], big[1:-1, 3:3 + C], big[:M, :C].t().contiguous().t()):
        got = ops.quantized_matmul(x, *ws, transpose=transpose, mode="mxfp4")
        check_sum(got, *_dense(x, W, transpose), C)


@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("M", [1, 3, 9, 40, 150])
def test_scales_at_the_ends_of_their_range(dev, M, transpose):
    """Powers of two far apart, a NaN scale, and subnormal weights."""
    say("matmul scales", M, transpose)
    g = _gen(6)
    N, K = 48, 96
    w, s = codes(g, N, K, lo=100, hi=150)
    s[5, 1] = 255
    s[6] = 0
    s[7] = 20
    x = _acts(g, M, K if transpose else N)
    got = ops.quantized_matmul(x.to(dev), w.to(dev), s.to(dev), transpose=transpose, mode="mxfp4")
    ref, mag = _dense(x, dequantize_ref(w, s), transpose)
    check_sum(got, ref, mag.nan_to_num(0), x.shape[1], (M, transpose))


@pytest.mark.parametrize("M", [1, 5, 80, 200])
def test_rows_do_not_mix(dev, M):
    """A row of NaN or infinities stays in its own row, whatever shares its tile."""
    say("rows", M)
    g = _gen(7)
    w, s = codes(g, 40, 64)
    x = _acts(g, M, 64)
    if M > 1:
        x[M // 2] = float("nan")
    x[0, 3] = float("inf")
    got = ops.quantized_matmul(x.to(dev), w.to(dev), s.to(dev), mode="mxfp4").cpu()
    fine = torch.ones(M, dtype=torch.bool)
    fine[[0, M // 2]] = False
    assert not torch.isfinite(got[0]).all() and (M == 1 or torch.isnan(got[M // 2]).all())
    ref, mag = _dense(x[fine], dequantize_ref(w, s), True)
    check_sum(got[fine], ref, mag, 64)


# --------------------------------------------------------------- experts


def _by_expert(x, W, e, transpose):
    x = x.detach().cpu().double()
    ref = torch.stack([(W[i].t() if transpose else W[i]).t() @ v for v, i in zip(x, e.tolist())]) if len(x) else x
    mag = torch.stack([(W[i].t() if transpose else W[i]).t().abs() @ v.abs() for v, i in zip(x, e.tolist())]) if len(x) else x
    return ref, mag


GATHER = [(1, 1, 3, 64, 40), (1, 10, 16, 2048, 96), (3, 2, 4, 96, 33), (8, 10, 32, 64, 48), (70, 2, 5, 160, 264),
          (200, 4, 16, 96, 72), (257, 1, 2, 64, 520), (40, 8, 8, 544, 100)]


@pytest.mark.parametrize("is_sorted", [False, True])
@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("T,k,E,K,N", GATHER)
def test_gather_qmm(dev, T, k, E, K, N, transpose, is_sorted):
    say("gather", T, k, E, K, N, transpose, is_sorted)
    g = _gen(T + k + E)
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(torch.int32)
    x = _acts(g, T, K if transpose else N)
    C = x.shape[1]
    w, s = w.to(dev), s.to(dev)
    if not is_sorted:
        got = ops.gather_qmm(x.to(dev).reshape(T, 1, 1, C), w, s, rhs_indices=ids.to(dev), transpose=transpose, mode="mxfp4")
        assert got.shape == (T, k, 1, N if transpose else K)
        ref, mag = _by_expert(x.repeat_interleave(k, 0), W, ids.reshape(-1), transpose)
        check_sum(got.reshape(T * k, -1), ref, mag, C)
        return
    order = torch.argsort(ids.reshape(-1), stable=True)
    e = ids.reshape(-1)[order]
    ref, mag = _by_expert(x[order // k], W, e, transpose)
    # rows taken by index, rows in hand, and with a table of the caller's
    got = ops.gather_qmm(x.to(dev).unsqueeze(1), w, s, lhs_indices=(order // k).to(dev), rhs_indices=e.to(dev),
                         transpose=transpose, mode="mxfp4", sorted_indices=True)
    check_sum(got.squeeze(1), ref, mag, C)
    xs = x[order // k].to(dev).unsqueeze(1)
    for tiles in (None, ops.build_tiles(e.to(dev), E)):
        again = ops.gather_qmm(xs, w, s, rhs_indices=e.to(dev), transpose=transpose, mode="mxfp4", sorted_indices=True,
                               tiles=tiles)
        assert torch.equal(again, got)


def test_gather_qmm_forms(dev):
    """The broadcasts of the batch: default experts, several rows a batch index, x's first dimension broadcast."""
    say("gather forms")
    g = _gen(9)
    E, K, N = 6, 64, 24
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s)
    wd, sd = w.to(dev), s.to(dev)

    def check(x, lhs, rhs, xi, e):
        kw = {} if rhs is None else {"rhs_indices": torch.tensor(rhs, dtype=torch.int64).to(dev)}
        if lhs is not None:
            kw["lhs_indices"] = torch.tensor(lhs, dtype=torch.int64).to(dev)
        got = ops.gather_qmm(x.to(dev), wd, sd, mode="mxfp4", **kw)
        M = x.shape[-2]
        x2 = x.reshape(-1, M, K)
        ref = torch.stack([x2[i].double() @ W[j].t() for i, j in zip(xi, e)])
        mag = torch.stack([x2[i].double().abs() @ W[j].t().abs() for i, j in zip(xi, e)])
        check_sum(got.reshape(-1, M, N), ref, mag, K)

    rows = lambda *shape: torch.randn(*shape, K, generator=g).to(BF)  # noqa: E731
    check(rows(E, 1), None, None, range(E), range(E))
    check(rows(1, 1), None, None, [0] * E, range(E))
    check(rows(1), None, [2, 2, 0], [0] * 3, [2, 2, 0])
    check(rows(3, 5), None, [5, 0, 3], range(3), [5, 0, 3])
    check(rows(3, 30), None, [5, 0, 3], range(3), [5, 0, 3])       # 90 rows: sorted inside
    check(rows(4, 1, 2), None, [[1, 5, 0]], [i // 3 for i in range(12)], [1, 5, 0] * 4)
    check(rows(1, 3, 2), None, [[1], [4]], [i % 3 for i in range(6)], [1, 1, 1, 4, 4, 4])
    check(rows(4, 2), [3, 3, 0, 1, 2], [0, 1, 1, 5, 5], [3, 3, 0, 1, 2], [0, 1, 1, 5, 5])
    check(rows(4, 20), [3, 3, 0, 1, 2], [0, 4, 1, 5, 5], [3, 3, 0, 1, 2], [0, 4, 1, 5, 5])
    got = ops.gather_qmm(rows(0, 1).to(dev), wd, sd, rhs_indices=torch.empty(0, dtype=torch.int32, device=dev), mode="mxfp4")
    assert got.shape == (0, 1, N)


@pytest.mark.parametrize("n", [63, 64, 300])
def test_sorted_rows_with_empty_and_full_experts(dev, n):
    say("skewed", n)
    g = _gen(11)
    E, K, N = 9, 96, 40
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s)
    x = _acts(g, n, K)
    for e in (torch.full((n,), 4), torch.tensor([0] * 3 + [8] * (n - 3)), torch.sort(torch.randint(2, 5, (n,), generator=g))[0]):
        got = ops.gather_qmm(x.to(dev).unsqueeze(1), w.to(dev), s.to(dev), rhs_indices=e.to(dev), mode="mxfp4",
                             sorted_indices=True)
        check_sum(got.squeeze(1), *_by_expert(x, W, e, True), K)


@pytest.mark.parametrize("n", [5, 70, 300])
@pytest.mark.parametrize("is_sorted", [False, True])
def test_indices_out_of_range_are_clamped(dev, n, is_sorted):
    """Memory stays in bounds and every row is computed, forward and backward, few rows and many."""
    say("clamped", n, is_sorted)
    g = _gen(41)
    E, K, N = 4, 64, 40
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s)
    e = torch.randint(-3, E + 3, (n,), generator=g)
    lhs = torch.randint(-2, n + 2, (n,), generator=g)
    if is_sorted:
        e = torch.sort(e)[0]
    x = _acts(g, n, K)
    inside = e.clamp(0, E - 1)
    xd = x.to(dev).unsqueeze(1).requires_grad_(True)
    for kw, xi in (({}, torch.arange(n)), ({"lhs_indices": lhs.to(dev)}, lhs.clamp(0, n - 1))):
        for ids in (e.to(dev), e.to(torch.int32).to(dev)):
            y = ops.gather_qmm(xd, w.to(dev), s.to(dev), rhs_indices=ids, mode="mxfp4", sorted_indices=is_sorted, **kw)
            check_sum(y.squeeze(1), *_by_expert(x[xi], W, inside, True), K)
            q = ops.gather_qqmm(xd.detach(), w.to(dev), s.to(dev), rhs_indices=ids, sorted_indices=is_sorted, **kw)
            check_sum(q.squeeze(1), *_by_expert(quantize_ref(x)[0][xi], W, inside, True), K)
        dy = _acts(g, n, N)
        (dx,) = torch.autograd.grad(y, xd, dy.to(dev).unsqueeze(1))
        ref, mag = _by_expert(dy, W, inside, False)
        zero = torch.zeros(n, K, dtype=torch.float64)
        check_sum(dx.squeeze(1), zero.index_add(0, xi, ref), zero.index_add(0, xi, mag), N + n)


# -------------------------------------------------------------- gradients


@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("M,K,N", [(1, 64, 40), (3, 96, 33), (6, 2048, 72), (70, 160, 65), (200, 544, 264)])
def test_matmul_gradient(dev, M, K, N, transpose):
    say("matmul grad", M, K, N, transpose)
    g = _gen(13)
    w, s = codes(g, N, K)
    W = dequantize_ref(w, s)
    x = _acts(g, M, K if transpose else N).to(dev).requires_grad_(True)
    y = ops.quantized_matmul(x, w.to(dev), s.to(dev), transpose=transpose, mode="mxfp4")
    dy = _acts(g, M, y.shape[1])
    (dx,) = torch.autograd.grad(y, x, dy.to(dev))
    check_sum(dx, *_dense(dy, W, not transpose), dy.shape[1])
    # the product is linear: its difference along a direction, in 64 bits, is what the gradient says
    d = torch.randn(x.shape, generator=g).double()
    W2 = W.t() if transpose else W
    want = ((d @ W2) * dy.double()).sum()
    got = (d * dx.cpu().double()).sum()
    slack = (d.abs() * (dy.double().abs() @ W2.t().abs())).sum() * ((dy.shape[1] + 8) * 2.0 ** -24 + 2.0 ** -8)
    assert abs(got - want) <= slack


@pytest.mark.parametrize("is_sorted", [False, True])
@pytest.mark.parametrize("transpose", [True, False])
@pytest.mark.parametrize("T,k,E,K,N", [(1, 3, 4, 64, 40), (9, 4, 8, 96, 33), (100, 4, 12, 160, 72)])
def test_gather_gradient(dev, T, k, E, K, N, transpose, is_sorted):
    """Token rows shared by k pairs: by broadcast, or by index."""
    say("gather grad", T, k, E, K, N, transpose, is_sorted)
    g = _gen(17)
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    C, O = (K, N) if transpose else (N, K)
    x = _acts(g, T, C).to(dev).requires_grad_(True)
    flat = ids.reshape(-1)
    tok = torch.arange(T).repeat_interleave(k)
    if is_sorted:
        order = torch.argsort(flat, stable=True)
        flat, tok = flat[order], tok[order]
        y = ops.gather_qmm(x.unsqueeze(1), w.to(dev), s.to(dev), lhs_indices=tok.to(dev), rhs_indices=flat.to(dev),
                           transpose=transpose, mode="mxfp4", sorted_indices=True)
    else:
        y = ops.gather_qmm(x.reshape(T, 1, 1, C), w.to(dev), s.to(dev), rhs_indices=ids.to(dev), transpose=transpose,
                           mode="mxfp4")
    dy = _acts(g, T * k, O)
    (dx,) = torch.autograd.grad(y, x, dy.to(dev).reshape(y.shape))
    ref, mag = _by_expert(dy, W, flat, not transpose)
    zero = torch.zeros(T, C, dtype=torch.float64)
    check_sum(dx, zero.index_add(0, tok, ref), zero.index_add(0, tok, mag), O + k)


def test_gradient_of_an_expanded_result(dev):
    """A gradient that arrives as an expanded view, and a row no pair takes."""
    say("grad expanded")
    g = _gen(19)
    w, s = codes(g, 2, 40, 64)
    W = dequantize_ref(w, s)
    x = _acts(g, 3, 64).to(dev).requires_grad_(True)
    y = ops.gather_qmm(x.unsqueeze(1), w.to(dev), s.to(dev), lhs_indices=torch.tensor([2, 0, 2], device=dev),
                       rhs_indices=torch.tensor([0, 1, 1], device=dev), mode="mxfp4")
    y.sum().backward()
    ref = torch.stack([W[1].sum(0), torch.zeros(64, dtype=torch.float64), W[0].sum(0) + W[1].sum(0)])
    mag = torch.stack([W[1].abs().sum(0), torch.zeros(64, dtype=torch.float64), (W[0].abs() + W[1].abs()).sum(0)])
    check_sum(x.grad, ref, mag, 42)
    assert not x.grad[1].any()


# ----------------------------------------------------------- both in 4 bits


@pytest.mark.parametrize("M,K,N", DENSE)
def test_qqmm(dev, M, K, N):
    say("qqmm", M, K, N)
    g = _gen(23)
    w, s = codes(g, N, K)
    x = _acts(g, M, K)
    got = ops.qqmm(x.to(dev), w.to(dev), s.to(dev))
    check_sum(got, *_dense(quantize_ref(x)[0], dequantize_ref(w, s), True), K)


@pytest.mark.parametrize("is_sorted", [False, True])
@pytest.mark.parametrize("T,k,E,K,N", GATHER)
def test_gather_qqmm(dev, T, k, E, K, N, is_sorted):
    say("gather qq", T, k, E, K, N, is_sorted)
    g = _gen(29)
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    x = _acts(g, T, K)
    xq = quantize_ref(x)[0]
    flat, tok = ids.reshape(-1), torch.arange(T).repeat_interleave(k)
    if is_sorted:
        order = torch.argsort(flat, stable=True)
        flat, tok = flat[order], tok[order]
        got = ops.gather_qqmm(x.to(dev).unsqueeze(1), w.to(dev), s.to(dev), lhs_indices=tok.to(dev),
                              rhs_indices=flat.to(dev), sorted_indices=True).squeeze(1)
    else:
        got = ops.gather_qqmm(x.to(dev).reshape(T, 1, 1, K), w.to(dev), s.to(dev), rhs_indices=ids.to(dev))
        assert got.shape == (T, k, 1, N)
        got = got.reshape(T * k, N)
    check_sum(got, *_by_expert(xq[tok], W, flat, True), K)


def test_qqmm_scales_at_the_ends_of_their_range(dev):
    say("qq scales")
    g = _gen(31)
    w, s = codes(g, 48, 96, lo=100, hi=150)
    s[5, 1], s[6] = 255, 0
    x = _acts(g, 70, 96)
    x[3] = 0
    x[4, 40] = float("nan")
    got = ops.qqmm(x.to(dev), w.to(dev), s.to(dev))
    ref, mag = _dense(quantize_ref(x)[0], dequantize_ref(w, s), True)
    check_sum(got, ref, mag.nan_to_num(0), 96)


def test_qqmm_refuses_a_gradient(dev):
    w, s = codes(_gen(1), 8, 32)
    x = torch.ones(2, 32, dtype=BF, device=dev, requires_grad=True)
    with pytest.raises(QmoeUnsupported, match="gradient"):
        ops.qqmm(x, w.to(dev), s.to(dev))
    with torch.no_grad():
        assert ops.qqmm(x, w.to(dev), s.to(dev)).shape == (2, 8)


# --------------------------------------------------- streams, graphs, repeats


@pytest.mark.parametrize("M", [1, 9, 150])
def test_repeats_on_streams_and_in_graphs(dev, M):
    """Bit-equal on another stream and in replayed graphs with new inputs, forward and gradient."""
    say("graph", M)
    g = _gen(37)
    w, s = (t.to(dev) for t in codes(g, 72, 96))
    w3, s3 = (t.to(dev) for t in codes(g, 3, 72, 96))
    e = torch.sort(torch.randint(0, 3, (M,), generator=g))[0].to(dev)
    x = _acts(g, M, 96).to(dev)
    dy = _acts(g, M, 72).to(dev)

    def step():
        q, sc = ops.quantize(x)
        return (ops.dequantize(q, sc, mode="mxfp4"), ops.quantized_matmul(x, w, s, mode="mxfp4"),
                ops.quantized_matmul(dy, w, s, transpose=False, mode="mxfp4"), ops.qqmm(x, w, s),
                ops.gather_qmm(x.unsqueeze(1), w3, s3, rhs_indices=e, mode="mxfp4", sorted_indices=True),
                ops.gather_qqmm(x.unsqueeze(1), w3, s3, rhs_indices=e, sorted_indices=True))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        if seed > 1:
            x.copy_(_acts(_gen(seed), M, 96))
            dy.copy_(_acts(_gen(seed + 10), M, 72))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed
        if seed == 1:
            assert all(torch.equal(a, b) for a, b in zip(first, want))


def _indexed(dev, seed, n_x, n, E, K):
    g = _gen(seed)
    lhs = torch.randint(0, n_x, (n,), generator=g)
    lhs[: n // 4] = lhs[n // 4: n // 4 * 2]  # the same row by several indices
    return lhs, torch.randint(0, E, (n,), generator=g), _acts(g, n_x, K), _acts(g, n, 40)


@pytest.mark.parametrize("is_sorted", [False, True])
@pytest.mark.parametrize("n_x,n", [(1, 90), (300, 700), (2049, 64), (5000, 700)])
def test_gradient_of_indexed_rows(dev, n_x, n, is_sorted):
    """Activation rows taken by index, few and many, in any order: eager, and captured and replayed with new inputs."""
    say("indexed rows", n_x, n, is_sorted)
    E, K, N = 5, 64, 40
    w, s = codes(_gen(43), E, N, K)
    W = dequantize_ref(w, s)
    wd, sd = w.to(dev), s.to(dev)

    def prepared(seed):
        lhs, e, x, dy = _indexed(dev, seed, n_x, n, E, K)
        return lhs, torch.sort(e)[0] if is_sorted else e, x, dy

    lhs, e, x, dy = (t.to(dev) for t in prepared(1))

    def step():
        xd = x.detach().unsqueeze(1).requires_grad_(True)
        y = ops.gather_qmm(xd, wd, sd, lhs_indices=lhs, rhs_indices=e, mode="mxfp4", sorted_indices=is_sorted)
        return torch.autograd.grad(y, xd, dy.unsqueeze(1))[0].squeeze(1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        fresh = prepared(seed)
        for t, f in zip((lhs, e, x, dy), fresh):
            t.copy_(f)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), seed
        ref, mag = _by_expert(fresh[3], W, fresh[1], False)
        zero = torch.zeros(n_x, K, dtype=torch.float64)
        check_sum(want, zero.index_add(0, fresh[0], ref), zero.index_add(0, fresh[0], mag), N + n)


@pytest.mark.parametrize("k", [1, 3])
def test_gradient_of_an_unsorted_call_in_a_graph(dev, k):
    """Rows that the call sorts by itself, each token's for k pairs: eager and replayed alike."""
    say("unsorted graph", k)
    T, E, K, N = 80, 6, 96, 33
    g = _gen(47)
    w, s = codes(g, E, N, K)
    W = dequantize_ref(w, s)
    wd, sd = w.to(dev), s.to(dev)
    x, ids, dy = _acts(g, T, K).to(dev), torch.zeros(T, k, dtype=torch.int32, device=dev), _acts(g, T * k, N).to(dev)

    def step():
        xd = x.detach().requires_grad_(True)
        y = ops.gather_qmm(xd.reshape(T, 1, 1, K), wd, sd, rhs_indices=ids, mode="mxfp4")
        return torch.autograd.grad(y, xd, dy.reshape(y.shape))[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2, 3):
        new = torch.randint(0, E, (T, k), generator=_gen(seed))
        ids.copy_(new)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), seed
        ref, mag = _by_expert(dy.cpu(), W, new.reshape(-1), False)
        tok = torch.arange(T).repeat_interleave(k)
        zero = torch.zeros(T, K, dtype=torch.float64)
        check_sum(want, zero.index_add(0, tok, ref), zero.index_add(0, tok, mag), N + k)


def test_refuses_forward_mode(dev):
    """A tangent is refused, not lost."""
    from torch.autograd import forward_ad

    w, s = (t.to(dev) for t in codes(_gen(1), 8, 32))
    x = torch.ones(2, 32, dtype=BF, device=dev)
    one = torch.arange(2, dtype=torch.int32, device=dev)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.quantized_matmul(d, w, s, mode="mxfp4"), lambda: ops.qqmm(d, w, s),
                     lambda: ops.gather_qmm(d.unsqueeze(1), w[None], s[None], rhs_indices=one * 0, mode="mxfp4"),
                     lambda: ops.sort_tokens(d, one, one), lambda: ops.unsort_tokens(d, one, one),
                     lambda: ops.unsort_tokens(d, one, one, torch.ones(2, 1, device=dev))):
            with pytest.raises(NotImplementedError, match="forward"):
                call()


# ------------------------------------------------- offsets past 32 bits


@pytest.fixture
def room(dev):
    """These tests hold 10 to 25 GB for a moment."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("less than 40 GiB of GPU memory free")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [3, 200])
def test_experts_past_four_gigabytes(dev, room, rows):
    say("experts past 4 GB", rows)
    E, N, K = 1100, 1024, 8192
    g = torch.Generator(device=dev).manual_seed(5)
    w = torch.randint(-(1 << 31), 1 << 31, (E, N, K // 8), generator=g, device=dev, dtype=torch.int32)
    s = torch.randint(116, 124, (E, N, K // 32), generator=g, device=dev, dtype=torch.int32).to(torch.uint8)
    assert w.numel() * 4 > 1 << 32
    used = torch.tensor([0, 511, 1030, 1099])  # the last two lie behind it
    e = torch.sort(used[torch.randint(0, 4, (rows,), generator=_gen(3))])[0]
    e[-1] = 1099
    W = dequantize_ref(w[used.to(dev)], s[used.to(dev)])
    at = (e.unsqueeze(1) == used).int().argmax(1)
    for transpose, C in ((True, K), (False, N)):
        x = _acts(_gen(9), rows, C)
        for is_sorted in (True, False):
            y = ops.gather_qmm(x.to(dev).unsqueeze(1), w, s, rhs_indices=e.to(dev), transpose=transpose, mode="mxfp4",
                               sorted_indices=is_sorted)
            check_sum(y.squeeze(1), *_by_expert(x, W, at, transpose), C)
    x = _acts(_gen(9), rows, K)
    y = ops.gather_qqmm(x.to(dev).unsqueeze(1), w, s, rhs_indices=e.to(dev), sorted_indices=True)
    check_sum(y.squeeze(1), *_by_expert(quantize_ref(x)[0], W, at, True), K)


def test_rows_past_four_gigabytes(dev, room):
    say("rows past 4 GB")
    M, N, K = 300_000, 8192, 32
    w, s = codes(_gen(51), N, K)
    W, wd, sd = dequantize_ref(w, s), w.to(dev), s.to(dev)
    some = torch.tensor([0, 131_071, 262_144, 262_145, M - 1])
    few = _acts(_gen(53), len(some), K)
    x = torch.zeros(M, K, dtype=BF, device=dev)
    x[some.to(dev)] = few.to(dev)
    for y, v in ((ops.quantized_matmul(x, wd, sd, mode="mxfp4"), few), (ops.qqmm(x, wd, sd), quantize_ref(few)[0])):
        check_sum(y[some.to(dev)], *_dense(v, W, True), K)
        assert not y[1:131_071].any()
        del y
    few = _acts(_gen(57), len(some), N)
    x = torch.zeros(M, N, dtype=BF, device=dev)
    x[some.to(dev)] = few.to(dev)
    y = ops.quantized_matmul(x, wd, sd, transpose=False, mode="mxfp4")
    check_sum(y[some.to(dev)], *_dense(few, W, False), N)
    q, b = ops.quantize(x)
    ref, ref_b = quantize_ref(few)
    assert torch.equal(b[some.to(dev)].cpu(), ref_b)
    back = ops.dequantize(q, b, mode="mxfp4", dtype=torch.float32)
    assert torch.equal(back[some.to(dev)].cpu().double(), ref) and not back[1:131_071].any()


def test_two_threads_at_once(dev):
    """Calls with gradients from two threads, each on a stream of its own, agree with the same calls alone."""
    import threading

    say("threads")
    w, s = (t.to(dev) for t in codes(_gen(61), 6, 72, 96))
    e = torch.sort(torch.randint(0, 6, (150,), generator=_gen(62)))[0].to(torch.int32).to(dev)
    xs = [_acts(_gen(63 + i), 150, 96).to(dev) for i in range(2)]
    dy = _acts(_gen(65), 150, 72).to(dev)

    def step(x):
        x = x.detach().requires_grad_(True)
        y = ops.gather_qmm(x.unsqueeze(1), w, s, rhs_indices=e, mode="mxfp4", sorted_indices=True)
        z = ops.gather_qqmm(x.detach().unsqueeze(1), w, s, rhs_indices=e, sorted_indices=True)
        return y.detach(), z, torch.autograd.grad(y, x, dy.unsqueeze(1))[0]

    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i].append(step(xs[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as err:  # noqa: BLE001 - reported by the test's own thread
            errors.append(err)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i in range(2):
        assert len(got[i]) == 20
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))
