"""The 8-bit GEMM at contractions that turn the rings of its stages several times,
with a last group of 128 that is not whole: every form of a unit, and units of
different forms one after the other in a block.  The sums are exact, so that a
group left out, taken twice or read before it has landed shows."""

import int8_oracle as o
import pytest
import torch

from titan_amd import ops

BF, HF, F4 = o.BF, o.HF, o.F4
pytestmark = pytest.mark.gpu


def _codes(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-128, 128, shape, generator=g, dtype=torch.int8), 0.001 + 0.01 * torch.rand(shape[:-1], generator=g))


@pytest.mark.parametrize("K", [400, 528, 656, 912, 2064])  # 4, 5, 6, 8 and 17 groups
@pytest.mark.parametrize("M,N", [(100, 9001),    # 64 x 128 units
                                 (520, 4100),    # 128 x 128 and 64 x 128
                                 (1030, 4098),   # 128 x 256 and 32 x 256
                                 (4000, 4091)])  # 256 x 256 and 192 x 256 (160 rows)
def test_dense(dev, M, N, K):
    x, sx = _codes((M, K), 1)
    w, sw = _codes((N, K), 2)
    want = o.product(x, sx, w, sw)
    xd, sxd, wd, swd = (t.to(dev) for t in (x, sx, w, sw))
    for out in (BF, F4):
        y = ops.qqmm((xd, sxd), wd, swd, mode="int8", dtype=out)
        o.assert_rounded(y, want, what=(M, N, K, out))


def _by_table(dev, counts, N, K, out, seed):
    """Products of experts with so many rows each, rows taken by index."""
    g = torch.Generator().manual_seed(seed)
    E, n = len(counts), sum(counts)
    x, sx = _codes((700, K), seed + 1)
    w, sw = _codes((E, N, K), seed + 2)
    ids = torch.arange(E).repeat_interleave(torch.tensor(counts))
    rows = torch.randint(0, 700, (n,), generator=g)
    want = torch.cat([o.product(x[rows[ids == e]], sx[rows[ids == e]], w[e], sw[e]) for e in range(E)])
    args = [t.to(dev) for t in (x.unsqueeze(1), sx.unsqueeze(1), w, sw, rows.int(), ids.int())]
    for t in out:
        y = ops.gather_qqmm((args[0], args[1]), args[2], args[3], lhs_indices=args[4], rhs_indices=args[5], mode="int8",
                            sorted_indices=True, dtype=t)
        o.assert_rounded(y.squeeze(1), want, what=(N, K, t))


# rows of an expert: units of each form, an expert's last of fewer rows, one expert without
COUNTS = [129, 160, 192, 193, 256, 300, 448, 1, 40, 65, 97, 128, 0, 225]


@pytest.mark.parametrize("K,out", [(400, (BF, F4)), (656, (BF, HF)), (1168, (BF,))])  # 4, 6 and 10 groups
def test_pairs_of_tiles(dev, K, out):
    """30 units of up to 256 rows by 20 of columns, three to a block, of all six forms in the order of their rows."""
    _by_table(dev, COUNTS + COUNTS[::-1], 5000, K, out, 10)


def test_pairs_of_tiles_with_every_second_xcd_reversed(dev):
    """120 units by nine of columns: more than four to a block."""
    _by_table(dev, (COUNTS + COUNTS[::-1]) * 4, 2300, 400, (BF,), 20)


@pytest.mark.parametrize("counts,N", [([250, 0, 190, 65, 70, 125], 300),  # 64 x 128 units
                                      ([1500, 64, 65, 1900, 2000], 333),  # 128 x 128
                                      ([4400, 33, 4500, 97], 500)])       # 128 x 256
@pytest.mark.parametrize("K", [528, 1168])  # 5 and 10 groups
def test_small_units(dev, counts, N, K):
    _by_table(dev, counts, N, K, (BF, F4), 30)


def test_pairs_of_tiles_of_two_experts(dev):
    """Long runs of rows of an expert: units of two tiles each, and both experts' ends."""
    g = torch.Generator().manual_seed(4)
    n0 = int(torch.randint(8000, 9000, (1,), generator=g))
    _by_table(dev, [n0, 17000 - n0], 600, 912, (BF, HF, F4), 40)
