"""Which activation row and which expert each output row of a gather call takes,
on the CPU: the rows before any launch, where the kernels clamp what is left."""

import pytest
import torch

from titan_amd import mxfp4, ops

BF = torch.bfloat16


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(ops, "_dev", lambda t, name: None)


def _taken(x, E, lhs, rhs):
    """(activation row, expert) of each output row as the kernels read them."""
    _, rows, order = mxfp4._gathered(x, E, lhs, rhs, False, None, 1 << 40)
    assert order is None
    n_x = x[..., 0].numel()
    xr = mxfp4._x_rows(rows, x.device)
    xr = torch.arange(rows.n, dtype=torch.int32) if xr is None else xr
    assert xr.dtype == rows.experts.dtype == torch.int32
    return xr.clamp(0, n_x - 1).tolist(), rows.experts.clamp(0, E - 1).tolist()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.int16])
@pytest.mark.parametrize("M", [1, 2, 5])
def test_an_index_out_of_range_takes_the_nearest_batch(M, dtype):
    """All M rows of the nearest batch of x, not its nearest row M times."""
    B, E = 4, 3
    lhs, rhs = [4, -1, 2, 9, -7, 3, 0], [0, 1, 2, 3, -1, 0, 7]
    got = _taken(torch.zeros(B, M, 32, dtype=BF), E, torch.tensor(lhs, dtype=dtype), torch.tensor(rhs, dtype=dtype))
    assert got == ([min(max(i, 0), B - 1) * M + m for i in lhs for m in range(M)],
                   [min(max(i, 0), E - 1) for i in rhs for _ in range(M)])


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32, torch.uint64])
@pytest.mark.parametrize("M", [1, 3])
def test_an_index_past_32_bits_takes_the_last_batch(M, dtype):
    """What 32 bits do not hold is out of range, not some other index."""
    B, E = 4, 3
    far = [1 << 31, (1 << 31) + 1, (1 << 32) - 1]
    if dtype != torch.uint32:
        far += [1 << 32, (1 << 32) + 2, (1 << 62) + 1]
    if dtype == torch.uint64:
        far += [1 << 63, (1 << 64) - 1]
    t = lambda v: torch.tensor(v, dtype=dtype)  # noqa: E731
    n = len(far)
    got = _taken(torch.zeros(B, M, 32, dtype=BF), E, t([*far, 1]), t([*far, 2]))
    assert got == ([B * M - M + m for _ in far for m in range(M)] + list(range(M, 2 * M)), [E - 1] * (n * M) + [2] * M)
    if dtype == torch.int64:
        got = _taken(torch.zeros(B, M, 32, dtype=BF), E, t([-i for i in far]), t([-i for i in far]))
        assert got == (list(range(M)) * n, [0] * (n * M))


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.uint16])
def test_narrow_indices(dtype):
    B, E = 300, 400
    v = [0, 5, 100]
    t = torch.tensor(v, dtype=dtype)
    assert _taken(torch.zeros(B, 2, 32, dtype=BF), E, t, t) == ([2 * i + m for i in v for m in (0, 1)], [i for i in v for _ in (0, 1)])


def test_bad_arguments_of_the_narrowing():
    from titan_amd import _lib

    L, one = _lib.load(), 4096
    assert L.qmoe_narrow_ids(one, -1, 4, one, None) == _lib.ERR_INVALID
    assert L.qmoe_narrow_ids(one, 3, -1, one, None) == _lib.ERR_INVALID
    assert L.qmoe_narrow_ids(None, 3, 4, one, None) == _lib.ERR_INVALID
    assert L.qmoe_narrow_ids(one, 3, 4, None, None) == _lib.ERR_INVALID
    assert L.qmoe_narrow_ids(None, 0, 4, None, None) == _lib.OK
    assert L.qmoe_narrow_ids(one, 1 << 40, 4, one, None) == _lib.ERR_UNSUPPORTED
