"""The overlay's self-check of its mxfp4 gathers, on the CPU: a kernel that disagrees
is found whatever the replaced function does."""

import pytest

from titan_amd import stock
from titan_amd.patches import _selfcheck


def _no_mode(x, w, scales, biases, *, rhs_indices, mode="affine", **kw):
    raise ValueError(f"mode={mode!r}")


def _no_mode_argument(x, w, scales, biases, rhs_indices=None, transpose=True, group_size=64, bits=4):
    raise AssertionError("not reached")


def _fails_on(rows):
    def previous(x, *args, **kw):
        if x.shape[0] == rows:
            raise RuntimeError("broken")
        return stock.gather_qmm(x, *args, **kw)

    return previous


PREVIOUS = [stock.gather_qmm, _no_mode, _no_mode_argument, _fails_on(96), _fails_on(3)]


def _wrong_on(rows):
    def fast(x, *args, **kw):
        y = stock.gather_qmm(x, *args, **kw)
        return y * 1.5 if x.shape[0] == rows else y

    return fast


@pytest.mark.parametrize("i", range(len(PREVIOUS)))
def test_finds_a_kernel_that_disagrees(i):
    assert _selfcheck.mxfp4_gather_matches(PREVIOUS[i], stock.gather_qmm, "cpu")
    for rows in (96, 3):
        assert not _selfcheck.mxfp4_gather_matches(PREVIOUS[i], _wrong_on(rows), "cpu")


def test_a_kernel_that_fails_is_reported():
    def fast(*args, **kw):
        raise RuntimeError("no launch")

    for previous in PREVIOUS:
        with pytest.raises(RuntimeError, match="no launch"):
            _selfcheck.mxfp4_gather_matches(previous, fast, "cpu")
