"""Pairs of codes and scales that hold something else are refused by type."""

import pytest
import torch

from titan_amd import ops
from titan_amd.int8 import Normed


@pytest.mark.parametrize("pair", [([[1, 2]], torch.ones(1)), (None, torch.ones(1)), (1, 2), Normed(None, None, None, None)])
def test_codes_that_are_no_tensor(pair):
    w, s, ids = torch.zeros(3, 16, dtype=torch.int8), torch.ones(3), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(TypeError, match="codes and scales"):
        ops.qqmm(pair, w, s, mode="int8")
    with pytest.raises(TypeError, match="codes and scales"):
        ops.gather_qqmm(pair, w[None], s[None], rhs_indices=ids, mode="int8")
