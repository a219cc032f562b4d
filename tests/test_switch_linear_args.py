"""Arguments that QuantizedSwitchLinear takes for 8-bit integers alone: refused with
codes of other kinds, not dropped."""

import pytest
import torch

from titan_amd.switch_layers import QuantizedSwitchLinear

BF = torch.bfloat16


def _linear(mode, E=3, N=16, K=64):
    w = torch.zeros(E, N, K // 8, dtype=torch.int32)
    if mode == "mxfp4":
        return QuantizedSwitchLinear(w, torch.full((E, N, K // 32), 127, dtype=torch.uint8), mode=mode)
    return QuantizedSwitchLinear(w, torch.ones(E, N, K // 64, dtype=BF), torch.zeros(E, N, K // 64, dtype=BF))


@pytest.mark.parametrize("is_sorted", [False, True])
@pytest.mark.parametrize("mode", ["affine", "mxfp4"])
def test_rows_and_dtype_are_refused(mode, is_sorted):
    """Without the refusal, index i would take x's row i (or the only row), not row rows[i]."""
    lin, x, ids = _linear(mode), torch.randn(4, 1, 64).to(BF), torch.tensor([0, 0, 1, 2], dtype=torch.int32)
    assert lin(x, ids, sorted_indices=is_sorted).shape == (4, 1, 16)
    for kw in ({"rows": torch.tensor([3, 2, 1, 0], dtype=torch.int32)}, {"dtype": torch.float32}, {"dtype": BF}):
        with pytest.raises(ValueError, match="8-bit integers"):
            lin(x, ids, sorted_indices=is_sorted, **kw)
