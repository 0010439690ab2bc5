"""Offsets that do not start at 0, decrease, or end after the rows: an error on the CPU."""
import pytest
import torch

from abacus_b200.ops import experts

BAD = {"late start": [2, 4, 6, 8], "decrease": [0, 6, 3, 8], "past the rows": [0, 3, 6, 9], "negative": [0, -1, 4, 8]}


@pytest.mark.parametrize("ends", BAD.values(), ids=BAD.keys())
def test_bad_offsets(ends):
    x, offsets = torch.randn(8, 4), torch.tensor(ends, dtype=torch.int32)
    mats = [torch.randn(3, 4, 4) for _ in range(3)]
    with pytest.raises(ValueError, match="offsets must start at 0"):
        experts.ragged_matmul(x, mats[0], offsets)
    with pytest.raises(ValueError, match="offsets must start at 0"):
        experts.ragged_swiglu_mlp(x, *mats, offsets)


@pytest.mark.parametrize("ends", [[0, 0, 0, 0], [0, 8, 8, 8], [0, 2, 2, 5]])
def test_good_offsets(ends):
    x, w = torch.randn(8, 4), torch.randn(3, 4, 4)
    y = experts.ragged_matmul(x, w, torch.tensor(ends, dtype=torch.int32))
    assert y.shape == (8, 4) and torch.all(y[ends[-1]:] == 0)
